// Gated projections of up to 16 rows: y[m][f] = act(sum_k x[m][k] g[f][k]) * (sum_k x[m][k] u[f][k]), weights [2 F][K] = g above u.
//
// The weights are read once and that bounds it: a workgroup owns 8 columns f, eight rows of g and the same rows of u, and its W waves share the
// sum: runs of UN * 128 bytes of every row go to the waves in turn.
// 16 bits: a load of a wave is 128 bytes, a whole line, of each of the eight rows, lane (row = lane % 8, part = lane / 8) the part's 16 bytes.  As an operand of a 16 x 16
// MFMA those are sixteen rows, each row of weights twice: its even parts and its odd ones.  The operand of x has the even parts of x's rows in one
// load and the odd ones in another, and is multiplied with both: of the results of the even parts the first eight rows count, of the odd ones the
// others, and the two halves of a wave add them up.  Half of the products are thrown away; the matrix units have time.  (A piece of 64 bytes of each of the
// sixteen rows of g and u a load, every product used: lines come in halves, which loads past the caches pay for twice; us so / now, one row of x and weights that are
// not in the caches: 4096 -> 11264 37.3 / 32.4, 5120 -> 13824 55.1 / 44.8, 2560 -> 6912 20.0 / 15.4.)
// float32: the products take four times as long, so the rows of g and of u are the sixteen rows of one operand and every product counts; a load is 64
// bytes of each row, through the caches, where the other half of the line waits for the next (4096 -> 4096 27.3 us, 30.8 past them).  A lane's four k feed four MFMAs of 4 k each; both
// operands use the same pairing.
// The waves' sums meet in LDS, where gate and up of a result meet too.
//
// us a call over weights that are not in the caches, floor at the rate of a large copy (5.19 TB/s; reads alone are faster): bfloat16 1 x 4096 -> 11264 32.4, 35.6; 1 x 5120 -> 13824
// 44.8, 54.6; 8 x 2048 -> 5632 12.7, 8.9; 1 x 8192 -> 1024, 128 workgroups on 256 units, 15.9, 6.5; float32 1 x 2048 -> 8192 24.2, 25.9.  With sixteen rows of g and of u a
// workgroup half as many workgroups leave some compute units with twice the others' work.  More rows of x wait for x: 16 x 4096 -> 11264 46.0; those go to tiles.
//
// Supplied by the host: TYPE, ACT, W, UN, BOTH (gate and up are wanted), Y (y is wanted), RAGGED (otherwise rows of x
// and of the weights are multiples of 16 bytes and begin at one).  Rows past the last are read from the last, their results are not stored.
// a[0] x  a[1] weights  a[2] y  a[3] both  a[4] M  a[5] F  a[6] K
struct Params { void* a[7]; };
typedef unsigned mjt_piece __attribute__((ext_vector_type(4)));
#if RAGGED
typedef unsigned mjt_there __attribute__((ext_vector_type(4), aligned(sizeof(typename mjt_el<TYPE>::raw))));      // a piece in memory
#else
typedef mjt_piece mjt_there;
#endif
typedef float mjt_f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 mjt_b16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 mjt_h16x8 __attribute__((ext_vector_type(8)));
#define EPL (TYPE == 2 ? 4 : 8)          // elements of a lane's 16 bytes
#define STEP (8 * EPL)                   // k of a line of 128 bytes

template <int V> struct mjt_ic { static constexpr int v = V; };
__device__ __forceinline__ mjt_f32x4 mjt_multiply(mjt_piece a, mjt_piece b, mjt_f32x4 c) {
#if TYPE == 0
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(mjt_b16x8, a), __builtin_bit_cast(mjt_b16x8, b), c, 0, 0, 0);
#elif TYPE == 1
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(mjt_h16x8, a), __builtin_bit_cast(mjt_h16x8, b), c, 0, 0, 0);
#else
#pragma unroll
    for (int j = 0; j < 4; j++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[j]), __uint_as_float(b[j]), c, 0, 0, 0);
    return c;
#endif
}

extern "C" __global__ __launch_bounds__(W * 64) void ENTRY(Params p) {
    typedef typename mjt_el<TYPE>::raw raw;
    const int M = (int)(long long)p.a[4], F = (int)(long long)p.a[5], K = (int)(long long)p.a[6];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int m16 = lane & 15, half = lane >> 4;
    const long long f0 = (long long)blockIdx.x * 8, f = f0 + lane % 8 < F ? f0 + lane % 8 : F - 1;
    const raw* x = (const raw*)p.a[0] + (long long)(m16 < M ? m16 : M - 1) * K;
    __shared__ float part[W][16][20];
    // fullc: the piece lies inside the row; otherwise what is behind its end is zero
    auto piece = [&](const raw* row, int k, auto fullc) {
        mjt_piece v = {0, 0, 0, 0};
        if (decltype(fullc)::v || k + EPL <= K) v = *(const mjt_there*)(row + k);
#if RAGGED
        else
#pragma unroll
            for (int j = 0; j < EPL; j++)
                if (k + j < K) ((raw*)&v)[j] = row[k + j];
#endif
        return v;
    };
#if TYPE == 2
    const raw* w = (const raw*)p.a[1] + (m16 < 8 ? f : F + f) * K;
    mjt_f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    auto run = [&](int k, auto nc, auto fullc) {
        constexpr int N = decltype(nc)::v;
        mjt_piece a[2 * N], b[2 * N];
#pragma unroll
        for (int i = 0; i < 2 * N; i++) {
            a[i] = piece(w, k + i * STEP / 2 + half * EPL, fullc);
            b[i] = piece(x, k + i * STEP / 2 + half * EPL, fullc);
        }
#pragma unroll
        for (int i = 0; i < 2 * N; i++) acc = mjt_multiply(a[i], b[i], acc);
    };
#else
    const raw *g = (const raw*)p.a[1] + f * K, *u = g + (long long)F * K;
    mjt_f32x4 ge = {0.0f, 0.0f, 0.0f, 0.0f}, go = ge, ue = ge, uo = ge;           // even and odd parts
    auto run = [&](int k, auto nc, auto fullc) {
        constexpr int N = decltype(nc)::v;
        mjt_piece a[N], b[N], even[N], odd[N];
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int kw = k + i * STEP + (lane >> 3) * EPL, kx = k + i * STEP + half * (2 * EPL);
            if (decltype(fullc)::v) {
                a[i] = __builtin_nontemporal_load((const mjt_there*)(g + kw));
                b[i] = __builtin_nontemporal_load((const mjt_there*)(u + kw));
            } else {
                a[i] = piece(g, kw, fullc);
                b[i] = piece(u, kw, fullc);
            }
            even[i] = piece(x, kx, fullc);
            odd[i] = piece(x, kx + EPL, fullc);
        }
#pragma unroll
        for (int i = 0; i < N; i++) {
            ge = mjt_multiply(a[i], even[i], ge);
            go = mjt_multiply(a[i], odd[i], go);
            ue = mjt_multiply(b[i], even[i], ue);
            uo = mjt_multiply(b[i], odd[i], uo);
        }
    };
#endif
    int k = wave * (UN * STEP);
    for (; k + UN * STEP <= K; k += W * UN * STEP) run(k, mjt_ic<UN>(), mjt_ic<1>());
    for (int end = k + UN * STEP; k < end && k < K; k += STEP) run(k, mjt_ic<1>(), mjt_ic<0>());      // (the last run of a row: it ends with one of the waves)
    // D of a 16 x 16 tile: lane holds column lane % 16 (a row of x), rows 4 * (lane / 16) + e
#pragma unroll
    for (int e = 0; e < 4; e++) {
#if TYPE == 2
        part[wave][4 * half + e][m16] = acc[e];
#else
        float gate = half < 2 ? ge[e] : go[e], up = half < 2 ? ue[e] : uo[e];
        gate += __shfl_xor(gate, 32, 64);
        up += __shfl_xor(up, 32, 64);
        part[wave][(half < 2 ? 0 : 8) + 4 * (half & 1) + e][m16] = half < 2 ? gate : up;
#endif
    }
    __syncthreads();
    const int c = threadIdx.x % 8, m = threadIdx.x / 8;
    if (m >= M || f0 + c >= F) return;
    float gate = part[0][c][m], up = part[0][8 + c][m];
#pragma unroll
    for (int s = 1; s < W; s++) gate += part[s][c][m], up += part[s][8 + c][m];
#if BOTH
    float* both = (float*)p.a[3] + (long long)m * 2 * F + f0 + c;
    both[0] = gate;
    both[F] = up;
#endif
#if Y
    ((raw*)p.a[2])[(long long)m * F + f0 + c] = mjt_el<TYPE>::down(mjt_activate(gate).a * up);
#endif
}

// Gated projections of up to 16 rows: y[m][f] = act(sum_k x[m][k] g[f][k]) * (sum_k x[m][k] u[f][k]), weights [2 F][K] = g above u.
//
// The weights are read once and that bounds it: a workgroup owns 8 columns f, eight rows of g and the same rows of u, which are the sixteen
// rows of one MFMA operand, and its W waves share the sum: pieces of 64 bytes of every row go to the waves in turn, UN of them at a time, so
// that a workgroup walks along its rows in runs of W * UN * 64 bytes.  A piece is the operand as it lies in memory: lane (row = lane % 16, part = lane / 16)
// loads 16 bytes, the 8 consecutive k (4 for float32) of its row and part.  The rows of x are the other operand, loaded the
// same way from the caches.  (float32: a lane's four k feed four MFMAs of 4 k each; both operands use the same pairing.)  The waves' sums meet
// in LDS, where gate and up of a result meet too.
//
// us a call over weights that are not in the caches, floor at the rate of a large copy (5.19 TB/s): bfloat16 1 x 4096 -> 11264 37.0, 35.6; 8 x 2048 -> 5632 12.6, 8.9;
// 1 x 8192 -> 1024 12.5, 6.5.  With sixteen rows of g and of u a workgroup and four waves 37.9 / 14.3 / 24.6: half as many workgroups leave
// some compute units with twice the others' work.  Four pieces at a time instead of two 38 / 13.2 / 14.0.  More than sixteen rows of x this way
// wait for x: 24 x 2048 -> 5632 16.5, 64 x 4096 -> 11264 74; those go to tiles.
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
#define STEP (4 * EPL)                   // k of a piece

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
    const int row = lane & 15, at = (lane >> 4) * EPL;
    const long long f0 = (long long)blockIdx.x * 8, f = f0 + row % 8 < F ? f0 + row % 8 : F - 1;
    const raw* w = (const raw*)p.a[1] + ((row < 8 ? 0 : (long long)F) + f) * K + at;
    const raw* x = (const raw*)p.a[0] + (long long)(row < M ? row : M - 1) * K + at;
    mjt_f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    int k = wave * (UN * STEP);
    for (; k + UN * STEP <= K; k += W * UN * STEP) {
        mjt_piece a[UN], b[UN];
#pragma unroll
        for (int u = 0; u < UN; u++) {
            a[u] = __builtin_nontemporal_load((const mjt_there*)(w + k + u * STEP));
            b[u] = *(const mjt_there*)(x + k + u * STEP);
        }
#pragma unroll
        for (int u = 0; u < UN; u++) acc = mjt_multiply(a[u], b[u], acc);
    }
    // the last run of the row ends with one of the waves: piece by piece, nothing past K
    for (int end = k + UN * STEP; k < end && k < K; k += STEP) {
        const int have = K - k - at;                           // elements that the lane's piece has
        mjt_piece a = {0, 0, 0, 0}, b = {0, 0, 0, 0};
        if (have >= EPL) a = *(const mjt_there*)(w + k), b = *(const mjt_there*)(x + k);
#if RAGGED
        else
#pragma unroll
            for (int j = 0; j < EPL; j++)
                if (j < have) ((raw*)&a)[j] = w[k + j], ((raw*)&b)[j] = x[k + j];
#endif
        acc = mjt_multiply(a, b, acc);
    }
    // D of a 16 x 16 tile: lane holds column lane % 16 (a row of x), rows 4 * (lane / 16) + e (g, then u)
    __shared__ float part[W][16][20];
#pragma unroll
    for (int e = 0; e < 4; e++) part[wave][4 * (lane >> 4) + e][row] = acc[e];
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

// Gated projections of few rows (up to 64): y[m][f] = act(sum_k x[m][k] g[f][k]) * (sum_k x[m][k] u[f][k]), weights [2 F][K] = g above u.
//
// The weights are read once and that bounds it: a workgroup owns 16 RB columns f, rows of g and the same rows of u, for all rows of x, and its W
// waves share the sum: pieces of 64 bytes of every row go to the waves in turn, UN of them at a time, so that a workgroup walks along
// its rows in runs of W * UN * 64 bytes.  A piece is one 16 x 16 MFMA operand as it lies in memory: lane (row = lane % 16, part = lane / 16)
// loads 16 bytes, the 8 consecutive k (4 for float32) of its row and part.  The rows of x, in blocks of 16, are the other operand, loaded the
// same way from the caches.  (float32: a lane's four k feed four MFMAs of 4 k each; both operands use the same pairing.)  The waves' sums meet
// in LDS, where gate and up of a result meet too.
//
// Supplied by the host: TYPE, ACT, W, RB, MB (blocks of 16 rows of x), UN, BOTH (gate and up are wanted), Y (y is wanted).  Rows of x
// and of the weights are multiples of 16 bytes and begin at one; rows past the last are read from the last, their results are not stored.
// a[0] x  a[1] weights  a[2] y  a[3] both  a[4] M  a[5] F  a[6] K
struct Params { void* a[7]; };
typedef unsigned mjt_piece __attribute__((ext_vector_type(4)));
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
    const long long f0 = (long long)blockIdx.x * (16 * RB);
    const raw* w[2][RB];
    const raw* x[MB];
#pragma unroll
    for (int r = 0; r < RB; r++) {
        const long long f = f0 + r * 16 + row < F ? f0 + r * 16 + row : F - 1;
        w[0][r] = (const raw*)p.a[1] + f * K + at;
        w[1][r] = (const raw*)p.a[1] + (F + f) * K + at;
    }
#pragma unroll
    for (int m = 0; m < MB; m++) x[m] = (const raw*)p.a[0] + (long long)(m * 16 + row < M ? m * 16 + row : M - 1) * K + at;

    mjt_f32x4 acc[2][RB][MB];
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int r = 0; r < RB; r++)
#pragma unroll
            for (int m = 0; m < MB; m++) acc[i][r][m] = (mjt_f32x4){0.0f, 0.0f, 0.0f, 0.0f};
    const int run = W * UN * STEP;
    int k = wave * (UN * STEP);
    for (; k + UN * STEP <= K; k += run) {
        mjt_piece a[UN][2][RB], b[UN][MB];
#pragma unroll
        for (int u = 0; u < UN; u++) {
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int r = 0; r < RB; r++) a[u][i][r] = __builtin_nontemporal_load((const mjt_piece*)(w[i][r] + k + u * STEP));
#pragma unroll
            for (int m = 0; m < MB; m++) b[u][m] = *(const mjt_piece*)(x[m] + k + u * STEP);
        }
#pragma unroll
        for (int u = 0; u < UN; u++)
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int r = 0; r < RB; r++)
#pragma unroll
                    for (int m = 0; m < MB; m++) acc[i][r][m] = mjt_multiply(a[u][i][r], b[u][m], acc[i][r][m]);
    }
    // the last run of the row ends with one of the waves: piece by piece, nothing past K
    for (int end = k + UN * STEP; k < end && k < K; k += STEP) {
        const bool in = k + at < K;
        const mjt_piece none = {0, 0, 0, 0};
#pragma unroll
        for (int m = 0; m < MB; m++) {
            const mjt_piece b = in ? *(const mjt_piece*)(x[m] + k) : none;
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int r = 0; r < RB; r++) acc[i][r][m] = mjt_multiply(in ? *(const mjt_piece*)(w[i][r] + k) : none, b, acc[i][r][m]);
        }
    }
    // D of a 16 x 16 tile: lane holds column lane % 16 (a row of x), rows 4 * (lane / 16) + e (columns f)
    constexpr int PITCH = MB * 16 + 4;
    __shared__ float part[W][2][RB * 16][PITCH];
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int r = 0; r < RB; r++)
#pragma unroll
            for (int m = 0; m < MB; m++)
#pragma unroll
                for (int e = 0; e < 4; e++) part[wave][i][r * 16 + 4 * (lane >> 4) + e][m * 16 + row] = acc[i][r][m][e];
    __syncthreads();
    for (int item = threadIdx.x; item < RB * 16 * MB * 16; item += W * 64) {
        const int c = item % (RB * 16), m = item / (RB * 16);
        float gate = part[0][0][c][m], up = part[0][1][c][m];
#pragma unroll
        for (int s = 1; s < W; s++) gate += part[s][0][c][m], up += part[s][1][c][m];
        if (m >= M || f0 + c >= F) continue;
#if BOTH
        float* both = (float*)p.a[3] + (long long)m * 2 * F + f0 + c;
        both[0] = gate;
        both[F] = up;
#endif
#if Y
        ((raw*)p.a[2])[(long long)m * F + f0 + c] = mjt_el<TYPE>::down(mjt_activate(gate).a * up);
#endif
    }
}

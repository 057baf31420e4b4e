// Dropout: y[e] = keep(e) ? x[e] / (1 - p) : 0, and with RES y[e] = residual[e] + that; the gradient is the same kernel on dy.
//
// keep(e) is u(e) >= T with T = round(p * 2^32) and a number u(e) of 32 bits that depends on the element's place, the key and the call
// alone, so the mask is never stored: the backward pass works it out again.  u comes from Philox4x32 with 10 rounds (J. Salmon,
// M. Moraes, R. Dror and D. Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011), whose counter is (e / 8, side and block, call): a
// block of 128 bits gives the upper 16 bits of eight neighbouring elements' numbers (word e / 2 % 4, the lower half for even e), a second block their
// lower 16.  The upper halves decide unless one of them equals T / 2^16, one element in 65536, so that a wave works out the second block
// for one pass in 128 (never where T's lower half is 0, p = 0.5 or 0.25): full resolution of p for half the arithmetic.
// A dropped element is 0 whatever it held, also an infinity or NaN.
//
// Supplied by the host: TYPE (element type), RES, WIDE (a lane's eight elements are whole aligned vectors), SIDE (in place in the counter's second
// word, which no element's place reaches there), STREAMS.  (As a parameter the side took 3 of 61 us of the case of 8192 x 4096 bfloat16 with a residual.)
// a[0] x  a[1] residual  a[2] y  a[3] elements  a[4] key  a[5] call  a[6] T  a[7] 1 / (1 - p) (double bits)
struct Params { void* a[8]; };

struct mjt_u4 { unsigned w[4]; };
// ten rounds of two multiplications of 32 bits to 64 and the key's Weyl steps
__device__ __forceinline__ mjt_u4 mjt_philox(unsigned c0, unsigned c1, unsigned c2, unsigned c3, unsigned k0, unsigned k1) {
#pragma unroll
    for (int r = 0; r < 10; r++) {
        const unsigned long long p0 = (unsigned long long)c0 * 0xD2511F53u, p1 = (unsigned long long)c2 * 0xCD9E8D57u;
        c0 = (unsigned)(p1 >> 32) ^ c1 ^ k0;
        c2 = (unsigned)(p0 >> 32) ^ c3 ^ k1;
        c1 = (unsigned)p1;
        c3 = (unsigned)p0;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return {{c0, c1, c2, c3}};
}
__device__ __forceinline__ unsigned mjt_half_of(const mjt_u4& w, int j) { return j & 1 ? w.w[j / 2] >> 16 : w.w[j / 2] & 0xffffu; }

// bit j: element j of group g is kept
__device__ __forceinline__ unsigned mjt_keep_bits(unsigned long long g, unsigned long long key, unsigned long long call, unsigned long long threshold) {
    const unsigned hi = (unsigned)(threshold >> 16), lo = (unsigned)(threshold & 0xffffu);        // hi up to 65536, for p = 1
    const unsigned k0 = (unsigned)key, k1 = (unsigned)(key >> 32), c2 = (unsigned)call, c3 = (unsigned)(call >> 32);
    const mjt_u4 a = mjt_philox((unsigned)g, (unsigned)(g >> 32) | SIDE, c2, c3, k0, k1);
    unsigned keep = 0, tie = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const unsigned u = mjt_half_of(a, j);
        keep |= (u >= hi ? 1u : 0u) << j;
        tie |= (u == hi ? 1u : 0u) << j;
    }
    if (lo != 0 && __any(tie != 0)) {
        const mjt_u4 b = mjt_philox((unsigned)g, (unsigned)(g >> 32) | SIDE | 0x80000000u, c2, c3, k0, k1);
#pragma unroll
        for (int j = 0; j < 8; j++)
            if ((tie >> j & 1) && mjt_half_of(b, j) < lo) keep &= ~(1u << j);
    }
    return keep;
}

extern "C" __global__ __launch_bounds__(256) void ENTRY(Params p) {
    typedef typename mjt_el<TYPE>::raw raw;
    const long long n = (long long)p.a[3], groups = (n + 7) / 8;
    const unsigned long long key = (unsigned long long)p.a[4], call = (unsigned long long)p.a[5], threshold = (unsigned long long)p.a[6];
    const float scale = (float)__longlong_as_double((long long)p.a[7]);
    const raw* __restrict__ x = (const raw*)p.a[0];
    const raw* __restrict__ res = (const raw*)p.a[1];
    raw* __restrict__ y = (raw*)p.a[2];
    for (long long g = (long long)blockIdx.x * 256 + threadIdx.x; g < groups; g += (long long)gridDim.x * 256) {
        const int have = n - g * 8 < 8 ? (int)(n - g * 8) : 8;
        mjt_els<TYPE, 8> in, add, out;
        if (WIDE && have == 8) {
            in = mjt_get<TYPE, 8>(x + g * 8);
            if (RES) add = mjt_get<TYPE, 8>(res + g * 8);
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                in.v[j] = j < have ? x[g * 8 + j] : raw(0);
                if (RES) add.v[j] = j < have ? res[g * 8 + j] : raw(0);
            }
        }
        const unsigned keep = threshold ? mjt_keep_bits((unsigned long long)g, key, call, threshold) : 0xffu;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            float v = keep >> j & 1 ? mjt_el<TYPE>::up(in.v[j]) * scale : 0.0f;
            if (RES) v += mjt_el<TYPE>::up(add.v[j]);
            out.v[j] = mjt_el<TYPE>::down(v);
        }
        if (WIDE && have == 8) mjt_set(y + g * 8, out);
        else
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (j < have) y[g * 8 + j] = out.v[j];
    }
}

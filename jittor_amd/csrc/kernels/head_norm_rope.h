// Norms of queries and keys for each head and the rotation of positions in one pass, from the joint projection x[token][head][D] whose
// heads are HQ queries, HK keys and HV values:
//   n = x * r,  r = 1 / sqrt(mean over D of x^2 + eps),  z = n * scale      (scale of the queries or of the keys; NORM 0: z = x)
//   y = z with its first ROT elements turned in pairs: (a, b) -> (a cos - b sin, a sin + b cos), cos and sin from table[position][pair]
// written as q, k and v [token][head][D], or with FIRST [batch][head][token][D]; values are copied.  Pairs are neighbours (PAIRED 1) or
// elements i and i + ROT / 2.  With several AXES every pair takes the position of its axis (ENDS: the first pair behind each axis).  A
// position outside the table makes the token's turned heads NaN.
// BACK: the gradient.  From dy of q, k and v (any of them may be missing: zero)
//   dz = dy turned back,  dscale += dz * n,  dn = dz * scale,  dx = r * (dn - n * mean(dn * n))
// with r from x again, dx whole [token][head][D], and the sums over rows of dscale: in the lane that owns the columns, then over the
// workgroup in LDS, one partial result a workgroup, which the fold kernel (FOLD) adds up in a fixed order.
//
// Memory bounds it: x once, y once (and dy).  LP lanes own a row, so that a row's sums need log2(LP) exchanges and a wave has 64 / LP
// rows; a lane has V pairs of the row in each of its NC chunks, as two pieces of V adjacent elements: both halves of its pairs, so
// turning takes no exchange.  A wave works on one token at a time: cos and sin are loaded once for all its heads.  IT rounds of rows
// are under way together.
//
// Supplied by the host: TYPE, STYPE (types of x and of the scales), D, ROT, V, LP, NC, IT, PAIRED, FIRST, NORM, AXES, ENDS, POS (positions are
// given), BACK, SUMS (BACK with gradients of the scales).
// a[0] x  a[1] q  a[2] k  a[3] v  (BACK: dq, dk, dv, null where missing; forward: null where not wanted)  a[4] scale of q  a[5] of k  a[6] table  a[7] positions
// a[8] tokens  a[9] tokens of a sequence  a[10] HQ  a[11] HK  a[12] HV  a[13] eps (double bits)  a[14] positions of an axis  a[15] rows of the table
// a[16] dx  a[17] partial sums [workgroup][2][D]
#ifndef FOLD
struct Params { void* a[18]; };
typedef typename mjt_el<TYPE>::raw raw;
typedef typename mjt_el<STYPE>::raw raws;
#define R (64 / LP)                    // rows of a wave

// the sum over the LP lanes of a row, in all of them
__device__ __forceinline__ float mjt_row_sum(float v) {
#pragma unroll
    for (int off = 1; off < LP; off *= 2) v += __shfl_xor(v, off, 64);
    return v;
}

extern "C" __global__ __launch_bounds__(256) void ENTRY(Params p) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int sub = lane / LP, own = lane % LP;
    const unsigned tokens = (unsigned)(unsigned long long)p.a[8], seq = (unsigned)(unsigned long long)p.a[9];
    const int HQ = (int)(long long)p.a[10], HK = (int)(long long)p.a[11], HV = (int)(long long)p.a[12], H = HQ + HK + HV;
    const float eps = (float)__longlong_as_double((long long)p.a[13]);
    const raw* __restrict__ x = (const raw*)p.a[0];
    // the lane's pieces of a row: V elements from first[c] and from second[c] on; chunks past the row are those of chunk 0 and count nothing
    int first[NC], second[NC], pair[NC];
    bool in[NC], turned[NC];
#pragma unroll
    for (int c = 0; c < NC; c++) {
        int at = (c * LP + own) * V;
        in[c] = at < D / 2;
        at = in[c] ? at : 0;
        turned[c] = ROT > 0 && at < ROT / 2;
        pair[c] = turned[c] ? at : 0;
        first[c] = turned[c] && !PAIRED ? at : 2 * at;
        second[c] = turned[c] && !PAIRED ? at + ROT / 2 : 2 * at + V;
    }
#if BACK && SUMS
    float dsq[NC][2][V], dsk[NC][2][V];
#pragma unroll
    for (int c = 0; c < NC; c++)
#pragma unroll
        for (int i = 0; i < V; i++) dsq[c][0][i] = dsq[c][1][i] = dsk[c][0][i] = dsk[c][1][i] = 0.0f;
#endif
    for (unsigned t = blockIdx.x * 4 + wave; t < tokens; t += gridDim.x * 4) {
        float cs[NC][V], sn[NC][V];
#if ROT > 0
        {
            const float* __restrict__ table = (const float*)p.a[6];
            const unsigned rows = (unsigned)(unsigned long long)p.a[15];
            const unsigned per = (unsigned)(unsigned long long)p.a[14];
            constexpr int ends[AXES] = ENDS;
            unsigned at[AXES];
#if POS
            const int* __restrict__ positions = (const int*)p.a[7];
#pragma unroll
            for (int a = 0; a < AXES; a++) at[a] = (unsigned)positions[(long long)a * per + t % per];
#else
#pragma unroll
            for (int a = 0; a < AXES; a++) at[a] = t % seq;
#endif
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int i = 0; i < V; i++) {
                    unsigned row = at[0];
#pragma unroll
                    for (int a = 1; a < AXES; a++) row = pair[c] + i >= ends[a - 1] ? at[a] : row;
                    const bool there = row < rows;
                    const float* f = table + ((long long)(there ? row : 0) * (ROT / 2) + pair[c] + i) * 2;
                    cs[c][i] = turned[c] ? there ? f[0] : __builtin_nanf("") : 1.0f;
                    sn[c][i] = turned[c] ? f[1] : 0.0f;
                }
        }
#else
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int i = 0; i < V; i++) cs[c][i] = 1.0f, sn[c][i] = 0.0f;
#endif
        const unsigned b = FIRST ? t / seq : 0, s = FIRST ? t - b * seq : 0;
        for (int h0 = blockIdx.y * (R * IT); h0 < H; h0 += gridDim.y * (R * IT)) {
            mjt_els<TYPE, V> a0[IT][NC], a1[IT][NC];
#if BACK
            mjt_els<TYPE, V> g0[IT][NC], g1[IT][NC];
            bool given[IT];
#endif
            long long place[IT];
#pragma unroll
            for (int it = 0; it < IT; it++) {
                const int h = h0 + it * R + sub < H ? h0 + it * R + sub : H - 1;
                const raw* from = x + ((long long)t * H + h) * D;
                // the row in q, k or v
                const int heads = h < HQ ? HQ : h < HQ + HK ? HK : HV, mine = h < HQ ? h : h < HQ + HK ? h - HQ : h - HQ - HK;
                place[it] = (FIRST ? ((long long)b * heads + mine) * seq + s : (long long)t * heads + mine) * D;
#if BACK
                const raw* dy = (const raw*)(h < HQ ? p.a[1] : h < HQ + HK ? p.a[2] : p.a[3]);
                given[it] = dy != nullptr;
                dy = given[it] ? dy + place[it] : from;
#endif
#pragma unroll
                for (int c = 0; c < NC; c++) {
                    a0[it][c] = *(const mjt_els<TYPE, V>*)(from + first[c]);
                    a1[it][c] = *(const mjt_els<TYPE, V>*)(from + second[c]);
#if BACK
                    g0[it][c] = *(const mjt_els<TYPE, V>*)(dy + first[c]);
                    g1[it][c] = *(const mjt_els<TYPE, V>*)(dy + second[c]);
#endif
                }
            }
#pragma unroll
            for (int it = 0; it < IT; it++) {
                const int h = h0 + it * R + sub;
                const bool real = h < H, query = h < HQ, value = h >= HQ + HK;
                float u[NC][2][V];
                float sum = 0.0f;
#pragma unroll
                for (int c = 0; c < NC; c++)
#pragma unroll
                    for (int i = 0; i < V; i++) {
                        u[c][0][i] = mjt_el<TYPE>::up(a0[it][c].v[i]);
                        u[c][1][i] = mjt_el<TYPE>::up(a1[it][c].v[i]);
                        const float both = u[c][0][i] * u[c][0][i] + u[c][1][i] * u[c][1][i];
                        sum += in[c] ? both : 0.0f;
                    }
                float sc[NC][2][V];
#if NORM
                const float r = 1.0f / sqrtf(mjt_row_sum(sum) * (1.0f / D) + eps);
                const raws* scale = (const raws*)(query ? p.a[4] : p.a[5]);
#pragma unroll
                for (int c = 0; c < NC; c++) {
                    const mjt_els<STYPE, V> s0 = *(const mjt_els<STYPE, V>*)(scale + first[c]), s1 = *(const mjt_els<STYPE, V>*)(scale + second[c]);
#pragma unroll
                    for (int i = 0; i < V; i++) sc[c][0][i] = mjt_el<STYPE>::up(s0.v[i]), sc[c][1][i] = mjt_el<STYPE>::up(s1.v[i]);
                }
#else
                const float r = 1.0f;
#pragma unroll
                for (int c = 0; c < NC; c++)
#pragma unroll
                    for (int i = 0; i < V; i++) sc[c][0][i] = sc[c][1][i] = 1.0f;
#endif
                mjt_els<TYPE, V> o0[NC], o1[NC];
#if !BACK
#pragma unroll
                for (int c = 0; c < NC; c++)
#pragma unroll
                    for (int j = 0; j < V; j++) {
                        // (neighbouring pairs: pair j of the chunk is elements 2 j and 2 j + 1 of its 2 V)
                        constexpr bool near = PAIRED;
                        const int h0_ = near ? 2 * j / V : 0, i0 = near ? 2 * j % V : j, h1_ = near ? (2 * j + 1) / V : 1, i1 = near ? (2 * j + 1) % V : j;
                        const float za = u[c][h0_][i0] * r * sc[c][h0_][i0], zb = u[c][h1_][i1] * r * sc[c][h1_][i1];
                        const float ya = za * cs[c][j] - zb * sn[c][j], yb = za * sn[c][j] + zb * cs[c][j];
                        const raw ra = mjt_el<TYPE>::down(ya), rb = mjt_el<TYPE>::down(yb);
                        (h0_ ? o1[c] : o0[c]).v[i0] = ra;
                        (h1_ ? o1[c] : o0[c]).v[i1] = rb;
                    }
                raw* to = (raw*)(query ? p.a[1] : value ? p.a[3] : p.a[2]);
                if (real && to) {
#pragma unroll
                    for (int c = 0; c < NC; c++)
                        if (in[c]) {
                            *(mjt_els<TYPE, V>*)(to + place[it] + first[c]) = value ? a0[it][c] : o0[c];
                            *(mjt_els<TYPE, V>*)(to + place[it] + second[c]) = value ? a1[it][c] : o1[c];
                        }
                }
#else
                float dn[NC][2][V], dot = 0.0f;
#pragma unroll
                for (int c = 0; c < NC; c++)
#pragma unroll
                    for (int j = 0; j < V; j++) {
                        constexpr bool near = PAIRED;
                        const int h0_ = near ? 2 * j / V : 0, i0 = near ? 2 * j % V : j, h1_ = near ? (2 * j + 1) / V : 1, i1 = near ? (2 * j + 1) % V : j;
                        const float ga = given[it] ? mjt_el<TYPE>::up((h0_ ? g1[it][c] : g0[it][c]).v[i0]) : 0.0f, gb = given[it] ? mjt_el<TYPE>::up((h1_ ? g1[it][c] : g0[it][c]).v[i1]) : 0.0f;
                        const float za = ga * cs[c][j] + gb * sn[c][j], zb = gb * cs[c][j] - ga * sn[c][j];
                        const float na = u[c][h0_][i0] * r, nb = u[c][h1_][i1] * r;
#if SUMS
                        const bool counts = real && in[c] && !value && given[it];
                        const float wa = counts ? za * na : 0.0f, wb = counts ? zb * nb : 0.0f;
                        dsq[c][h0_][i0] += query ? wa : 0.0f, dsq[c][h1_][i1] += query ? wb : 0.0f;
                        dsk[c][h0_][i0] += query ? 0.0f : wa, dsk[c][h1_][i1] += query ? 0.0f : wb;
#endif
                        dn[c][h0_][i0] = za * sc[c][h0_][i0];
                        dn[c][h1_][i1] = zb * sc[c][h1_][i1];
                        const float both = dn[c][h0_][i0] * na + dn[c][h1_][i1] * nb;
                        dot += in[c] ? both : 0.0f;
                    }
                const float m = NORM ? mjt_row_sum(dot) * (1.0f / D) : 0.0f;
#pragma unroll
                for (int c = 0; c < NC; c++)
#pragma unroll
                    for (int i = 0; i < V; i++) {
                        o0[c].v[i] = mjt_el<TYPE>::down(NORM ? r * (dn[c][0][i] - u[c][0][i] * r * m) : dn[c][0][i]);
                        o1[c].v[i] = mjt_el<TYPE>::down(NORM ? r * (dn[c][1][i] - u[c][1][i] * r * m) : dn[c][1][i]);
                        if (value || !given[it]) {                            // (no gradient is none, whatever the position's angles are)
                            o0[c].v[i] = given[it] ? g0[it][c].v[i] : raw(0);
                            o1[c].v[i] = given[it] ? g1[it][c].v[i] : raw(0);
                        }
                    }
                raw* to = (raw*)p.a[16];
                if (real && to) {
                    to += ((long long)t * H + h) * D;
#pragma unroll
                    for (int c = 0; c < NC; c++)
                        if (in[c]) {
                            *(mjt_els<TYPE, V>*)(to + first[c]) = o0[c];
                            *(mjt_els<TYPE, V>*)(to + second[c]) = o1[c];
                        }
                }
#endif
            }
        }
    }
#if BACK && SUMS
    __shared__ float part[4][2][D];
#pragma unroll
    for (int c = 0; c < NC; c++)
#pragma unroll
        for (int e = 0; e < 2; e++)
#pragma unroll
            for (int i = 0; i < V; i++) {
                float q = dsq[c][e][i], k = dsk[c][e][i];
#pragma unroll
                for (int off = LP; off < 64; off *= 2) q += __shfl_xor(q, off, 64), k += __shfl_xor(k, off, 64);
                if (sub == 0 && in[c]) {
                    part[wave][0][(e ? second[c] : first[c]) + i] = q;
                    part[wave][1][(e ? second[c] : first[c]) + i] = k;
                }
            }
    __syncthreads();
    float* mine = (float*)p.a[17] + (long long)blockIdx.x * 2 * D;
    for (int i = threadIdx.x; i < 2 * D; i += 256) mine[i] = ((part[0][0][i] + part[1][0][i]) + (part[2][0][i] + part[3][0][i]));
#endif
}
#else
// dscale[e] = sum over workgroups of part[w][e], e in 0 .. 2 D (the queries' first): 32 columns a workgroup, 32 strips of partial results,
// joined in LDS in a fixed order.
// a[0] part  a[1] dscale of q  a[2] of k (null where not wanted)  a[3] partial results  a[4] D
struct Params { void* a[5]; };
extern "C" __global__ __launch_bounds__(1024) void ENTRY(Params p) {
    const float* __restrict__ part = (const float*)p.a[0];
    const int n = (int)(long long)p.a[3], D = (int)(long long)p.a[4];
    const int strip = threadIdx.x / 32, col = blockIdx.x * 32 + threadIdx.x % 32;
    float sum = 0.0f;
    if (col < 2 * D)
#pragma unroll 8
        for (int w = strip; w < n; w += 32) sum += part[(long long)w * 2 * D + col];
    __shared__ float sums[32][33];
    sums[strip][threadIdx.x % 32] = sum;
    __syncthreads();
    if (strip == 0 && col < 2 * D) {
        float total = 0.0f;
#pragma unroll
        for (int s = 0; s < 32; s++) total += sums[s][threadIdx.x];
        typename mjt_el<STYPE>::raw* to = (typename mjt_el<STYPE>::raw*)(col < D ? p.a[1] : p.a[2]);
        if (to) to[col < D ? col : col - D] = mjt_el<STYPE>::down(total);
    }
}
#endif

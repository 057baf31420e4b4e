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
// Memory bounds it: x once, y once (and dy).  LP lanes own a row, so that a row's sums need log2(LP) exchanges and a wave has R = 64 / LP
// rows; a lane has V pairs of the row in each of its NC chunks, as two pieces of V adjacent elements: both halves of its pairs, so
// turning takes no exchange.  A wave works on one token at a time, R heads of one kind in a round: cos and sin are loaded once for all heads,
// what a round does is the same for all its lanes, and values pass without arithmetic.  IT rounds are read before the first is worked on.
// us, floor at the rate of a large copy (5.19 TB/s): 48 heads of 128 bfloat16, 8192 tokens, heads first 38.4, 38.8, its gradient 59.5, 58.2; 48 heads of 64 float32,
// 4096 tokens 20.2, 19.4 and 27.0, 29.1; 24 heads of 80 bfloat16 on three axes, 9477 tokens 18.0, 14.0 and 30.5, 21.0 (22.5 and 31.8 in a
// training step, whose other tensors leave less of these in the caches): a row of 80 keeps ten of sixteen lanes busy, and arithmetic bounds its gradient.
//
// Supplied by the host: TYPE, STYPE (types of x and of the scales), D, ROT, V, LP, NC, IT, PAIRED, FIRST, NORM, STREAMS, AXES, ENDS, POS (positions are
// given), BACK, SUMS (BACK with gradients of the scales).
// a[0] x  a[1] q  a[2] k  a[3] v  (BACK: dq, dk, dv, null where missing; forward: null where not wanted)  a[4] scale of q  a[5] of k  a[6] table  a[7] positions
// a[8] tokens  a[9] tokens of a sequence  a[10] HQ  a[11] HK  a[12] HV  a[13] eps (double bits)  a[14] positions of an axis  a[15] rows of the table
// a[16] dx  a[17] partial sums [workgroup][2][D]
// Waves of the grid's x axis take tokens, its y axis the rounds of a token.
#ifndef FOLD
struct Params { void* a[18]; };
typedef typename mjt_el<TYPE>::raw raw;
typedef typename mjt_el<STYPE>::raw raws;
#define R (64 / LP)                    // rows of a wave

// A chunk's V pairs are one group of neighbours; or with PAIRED, where both elements of a pair lie in one piece, one of each piece, which are then half a
// row apart if they are whole 16-byte accesses: side by side every access of a wave takes half of each line, and those past the caches read
// lines twice (us side by side / apart: 48 heads of 128 bfloat16, 8192 tokens 47.4 / 38.9, 48 heads of 64 float32, 4096 tokens 23.4 / 19.8, gradient 32.5 / 26.9).
// Smaller pieces side by side are one access (24 heads of 80 bfloat16 on three axes, 9477 tokens 18.0 / 18.7, gradient 30.5 / 32.1).
constexpr bool APART = V * sizeof(raw) >= 16;
constexpr int GN = PAIRED && APART ? 2 : 1, G = V / GN;

// whether every axis ends with a whole group
template <int N> constexpr bool mjt_whole(const int (&ends)[N]) {
    for (int a = 0; a < N; a++)
        if (ends[a] % G) return false;
    return true;
}
template <int CTRL> __device__ __forceinline__ float mjt_dpp(float v) { return __uint_as_float((unsigned)__builtin_amdgcn_mov_dpp((int)__float_as_uint(v), CTRL, 0xf, 0xf, true)); }
// The sum over the LP lanes of a row, in all of them: neighbours, pairs, and then mirrors of 8 and 16 lanes, whose halves are uniform by then.
__device__ __forceinline__ float mjt_row_sum(float v) {
    if (LP > 1) v += mjt_dpp<0xB1>(v);
    if (LP > 2) v += mjt_dpp<0x4E>(v);
    if (LP > 4) v += mjt_dpp<0x141>(v);
    if (LP > 8) v += mjt_dpp<0x140>(v);
#pragma unroll
    for (int off = 16; off < LP; off *= 2) v += __shfl_xor(v, off, 64);
    return v;
}
// (the instruction takes a subnormal number for zero: without eps, rows of elements below 1e-19)
__device__ __forceinline__ float mjt_rsqrt(float v) {
    const bool low = v < 0x1p-96f;
    const float r = __builtin_amdgcn_rsqf(low ? v * 0x1p64f : v);
    return low ? r * 0x1p32f : r;
}
template <int I> struct mjt_ic { static constexpr int v = I; };
template <int I, int N, class F> __device__ __forceinline__ void mjt_each(F&& f) {
    if constexpr (I < N) {
        f(mjt_ic<I>());
        mjt_each<I + 1, N>(f);
    }
}

extern "C" __global__ __launch_bounds__(256) void ENTRY(Params p) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int sub = lane / LP, own = lane % LP;
    const unsigned tokens = (unsigned)(unsigned long long)p.a[8], seq = (unsigned)(unsigned long long)p.a[9];
    const int HQ = (int)(long long)p.a[10], HK = (int)(long long)p.a[11], HV = (int)(long long)p.a[12], H = HQ + HK + HV;
    const int rounds_q = (HQ + R - 1) / R, rounds_k = rounds_q + (HK + R - 1) / R, rounds = rounds_k + (HV + R - 1) / R;
    const float eps = (float)__longlong_as_double((long long)p.a[13]);
    const raw* __restrict__ x = (const raw*)p.a[0];
    // the lane's pieces of a row: V elements from first[c] and from second[c] on; chunks past the row are those of chunk 0 and count nothing
    int first[NC], second[NC], pair[NC][GN];
    bool in[NC], turned[NC][GN];
#pragma unroll
    for (int c = 0; c < NC; c++) {
        int at = (c * LP + own) * V;
        in[c] = at < D / 2;
        at = in[c] ? at : 0;
        // pieces of a pair's halves; of neighbours, or of what is not turned, in front and behind where they are whole accesses, otherwise side by side
        const bool halves = !PAIRED && at < ROT / 2;
        first[c] = halves || GN == 2 ? at : APART ? at + ROT / 2 : 2 * at;
        second[c] = halves ? at + ROT / 2 : APART ? at + D / 2 : 2 * at + V;
#pragma unroll
        for (int g = 0; g < GN; g++) {
            const int p0 = GN == 2 ? (g ? second[c] : first[c]) / 2 : at;
            turned[c][g] = p0 < ROT / 2;
            pair[c][g] = turned[c][g] ? p0 : 0;
        }
    }
    // element i of piece e of a chunk, e and i of pair j's two elements: its piece's j-th each, or (neighbours) elements 2 j and 2 j + 1 of the 2 V
    constexpr auto piece = [](int j, int e) { return PAIRED ? (2 * j + e) / V : e; };
    constexpr auto place = [](int j, int e) { return PAIRED ? (2 * j + e) % V : j; };
#if BACK && SUMS
    float ds[2][NC][2][V];
#pragma unroll
    for (int k = 0; k < 2; k++)
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int i = 0; i < V; i++) ds[k][c][0][i] = ds[k][c][1][i] = 0.0f;
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
            constexpr bool whole = mjt_whole(ends);
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int g = 0; g < GN; g++) {
                    if constexpr (whole) {                      // the group's pairs lie on one axis
                        unsigned row = at[0];
#pragma unroll
                        for (int a = 1; a < AXES; a++) row = pair[c][g] >= ends[a - 1] ? at[a] : row;
                        const bool there = row < rows;
                        const mjt_els<2, 2 * G> f = *(const mjt_els<2, 2 * G>*)(table + ((long long)(there ? row : 0) * (ROT / 2) + pair[c][g]) * 2);
#pragma unroll
                        for (int i = 0; i < G; i++) {
                            cs[c][g * G + i] = turned[c][g] ? there ? f.v[2 * i] : __builtin_nanf("") : 1.0f;
                            sn[c][g * G + i] = turned[c][g] ? f.v[2 * i + 1] : 0.0f;
                        }
                    } else
#pragma unroll
                        for (int i = 0; i < G; i++) {
                            unsigned row = at[0];
#pragma unroll
                            for (int a = 1; a < AXES; a++) row = pair[c][g] + i >= ends[a - 1] ? at[a] : row;
                            const bool there = row < rows;
                            const float* f = table + ((long long)(there ? row : 0) * (ROT / 2) + pair[c][g] + i) * 2;
                            cs[c][g * G + i] = turned[c][g] ? there ? f[0] : __builtin_nanf("") : 1.0f;
                            sn[c][g * G + i] = turned[c][g] ? f[1] : 0.0f;
                        }
                }
        }
#else
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int i = 0; i < V; i++) cs[c][i] = 1.0f, sn[c][i] = 0.0f;
#endif
        const unsigned b = FIRST ? t / seq : 0, s = FIRST ? t - b * seq : 0;
        for (int q0 = blockIdx.y * IT; q0 < rounds; q0 += gridDim.y * IT) {
        // what IT rounds read is asked for before the first of them is worked on: R heads of one kind each, those past the last repeat it
        mjt_els<TYPE, V> in0[IT][NC], in1[IT][NC];
#if BACK
        mjt_els<TYPE, V> g0[IT][NC], g1[IT][NC];
#endif
        raw* to[IT];                                           // where the lane's row goes, null where nowhere
        bool real[IT], given[IT];
#pragma unroll
        for (int it = 0; it < IT; it++) {
            const int q = q0 + it < rounds ? q0 + it : rounds - 1;
            const int kind = q < rounds_q ? 0 : q < rounds_k ? 1 : 2, h0 = (q - (kind == 0 ? 0 : kind == 1 ? rounds_q : rounds_k)) * R;
            const int heads = kind == 0 ? HQ : kind == 1 ? HK : HV, before = kind == 0 ? 0 : kind == 1 ? HQ : HQ + HK;
            raw* part = (raw*)(kind == 0 ? p.a[1] : kind == 1 ? p.a[2] : p.a[3]);             // the kind's result, or its gradient
            given[it] = part != nullptr;
            real[it] = h0 + sub < heads && q0 + it < rounds;
            const int h = h0 + sub < heads ? h0 + sub : heads - 1;
            const raw* from = x + ((long long)t * H + before + h) * D;
            part += (FIRST ? ((long long)b * heads + h) * seq + s : (long long)t * heads + h) * D;
#if BACK
            const raw* grad = given[it] ? part : from;
            to[it] = real[it] && p.a[16] ? (raw*)p.a[16] + ((long long)t * H + before + h) * D : nullptr;
            if (kind == 2) from = grad;                        // (nothing of the values themselves is needed)
#else
            to[it] = real[it] && given[it] ? part : nullptr;
#endif
#pragma unroll
            for (int c = 0; c < NC; c++) {
                in0[it][c] = mjt_get<TYPE, V>(from + first[c]);
                in1[it][c] = mjt_get<TYPE, V>(from + second[c]);
#if BACK
                g0[it][c] = mjt_get<TYPE, V>(grad + first[c]);
                g1[it][c] = mjt_get<TYPE, V>(grad + second[c]);
#endif
            }
        }
        auto write = [&](raw* at, const mjt_els<TYPE, V> (&o)[NC][2]) {
            if (at)
#pragma unroll
                for (int c = 0; c < NC; c++)
                    if (in[c]) {
                        mjt_set(at + first[c], o[c][0]);
                        mjt_set(at + second[c], o[c][1]);
                    }
        };
        auto copy = [&](auto itc) {                            // a row of values, or of zeros where no gradient arrives
            constexpr int it = decltype(itc)::v;
            mjt_els<TYPE, V> o[NC][2];
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int i = 0; i < V; i++) {
                    o[c][0].v[i] = !BACK || given[it] ? in0[it][c].v[i] : raw(0);
                    o[c][1].v[i] = !BACK || given[it] ? in1[it][c].v[i] : raw(0);
                }
            write(to[it], o);
        };
        auto normed = [&](auto itc, auto kindc) {
            constexpr int it = decltype(itc)::v, K = decltype(kindc)::v;
            float u[NC][2][V], sc[NC][2][V];
#if NORM
            const raws* scale = (const raws*)p.a[4 + K];
#pragma unroll
            for (int c = 0; c < NC; c++) {
                const mjt_els<STYPE, V> s0 = *(const mjt_els<STYPE, V>*)(scale + first[c]), s1 = *(const mjt_els<STYPE, V>*)(scale + second[c]);
#pragma unroll
                for (int i = 0; i < V; i++) sc[c][0][i] = mjt_el<STYPE>::up(s0.v[i]), sc[c][1][i] = mjt_el<STYPE>::up(s1.v[i]);
            }
#else
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int i = 0; i < V; i++) sc[c][0][i] = sc[c][1][i] = 1.0f;
#endif
            float sum = 0.0f;
#pragma unroll
            for (int c = 0; c < NC; c++) {
                float mine = 0.0f;
#pragma unroll
                for (int i = 0; i < V; i++) {
                    u[c][0][i] = mjt_el<TYPE>::up(in0[it][c].v[i]);
                    u[c][1][i] = mjt_el<TYPE>::up(in1[it][c].v[i]);
                    mine += u[c][0][i] * u[c][0][i] + u[c][1][i] * u[c][1][i];
                }
                sum += in[c] ? mine : 0.0f;
            }
            const float r = NORM ? mjt_rsqrt(mjt_row_sum(sum) * (1.0f / D) + eps) : 1.0f;
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int i = 0; i < V; i++) u[c][0][i] *= r, u[c][1][i] *= r;              // n
            mjt_els<TYPE, V> o[NC][2];
#if !BACK
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int j = 0; j < V; j++) {
                    const float za = u[c][piece(j, 0)][place(j, 0)] * sc[c][piece(j, 0)][place(j, 0)], zb = u[c][piece(j, 1)][place(j, 1)] * sc[c][piece(j, 1)][place(j, 1)];
                    o[c][piece(j, 0)].v[place(j, 0)] = mjt_el<TYPE>::down(za * cs[c][j] - zb * sn[c][j]);
                    o[c][piece(j, 1)].v[place(j, 1)] = mjt_el<TYPE>::down(za * sn[c][j] + zb * cs[c][j]);
                }
            write(to[it], o);
#else
            float dn[NC][2][V], dot = 0.0f;
#pragma unroll
            for (int c = 0; c < NC; c++) {
                float mine = 0.0f;
#pragma unroll
                for (int j = 0; j < V; j++) {
                    const float ga = mjt_el<TYPE>::up((piece(j, 0) ? g1 : g0)[it][c].v[place(j, 0)]), gb = mjt_el<TYPE>::up((piece(j, 1) ? g1 : g0)[it][c].v[place(j, 1)]);
                    dn[c][piece(j, 0)][place(j, 0)] = ga * cs[c][j] + gb * sn[c][j];
                    dn[c][piece(j, 1)][place(j, 1)] = gb * cs[c][j] - ga * sn[c][j];
                }
#pragma unroll
                for (int e = 0; e < 2; e++)
#pragma unroll
                    for (int i = 0; i < V; i++) {
#if SUMS
                        // (a lane of a head past the last repeats the last one's, and is left out)
                        ds[K][c][e][i] += real[it] ? dn[c][e][i] * u[c][e][i] : 0.0f;
#endif
                        dn[c][e][i] *= sc[c][e][i];
                        mine += dn[c][e][i] * u[c][e][i];
                    }
                dot += in[c] ? mine : 0.0f;
            }
            const float m = NORM ? mjt_row_sum(dot) * (1.0f / D) : 0.0f;
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int e = 0; e < 2; e++)
#pragma unroll
                    for (int i = 0; i < V; i++) o[c][e].v[i] = mjt_el<TYPE>::down(NORM ? r * (dn[c][e][i] - u[c][e][i] * m) : dn[c][e][i]);
            write(to[it], o);
#endif
        };
        mjt_each<0, IT>([&](auto itc) {                        // (what a round is, is the same for the whole wave)
            constexpr int it = decltype(itc)::v;
            const int q = q0 + it;
            if (q >= rounds) return;
            if (q >= rounds_k || (BACK && !given[it])) copy(itc);
            else if (q < rounds_q) normed(itc, mjt_ic<0>());
            else normed(itc, mjt_ic<1>());
        });
        }
    }
#if BACK && SUMS
    __shared__ float part[4][2][D];
#pragma unroll
    for (int k = 0; k < 2; k++)
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int e = 0; e < 2; e++)
#pragma unroll
                for (int i = 0; i < V; i++) {
                    float v = ds[k][c][e][i];
#pragma unroll
                    for (int off = LP; off < 64; off *= 2) v += __shfl_xor(v, off, 64);
                    if (sub == 0 && in[c]) part[wave][k][(e ? second[c] : first[c]) + i] = v;
                }
    __syncthreads();
    float* mine = (float*)p.a[17] + ((long long)blockIdx.y * gridDim.x + blockIdx.x) * 2 * D;
    for (int i = threadIdx.x; i < 2 * D; i += 256) mine[i] = (part[0][0][i] + part[1][0][i]) + (part[2][0][i] + part[3][0][i]);
#endif
}
#else
// dscale[e] = sum over workgroups of part[w][e], e in 0 .. 2 D (the queries' first): 16 columns a workgroup, 64 strips of partial results,
// joined in LDS in a fixed order.
// a[0] part  a[1] dscale of q  a[2] of k (null where not wanted)  a[3] partial results  a[4] D
struct Params { void* a[5]; };
extern "C" __global__ __launch_bounds__(1024) void ENTRY(Params p) {
    const float* __restrict__ part = (const float*)p.a[0];
    const int n = (int)(long long)p.a[3], D = (int)(long long)p.a[4];
    const int strip = threadIdx.x / 16, col = blockIdx.x * 16 + threadIdx.x % 16;
    float sum = 0.0f;
    if (col < 2 * D)
#pragma unroll 8
        for (int w = strip; w < n; w += 64) sum += part[(long long)w * 2 * D + col];
    __shared__ float sums[64][17];
    sums[strip][threadIdx.x % 16] = sum;
    __syncthreads();
    if (strip == 0 && col < 2 * D) {
        float total = 0.0f;
#pragma unroll
        for (int s = 0; s < 64; s++) total += sums[s][threadIdx.x];
        typename mjt_el<STYPE>::raw* to = (typename mjt_el<STYPE>::raw*)(col < D ? p.a[1] : p.a[2]);
        if (to) to[col < D ? col : col - D] = mjt_el<STYPE>::down(total);
    }
}
#endif

// Element-wise halves of a gated layer whose product is a kernel of its own.  both[row][2 F] holds gate and up side by side in 32 bits.
// BACK 0:  y[row][f] = act(gate) * up
// BACK 1:  d[row][f] = dy * up * act'(gate),  d[row][F + f] = dy * act(gate)
// d is rounded to the operands' type: dx and dw are products of 16-bit operands then, and twice as many MFMAs if it were not (d as two parts).  It makes the error of
// dx and dw against 64 bits 1.35 to 1.4 times that of products of an exact d, whose results are rounded all the same.  float32 rounds nothing here.
// Memory bounds it: 8192 x 5632 bfloat16 with dy, 646 MB, 101 us (6.4 TB/s; 110 to 130 through the caches).
// Supplied by the host: TYPE (type of y, dy and d), V (adjacent elements a lane takes: 4 or 1), ACT, BACK, STREAMS.
// a[0] both  a[1] y or dy  a[2] d  a[3] rows * F / V  a[4] F / V
struct Params { void* a[5]; };

extern "C" __global__ __launch_bounds__(256) void ENTRY(Params p) {
    typedef typename mjt_el<TYPE>::raw raw;
    const long long n = (long long)p.a[3], per = (long long)p.a[4];
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
        const long long row = i / per, at = (i - row * per) * V, F = per * V;
        const float* both = (const float*)p.a[0] + row * 2 * F + at;
        const mjt_els<2, V> gate = mjt_get<2, V>(both), up = mjt_get<2, V>(both + F);
        mjt_els<TYPE, V>* y = (mjt_els<TYPE, V>*)((raw*)p.a[1] + row * F + at);
        mjt_els<TYPE, V> o, o2;
#if BACK
        const mjt_els<TYPE, V> dy = mjt_get<TYPE, V>(y);
#endif
#pragma unroll
        for (int j = 0; j < V; j++) {
            const mjt_gate a = mjt_activate(gate.v[j]);
#if BACK
            const float g = mjt_el<TYPE>::up(dy.v[j]);
            o.v[j] = mjt_el<TYPE>::down(g * up.v[j] * a.d);
            o2.v[j] = mjt_el<TYPE>::down(g * a.a);
#else
            o.v[j] = mjt_el<TYPE>::down(a.a * up.v[j]);
#endif
        }
#if BACK
        raw* d = (raw*)p.a[2] + row * 2 * F + at;
        mjt_set(d, o);
        mjt_set(d + F, o2);
#else
        mjt_set(y, o);
#endif
    }
}

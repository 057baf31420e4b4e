// The activations of gated layers, and the element-wise passes around their products where those are kernels of their own.
//   ACT: 0 silu g s(g)   1 gelu g P(g)   2 relu max(g, 0)   3 sigmoid s(g);   s(g) = 1 / (1 + exp(-g)), P the normal distribution's mass below g
// 32 bits throughout.  exp overflows to infinity for very negative g, where s is 0; silu's g s(g) would be -inf * 0 at g = -inf and
// is 0 there as its limit; gelu's likewise.
struct mjt_gate { float a, d; };           // the activation and its derivative

__device__ __forceinline__ mjt_gate mjt_activate(float g) {
#if ACT == 2
    return {g < 0.0f ? 0.0f : g, g > 0.0f ? 1.0f : 0.0f};                     // (a NaN stays one)
#elif ACT == 1
    const float below = 0.5f * erfcf(-0.70710678118654752f * g), at = 0.39894228040143268f * expf(-0.5f * g * g);
    const bool none = below == 0.0f;                                          // far below zero
    return {none ? 0.0f : g * below, none || at == 0.0f ? below : below + g * at};
#else
    const float e = expf(-g), s = 1.0f / (1.0f + e);
    const bool none = s == 0.0f;
    const float rest = none ? 1.0f : e * s;                                   // 1 - s without its cancellation
#if ACT == 3
    return {s, s * rest};
#else
    return {none ? 0.0f : g * s, none ? 0.0f : rest == 0.0f ? s : s * (1.0f + g * rest)};
#endif
#endif
}

// The activations of gated layers, and the element-wise passes around their products where those are kernels of their own.
//   ACT: 0 silu g s(g)   1 gelu g P(g)   2 relu max(g, 0)   3 sigmoid s(g);   s(g) = 1 / (1 + exp(-g)), P the normal distribution's mass below g
// 32 bits throughout.  exp overflows to infinity for very negative g, where s is 0; silu's g s(g) would be -inf * 0 at g = -inf and
// is 0 there as its limit; gelu's likewise.
struct mjt_gate { float a, d; };           // the activation and its derivative

__device__ __forceinline__ mjt_gate mjt_activate(float g) {
#if ACT == 2
    return {g < 0.0f ? 0.0f : g, g > 0.0f ? 1.0f : 0.0f};                     // (a NaN stays one)
#elif ACT == 1
    // P(-z) = exp(-z^2 / 2) q(1 / (1 + 0.3 z)) for z >= 0: q, a polynomial of degree 8, is fitted to the scaled complementary error function with the
    // least largest relative error, 5.8e-8 up to z = 14.4, where P leaves the range.  (erfcf and expf here took 414 us for 8192 x 2048 -> 5632 bfloat16,
    // silu 344.)
    const float z = __builtin_fabsf(g), t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3f, z, 1.0f)), bell = __builtin_amdgcn_exp2f(-0.72134752044448170f * g * g);
    const float q = __builtin_fmaf(__builtin_fmaf(__builtin_fmaf(__builtin_fmaf(__builtin_fmaf(__builtin_fmaf(__builtin_fmaf(__builtin_fmaf(0.0384075716f, t, -0.169308305f), t, 0.228953421f), t, -0.0768414438f), t, 0.142766431f), t, 0.0945854038f), t, 0.121945374f), t, 0.119484194f), t, 7.37314485e-06f);
    const float tail = bell == 0.0f ? 0.0f : bell * q, below = g < 0.0f ? tail : 1.0f - tail, at = 0.39894228040143268f * bell;
    const bool none = g < 0.0f && tail == 0.0f;                               // far below zero
    return {none ? 0.0f : g * below, at == 0.0f ? below : below + g * at};
#else
    // exp and the quotient from the hardware's exp2 and reciprocal, one unit in the last place each: with expf and a division an epilogue of
    // 256 x 128 results took 8 us, a tenth of its products
    const float e = __builtin_amdgcn_exp2f(-1.44269504088896341f * g), s = __builtin_amdgcn_rcpf(1.0f + e);
    const bool none = s == 0.0f;
    const float rest = none ? 1.0f : e * s;                                   // 1 - s without its cancellation
#if ACT == 3
    return {s, s * rest};
#else
    return {none ? 0.0f : g * s, none ? 0.0f : rest == 0.0f ? s : s * (1.0f + g * rest)};
#endif
#endif
}

// Elements of the kernels for transformer layers: float types by number (0 bfloat16, 1 float16, 2 float32), computed with in 32 bits and
// rounded to nearest even where they are stored (these results are new ones, so nothing asks for the truncation to bfloat16 that the
// element-wise vocabulary keeps; half its error, and no drift towards zero in sums of gradients).
template <int T> struct mjt_el;
template <> struct mjt_el<0> {
    typedef unsigned short raw;
    static __device__ __forceinline__ float up(raw v) { return __uint_as_float((unsigned)v << 16); }
    static __device__ __forceinline__ raw down(float v) { return __builtin_bit_cast(raw, (__bf16)v); }
};
template <> struct mjt_el<1> {
    typedef unsigned short raw;
    static __device__ __forceinline__ float up(raw v) { return (float)__builtin_bit_cast(_Float16, v); }
    static __device__ __forceinline__ raw down(float v) { return __builtin_bit_cast(raw, (_Float16)v); }
};
template <> struct mjt_el<2> {
    typedef float raw;
    static __device__ __forceinline__ float up(raw v) { return v; }
    static __device__ __forceinline__ raw down(float v) { return v; }
};
// N adjacent elements, one access (two of 16 bytes for 32)
template <int T, int N> struct alignas(N * sizeof(typename mjt_el<T>::raw)) mjt_els {
    typename mjt_el<T>::raw v[N];
};

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

// Reads and writes of a kernel that passes over more memory than the caches hold, once (STREAMS 1, which the host sets from 32 MB on): past
// the caches' replacement, so that what is read does not drive out what is being written (us, dropout of 8192 x 4096 bfloat16 with a residual, ordinary /
// loads so / both so 46.4 / 35.9 / 31.8; without one 37.7 / 28.1 / 25.4; float32 51.9 / 59.2 / 49.7).
#ifndef STREAMS
#define STREAMS 0
#endif
typedef unsigned mjt_words1;
typedef unsigned mjt_words2 __attribute__((ext_vector_type(2)));
typedef unsigned mjt_words4 __attribute__((ext_vector_type(4)));
template <class Words, class E> __device__ __forceinline__ void mjt_stream_in(E& to, const void* from) {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(E) / sizeof(Words)); i++) ((Words*)&to)[i] = __builtin_nontemporal_load((const Words*)from + i);
}
template <class Words, class E> __device__ __forceinline__ void mjt_stream_out(void* to, const E& from) {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(E) / sizeof(Words)); i++) __builtin_nontemporal_store(((const Words*)&from)[i], (Words*)to + i);
}
template <int T, int N> __device__ __forceinline__ mjt_els<T, N> mjt_get(const void* from) {
    constexpr int BYTES = (int)sizeof(mjt_els<T, N>);
    mjt_els<T, N> v;
    if constexpr (!STREAMS || BYTES < 4) v = *(const mjt_els<T, N>*)from;
    else if constexpr (BYTES % 16 == 0) mjt_stream_in<mjt_words4>(v, from);
    else if constexpr (BYTES % 8 == 0) mjt_stream_in<mjt_words2>(v, from);
    else mjt_stream_in<mjt_words1>(v, from);
    return v;
}
template <int T, int N> __device__ __forceinline__ void mjt_set(void* to, const mjt_els<T, N>& v) {
    constexpr int BYTES = (int)sizeof(mjt_els<T, N>);
    if constexpr (!STREAMS || BYTES < 4) *(mjt_els<T, N>*)to = v;
    else if constexpr (BYTES % 16 == 0) mjt_stream_out<mjt_words4>(to, v);
    else if constexpr (BYTES % 8 == 0) mjt_stream_out<mjt_words2>(to, v);
    else mjt_stream_out<mjt_words1>(to, v);
}

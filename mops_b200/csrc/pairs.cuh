// Two values at a time: sm_100 multiplies and adds pairs of f32 in one instruction (fma.rn.f32x2), each value rounded as by itself.
#ifndef MOPS_B200_PAIRS_CUH
#define MOPS_B200_PAIRS_CUH

#include "arrays.hpp"

namespace mops_b200 {

template <typename S> struct Pair {
    S x, y;
};

template <typename S> __device__ __forceinline__ Pair<S> both(S v) { return {v, v}; }
template <typename S> __device__ __forceinline__ S total(Pair<S> v) { return v.x + v.y; }

__device__ __forceinline__ uint64_t packed(Pair<float> v) {
    uint64_t u;
    asm("mov.b64 %0, {%1, %2};" : "=l"(u) : "f"(v.x), "f"(v.y));
    return u;
}
__device__ __forceinline__ Pair<float> unpacked(uint64_t u) {
    Pair<float> v;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(u));
    return v;
}
// a b + c
__device__ __forceinline__ Pair<float> fma2(Pair<float> a, Pair<float> b, Pair<float> c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(packed(a)), "l"(packed(b)), "l"(packed(c)));
    return unpacked(d);
}
__device__ __forceinline__ Pair<float> operator*(Pair<float> a, Pair<float> b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(packed(a)), "l"(packed(b)));
    return unpacked(d);
}
__device__ __forceinline__ Pair<float> operator+(Pair<float> a, Pair<float> b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(packed(a)), "l"(packed(b)));
    return unpacked(d);
}
__device__ __forceinline__ Pair<double> fma2(Pair<double> a, Pair<double> b, Pair<double> c) {
    return {fma(a.x, b.x, c.x), fma(a.y, b.y, c.y)};
}
__device__ __forceinline__ Pair<double> operator*(Pair<double> a, Pair<double> b) { return {a.x * b.x, a.y * b.y}; }
__device__ __forceinline__ Pair<double> operator+(Pair<double> a, Pair<double> b) { return {a.x + b.x, a.y + b.y}; }
template <typename S> __device__ __forceinline__ Pair<S> operator*(Pair<S> a, S b) { return a * both(b); }

// Two neighbouring values of an array, and back.
template <typename T> __device__ __forceinline__ Pair<Sum<T>> widen2(const T* v) { return {widen(v[0]), widen(v[1])}; }
template <> __device__ __forceinline__ Pair<float> widen2<__nv_bfloat16>(const __nv_bfloat16* v) {
    const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(v));
    return {f.x, f.y};
}
template <> __device__ __forceinline__ Pair<float> widen2<__half>(const __half* v) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(v));
    return {f.x, f.y};
}
template <typename T> __device__ __forceinline__ void narrow2(T* to, Pair<Sum<T>> v) { to[0] = narrow<T>(v.x), to[1] = narrow<T>(v.y); }
template <> __device__ __forceinline__ void narrow2<__nv_bfloat16>(__nv_bfloat16* to, Pair<float> v) {
    *reinterpret_cast<__nv_bfloat162*>(to) = __floats2bfloat162_rn(v.x, v.y);
}
template <> __device__ __forceinline__ void narrow2<__half>(__half* to, Pair<float> v) {
    *reinterpret_cast<__half2*>(to) = __floats2half2_rn(v.x, v.y);
}

} // namespace mops_b200

#endif

// Elements of activation rows (f32, f16, bf16) as floats, one or several at a time.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

namespace qb {

template <class T>
__device__ __forceinline__ float to_float(T x);
template <>
__device__ __forceinline__ float to_float(float x) { return x; }
template <>
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

// One rounding to nearest.
template <class T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float(float x) { return x; }
template <>
__device__ __forceinline__ __half from_float(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float(float x) { return __float2bfloat16_rn(x); }

// N consecutive elements as one access (N * sizeof(T) <= 16) or, above that, as 16-byte ones.
template <class T, int N>
struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) Pack {
    T v[N];
};

// The elements as floats, and floats with one rounding each, two 16-bit ones in one conversion.
template <class T, int N>
__device__ __forceinline__ void to_floats(const Pack<T, N>& w, float (&x)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = to_float(w.v[i]);
}
template <int N>
__device__ __forceinline__ Pack<float, N> from_floats(const float (&x)[N], float) {
    Pack<float, N> w;
#pragma unroll
    for (int i = 0; i < N; ++i) w.v[i] = x[i];
    return w;
}
template <int N>
__device__ __forceinline__ Pack<__half, N> from_floats(const float (&x)[N], __half) {
    Pack<__half, N> w;
    if constexpr (N == 1) {
        w.v[0] = __float2half_rn(x[0]);
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 2) *reinterpret_cast<__half2*>(&w.v[i]) = __floats2half2_rn(x[i], x[i + 1]);
    }
    return w;
}
template <int N>
__device__ __forceinline__ Pack<__nv_bfloat16, N> from_floats(const float (&x)[N], __nv_bfloat16) {
    Pack<__nv_bfloat16, N> w;
    if constexpr (N == 1) {
        w.v[0] = __float2bfloat16_rn(x[0]);
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 2) *reinterpret_cast<__nv_bfloat162*>(&w.v[i]) = __floats2bfloat162_rn(x[i], x[i + 1]);
    }
    return w;
}

template <class T, int N>
__device__ __forceinline__ void store_row(T* p, const float (&x)[N], bool aligned) {
    if (aligned) {
        *reinterpret_cast<Pack<T, N>*>(p) = from_floats(x, T());
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) p[i] = from_float<T>(x[i]);
    }
}

// max that keeps a NaN
__device__ __forceinline__ float max_or_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

}  // namespace qb

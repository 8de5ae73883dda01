// Element types of the operators beside the engine: fp32, fp16 (results saturate) and bf16 arrays, a 16-byte piece at a time.
#pragma once
#include "common.cuh"

namespace ts2 {

template <class T>
__device__ __forceinline__ float widen(T v) { return (float)v; }
template <class T>
__device__ __forceinline__ T narrow(float v);
template <>
__device__ __forceinline__ float narrow<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half narrow<__half>(float v) { return __low2half(sat_half2(v, v)); }
template <>
__device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <class T, int VEC>
struct alignas(VEC * sizeof(T)) Piece {
    T v[VEC];
};

} // namespace ts2

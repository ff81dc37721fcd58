// zq_elem.cuh -- fp32 / fp16 / bf16 element access shared by the operators
// around the quantized matmul (norm, low-rank adapters, log probabilities).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

namespace zq {

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

template <class T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Elements of T in a 16-byte access.
template <class T>
constexpr int kElemsPer16 = 16 / (int)sizeof(T);

// N elements as one naturally aligned memory access (N * sizeof(T) <= 16).
template <class T, int N>
struct alignas(N * sizeof(T)) Pack {
    T e[N];
};

}  // namespace zq

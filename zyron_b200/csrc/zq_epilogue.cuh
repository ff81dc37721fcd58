// zq_epilogue.cuh -- what a matmul does with a finished value before it is
// stored (zq_matmul_epilogue), shared by the kernels of every size:
//
//   y = round_T( act( fl(fl(acc * s_row) * s_col) (+ bias) ) + residual )
//
//   gelu(v) = v / (1 + exp(-2 sqrt(2/pi) (v + 0.044715 v^3)))
//   silu(v) = v / (1 + exp(-v)),  relu(v) = max(v, 0)
//
// gelu is the tanh form, 0.5 v (1 + tanh(u)) = v / (1 + exp(-2u)): the quotient
// needs one exponential and one reciprocal and, unlike 1 + tanh(u), loses
// nothing where v is far below 0.  Everything is fp32; the one rounding to the
// stored type is the last step.
#pragma once

#include "zq_common.cuh"
#include "zq_elem.cuh"
#include "zq_kernels.h"

namespace zq {

__device__ __forceinline__ float epi_gelu(float v) {
    // -2 sqrt(2/pi) and -2 sqrt(2/pi) 0.044715
    const float t = v * fmaf(-0.07135481627f, v * v, -1.59576912161f);
    return __fdividef(v, 1.0f + expf(t));
}
__device__ __forceinline__ float epi_silu(float v) { return __fdividef(v, 1.0f + expf(-v)); }
__device__ __forceinline__ float epi_relu(float v) { return v < 0.0f ? 0.0f : v; }  // NaN stays

template <int N>
__device__ __forceinline__ void epi_activate(int activation, float (&v)[N]) {
    if (activation == ZQ_ACT_GELU) {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = epi_gelu(v[j]);
    } else if (activation == ZQ_ACT_SILU) {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = epi_silu(v[j]);
    } else if (activation == ZQ_ACT_RELU) {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = epi_relu(v[j]);
    }
}

// Element i of the residual, and one result stored at i, in the stored type.
__device__ __forceinline__ float epi_residual(const Epilogue& e, size_t i) {
    if (e.dtype == ZQ_DTYPE_F32) return load_l2(static_cast<const float*>(e.residual) + i);
    if (e.dtype == ZQ_DTYPE_F16) return to_float(load_l2(static_cast<const __half*>(e.residual) + i));
    return to_float(load_l2(static_cast<const __nv_bfloat16*>(e.residual) + i));
}
__device__ __forceinline__ void epi_store(const Epilogue& e, void* y, size_t i, float v) {
    if (e.dtype == ZQ_DTYPE_F32)
        static_cast<float*>(y)[i] = v;
    else if (e.dtype == ZQ_DTYPE_F16)
        static_cast<__half*>(y)[i] = __float2half_rn(v);
    else
        static_cast<__nv_bfloat16*>(y)[i] = __float2bfloat16_rn(v);
}

// Activation, residual and store of one value at (row, col) of y [M][n].
__device__ __forceinline__ void epi_finish(const Epilogue& e, void* y, int n, int row, int col, float value) {
    float v[1] = {value};
    epi_activate(e.activation, v);
    if (e.residual) v[0] += epi_residual(e, (size_t)row * (size_t)e.ld_residual + (size_t)col);
    epi_store(e, y, (size_t)row * (size_t)n + (size_t)col, v[0]);
}

// 16 consecutive elements of a row on the 16-byte grid: raw residual words
// (four 16-byte loads of fp32, two of 16-bit types), and the sum and store.
struct Epi16 {
    uint4 w[4];
};
__device__ __forceinline__ void epi_load16(const Epilogue& e, size_t i, Epi16& r) {
    const bool full = e.dtype == ZQ_DTYPE_F32;
    const uint4* p = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(e.residual) + i * (full ? 4 : 2));
    r.w[0] = load_l2(p);
    r.w[1] = load_l2(p + 1);
    if (full) {
        r.w[2] = load_l2(p + 2);
        r.w[3] = load_l2(p + 3);
    }
}
template <class T>
__device__ __forceinline__ void epi_add_halves(const Epi16& r, float (&v)[16]) {
    Pack<T, 8> p;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        memcpy(&p, &r.w[k], 16);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[8 * k + j] += to_float(p.e[j]);
    }
}
template <class T>
__device__ __forceinline__ void epi_store_halves(void* y, size_t i, const float (&v)[16]) {
    Pack<T, 8> p;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
        for (int j = 0; j < 8; ++j) p.e[j] = from_float<T>(v[8 * k + j]);
        reinterpret_cast<Pack<T, 8>*>(static_cast<T*>(y) + i)[k] = p;
    }
}
__device__ __forceinline__ void epi_add16(const Epilogue& e, const Epi16& r, float (&v)[16]) {
    if (e.dtype == ZQ_DTYPE_F32) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            v[4 * k] += __uint_as_float(r.w[k].x);
            v[4 * k + 1] += __uint_as_float(r.w[k].y);
            v[4 * k + 2] += __uint_as_float(r.w[k].z);
            v[4 * k + 3] += __uint_as_float(r.w[k].w);
        }
    } else if (e.dtype == ZQ_DTYPE_F16) {
        epi_add_halves<__half>(r, v);
    } else {
        epi_add_halves<__nv_bfloat16>(r, v);
    }
}
__device__ __forceinline__ void epi_store16(const Epilogue& e, void* y, size_t i, const float (&v)[16]) {
    if (e.dtype == ZQ_DTYPE_F32) {
        float4* p = reinterpret_cast<float4*>(static_cast<float*>(y) + i);
#pragma unroll
        for (int k = 0; k < 4; ++k) p[k] = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
    } else if (e.dtype == ZQ_DTYPE_F16) {
        epi_store_halves<__half>(y, i, v);
    } else {
        epi_store_halves<__nv_bfloat16>(y, i, v);
    }
}

}  // namespace zq

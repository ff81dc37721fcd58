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

// float(acc) * s_row * s_col, each product rounded, a NaN being any NaN.
__device__ __forceinline__ float epi_value(int32_t acc, float s_row, float s_col) {
    return __fmul_rn(__fmul_rn(__int2float_rn(acc), s_row), s_col);
}

// v / (1 + 2^t): the base-2 exponential and the reciprocal of the special
// function unit (2^-22.5 and 2^-23 off), each one instruction.  A quotient below
// 2^-126 is 0, so gelu and silu are 0 from about -10.0 and -87.3 down, where they
// are 2^-122 and 2^-119.
__device__ __forceinline__ float epi_logistic(float v, float t) {
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    return v * r;
}
__device__ __forceinline__ float epi_gelu(float v) {
    // log2(e) times -2 sqrt(2/pi) 0.044715 and -2 sqrt(2/pi)
    return epi_logistic(v, v * fmaf(-0.10294324f, v * v, -2.3022082f));
}
__device__ __forceinline__ float epi_silu(float v) { return epi_logistic(v, v * -1.4426950f); }
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

// A warp's block of 32 rows x 16 columns whose rows lie on no grid: turned
// around in shared memory, so that 16 lanes take one row's columns and their
// accesses merge (333 x 2050 x 1003 with an fp32 residual took 36 us row by
// lane).  `stage` is the warp's own 32 x kEpiPitch16 floats.
constexpr int kEpiPitch16 = 17;
__device__ __forceinline__ void epi_finish_block(const Epilogue& e, void* y, int n, int row0, int rows, int col0,
                                                 const float (&v)[16], float* stage) {
    const int lane = threadIdx.x & 31;
    __syncwarp();  // the block before has been read
#pragma unroll
    for (int j = 0; j < 16; ++j) stage[lane * kEpiPitch16 + j] = v[j];
    __syncwarp();
    const int col = col0 + (lane & 15), sub = lane >> 4;
    if (col >= n) return;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        float r[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int row = half * 16 + i * 2 + sub;
            r[i] = e.residual && row < rows ? epi_residual(e, (size_t)(row0 + row) * (size_t)e.ld_residual + col) : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int row = half * 16 + i * 2 + sub;
            if (row < rows)
                epi_store(e, y, (size_t)(row0 + row) * (size_t)n + col, stage[row * kEpiPitch16 + (lane & 15)] + r[i]);
        }
    }
}

// The same on the 16-byte grid, 16 bytes a lane: four lanes a row of fp32, two of
// 16 bits, so that the residual's sectors are read once.  Row by lane, every
// 16-byte access of a warp touches 32 rows, and half of each sector that it
// brings is asked for again: 4096 x 4096 x 11008 with an fp32 residual took
// 321 us.  `stage` is 32 x kEpiPitchWide floats.
constexpr int kEpiPitchWide = 20;
struct EpiWide {
    uint4 w[4];
};
__device__ __forceinline__ void epi_load_wide(const Epilogue& e, int row0, int rows, int col0, EpiWide& r) {
    const int lane = threadIdx.x & 31;
    const bool full = e.dtype == ZQ_DTYPE_F32;
    const int sub = full ? lane >> 2 : lane >> 1, each = full ? 8 : 16;
    const int col = col0 + (full ? 4 * (lane & 3) : 8 * (lane & 1));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = i * each + sub;
        if ((full || i < 2) && row < rows)
            r.w[i] = load_l2(reinterpret_cast<const uint4*>(
                static_cast<const uint8_t*>(e.residual) +
                ((size_t)(row0 + row) * (size_t)e.ld_residual + (size_t)col) * (full ? 4 : 2)));
    }
}
template <class T>
__device__ __forceinline__ void epi_put_halves(const Epilogue& e, void* y, int n, int row0, int rows, int col0,
                                               const EpiWide& r, const float* stage) {
    const int lane = threadIdx.x & 31, col = 8 * (lane & 1);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int row = i * 16 + (lane >> 1);
        if (row >= rows) continue;
        const float4 a = *reinterpret_cast<const float4*>(stage + row * kEpiPitchWide + col);
        const float4 b = *reinterpret_cast<const float4*>(stage + row * kEpiPitchWide + col + 4);
        float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        Pack<T, 8> p;
        if (e.residual) {
            memcpy(&p, &r.w[i], 16);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] += to_float(p.e[j]);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) p.e[j] = from_float<T>(v[j]);
        *reinterpret_cast<Pack<T, 8>*>(static_cast<T*>(y) + (size_t)(row0 + row) * (size_t)n + col0 + col) = p;
    }
}
__device__ __forceinline__ void epi_finish_wide(const Epilogue& e, void* y, int n, int row0, int rows, int col0,
                                                const float (&v)[16], const EpiWide& r, float* stage) {
    const int lane = threadIdx.x & 31;
    __syncwarp();  // the block before has been read
#pragma unroll
    for (int j = 0; j < 4; ++j)
        *reinterpret_cast<float4*>(stage + lane * kEpiPitchWide + 4 * j) =
            make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
    __syncwarp();
    if (e.dtype == ZQ_DTYPE_F16) return epi_put_halves<__half>(e, y, n, row0, rows, col0, r, stage);
    if (e.dtype == ZQ_DTYPE_BF16) return epi_put_halves<__nv_bfloat16>(e, y, n, row0, rows, col0, r, stage);
    const int col = 4 * (lane & 3);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = i * 8 + (lane >> 2);
        if (row >= rows) continue;
        float4 o = *reinterpret_cast<const float4*>(stage + row * kEpiPitchWide + col);
        if (e.residual) {
            o.x += __uint_as_float(r.w[i].x);
            o.y += __uint_as_float(r.w[i].y);
            o.z += __uint_as_float(r.w[i].z);
            o.w += __uint_as_float(r.w[i].w);
        }
        *reinterpret_cast<float4*>(static_cast<float*>(y) + (size_t)(row0 + row) * (size_t)n + col0 + col) = o;
    }
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

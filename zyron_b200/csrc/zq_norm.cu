// zq_norm.cu -- root-mean-square norm with the residual's addition and the
// activation quantizer's output (zq_rms_norm_quantize).
//
//   s = x + residual, rounded to the type it is stored in
//   r = fl32(1 / sqrt(mean(s^2) + eps))          mean in 64 bits
//   v = fl32(fl32(s * r) * w)
//   scale = max|v| / 127 (1 for a row of zeros), code = round(v / scale)
//
// The codes and scales are those of quantize_rows over v, bit for bit.  The
// only quantity that depends on the order of a sum is the mean of squares.
// It is summed in 64 bits, where fp32 squares are exact, so r -- and with it
// every code -- does not depend on the launch shape: a last-bit change of r
// would carry values across the codes' rounding borders.
//
// Bound: one read of x and residual and one write of the sum and the codes,
// at about 20 operations an element, so memory bandwidth.  A row stays in the
// registers of one group of threads from its load to its stores.
#include "zq_common.cuh"
#include "zq_elem.cuh"
#include "zq_kernels.h"

namespace zq {

namespace {

// Sum (64-bit) and maximum over the kWarps warps of a row's group.  `part`
// holds one value per warp of the block; each call needs its own.
template <int kWarps>
__device__ __forceinline__ double group_sum(double v, double* part) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (kWarps > 1) {
        const int warp = threadIdx.x >> 5;
        if ((threadIdx.x & 31) == 0) part[warp] = v;
        __syncthreads();
        const int first = warp / kWarps * kWarps;
        v = 0.0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) v += part[first + w];
    }
    return v;
}

template <int kWarps>
__device__ __forceinline__ float group_max(float v, float* part) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    if (kWarps > 1) {
        const int warp = threadIdx.x >> 5;
        if ((threadIdx.x & 31) == 0) part[warp] = v;
        __syncthreads();
        const int first = warp / kWarps * kWarps;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) v = fmaxf(v, part[first + w]);
    }
    return v;
}

__device__ __forceinline__ float row_rstd(double sum, int K, double eps) {
    return (float)__ddiv_rn(1.0, __dsqrt_rn(sum / (double)K + eps));
}

__device__ __forceinline__ float norm_value(float s, float rstd, float w) {
    return __fmul_rn(__fmul_rn(s, rstd), w);
}

// A row of at most 32 * kWarps * kPacks packs of kN elements, held in the
// registers of kWarps warps.  kN is what one memory access carries: 16 bytes
// of T where every row and width allows it, else one element.
template <class T, int kN, int kWarps, int kPacks>
__global__ void __launch_bounds__(kWarps > 8 ? kWarps * 32 : 256)
    rms_norm_quantize_kernel(const NormArgs a) {
    pdl_launch_dependents();
    pdl_wait_primary();
    constexpr int kBlockWarps = kWarps > 8 ? kWarps : 8;
    constexpr int kThreads = 32 * kWarps;
    __shared__ double part_sum[kBlockWarps];
    __shared__ float part_max[kBlockWarps];
    const long long row = (long long)blockIdx.x * (kBlockWarps / kWarps) + threadIdx.x / kThreads;
    const int t = threadIdx.x % kThreads;
    const bool live = row < a.m;
    const int packs = a.k / kN;
    using P = Pack<T, kN>;
    const P* x = reinterpret_cast<const P*>(static_cast<const T*>(a.x) + (live ? row : 0) * a.ldx);
    const P* res = reinterpret_cast<const P*>(static_cast<const T*>(a.residual) + (live ? row : 0) * a.ld_residual);
    P* sum_out = reinterpret_cast<P*>(static_cast<T*>(a.residual_out) + (live ? row : 0) * a.ld_residual_out);

    P v[kPacks];
#pragma unroll
    for (int i = 0; i < kPacks; ++i) {
        const int p = t + i * kThreads;
        if (live && p < packs)
            v[i] = x[p];
        else
#pragma unroll
            for (int j = 0; j < kN; ++j) v[i].e[j] = from_float<T>(0.0f);
    }
    if (a.residual) {
        P r[kPacks];
#pragma unroll
        for (int i = 0; i < kPacks; ++i) {
            const int p = t + i * kThreads;
            if (live && p < packs) r[i] = res[p];
        }
#pragma unroll
        for (int i = 0; i < kPacks; ++i) {
            const int p = t + i * kThreads;
            if (live && p < packs) {
#pragma unroll
                for (int j = 0; j < kN; ++j)
                    v[i].e[j] = from_float<T>(__fadd_rn(to_float(v[i].e[j]), to_float(r[i].e[j])));
                sum_out[p] = v[i];
            }
        }
    }
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < kPacks; ++i)
#pragma unroll
        for (int j = 0; j < kN; ++j) {
            const double d = (double)to_float(v[i].e[j]);
            sum = __fma_rn(d, d, sum);
        }
    sum = group_sum<kWarps>(sum, part_sum);
    const float rstd = row_rstd(sum, a.k, a.eps);

    float n[kPacks][kN];
    float absmax = 0.0f;
#pragma unroll
    for (int i = 0; i < kPacks; ++i) {
        const int p = t + i * kThreads;
        if (!live || p >= packs) continue;
        Pack<float, kN == 1 ? 1 : 4> w[kN == 1 ? 1 : kN / 4];
#pragma unroll
        for (int j = 0; j < (kN == 1 ? 1 : kN / 4); ++j)
            if (a.weight) w[j] = reinterpret_cast<const Pack<float, kN == 1 ? 1 : 4>*>(a.weight + (size_t)p * kN)[j];
#pragma unroll
        for (int j = 0; j < kN; ++j) {
            n[i][j] = norm_value(to_float(v[i].e[j]), rstd, a.weight ? w[j / 4].e[j % 4] : 1.0f);
            absmax = fmaxf(absmax, fabsf(n[i][j]));
        }
    }
    absmax = group_max<kWarps>(absmax, part_max);
    if (!live) return;
    const float scale = zq_scale_from_absmax(absmax, 127.0f);
    const float rcp = zq_quant_rcp(scale);
    if (t == 0) a.row_scale[row] = scale;
    int8_t* q = a.q + row * a.ldq;
    T* normed = a.normed ? static_cast<T*>(a.normed) + row * a.ld_normed : nullptr;
#pragma unroll
    for (int i = 0; i < kPacks; ++i) {
        const int p = t + i * kThreads;
        if (p >= packs) continue;
        Pack<int8_t, kN> c;
        P o;
#pragma unroll
        for (int j = 0; j < kN; ++j) {
            c.e[j] = (int8_t)zq_quantize_value_rcp(n[i][j], scale, rcp, 127);
            o.e[j] = from_float<T>(n[i][j]);
        }
        reinterpret_cast<Pack<int8_t, kN>*>(q)[p] = c;
        if (normed) reinterpret_cast<P*>(normed)[p] = o;
    }
    for (int j = a.k + t; j < a.ldq; j += kThreads) q[j] = 0;
}

// Rows too long for the registers: one block a row that reads the sum three
// times (the second and third time mostly from L2).  Every element stays with
// one thread, so an output may be its own input's buffer.
template <class T>
__global__ void __launch_bounds__(1024) rms_norm_quantize_long_kernel(const NormArgs a) {
    pdl_launch_dependents();
    pdl_wait_primary();
    __shared__ double part_sum[32];
    __shared__ float part_max[32];
    const long long row = blockIdx.x;
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    const T* res = a.residual ? static_cast<const T*>(a.residual) + row * a.ld_residual : nullptr;
    T* sum_out = a.residual ? static_cast<T*>(a.residual_out) + row * a.ld_residual_out : nullptr;
    double sum = 0.0;
    for (int i = threadIdx.x; i < a.k; i += 1024) {
        T v = x[i];
        if (res) {
            v = from_float<T>(__fadd_rn(to_float(v), to_float(res[i])));
            sum_out[i] = v;
        }
        const double d = (double)to_float(v);
        sum = __fma_rn(d, d, sum);
    }
    const float rstd = row_rstd(group_sum<32>(sum, part_sum), a.k, a.eps);
    const T* s = res ? sum_out : x;
    float absmax = 0.0f;
    for (int i = threadIdx.x; i < a.k; i += 1024)
        absmax = fmaxf(absmax, fabsf(norm_value(to_float(s[i]), rstd, a.weight ? a.weight[i] : 1.0f)));
    absmax = group_max<32>(absmax, part_max);
    const float scale = zq_scale_from_absmax(absmax, 127.0f);
    const float rcp = zq_quant_rcp(scale);
    if (threadIdx.x == 0) a.row_scale[row] = scale;
    int8_t* q = a.q + row * a.ldq;
    T* normed = a.normed ? static_cast<T*>(a.normed) + row * a.ld_normed : nullptr;
    for (int i = threadIdx.x; i < a.k; i += 1024) {
        const float n = norm_value(to_float(s[i]), rstd, a.weight ? a.weight[i] : 1.0f);
        q[i] = (int8_t)zq_quantize_value_rcp(n, scale, rcp, 127);
        if (normed) normed[i] = from_float<T>(n);
    }
    for (long long i = a.k + threadIdx.x; i < a.ldq; i += 1024) q[i] = 0;
}

template <class T, int kN, int kWarps, int kPacks>
cudaError_t launch_rows(const NormArgs& a, cudaStream_t stream) {
    constexpr int kRows = kWarps > 8 ? 1 : 8 / kWarps;
    return launch_pdl_kernel(rms_norm_quantize_kernel<T, kN, kWarps, kPacks>,
                             dim3((unsigned)((a.m + kRows - 1) / kRows)), dim3(kWarps > 8 ? kWarps * 32 : 256), 0,
                             stream, a);
}

template <class T, int kN>
cudaError_t launch_width(const NormArgs& a, cudaStream_t stream) {
    // Up to 32 elements a thread; the fewest warps that hold the row.
    constexpr int kPacks = 32 / kN;
    const int packs = a.k / kN;
    if (packs <= 32 * kPacks) return launch_rows<T, kN, 1, kPacks>(a, stream);
    if (packs <= 64 * kPacks) return launch_rows<T, kN, 2, kPacks>(a, stream);
    if (packs <= 128 * kPacks) return launch_rows<T, kN, 4, kPacks>(a, stream);
    if (packs <= 256 * kPacks) return launch_rows<T, kN, 8, kPacks>(a, stream);
    if (packs <= 512 * kPacks) return launch_rows<T, kN, 16, kPacks>(a, stream);
    if (packs <= 1024 * kPacks) return launch_rows<T, kN, 32, kPacks>(a, stream);
    return launch_pdl_kernel(rms_norm_quantize_long_kernel<T>, dim3((unsigned)a.m), dim3(1024), 0, stream, a);
}

bool aligned(const void* p, long long pitch_bytes, size_t to) {
    return (reinterpret_cast<uintptr_t>(p) | (uintptr_t)pitch_bytes) % to == 0;
}

template <class T>
cudaError_t launch_type(const NormArgs& a, cudaStream_t stream) {
    constexpr int kN = kElemsPer16<T>;
    constexpr long long b = sizeof(T);
    const bool wide = a.k % kN == 0 && aligned(a.x, a.ldx * b, 16) && aligned(a.q, a.ldq, kN) &&
                      aligned(a.weight, 0, 16) &&
                      (!a.residual ||
                       (aligned(a.residual, a.ld_residual * b, 16) && aligned(a.residual_out, a.ld_residual_out * b, 16))) &&
                      (!a.normed || aligned(a.normed, a.ld_normed * b, 16));
    return wide ? launch_width<T, kN>(a, stream) : launch_width<T, 1>(a, stream);
}

}  // namespace

cudaError_t launch_rms_norm_quantize(const NormArgs& a, int dtype, cudaStream_t stream) {
    if (dtype == ZQ_DTYPE_F32) return launch_type<float>(a, stream);
    if (dtype == ZQ_DTYPE_F16) return launch_type<__half>(a, stream);
    return launch_type<__nv_bfloat16>(a, stream);
}

}  // namespace zq

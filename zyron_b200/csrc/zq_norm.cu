// zq_norm.cu -- root-mean-square norm with the residual's addition and the
// activation quantizer's output (zq_rms_norm_quantize).
//
//   s = x + residual, rounded to the type it is stored in
//   r = fl32(1 / sqrt(mean(s^2) + eps))          mean in 64 bits
//   v = fl32(fl32(s * r) * w)
//   scale = max|v| / 127 (1 for a row of zeros), code = round(v / scale)
//   (or scale = max|v| * fl32(1 / 127) where the caller asks for it)
//
// With the quotient the codes and scales are those of quantize_rows over v, bit
// for bit.  The
// only quantity that depends on the order of a sum is the mean of squares.
// It is summed in 64 bits, where fp32 squares are exact, so r -- and with it
// every code -- does not depend on the launch shape: a last-bit change of r
// would carry values across the codes' rounding borders.
//
// Bound: one read of x and residual and one write of the sum and the codes:
// memory bandwidth, if an element takes few instructions (at 16 bits and 8192
// columns there is time for about 25 of them).  So a row stays in the registers
// of one group of threads from its load to its stores, 16-bit sums are added
// in pairs, and a code is read off a sum with 1.5 * 2^23 unless it is near a
// tie.
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

// fl32(1 / sqrt(sum / k + eps)).  Two Newton steps from the hardware's estimate
// (2^-20) leave the 64-bit value within a few of its last bits: the fp32
// rounding is that of the division's result unless it lies within 2^-50 of a
// border between two fp32 values.
__device__ __forceinline__ float row_rstd(double sum, double inv_k, double eps) {
    const double a = fma(sum, inv_k, eps);
    if (!(a > 1e-290 && a < 1e290)) return (float)__ddiv_rn(1.0, __dsqrt_rn(a));
    double y;
    asm("rsqrt.approx.ftz.f64 %0, %1;" : "=d"(y) : "d"(a));
    const double h = 0.5 * a;
    y = y * fma(-h * y, y, 1.5);
    y = y * fma(-h * y, y, 1.5);
    return (float)y;
}

__device__ __forceinline__ float row_scale_of(const NormArgs& a, float absmax) {
    return a.reciprocal && absmax > 0.0f ? __fmul_rn(absmax, 1.0f / 127.0f) : zq_scale_from_absmax(absmax, 127.0f);
}

__device__ __forceinline__ float norm_value(float s, float rstd, float w) {
    return __fmul_rn(__fmul_rn(s, rstd), w);
}

// a + b, rounded to the type.  16-bit sums in pairs: rounding the exact sum
// once equals rounding it to fp32 first, since a sum that fp32 cannot hold has
// one term below the other's last 16-bit place.
template <int kN>
__device__ __forceinline__ void add_packs(Pack<float, kN>& a, const Pack<float, kN>& b) {
#pragma unroll
    for (int j = 0; j < kN; ++j) a.e[j] = __fadd_rn(a.e[j], b.e[j]);
}
template <int kN>
__device__ __forceinline__ void add_packs(Pack<__half, kN>& a, const Pack<__half, kN>& b) {
#pragma unroll
    for (int j = 0; j + 1 < kN; j += 2) {
        const __half2 s = __hadd2_rn(__halves2half2(a.e[j], a.e[j + 1]), __halves2half2(b.e[j], b.e[j + 1]));
        a.e[j] = __low2half(s), a.e[j + 1] = __high2half(s);
    }
}
template <int kN>
__device__ __forceinline__ void add_packs(Pack<__nv_bfloat16, kN>& a, const Pack<__nv_bfloat16, kN>& b) {
#pragma unroll
    for (int j = 0; j + 1 < kN; j += 2) {
        const __nv_bfloat162 s =
            __hadd2_rn(__halves2bfloat162(a.e[j], a.e[j + 1]), __halves2bfloat162(b.e[j], b.e[j + 1]));
        a.e[j] = __low2bfloat16(s), a.e[j + 1] = __high2bfloat16(s);
    }
}

__device__ __noinline__ int divided_code(float n, float scale) { return zq_quantize_value(n, scale, 127); }

// The codes of n[0..kN), as zq_quantize_value gives them.  y = n * rcp lies
// within 2.3e-5 of the quotient that is to be rounded (zq_quantize_value_rcp),
// and at most at 127 (1 + 2^-22).  y + 1.5 * 2^23 rounds y to a whole number,
// which its low bits hold.  Nearer than 3e-5 to a tie, and for NaN, the
// division decides.
template <int kN>
__device__ __forceinline__ Pack<int8_t, kN> codes_of(const float (&n)[kN], float scale, float rcp) {
    constexpr float kMagic = 12582912.0f;
    float t[kN];
    bool clear = true;
#pragma unroll
    for (int j = 0; j < kN; ++j) {
        const float y = __fmul_rn(n[j], rcp);
        t[j] = __fadd_rn(y, kMagic);
        clear = clear && fabsf(__fadd_rn(y, -__fadd_rn(t[j], -kMagic))) < 0.5f - 3.0e-5f;
    }
    Pack<int8_t, kN> c;
    if (clear) {
        if constexpr (kN % 4 == 0) {
#pragma unroll
            for (int j = 0; j < kN; j += 4) {
                const uint32_t w = __byte_perm(__byte_perm(__float_as_uint(t[j]), __float_as_uint(t[j + 1]), 0x0040),
                                               __byte_perm(__float_as_uint(t[j + 2]), __float_as_uint(t[j + 3]), 0x0040),
                                               0x5410);
                memcpy(&c.e[j], &w, 4);
            }
        } else {
#pragma unroll
            for (int j = 0; j < kN; ++j) c.e[j] = (int8_t)__float_as_uint(t[j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < kN; ++j) c.e[j] = (int8_t)divided_code(n[j], scale);
    }
    return c;
}

// The kN elements of a row from p * kN on, as far as k; zeros behind.  kAligned:
// rows start on 16 bytes and k is a multiple of kN.  Else a lane's elements
// come one by one, out of lines that its first access brought to L1 (such a kernel
// neither starts early nor lets others, launch_kernel; 1537 x 4099 fp32: 20.7 us,
// with an early start and load_l2 22.4 us).  (Aligned loads shifted into place
// with a neighbour's took longer: 94 us against 79 us at 4000 x 4099 bf16 when
// they were tried.)
template <bool kAligned, class T, int kN>
__device__ __forceinline__ Pack<T, kN> load_pack(const T* row, int p, int k) {
    Pack<T, kN> v;
    if (kAligned) {
        v = load_l2(reinterpret_cast<const Pack<T, kN>*>(row) + p);
    } else {
#pragma unroll
        for (int j = 0; j < kN; ++j) v.e[j] = p * kN + j < k ? row[p * kN + j] : T(0.0f);
    }
    return v;
}
// kAligned or `wide`: whole packs of the row lie on their own size.
template <bool kAligned, class T, int kN>
__device__ __forceinline__ void store_pack(T* row, int p, int k, const Pack<T, kN>& v, bool wide) {
    if (kAligned || (wide && (p + 1) * kN <= k)) {
        reinterpret_cast<Pack<T, kN>*>(row)[p] = v;
    } else {
#pragma unroll
        for (int j = 0; j < kN; ++j)
            if (p * kN + j < k) row[p * kN + j] = v.e[j];
    }
}

// A row of at most 32 * kWarps * kPacks packs of 16 bytes, held in the
// registers of kWarps warps.
template <class T, int kWarps, int kPacks, bool kAligned>
__global__ void __launch_bounds__(kWarps > 8 ? kWarps * 32 : 256, kWarps > 8 ? 1 : 3)
    rms_norm_quantize_kernel(const NormArgs a) {
    if (kAligned) pdl_launch_dependents();
    pdl_wait_primary();
    constexpr int kN = kElemsPer16<T>;
    constexpr int kBlockWarps = kWarps > 8 ? kWarps : 8;
    constexpr int kThreads = 32 * kWarps;
    __shared__ double part_sum[kBlockWarps];
    __shared__ float part_max[kBlockWarps];
    const long long row = (long long)blockIdx.x * (kBlockWarps / kWarps) + threadIdx.x / kThreads;
    const int t = threadIdx.x % kThreads;
    const bool live = row < a.m;
    const int packs = live ? (a.k + kN - 1) / kN : 0;
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    const T* res = static_cast<const T*>(a.residual) + row * a.ld_residual;
    T* sum_out = static_cast<T*>(a.residual_out) + row * a.ld_residual_out;
    using P = Pack<T, kN>;

    P v[kPacks];
#pragma unroll
    for (int i = 0; i < kPacks; ++i) {
        const int p = t + i * kThreads;
        if (p < packs)
            v[i] = load_pack<kAligned, T, kN>(x, p, a.k);
        else
#pragma unroll
            for (int j = 0; j < kN; ++j) v[i].e[j] = T(0.0f);
    }
    if (a.residual) {
        P r[kPacks];
#pragma unroll
        for (int i = 0; i < kPacks; ++i) {
            const int p = t + i * kThreads;
            if (p < packs) r[i] = load_pack<kAligned, T, kN>(res, p, a.k);
        }
#pragma unroll
        for (int i = 0; i < kPacks; ++i) {
            const int p = t + i * kThreads;
            if (p < packs) {
                add_packs(v[i], r[i]);
                store_pack<kAligned, T, kN>(sum_out, p, a.k, v[i], a.wide_sum);
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
    const float rstd = row_rstd(sum, a.inv_k, a.eps);

    float n[kPacks][kN];
    float absmax = 0.0f;
#pragma unroll
    for (int i = 0; i < kPacks; ++i) {
        const int p = t + i * kThreads;
        if (p >= packs) continue;
        Pack<float, 4> w[kN / 4];
#pragma unroll
        for (int j = 0; j < kN / 4; ++j) {
            w[j] = Pack<float, 4>{{1.0f, 1.0f, 1.0f, 1.0f}};
            if (a.weight) {
                const int from = p * kN + 4 * j;
                if (kAligned || (a.wide_weight && from + 4 <= a.k)) {
                    w[j] = *reinterpret_cast<const Pack<float, 4>*>(a.weight + from);
                } else {
#pragma unroll
                    for (int u = 0; u < 4; ++u) w[j].e[u] = from + u < a.k ? a.weight[from + u] : 0.0f;
                }
            }
        }
#pragma unroll
        for (int j = 0; j < kN; ++j) {
            n[i][j] = norm_value(to_float(v[i].e[j]), rstd, w[j / 4].e[j % 4]);
            // behind the row 0 * rstd is NaN for an infinite rstd: no maximum
            absmax = fmaxf(absmax, fabsf(n[i][j]));
        }
    }
    absmax = group_max<kWarps>(absmax, part_max);
    if (!live) return;
    const float scale = row_scale_of(a, absmax);
    const float rcp = zq_quant_rcp(scale);
    if (t == 0) a.row_scale[row] = scale;
    int8_t* q = a.q + row * a.ldq;
    T* normed = a.normed ? static_cast<T*>(a.normed) + row * a.ld_normed : nullptr;
#pragma unroll
    for (int i = 0; i < kPacks; ++i) {
        const int p = t + i * kThreads;
        if (p >= packs) continue;
        store_pack<kAligned, int8_t, kN>(q, p, a.k, codes_of(n[i], scale, rcp), a.wide_codes);
        if (normed) {
            P o;
#pragma unroll
            for (int j = 0; j < kN; ++j) o.e[j] = from_float<T>(n[i][j]);
            store_pack<kAligned, T, kN>(normed, p, a.k, o, a.wide_normed);
        }
    }
    for (long long j = a.k + t; j < a.ldq; j += kThreads) q[j] = 0;  // ldq may be the last int
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
        T v = load_l2(x + i);
        if (res) {
            v = from_float<T>(__fadd_rn(to_float(v), to_float(load_l2(res + i))));
            sum_out[i] = v;
        }
        const double d = (double)to_float(v);
        sum = __fma_rn(d, d, sum);
    }
    const float rstd = row_rstd(group_sum<32>(sum, part_sum), a.inv_k, a.eps);
    const T* s = res ? sum_out : x;
    float absmax = 0.0f;
    for (int i = threadIdx.x; i < a.k; i += 1024)
        absmax = fmaxf(absmax, fabsf(norm_value(to_float(load_l2(s + i)), rstd, a.weight ? a.weight[i] : 1.0f)));
    absmax = group_max<32>(absmax, part_max);
    const float scale = row_scale_of(a, absmax);
    const float rcp = zq_quant_rcp(scale);
    if (threadIdx.x == 0) a.row_scale[row] = scale;
    int8_t* q = a.q + row * a.ldq;
    T* normed = a.normed ? static_cast<T*>(a.normed) + row * a.ld_normed : nullptr;
    for (int i = threadIdx.x; i < a.k; i += 1024) {
        const float n = norm_value(to_float(load_l2(s + i)), rstd, a.weight ? a.weight[i] : 1.0f);
        q[i] = (int8_t)zq_quantize_value_rcp(n, scale, rcp, 127);
        if (normed) normed[i] = from_float<T>(n);
    }
    for (long long i = a.k + threadIdx.x; i < a.ldq; i += 1024) q[i] = 0;
}

template <class T, int kWarps, int kPacks, bool kAligned>
cudaError_t launch_rows(const NormArgs& a, cudaStream_t stream) {
    constexpr int kRows = kWarps > 8 ? 1 : 8 / kWarps;
    return launch_kernel(kAligned, rms_norm_quantize_kernel<T, kWarps, kPacks, kAligned>,
                         dim3((unsigned)((a.m + kRows - 1) / kRows)), dim3(kWarps > 8 ? kWarps * 32 : 256), 0, stream,
                         a);
}

template <class T, int kPacks, bool kAligned>
cudaError_t launch_width(const NormArgs& a, cudaStream_t stream) {
    // The fewest warps that hold the row at kPacks packs a thread.
    const int packs = (a.k + kElemsPer16<T> - 1) / kElemsPer16<T>;
    if (packs <= 32 * kPacks) return launch_rows<T, 1, kPacks, kAligned>(a, stream);
    if (packs <= 64 * kPacks) return launch_rows<T, 2, kPacks, kAligned>(a, stream);
    if (packs <= 128 * kPacks) return launch_rows<T, 4, kPacks, kAligned>(a, stream);
    if (packs <= 256 * kPacks) return launch_rows<T, 8, kPacks, kAligned>(a, stream);
    if (packs <= 512 * kPacks) return launch_rows<T, 16, kPacks, kAligned>(a, stream);
    if (packs <= 1024 * kPacks) return launch_rows<T, 32, kPacks, kAligned>(a, stream);
    // 32 elements a thread reach furthest
    if constexpr (kPacks < 32 / kElemsPer16<T>) return launch_width<T, 32 / kElemsPer16<T>, kAligned>(a, stream);
    return launch_pdl_kernel(rms_norm_quantize_long_kernel<T>, dim3((unsigned)a.m), dim3(1024), 0, stream, a);
}

bool aligned(const void* p, long long pitch_bytes, size_t to) {
    return (reinterpret_cast<uintptr_t>(p) | (uintptr_t)pitch_bytes) % to == 0;
}

template <class T>
cudaError_t launch_type(NormArgs a, cudaStream_t stream) {
    constexpr int kN = kElemsPer16<T>;
    constexpr long long b = sizeof(T);
    a.inv_k = 1.0 / a.k;
    a.wide_weight = aligned(a.weight, 0, 16);
    a.wide_codes = aligned(a.q, a.ldq, kN);
    a.wide_sum = aligned(a.residual_out, a.ld_residual_out * b, 16);
    a.wide_normed = aligned(a.normed, a.ld_normed * b, 16);
    const bool whole = a.k % kN == 0 && aligned(a.x, a.ldx * b, 16) && a.wide_weight && a.wide_codes &&
                       (!a.residual || (aligned(a.residual, a.ld_residual * b, 16) && a.wide_sum)) &&
                       (!a.normed || a.wide_normed);
    // Elements a thread.  Many rows: 32, since what a thread does once a row
    // (two reductions, the root) then weighs least (8192 x 8192 bf16: 86 us, 16
    // a thread 125 us, 64 a thread, with fewer loads under way, 111 us; rows off
    // the 16-byte grid, 1537 x 4099 fp32: 21 us, 16 a thread 26 us).  A row an SM
    // or fewer: 8, the shortest chains (one row of 4096 fp32: 2.7 us against
    // 3.4 us with 16).  Off the grid a warp's lanes should all have elements
    // (30000 x 100 bf16: 20 us with 8, 27 us with 16, 41 us with 32).
    const bool few = a.m <= sm_count();
    if (whole) return few ? launch_width<T, 8 / kN, true>(a, stream) : launch_width<T, 32 / kN, true>(a, stream);
    if (few || a.k <= 256) return launch_width<T, 8 / kN, false>(a, stream);
    return a.k <= 512 ? launch_width<T, 16 / kN, false>(a, stream) : launch_width<T, 32 / kN, false>(a, stream);
}

}  // namespace

cudaError_t launch_rms_norm_quantize(const NormArgs& a, int dtype, cudaStream_t stream) {
    if (dtype == ZQ_DTYPE_F32) return launch_type<float>(a, stream);
    if (dtype == ZQ_DTYPE_F16) return launch_type<__half>(a, stream);
    return launch_type<__nv_bfloat16>(a, stream);
}

}  // namespace zq

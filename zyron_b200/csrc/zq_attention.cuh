// zq_attention.cuh -- what the attention kernels share: where unfinished sums
// lie, and how they are joined.
#pragma once

#include "zq_elem.cuh"
#include "zq_paged.cuh"

namespace zq {
namespace attn {

// Sums are kept as the unscaled output row, with the maximum (base 2) that its
// weights are relative to and their sum.
struct Workspace {
    float* part_sums;    // parts of cut items: [block][2][rows of a tile][width]
    float* part_stats;   // [block][2][rows of a tile][2]
    float* row_sums[2];  // with a prefix: own and prefix sums of every row, [rows][heads][dim]
    float* row_stats[2]; // [rows][heads][2]
};

template <class T>
constexpr bool kIsHalf = false;
template <>
constexpr bool kIsHalf<__half> = true;

__device__ __forceinline__ float exp2_approx(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

// Two fp32 values as packed pairs of 16-bit parts whose sum they are (to 2^-17
// of bf16, 2^-22 of fp16).
template <class T>
__device__ __forceinline__ void split_pair(float x, float y, uint32_t& hi, uint32_t& lo) {
    const T hx = from_float<T>(x), hy = from_float<T>(y);
    const T lx = from_float<T>(x - to_float(hx)), ly = from_float<T>(y - to_float(hy));
    Pack<T, 2> h{{hx, hy}}, l{{lx, ly}};
    memcpy(&hi, &h, 4);
    memcpy(&lo, &l, 4);
}

// Whether a warp's 16 keys' values in shared memory hold an infinity or NaN: an
// exponent of all ones in either half of a word.
template <class T, int kD>
__device__ __forceinline__ bool wild_values(uint32_t v_u, int lane) {
    constexpr uint32_t kOnes = kIsHalf<T> ? 0x7C007C00u : 0x7F807F80u;
    bool wild = false;
    for (int i = lane; i < 16 * kD / 8; i += 32) {
        uint32_t w[4];
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                     : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                     : "r"(v_u + i * 16)
                     : "memory");
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t e = w[j] & kOnes;
            wild |= (e & 0xFFFF0000u) == (kOnes & 0xFFFF0000u) || (e & 0xFFFFu) == (kOnes & 0xFFFFu);
        }
    }
    return __any_sync(0xffffffffu, wild);
}

// Rows of the call that some request may own: all requests' last row on.
__device__ __forceinline__ int live_rows(const PagedBatch& p) {
    if (!p.starts) return p.rows;
    return min(max(load_l2(p.starts + p.requests), 0), p.rows);
}

// Four elements of a part.
__device__ __forceinline__ void put_part(const Workspace& ws, long long row, int width, int d, const float (&v)[4],
                                         float most, float total) {
    *reinterpret_cast<float4*>(ws.part_sums + row * width + d) = make_float4(v[0], v[1], v[2], v[3]);
    if (d == 0) {
        ws.part_stats[2 * row] = most;
        ws.part_stats[2 * row + 1] = total;
    }
}

// Four elements of a row's output.  A row that sees no key is zero.
template <class T>
__device__ __forceinline__ void put_out(const AttentionArgs& a, int row, int head, int d, const float (&v)[4],
                                        float total) {
    const float scale = total == 0.0f ? 0.0f : 1.0f / total;
    Pack<T, 4> o;
#pragma unroll
    for (int j = 0; j < 4; ++j) o.e[j] = from_float<T>(total == 0.0f ? 0.0f : v[j] * scale);
    *reinterpret_cast<Pack<T, 4>*>(static_cast<T*>(a.out) + (long long)row * a.ld_out + (long long)head * a.batch.dim +
                                   d) = o;
}

// A row's whole own or prefix result: the output, or with a prefix its sums.
template <class T>
__device__ __forceinline__ void put_row(const AttentionArgs& a, const Workspace& ws, bool prefix, int row, int head,
                                        int d, const float (&v)[4], float most, float total) {
    if (a.prefix_length == 0) return put_out<T>(a, row, head, d, v, total);
    const long long at = (long long)row * a.heads + head;
    *reinterpret_cast<float4*>((prefix ? ws.row_sums[1] : ws.row_sums[0]) + at * a.batch.dim + d) =
        make_float4(v[0], v[1], v[2], v[3]);
    if (d == 0) {
        float* s = (prefix ? ws.row_stats[1] : ws.row_stats[0]) + 2 * at;
        s[0] = most;
        s[1] = total;
    }
}

// Sums of several parts of the same keys' row, in a fixed order.
struct Joined {
    float most = -INFINITY, total = 0.0f, v[4] = {0.0f, 0.0f, 0.0f, 0.0f};

    __device__ __forceinline__ void add_row(const float* stats, const float* sums, long long row, int width, int d) {
        const float m = load_l2(stats + 2 * row), l = load_l2(stats + 2 * row + 1);
        const float4 x = load_l2(reinterpret_cast<const float4*>(sums + row * width + d));
        const float now = fmaxf(most, m);
        const float ref = now == -INFINITY ? 0.0f : now;
        const float keep = exp2_approx(most - ref), weight = exp2_approx(m - ref);
        most = now;
        total = total * keep + l * weight;
        v[0] = v[0] * keep + x.x * weight;
        v[1] = v[1] * keep + x.y * weight;
        v[2] = v[2] * keep + x.z * weight;
        v[3] = v[3] * keep + x.w * weight;
    }
    __device__ __forceinline__ void add(const Workspace& ws, long long row, int width, int d) {
        add_row(ws.part_stats, ws.part_sums, row, width, d);
    }
};

}  // namespace attn
}  // namespace zq

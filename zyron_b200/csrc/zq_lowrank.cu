// zq_lowrank.cu -- low-rank adapters of many requests added onto a shared
// projection's output (zq_add_low_rank).
//
//   y[i] += scale_s * B_s (A_s x[i]),   s = ids[i]
//
// Rows of one adapter are taken 16 at a time.  One cluster of CTAs does such
// a tile in a single launch: the CTAs split k for h = A x, sum their parts
// through distributed shared memory, and split the output columns for B h.
// So an adapter's weights are read once a tile, spread over the cluster's SMs,
// and h never leaves the chip.
//
// Few rows (kDirectRows): cluster c belongs to row c and works if an even
// multiple of 16 earlier rows have the same adapter; it takes that row and the
// next 15 of its adapter.  More rows: a plan kernel sorts the rows by adapter
// into tiles first.
//
// Both products run on the tensor cores (m16n8k16, bf16 in, fp32 out).  fp32
// and fp16 values enter as sums of bf16 parts, cut off at 8 bits each, so the
// parts add up to the value exactly (fp32: three, fp16: two, bf16: one) and
// every product is exact; sums are fp32.
//
// The sums over k and over the rank do not care in which order the operands'
// elements come, as long as both have the same: a lane takes 8 elements that
// lie side by side in memory, and their pairs go to the two MMAs of a chunk of
// 32.  In the same way the columns of two n8 tiles are dealt so that a lane
// ends up with 4 neighbouring outputs of a row.
//
// Bound: the used adapters once, x once, y read and written.
#include <cooperative_groups.h>

#include "zq_common.cuh"
#include "zq_elem.cuh"
#include "zq_kernels.h"

namespace zq {

namespace {

namespace cg = cooperative_groups;

constexpr int kTileRows = 16;
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kCluster = 8;
constexpr int kDirectRows = 256;
constexpr int kRankPass = 64;  // ranks whose sums a warp holds at once
static_assert(kDirectRows <= kThreads, "one row a thread when a cluster looks for its tile");

struct Tile {
    int slot, first, rows, pad;
};

// Workspace of the sorted form: tile count, tiles, row order.
__host__ __device__ size_t max_tiles(size_t m, size_t slots) { return m / kTileRows + (slots < m ? slots : m); }
struct Plan {
    int* count;
    Tile* tiles;
    int* order;
};
__host__ __device__ Plan plan_at(void* ws, size_t m, size_t slots) {
    uint8_t* p = static_cast<uint8_t*>(ws);
    Plan r;
    r.count = reinterpret_cast<int*>(p);
    r.tiles = reinterpret_cast<Tile*>(p + 256);
    r.order = reinterpret_cast<int*>(p + 256 + max_tiles(m, slots) * sizeof(Tile));
    return r;
}

// ---- bf16 parts ------------------------------------------------------------

template <class T>
constexpr int kParts = sizeof(T) == 4 ? 3 : 2;
template <>
constexpr int kParts<__nv_bfloat16> = 1;

// Cuts v into bf16 bit patterns part[0..kP), highest bits first.
template <int kP>
__device__ __forceinline__ void cut(float v, uint32_t (&part)[kP]) {
#pragma unroll
    for (int p = 0; p < kP; ++p) {
        const uint32_t top = __float_as_uint(v) & 0xFFFF0000u;
        part[p] = top >> 16;
        const float rest = v - __uint_as_float(top);
        if (p == 0 && rest != rest) {  // inf and NaN have one part
            part[0] = v != v ? 0x7FC0u : part[0];
            v = 0.0f;
        } else {
            v = rest;
        }
    }
}

// 8 neighbouring elements as packed pairs of each part: pair[p][i] holds
// elements 2i (low half) and 2i + 1.
template <class T>
struct Pairs {
    uint32_t pair[kParts<T>][4];
};

__device__ __forceinline__ void to_pairs(const float (&v)[8], Pairs<float>& o) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t a[3], b[3];
        cut(v[2 * i], a);
        cut(v[2 * i + 1], b);
#pragma unroll
        for (int p = 0; p < 3; ++p) o.pair[p][i] = a[p] | b[p] << 16;
    }
}
__device__ __forceinline__ void to_pairs(const __half (&v)[8], Pairs<__half>& o) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t a[2], b[2];
        cut(__half2float(v[2 * i]), a);
        cut(__half2float(v[2 * i + 1]), b);
#pragma unroll
        for (int p = 0; p < 2; ++p) o.pair[p][i] = a[p] | b[p] << 16;
    }
}
__device__ __forceinline__ void to_pairs(const __nv_bfloat16 (&v)[8], Pairs<__nv_bfloat16>& o) {
    memcpy(o.pair, v, 16);
}

// Elements [0, n) of p (n may be <= 0 or above 8), zeros behind them.  kVec:
// p is 16-byte aligned and, where n > 0, all 8 may be read.
template <class T, bool kVec>
__device__ __forceinline__ void load8(const T* p, int n, T (&v)[8]) {
    constexpr int kN = kElemsPer16<T>;
    if (kVec) {
#pragma unroll
        for (int i = 0; i < 8 / kN; ++i) {
            uint4 w = make_uint4(0, 0, 0, 0);
            if (n > 0) w = __ldg(reinterpret_cast<const uint4*>(p) + i);
            memcpy(&v[i * kN], &w, 16);
        }
        if (n < 8)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i >= n) v[i] = from_float<T>(0.0f);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : from_float<T>(0.0f);
    }
}

__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// d += (rows lo, hi) x (column b) over a chunk of 32, every part with every
// part, the smallest products first.
template <int kPA, int kPB>
__device__ __forceinline__ void mma_chunk(float (&d)[4], const uint32_t (&lo)[kPA][4], const uint32_t (&hi)[kPA][4],
                                          const uint32_t (&b)[kPB][4]) {
#pragma unroll
    for (int p = kPA - 1; p >= 0; --p)
#pragma unroll
        for (int q = kPB - 1; q >= 0; --q)
#pragma unroll
            for (int s = 0; s < 4; s += 2)
                mma_bf16(d, lo[p][s], hi[p][s], lo[p][s + 1], hi[p][s + 1], b[q][s], b[q][s + 1]);
}

// ---- shared memory ---------------------------------------------------------

// Bytes of a row of one part of h: a multiple of 32 ranks, 64 bytes past a
// multiple of 128 so that the rows' 16-byte reads fall into all banks.
__host__ __device__ int h_pitch(int max_rank) {
    const int b = (max_rank + 31) / 32 * 64;
    return b % 128 == 64 ? b : b + 64;
}
__host__ __device__ int pass_width(int max_rank) {
    const int r = (max_rank + 7) / 8 * 8;
    return r < kRankPass ? r : kRankPass;
}
// The warps' sums of one pass and, later, h's three parts share one region.
__host__ __device__ int region_bytes(int max_rank) {
    const int sums = kWarps * kTileRows * pass_width(max_rank) * 4;
    const int parts = 3 * kTileRows * h_pitch(max_rank);
    return sums > parts ? sums : parts;
}
__host__ __device__ int cta_h_pitch(int max_rank) { return (max_rank + 7) / 8 * 8; }
__host__ __device__ int smem_bytes(int max_rank) {
    return region_bytes(max_rank) + kTileRows * cta_h_pitch(max_rank) * 4;
}

// kVecX, kVecB: rows of x and of A, and rows of B, start on 16 bytes and are
// whole 16-byte packs of 8 elements.  kVecY: 16-byte access to y.
template <class TX, class TW, bool kVecX, bool kVecB, bool kVecY>
__global__ void __launch_bounds__(kThreads) add_low_rank_kernel(const LowRankArgs a, void* workspace) {
    cg::cluster_group cluster = cg::this_cluster();
    pdl_launch_dependents();
    pdl_wait_primary();
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int row_of[kTileRows];
    __shared__ uint32_t same[kDirectRows / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, t = lane & 3;
    const int ctas = (int)cluster.num_blocks();
    const int tile = blockIdx.x / ctas;

    // ---- which rows ----
    int slot, rows;
    if (threadIdx.x < kTileRows) row_of[threadIdx.x] = -1;
    if (a.m <= kDirectRows) {
        slot = a.ids[tile];
        const bool mine = (int)threadIdx.x < a.m && a.ids[threadIdx.x] == slot;
        const uint32_t votes = __ballot_sync(0xffffffffu, mine);
        if (lane == 0) same[warp] = votes;
        __syncthreads();
        int before = 0, rank_in = 0, all = 0;
        for (int w = 0; w < kWarps; ++w) {
            const uint32_t v = same[w];
            const uint32_t below = w * 32 > tile ? 0u : tile - w * 32 >= 32 ? ~0u : (1u << (tile - w * 32)) - 1;
            before += __popc(v & below);
            if (w < warp) rank_in += __popc(v);
            all += __popc(v);
        }
        if (slot < 0 || slot >= a.slots || before % kTileRows != 0) return;
        rank_in += __popc(votes & ((1u << lane) - 1)) - before;
        if (mine && rank_in >= 0 && rank_in < kTileRows) row_of[rank_in] = threadIdx.x;
        rows = min(kTileRows, all - before);
    } else {
        const Plan plan = plan_at(workspace, (size_t)a.m, (size_t)a.slots);
        if (tile >= *plan.count) return;
        const Tile what = plan.tiles[tile];
        slot = what.slot;
        rows = what.rows;
        if ((int)threadIdx.x < rows) row_of[threadIdx.x] = plan.order[what.first + threadIdx.x];
    }
    const int rank = a.ranks ? min(max(a.ranks[slot], 0), a.max_rank) : a.max_rank;
    if (rank == 0) return;
    __syncthreads();
    const int gw = (int)cluster.block_rank() * kWarps + warp, all_warps = ctas * kWarps;
    const long long row_lo = row_of[g], row_hi = row_of[g + 8];

    // ---- h = A x: this CTA's share of k ----
    float* sums = reinterpret_cast<float*>(smem);
    float* cta_h = reinterpret_cast<float*>(smem + region_bytes(a.max_rank));
    const int hp = cta_h_pitch(a.max_rank), width = pass_width(a.max_rank);
    const TX* x_lo = static_cast<const TX*>(a.x) + (row_lo < 0 ? 0 : row_lo) * a.ldx;
    const TX* x_hi = static_cast<const TX*>(a.x) + (row_hi < 0 ? 0 : row_hi) * a.ldx;
    const TW* wa = static_cast<const TW*>(a.a) + (long long)slot * a.max_rank * a.k;
    for (int r0 = 0; r0 < rank; r0 += kRankPass) {
        float acc[kRankPass / 8][4] = {};
        for (int k0 = gw * 32; k0 < a.k; k0 += all_warps * 32) {
            const int k = k0 + 8 * t;
            TX v[8];
            Pairs<TX> lo, hi;
            load8<TX, kVecX>(x_lo + k, row_lo < 0 ? 0 : a.k - k, v);
            to_pairs(v, lo);
            load8<TX, kVecX>(x_hi + k, row_hi < 0 ? 0 : a.k - k, v);
            to_pairs(v, hi);
#pragma unroll
            for (int j = 0; j < kRankPass / 8; ++j) {
                if (r0 + 8 * j >= rank) continue;
                const int r = r0 + 8 * j + g;
                TW u[8];
                Pairs<TW> b;
                load8<TW, kVecX>(wa + (long long)r * a.k + k, r < rank ? a.k - k : 0, u);
                to_pairs(u, b);
                mma_chunk(acc[j], lo.pair, hi.pair, b.pair);
            }
        }
        if (r0) __syncthreads();
#pragma unroll
        for (int j = 0; j < kRankPass / 8; ++j) {
            if (8 * j >= width) continue;
            float* s = sums + warp * kTileRows * width + 8 * j + 2 * t;
            *reinterpret_cast<float2*>(s + g * width) = make_float2(acc[j][0], acc[j][1]);
            *reinterpret_cast<float2*>(s + (g + 8) * width) = make_float2(acc[j][2], acc[j][3]);
        }
        __syncthreads();
        for (int i = threadIdx.x; i < kTileRows * width; i += kThreads) {
            const int r = i / width, c = i % width;
            if (r0 + c >= hp) continue;
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) s += sums[w * kTileRows * width + i];
            cta_h[r * hp + r0 + c] = s;
        }
    }

    // ---- the cluster's sum, scaled, as three bf16 parts ----
    cluster.sync();
    const float scale = a.scales ? a.scales[slot] : 1.0f;
    const int pitch = h_pitch(a.max_rank), rank32 = (rank + 31) / 32 * 32;
    for (int i = threadIdx.x; i < kTileRows * rank32; i += kThreads) {
        const int r = i / rank32, c = i % rank32;
        uint32_t part[3] = {0, 0, 0};
        if (c < rank && r < rows) {
            float s = 0.0f;
            for (int w = 0; w < ctas; ++w) s += cluster.map_shared_rank(cta_h, w)[r * hp + c];
            cut(s * scale, part);
        }
#pragma unroll
        for (int p = 0; p < 3; ++p)
            *reinterpret_cast<uint16_t*>(smem + (p * kTileRows + r) * pitch + 2 * c) = (uint16_t)part[p];
    }
    cluster.barrier_arrive();  // no more reads of the other CTAs' sums
    __syncthreads();

    // ---- y += B h: this CTA's share of the columns ----
    const TW* wb = static_cast<const TW*>(a.b) + (long long)slot * a.n * a.max_rank;
    float* y_lo = a.y + (row_lo < 0 ? 0 : row_lo) * a.ldy;
    float* y_hi = a.y + (row_hi < 0 ? 0 : row_hi) * a.ldy;
    const uint8_t* h_lo = smem + g * pitch + 16 * t;
    for (int c0 = gw * 16; c0 < a.n; c0 += all_warps * 16) {
        const int col = c0 + 4 * t;  // of the 4 outputs that this lane gets
        float4 was_lo = make_float4(0, 0, 0, 0), was_hi = was_lo;
        if (kVecY) {
            if (row_lo >= 0 && col < a.n) was_lo = *reinterpret_cast<const float4*>(y_lo + col);
            if (row_hi >= 0 && col < a.n) was_hi = *reinterpret_cast<const float4*>(y_hi + col);
        }
        float acc[2][4] = {};
        for (int r0 = 0; r0 < rank; r0 += 32) {
            uint32_t lo[3][4], hi[3][4];
#pragma unroll
            for (int p = 0; p < 3; ++p) {
                const uint8_t* h = h_lo + p * kTileRows * pitch + 2 * r0;
                memcpy(lo[p], __builtin_assume_aligned(h, 16), 16);
                memcpy(hi[p], __builtin_assume_aligned(h + 8 * pitch, 16), 16);
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int bc = c0 + 4 * (g >> 1) + (g & 1) + 2 * j;
                const int r = r0 + 8 * t;
                TW u[8];
                Pairs<TW> b;
                load8<TW, kVecB>(wb + (long long)bc * a.max_rank + r, bc < a.n ? rank - r : 0, u);
                to_pairs(u, b);
                mma_chunk(acc[j], lo, hi, b.pair);
            }
        }
        const float d_lo[4] = {acc[0][0], acc[0][1], acc[1][0], acc[1][1]};
        const float d_hi[4] = {acc[0][2], acc[0][3], acc[1][2], acc[1][3]};
        if (kVecY) {
            if (row_lo >= 0 && col < a.n)
                *reinterpret_cast<float4*>(y_lo + col) =
                    make_float4(was_lo.x + d_lo[0], was_lo.y + d_lo[1], was_lo.z + d_lo[2], was_lo.w + d_lo[3]);
            if (row_hi >= 0 && col < a.n)
                *reinterpret_cast<float4*>(y_hi + col) =
                    make_float4(was_hi.x + d_hi[0], was_hi.y + d_hi[1], was_hi.z + d_hi[2], was_hi.w + d_hi[3]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (row_lo >= 0 && col + i < a.n) y_lo[col + i] += d_lo[i];
                if (row_hi >= 0 && col + i < a.n) y_hi[col + i] += d_hi[i];
            }
        }
    }
    cluster.barrier_wait();
}

// Sorts the rows by adapter: order[] lists the rows of slot 0, then 1, ...,
// each slot's rows cut into tiles of kTileRows.  The order of a slot's rows
// varies from run to run; their results do not depend on it.
constexpr int kPlanThreads = 1024;
__global__ void __launch_bounds__(kPlanThreads) plan_rows_kernel(const int32_t* ids, int m, int slots, void* workspace) {
    pdl_launch_dependents();
    pdl_wait_primary();
    extern __shared__ int counts[];  // [slots]
    __shared__ int2 warp_sum[kPlanThreads / 32];
    const Plan plan = plan_at(workspace, (size_t)m, (size_t)slots);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int s = threadIdx.x; s < slots; s += kPlanThreads) counts[s] = 0;
    __syncthreads();
    // Neighbouring rows mostly share an adapter: one atomic for a warp's equals.
    for (int i = threadIdx.x; i < (m + 31) / 32 * 32; i += kPlanThreads) {
        const int id = i < m ? ids[i] : -1;
        const bool ok = id >= 0 && id < slots;
        const uint32_t peers = __match_any_sync(0xffffffffu, ok ? id : -1);
        if (ok && lane == __ffs(peers) - 1) atomicAdd(&counts[id], __popc(peers));
    }
    __syncthreads();
    // Where each slot's rows and tiles begin: a scan over runs of slots.
    const int run = (slots + kPlanThreads - 1) / kPlanThreads;
    const int s0 = min(slots, (int)threadIdx.x * run), s1 = min(slots, s0 + run);
    int2 sum = make_int2(0, 0);
    for (int s = s0; s < s1; ++s) {
        sum.x += counts[s];
        sum.y += (counts[s] + kTileRows - 1) / kTileRows;
    }
    int2 at = sum;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const int x = __shfl_up_sync(0xffffffffu, at.x, o), y = __shfl_up_sync(0xffffffffu, at.y, o);
        if (lane >= o) at.x += x, at.y += y;
    }
    if (lane == 31) warp_sum[warp] = at;
    __syncthreads();
    at.x -= sum.x;
    at.y -= sum.y;
    for (int w = 0; w < warp; ++w) at.x += warp_sum[w].x, at.y += warp_sum[w].y;
    if (threadIdx.x == kPlanThreads - 1) *plan.count = at.y + sum.y;
    for (int s = s0; s < s1; ++s) {
        const int n = counts[s];
        for (int i = 0; i < n; i += kTileRows)
            plan.tiles[at.y++] = Tile{s, at.x + i, min(kTileRows, n - i), 0};
        counts[s] = at.x;
        at.x += n;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < (m + 31) / 32 * 32; i += kPlanThreads) {
        const int id = i < m ? ids[i] : -1;
        const bool ok = id >= 0 && id < slots;
        const uint32_t peers = __match_any_sync(0xffffffffu, ok ? id : -1);
        const int leader = __ffs(peers) - 1;
        int first = 0;
        if (ok && lane == leader) first = atomicAdd(&counts[id], __popc(peers));
        first = __shfl_sync(0xffffffffu, first, leader);
        if (ok) plan.order[first + __popc(peers & ((1u << lane) - 1))] = i;
    }
}

template <class TX, class TW, bool kVecX, bool kVecB, bool kVecY>
cudaError_t launch(const LowRankArgs& a, void* workspace, cudaStream_t stream) {
    size_t tiles = (size_t)a.m;
    if (a.m > kDirectRows) {
        tiles = max_tiles((size_t)a.m, (size_t)a.slots);
        const size_t smem = (size_t)a.slots * sizeof(int);
        const cudaError_t e =
            launch_pdl_kernel(plan_rows_kernel, dim3(1), dim3(kPlanThreads), smem, stream, a.ids, (int)a.m, a.slots,
                              workspace);
        if (e != cudaSuccess) return e;
    }
    auto kern = add_low_rank_kernel<TX, TW, kVecX, kVecB, kVecY>;
    const size_t smem = (size_t)smem_bytes(a.max_rank);
    if (smem > 47 * 1024) {  // with the static arrays past the 48 KiB that need no attribute
        const cudaError_t e = ensure_smem_attr(kern, smem);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(tiles * kCluster));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = kCluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kern, a, workspace);
}

bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <class TX, class TW>
cudaError_t launch_types(const LowRankArgs& a, void* ws, cudaStream_t stream) {
    const bool vx = a.k % 8 == 0 && on16(a.x) && a.ldx * sizeof(TX) % 16 == 0 && on16(a.a);
    const bool vb = a.max_rank % 8 == 0 && on16(a.b);
    const bool vy = a.n % 4 == 0 && on16(a.y) && a.ldy % 4 == 0;
    if (vx && vb && vy) return launch<TX, TW, true, true, true>(a, ws, stream);
    if (vx && vb) return launch<TX, TW, true, true, false>(a, ws, stream);
    if (vx && vy) return launch<TX, TW, true, false, true>(a, ws, stream);
    if (vx) return launch<TX, TW, true, false, false>(a, ws, stream);
    return launch<TX, TW, false, false, false>(a, ws, stream);
}

template <class TX>
cudaError_t launch_x(const LowRankArgs& a, int w_dtype, void* ws, cudaStream_t stream) {
    return w_dtype == ZQ_DTYPE_F16 ? launch_types<TX, __half>(a, ws, stream)
                                   : launch_types<TX, __nv_bfloat16>(a, ws, stream);
}

}  // namespace

size_t low_rank_workspace_bytes(size_t m, size_t slots) {
    if (m <= (size_t)kDirectRows) return 0;
    return (256 + max_tiles(m, slots) * sizeof(Tile) + m * sizeof(int) + 255) & ~size_t(255);
}

cudaError_t launch_add_low_rank(const LowRankArgs& a, int x_dtype, int w_dtype, void* workspace, cudaStream_t stream) {
    if (x_dtype == ZQ_DTYPE_F32) return launch_x<float>(a, w_dtype, workspace, stream);
    if (x_dtype == ZQ_DTYPE_F16) return launch_x<__half>(a, w_dtype, workspace, stream);
    return launch_x<__nv_bfloat16>(a, w_dtype, workspace, stream);
}

}  // namespace zq

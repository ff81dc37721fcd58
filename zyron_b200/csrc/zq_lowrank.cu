// zq_lowrank.cu -- low-rank adapters of many requests added onto a shared
// projection's output (zq_add_low_rank).
//
//   y[i] += scale_s * B_s (A_s x[i]),   s = ids[i]
//
// Rows of one adapter are taken in tiles, so that its weights serve several
// rows.  Up to kDirectRows rows, tile c belongs to row c and has work if a
// multiple of 16 earlier rows have its adapter: it takes row c and the next 15
// of the adapter.  More rows are sorted by adapter first (plan_rows_kernel).
// Then two launches: shrink computes h = A x, a grid of tiles x shares of k,
// each share's sums to the workspace; expand adds the shares up and computes
// y += B h, a grid of tiles x shares of the columns.  h of a row is small (its
// shares stay in L2), and with two grids each splits where it is long: one
// cluster a tile that did both measured 190 us at 4096 x 4096 x 4096 of rank
// 64, waiting in turn for x, the other CTAs' sums and y.
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
// ends up with 4 neighbouring outputs of a row.  So both operands come from
// global memory straight into fragments; the kMT warps of a block that share
// weights and differ in rows meet in L1.
//
// Bound: the used adapters once, x once, y read and written.  A block prefetches
// its shares into L2 as soon as it knows its rows: in expand that is before h is
// there.
#include <type_traits>

#include "zq_common.cuh"
#include "zq_elem.cuh"
#include "zq_kernels.h"

namespace zq {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kDirectRows = 256;
constexpr int kSortedTiles = 2;  // 16-row tiles of a block when the rows are sorted
constexpr int kWarpCols = 32;   // columns that a warp computes at once
constexpr int kRankPass = 64;  // ranks whose sums a warp holds at once
static_assert(kDirectRows <= kThreads, "one row a thread when a block looks for its tile");

struct Tile {
    int slot, first, rows, pad;
};

// Workspace: the shares of h [shares][m][rank_pitch] and, for the sorted form,
// the tile count, the tiles, the row order and the rows' places in their slots.
__host__ __device__ int rank_pitch(int max_rank) { return (max_rank + 7) / 8 * 8; }
__host__ __device__ size_t max_tiles(size_t m, size_t slots, int tile_rows) {
    return m / tile_rows + (slots < m ? slots : m);
}
struct Workspace {
    float* h;
    int* count;
    Tile* tiles;
    int* order;
    int* place;
};
__host__ __device__ size_t align256(size_t v) { return (v + 255) & ~size_t(255); }
__host__ __device__ size_t h_bytes(size_t m, int shares, int max_rank) {
    return align256((size_t)shares * m * rank_pitch(max_rank) * sizeof(float));
}

// How a call is cut up.
struct Shape {
    int mt;          // 16-row tiles of a block
    int shares;      // of k
    int k_span;      // k of a share, a multiple of 32
    int col_shares;  // of the columns
    int col_span;    // columns of a share, a multiple of 16
};
__host__ __device__ Workspace workspace_at(void* ws, size_t m, size_t slots, int shares, int max_rank, int mt) {
    uint8_t* p = static_cast<uint8_t*>(ws);
    Workspace r;
    r.h = reinterpret_cast<float*>(p);
    p += h_bytes(m, shares, max_rank);
    r.count = reinterpret_cast<int*>(p);
    r.tiles = reinterpret_cast<Tile*>(p + 256);
    r.order = reinterpret_cast<int*>(p + 256 + max_tiles(m, slots, 16 * mt) * sizeof(Tile));
    r.place = r.order + m;
    return r;
}

// ---- bf16 parts ------------------------------------------------------------

template <class T>
constexpr int kParts = sizeof(T) == 4 ? 3 : 2;
template <>
constexpr int kParts<__nv_bfloat16> = 1;

// 8 neighbouring elements as packed pairs of each part: pair[p][i] holds
// elements 2i (low half) and 2i + 1.
template <class T>
struct Pairs {
    uint32_t pair[kParts<T>][4];
};

// Cuts a and b into bf16 parts: the upper halves of the fp32 values, then of
// what they leave (exact), the highest bits first.  An infinite or NaN value
// leaves NaN, so some part is NaN.
template <int kP>
__device__ __forceinline__ void cut_pair(float a, float b, uint32_t (&part)[kP]) {
#pragma unroll
    for (int p = 0; p < kP; ++p) {
        const uint32_t ua = __float_as_uint(a), ub = __float_as_uint(b);
        part[p] = __byte_perm(ua, ub, 0x7632);
        a -= __uint_as_float(ua & 0xFFFF0000u);
        b -= __uint_as_float(ub & 0xFFFF0000u);
    }
}

__device__ __forceinline__ void to_pairs(const uint4 (&raw)[2], Pairs<float>& o) {
    const uint32_t w[8] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w, raw[1].x, raw[1].y, raw[1].z, raw[1].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t part[3];
        cut_pair(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]), part);
#pragma unroll
        for (int p = 0; p < 3; ++p) o.pair[p][i] = part[p];
    }
}
__device__ __forceinline__ void to_pairs(const uint4 (&raw)[1], Pairs<__half>& o) {
    const uint32_t w[4] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        uint32_t part[2];
        cut_pair(f.x, f.y, part);
        o.pair[0][i] = part[0];
        o.pair[1][i] = part[1];
    }
}
__device__ __forceinline__ void to_pairs(const uint4 (&raw)[1], Pairs<__nv_bfloat16>& o) {
    o.pair[0][0] = raw[0].x;
    o.pair[0][1] = raw[0].y;
    o.pair[0][2] = raw[0].z;
    o.pair[0][3] = raw[0].w;
}

template <class T>
constexpr int kRaw = 8 / kElemsPer16<T>;

// Elements [0, n) of p (n may be <= 0 or above 8) as raw packs, zeros behind
// them.  kVec: p is 16-byte aligned and, where n > 0, all 8 may be read; with
// kWhole all 8 count.  kL2: p is data of earlier kernels (one by one its
// elements share lines in L1, and the kernel neither starts early nor lets
// others; launch_kernel).
template <class T, bool kVec, bool kWhole = false, bool kL2 = false>
__device__ __forceinline__ void load8(const T* p, int n, uint4 (&raw)[kRaw<T>]) {
    constexpr int kN = kElemsPer16<T>;
    if (kVec) {
#pragma unroll
        for (int i = 0; i < kRaw<T>; ++i) {
            raw[i] = make_uint4(0, 0, 0, 0);
            if (n > 0) {
                const uint4* q = reinterpret_cast<const uint4*>(p) + i;
                raw[i] = kL2 ? load_l2_once(q) : __ldg(q);
            }
        }
        if (!kWhole && n > 0 && n < 8) {
#pragma unroll
            for (int i = 0; i < kRaw<T>; ++i) {
                Pack<T, kN> v;
                memcpy(&v, &raw[i], 16);
#pragma unroll
                for (int j = 0; j < kN; ++j)
                    if (i * kN + j >= n) v.e[j] = from_float<T>(0.0f);
                memcpy(&raw[i], &v, 16);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < kRaw<T>; ++i) {
            Pack<T, kN> v;
#pragma unroll
            for (int j = 0; j < kN; ++j) v.e[j] = i * kN + j < n ? p[i * kN + j] : from_float<T>(0.0f);
            memcpy(&raw[i], &v, 16);
        }
    }
}

// Part q alone of 8 raw 16-bit elements.
__device__ __forceinline__ void part_of(const uint4& raw, int q, __nv_bfloat16, uint32_t (&pair)[4]) {
    pair[0] = raw.x, pair[1] = raw.y, pair[2] = raw.z, pair[3] = raw.w;
}
__device__ __forceinline__ void part_of(const uint4& raw, int q, __half, uint32_t (&pair)[4]) {
    Pairs<__half> all;
    const uint4 one[1] = {raw};
    to_pairs(one, all);
#pragma unroll
    for (int i = 0; i < 4; ++i) pair[i] = all.pair[q][i];
}

__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Tensor cores cut sums off instead of rounding them, which adds up along a
// chain of products; so a chain ends after kChainMmas of them, and chains are
// added with rounding.
constexpr int kChainMmas = 24;

// d[j] += (rows lo, hi) x (column j of a chunk's 16-bit weights) over a chunk of
// 32, every part with every part, the smallest products first; the same step
// of all columns in a row, since each waits for its column's last.
template <class TW, int kN, int kPA>
__device__ __forceinline__ void mma_chunk(float (*d)[4], const uint32_t (&lo)[kPA][4], const uint32_t (&hi)[kPA][4],
                                          const uint4 (*raw)[1]) {
#pragma unroll
    for (int q = kParts<TW> - 1; q >= 0; --q) {
        uint32_t b[kN][4];
#pragma unroll
        for (int j = 0; j < kN; ++j) part_of(raw[j][0], q, TW{}, b[j]);
#pragma unroll
        for (int p = kPA - 1; p >= 0; --p)
#pragma unroll
            for (int s = 0; s < 4; s += 2)
#pragma unroll
                for (int j = 0; j < kN; ++j)
                    mma_bf16(d[j], lo[p][s], hi[p][s], lo[p][s + 1], hi[p][s + 1], b[j][s], b[j][s + 1]);
    }
}

// Fetches `bytes` (a multiple of 16; 1 MiB of them at most) at p (16-byte
// aligned) into L2.
__device__ __forceinline__ void prefetch(const void* p, long long bytes) {
    const uint32_t n = (uint32_t)(bytes < (1 << 20) ? bytes : (1 << 20));
    if (n) asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(n) : "memory");
}

// The tile of block `tile`: its rows (-1 behind the last) and their count, 0
// where it has none.  Every thread of the block calls it.
template <int kMT>
__device__ __forceinline__ int find_rows(const LowRankArgs& a, const Workspace& ws, int tile, int* row_of, int* slot) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (kMT == 1 && a.m <= kDirectRows) {
        __shared__ uint32_t same[kWarps];
        const int id = load_l1(a.ids + tile);
        *slot = id;
        if (threadIdx.x < 16) row_of[threadIdx.x] = -1;
        const bool mine = (int)threadIdx.x < a.m && load_l1(a.ids + threadIdx.x) == id;
        const uint32_t votes = __ballot_sync(0xffffffffu, mine);
        if (lane == 0) same[warp] = votes;
        __syncthreads();
        int before = 0, place = 0, all = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const uint32_t v = same[w];
            const int left = tile - 32 * w;  // rows of this word before the tile's
            before += __popc(left >= 32 ? v : left <= 0 ? 0u : v & ((1u << left) - 1));
            if (w < warp) place += __popc(v);
            all += __popc(v);
        }
        if (id < 0 || id >= a.slots || before % 16 != 0) return 0;
        place += __popc(votes & ((1u << lane) - 1)) - before;
        if (mine && place >= 0 && place < 16) row_of[place] = threadIdx.x;
        __syncthreads();
        return min(16, all - before);
    }
    if (tile >= load_l2_once(ws.count)) return 0;
    const Tile t = load_l2_once(ws.tiles + tile);
    *slot = t.slot;
    if (threadIdx.x < 16 * kMT) row_of[threadIdx.x] = (int)threadIdx.x < t.rows ? load_l2_once(ws.order + t.first + threadIdx.x) : -1;
    __syncthreads();
    return t.rows;
}

__device__ __forceinline__ int rank_of(const LowRankArgs& a, int slot) {
    return a.ranks ? min(max(load_l1(a.ranks + slot), 0), a.max_rank) : a.max_rank;
}

// ---- h = A x -----------------------------------------------------------------

__host__ __device__ int pass_width(int max_rank) { return rank_pitch(max_rank) < kRankPass ? rank_pitch(max_rank) : kRankPass; }

// kVec: rows of x and of A start on 16 bytes and are whole packs of 8.
template <class TX, class TW, bool kVec, int kMT>
__global__ void __launch_bounds__(kThreads, 2) shrink_kernel(const LowRankArgs a, void* workspace, const Shape shape) {
    // The kernels before have completed when this one's blocks let expand
    // start, so expand may read everything but h before its own wait.
    pdl_wait_primary();
    if (kVec) pdl_launch_dependents();
    constexpr int kGroups = kWarps / kMT;  // warps that split a tile's k
    __shared__ int row_of[16 * kMT];
    extern __shared__ float sums[];  // [kGroups][16 * kMT][width]
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, t = lane & 3;
    const int mt = warp % kMT, group = warp / kMT;
    const Workspace ws = workspace_at(workspace, (size_t)a.m, (size_t)a.slots, shape.shares, a.max_rank, kMT);
    int slot = 0;
    const int rows = find_rows<kMT>(a, ws, blockIdx.x, row_of, &slot);
    if (rows == 0) return;
    const int rank = rank_of(a, slot);
    if (rank == 0) return;
    const int k_begin = blockIdx.y * shape.k_span, k_end = min(a.k, k_begin + shape.k_span);
    const TW* wa = static_cast<const TW*>(a.a) + (long long)slot * a.max_rank * a.k;
    if (kVec) {
        for (int i = threadIdx.x; i < rows + rank; i += kThreads) {
            if (i < rows)
                prefetch(static_cast<const TX*>(a.x) + row_of[i] * a.ldx + k_begin, (k_end - k_begin) * (long long)sizeof(TX));
            else
                prefetch(wa + (long long)(i - rows) * a.k + k_begin, (k_end - k_begin) * (long long)sizeof(TW));
        }
    }
    // Rows behind the tile's last and ranks behind the adapter's last are taken
    // as the last: what comes out for them is not used.
    const int width = pass_width(a.max_rank), hp = rank_pitch(a.max_rank);
    const TX* x_lo = static_cast<const TX*>(a.x) + row_of[min(16 * mt + g, rows - 1)] * a.ldx;
    const TX* x_hi = static_cast<const TX*>(a.x) + row_of[min(16 * mt + g + 8, rows - 1)] * a.ldx;
    const int hi_end = 16 * mt + 8 < rows ? k_end : 0;  // no loads for an upper half without rows
    constexpr int kStep = 32 * kGroups;
    for (int r0 = 0; r0 < rank; r0 += kRankPass) {
        if (r0) __syncthreads();  // the pass before has been read
        float acc[kRankPass / 8][4] = {};
        // One chunk of 32: its elements are at hand, and the next chunk's are
        // fetched into the places that its products leave; with 8 columns there
        // are no registers for that, and A's come at the chunk's start (4096 x
        // 4096 x 4096, rank 16: 51 us, without it 54; rank 64: 78 us, with it,
        // spilling, 87).  k is a whole number of packs where kVec.
        uint4 raw_lo[kRaw<TX>], raw_hi[kRaw<TX>], raw_a[kRankPass / 8][1];
        auto fetch_x = [&](int k) {
            load8<TX, kVec, kVec, true>(x_lo + k, k_end - k, raw_lo);
            load8<TX, kVec, kVec, true>(x_hi + k, hi_end - k, raw_hi);
        };
        auto fetch_a = [&](int k, int j) {
            const int r = min(r0 + 8 * j + g, rank - 1);
            load8<TW, kVec, kVec>(wa + (long long)r * a.k + k, k_end - k, raw_a[j]);
        };
        auto chunk = [&](int k0, auto columns) {
            constexpr int kN = decltype(columns)::value;  // 8-rank columns
            constexpr bool kAhead = kN < 8;
            const int next = k0 + kStep + 8 * t;
            Pairs<TX> lo, hi;
            to_pairs(raw_lo, lo);
            to_pairs(raw_hi, hi);
            // two-part weights: 2 columns' parts at a time (4096 rows of rank 64:
            // 126 us, 4 columns at a time with their loads 140 us)
            constexpr int kAtOnce = kAhead || kParts<TW> == 1 ? kN : 2;
            if (!kAhead) {
#pragma unroll
                for (int j = 0; j < kN; ++j) fetch_a(k0 + 8 * t, j);
            }
            fetch_x(next);
#pragma unroll
            for (int j0 = 0; j0 < kN; j0 += kAtOnce)
                mma_chunk<TW, kAtOnce>(acc + j0, lo.pair, hi.pair, raw_a + j0);
            if (kAhead) {
#pragma unroll
                for (int j = 0; j < kN; ++j) fetch_a(next, j);
            }
        };
        // A chain's sums to the warp's place in shared memory (4096 x 4096 x 4096
        // of rank 64: the sums' error 1.2e-6 in chains of 96, 3.5e-7 in chains of
        // 24, at 79 us against 77 us).
        constexpr int kChain = kChainMmas / (2 * kParts<TX> * kParts<TW>);  // chunks
        float* place = sums + (group * 16 * kMT + 16 * mt) * width + 2 * t;
        auto put = [&](auto columns, bool add) {
            constexpr int kN = decltype(columns)::value;
#pragma unroll
            for (int j = 0; j < kN; ++j) {
                if (8 * j >= width) break;
                float2* lo = reinterpret_cast<float2*>(place + g * width + 8 * j);
                float2* hi = reinterpret_cast<float2*>(place + (g + 8) * width + 8 * j);
                const float2 l = add ? *lo : make_float2(0.0f, 0.0f), h = add ? *hi : make_float2(0.0f, 0.0f);
                *lo = make_float2(l.x + acc[j][0], l.y + acc[j][1]);
                *hi = make_float2(h.x + acc[j][2], h.y + acc[j][3]);
                acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.0f;
            }
        };
        auto share = [&](auto columns) {
            int k0 = k_begin + 32 * group;
            fetch_x(k0 + 8 * t);
            constexpr int kN = decltype(columns)::value;
            if (kN < 8) {
#pragma unroll
                for (int j = 0; j < kN; ++j) fetch_a(k0 + 8 * t, j);
            }
            bool add = false;
            for (int n = 1; k0 < k_end; k0 += kStep, ++n) {
                chunk(k0, columns);
                if (n % kChain == 0) {
                    put(columns, add);
                    add = true;
                }
            }
            put(columns, add);
        };
        if (16 * mt < rows) {
            if (rank - r0 <= 8)
                share(std::integral_constant<int, 1>{});
            else if (rank - r0 <= 16)
                share(std::integral_constant<int, 2>{});
            else if (rank - r0 <= 32)
                share(std::integral_constant<int, 4>{});
            else
                share(std::integral_constant<int, 8>{});
        }
        __syncthreads();
        for (int r = warp; r < rows; r += kWarps) {
            float* h = ws.h + ((size_t)blockIdx.y * a.m + row_of[r]) * hp + r0;
            for (int c = lane; c < width && r0 + c < hp; c += 32) {
                float s = 0.0f;
#pragma unroll
                for (int w = 0; w < kGroups; ++w) s += sums[(w * 16 * kMT + r) * width + c];
                h[c] = s;
            }
        }
    }
}

// ---- y += B h ----------------------------------------------------------------

// Bytes of a row of one part of h in shared memory: a multiple of 32 ranks, 64
// bytes past a multiple of 128 so that the rows' 16-byte reads fall into all
// banks.
__host__ __device__ int part_pitch(int max_rank) {
    const int b = (max_rank + 31) / 32 * 64;
    return b % 128 == 64 ? b : b + 64;
}

// y[0..4) += v, added in L2: nothing waits for y to arrive, and no sector of y
// that another block adds to comes to L1.  Each element is added to once, so the
// result does not depend on any order.  (The addition in L2 takes subnormal
// values as 0.)
__device__ __forceinline__ void add4(float* y, float v0, float v1, float v2, float v3) {
    asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(y), "f"(v0), "f"(v1), "f"(v2), "f"(v3) : "memory");
}

__device__ __forceinline__ void add1(float* y, float v) {
    asm volatile("red.global.add.f32 [%0], %1;" ::"l"(y), "f"(v) : "memory");
}

// kVecB: rows of B start on 16 bytes and are whole packs of 8; kVecY: 16-byte
// access to y.
template <class TW, bool kVecB, bool kVecY, int kMT>
__global__ void __launch_bounds__(kThreads, 2) expand_kernel(const LowRankArgs a, void* workspace, const Shape shape) {
    constexpr int kGroups = kWarps / kMT;  // warps that split a tile's columns
    __shared__ int row_of[16 * kMT];
    extern __shared__ __align__(128) uint8_t parts[];  // [3][16 * kMT][pitch], sums of chains
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, t = lane & 3;
    const int mt = warp % kMT, group = warp / kMT;
    const Workspace ws = workspace_at(workspace, (size_t)a.m, (size_t)a.slots, shape.shares, a.max_rank, kMT);
    int slot = 0;
    const int rows = find_rows<kMT>(a, ws, blockIdx.x, row_of, &slot);
    const int rank = rows ? rank_of(a, slot) : 0;
    const int c_begin = blockIdx.y * shape.col_span, c_end = min(a.n, c_begin + shape.col_span);
    const TW* wb = static_cast<const TW*>(a.b) + (long long)slot * a.n * a.max_rank;
    if (rank) {
        if (kVecY)
            for (int i = threadIdx.x; i < rows; i += kThreads)
                prefetch(a.y + row_of[i] * a.ldy + c_begin, (c_end - c_begin) * 4LL);
        if (kVecB && threadIdx.x == kThreads - 1)
            prefetch(wb + (long long)c_begin * a.max_rank, (long long)(c_end - c_begin) * a.max_rank * (long long)sizeof(TW));
    }
    pdl_wait_primary();
    pdl_launch_dependents();  // no earlier: shrink may have brought x to L1
    if (rank == 0) return;

    // h: the shares' sum, scaled, as three bf16 parts
    const float scale = a.scales ? load_l1(a.scales + slot) : 1.0f;
    const int pitch = part_pitch(a.max_rank), hp = rank_pitch(a.max_rank);
    for (int r = threadIdx.x >> 3; r < 16 * kMT; r += kThreads / 8)
        for (int c = (threadIdx.x & 7) * 4; c < rank; c += 32) {
            float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (r < rows) {
                const float* h = ws.h + (size_t)row_of[r] * hp + c;
#pragma unroll 8
                for (int w = 0; w < shape.shares; ++w) {
                    const float4 v = load_l2_once(reinterpret_cast<const float4*>(h + (size_t)w * a.m * hp));
                    s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
                }
            }
            uint32_t first[3], second[3];
            cut_pair(s.x * scale, c + 1 < rank ? s.y * scale : 0.0f, first);
            cut_pair(c + 2 < rank ? s.z * scale : 0.0f, c + 3 < rank ? s.w * scale : 0.0f, second);
#pragma unroll
            for (int p = 0; p < 3; ++p)
                *reinterpret_cast<uint2*>(parts + (p * 16 * kMT + r) * pitch + 2 * c) = make_uint2(first[p], second[p]);
        }
    // zeros up to the next multiple of 32 ranks
    for (int r = threadIdx.x >> 3; r < 16 * kMT; r += kThreads / 8) {
        const int c = (rank + 3) / 4 * 4 + (threadIdx.x & 7) * 4;
        if (c < (rank + 31) / 32 * 32)
#pragma unroll
            for (int p = 0; p < 3; ++p)
                *reinterpret_cast<uint2*>(parts + (p * 16 * kMT + r) * pitch + 2 * c) = make_uint2(0, 0);
    }
    __syncthreads();
    if (16 * mt >= rows) return;

    const bool has_lo = 16 * mt + g < rows, has_hi = 16 * mt + g + 8 < rows;
    float* y_lo = a.y + row_of[min(16 * mt + g, rows - 1)] * a.ldy;
    float* y_hi = a.y + row_of[min(16 * mt + g + 8, rows - 1)] * a.ldy;
    const uint8_t* h_lo = parts + (16 * mt + g) * pitch + 16 * t;
    constexpr int kStep = kWarpCols * kGroups;
    const int first = c_begin + kWarpCols * group;  // of the columns, kWarpCols at a time
    const TW* b_lane = wb + (long long)(first + 4 * (g >> 1) + (g & 1)) * a.max_rank;  // this lane's first
    // This lane's elements of kWarpCols columns of B over ranks r0 to r0 + 31.
    // kWhole: all columns exist and rows of B are whole packs; packs past the
    // rank meet zeros of h, so the first pack stands in for them, and what a
    // pack holds past the rank (`in_rank` masks the last step's) is made zero.
    // `cols`: else the columns that exist, of kWarpCols.
    auto fetch_b = [&](uint4(&raw)[kWarpCols / 8][1], const TW* b0, int r0, int cols, auto whole) {
        constexpr bool kWhole = decltype(whole)::value;
        const int r = r0 + 8 * t, at = kWhole && r >= rank ? 0 : r;
#pragma unroll
        for (int j = 0; j < kWarpCols / 8; ++j) {
            const int bc = 16 * (j >> 1) + 2 * (j & 1);
            const bool in = kWhole || bc + 4 * (g >> 1) + (g & 1) < cols;
            load8<TW, kVecB, kWhole>(b0 + bc * a.max_rank + at, kWhole ? 8 : in ? rank - r : 0, raw[j]);
        }
    };
    const bool ragged = rank % 8 != 0;
    uint32_t in_rank[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = (rank - 1) / 32 * 32 + 8 * t + 2 * i;
        in_rank[i] = (r < rank ? 0xFFFFu : 0u) | (r + 1 < rank ? 0xFFFF0000u : 0u);
    }
    // d += this lane's h over those ranks x the columns
    auto product = [&](float(&acc)[kWarpCols / 8][4], const uint4(&raw)[kWarpCols / 8][1], int r0) {
        uint32_t lo[3][4], hi[3][4];
#pragma unroll
        for (int p = 0; p < 3; ++p) {
            const uint8_t* h = h_lo + p * 16 * kMT * pitch + 2 * r0;
            memcpy(lo[p], __builtin_assume_aligned(h, 16), 16);
            memcpy(hi[p], __builtin_assume_aligned(h + 8 * pitch, 16), 16);
        }
        mma_chunk<TW, kWarpCols / 8>(acc, lo, hi, raw);
    };
    auto store = [&](const float(&acc)[kWarpCols / 8][4], int c0, int cols) {
#pragma unroll
        for (int u = 0; u < kWarpCols / 16; ++u) {
            const int at = 16 * u + 4 * t, col = c0 + at;
            if (kVecY) {
                const bool in = at < cols;
                if (has_lo && in) add4(y_lo + col, acc[2 * u][0], acc[2 * u][1], acc[2 * u + 1][0], acc[2 * u + 1][1]);
                if (has_hi && in) add4(y_hi + col, acc[2 * u][2], acc[2 * u][3], acc[2 * u + 1][2], acc[2 * u + 1][3]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (has_lo && at + i < cols) add1(y_lo + col + i, acc[2 * u + i / 2][i % 2]);
                    if (has_hi && at + i < cols) add1(y_hi + col + i, acc[2 * u + i / 2][2 + i % 2]);
                }
            }
        }
    };
    // A chain's sums wait in shared memory, behind the parts of h, for the next
    // one's.  Ranks of one chain need none of it.  (4096 x 4096 x 4096 of rank 256:
    // 248 us, in one chain 246 us; sums of one sign lose 1.1e-6, in one chain
    // 2.8e-6, with fp16 weights 5.4e-7 and 4.3e-6.)
    constexpr int kChain = 32 * kChainMmas / (2 * 3 * kParts<TW>);  // ranks
    float* parked = reinterpret_cast<float*>(parts + 3 * 16 * kMT * pitch) + threadIdx.x;
    auto end_chain = [&](float(&acc)[kWarpCols / 8][4], int r0) {
        if ((r0 + 32) % kChain != 0 && r0 + 32 < rank) return;
        const bool add = r0 >= kChain, last = r0 + 32 >= rank;
#pragma unroll
        for (int i = 0; i < kWarpCols / 2; ++i) {
            float& v = acc[i / 4][i % 4];
            if (add) v += parked[i * kThreads];
            if (!last) {
                parked[i * kThreads] = v;
                v = 0.0f;
            }
        }
    };
    int c0 = first;
    const long long b_step = (long long)kStep * a.max_rank;
    if (kVecB && c0 + kWarpCols <= c_end) {
        // the next step's elements are fetched while this one's products run
        uint4 raw[kWarpCols / 8][1];
        fetch_b(raw, b_lane, 0, kWarpCols, std::true_type{});
        for (; c0 + kWarpCols <= c_end; c0 += kStep, b_lane += b_step) {
            float acc[kWarpCols / 8][4] = {};
            for (int r0 = 0; r0 < rank; r0 += 32) {
                uint4 next[kWarpCols / 8][1];
                if (r0 + 32 < rank)
                    fetch_b(next, b_lane, r0 + 32, kWarpCols, std::true_type{});
                else if (c0 + kStep + kWarpCols <= c_end)
                    fetch_b(next, b_lane + b_step, 0, kWarpCols, std::true_type{});
                if (ragged && r0 + 32 >= rank) {
#pragma unroll
                    for (int j = 0; j < kWarpCols / 8; ++j) {
                        raw[j][0].x &= in_rank[0], raw[j][0].y &= in_rank[1];
                        raw[j][0].z &= in_rank[2], raw[j][0].w &= in_rank[3];
                    }
                }
                product(acc, raw, r0);
                if (rank > kChain) end_chain(acc, r0);
#pragma unroll
                for (int j = 0; j < kWarpCols / 8; ++j) raw[j][0] = next[j][0];
            }
            store(acc, c0, kWarpCols);
        }
    }
    for (; c0 < c_end; c0 += kStep, b_lane += b_step) {
        float acc[kWarpCols / 8][4] = {};
        for (int r0 = 0; r0 < rank; r0 += 32) {
            uint4 raw[kWarpCols / 8][1];
            fetch_b(raw, b_lane, r0, c_end - c0, std::false_type{});
            product(acc, raw, r0);
            if (rank > kChain) end_chain(acc, r0);
        }
        store(acc, c0, c_end - c0);
    }
}

// ---- sorting -----------------------------------------------------------------

// Sorts the rows by adapter: order[] lists the rows of slot 0, then 1, ...,
// each slot's rows cut into tiles of tile_rows.  The order of a slot's rows
// varies from run to run; their results do not depend on it.
constexpr int kPlanThreads = 1024;
constexpr int kPlanHeld = 8;  // rows of a thread that stay in its registers
__global__ void __launch_bounds__(kPlanThreads)
    plan_rows_kernel(const int32_t* ids, int m, int slots, int tile_rows, const Workspace ws) {
    pdl_wait_primary();
    pdl_launch_dependents();
    extern __shared__ int counts[];  // [slots]
    __shared__ int2 warp_sum[kPlanThreads / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int id[kPlanHeld], place[kPlanHeld];  // slot, -1: none; and the row's place in it
#pragma unroll
    for (int u = 0; u < kPlanHeld; ++u) {
        const int i = u * kPlanThreads + threadIdx.x;
        id[u] = i < m ? load_l1(ids + i) : -1;
        if (id[u] >= slots || id[u] < 0) id[u] = -1;
    }
    for (int s = threadIdx.x; s < slots; s += kPlanThreads) counts[s] = 0;
    __syncthreads();
    // Neighbouring rows mostly share an adapter: one atomic for a warp's equals.
    auto count = [&](int slot) {
        const uint32_t peers = __match_any_sync(0xffffffffu, slot);
        const int leader = __ffs(peers) - 1;
        int first = 0;
        if (slot >= 0 && lane == leader) first = atomicAdd(&counts[slot], __popc(peers));
        return __shfl_sync(0xffffffffu, first, leader) + __popc(peers & ((1u << lane) - 1));
    };
#pragma unroll
    for (int u = 0; u < kPlanHeld; ++u)
        if (u * kPlanThreads < m) place[u] = count(id[u]);
    for (int i = kPlanHeld * kPlanThreads + threadIdx.x; i < (m + 31) / 32 * 32; i += kPlanThreads) {
        const int slot = i < m ? load_l1(ids + i) : -1;
        const int at = count(slot < 0 || slot >= slots ? -1 : slot);
        if (i < m) ws.place[i] = at;
    }
    __syncthreads();
    // Where each slot's rows and tiles begin: a scan over runs of slots.
    const int run = (slots + kPlanThreads - 1) / kPlanThreads;
    const int s0 = min(slots, (int)threadIdx.x * run), s1 = min(slots, s0 + run);
    int2 sum = make_int2(0, 0);
    for (int s = s0; s < s1; ++s) {
        sum.x += counts[s];
        sum.y += (counts[s] + tile_rows - 1) / tile_rows;
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
    if (threadIdx.x == kPlanThreads - 1) *ws.count = at.y + sum.y;
    for (int s = s0; s < s1; ++s) {
        const int n = counts[s];
        for (int i = 0; i < n; i += tile_rows)
            ws.tiles[at.y++] = Tile{s, at.x + i, min(tile_rows, n - i), 0};
        counts[s] = at.x;
        at.x += n;
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kPlanHeld; ++u)
        if (u * kPlanThreads < m && id[u] >= 0) ws.order[counts[id[u]] + place[u]] = u * kPlanThreads + threadIdx.x;
    for (int i = kPlanHeld * kPlanThreads + threadIdx.x; i < m; i += kPlanThreads) {
        const int slot = load_l1(ids + i);
        if (slot >= 0 && slot < slots) ws.order[counts[slot] + ws.place[i]] = i;
    }
}

// ---- launches ----------------------------------------------------------------

Shape shape_of(const LowRankArgs& a) {
    Shape s;
    const bool direct = a.m <= kDirectRows;
    s.mt = direct ? 1 : kSortedTiles;
    // Blocks a tile, so that each grid fills the SMs twice over, which is what
    // fits at once: a part of a third block an SM costs as much as a whole one
    // (4096 x 4096 x 4096 of rank 64: 82 us, with 3 an SM 94 us, with 1 119
    // us).  No share is smaller than one chunk a warp.  How many tiles have
    // rows is only known on the device; full tiles and one in part for every
    // slot (for every second, where many rows are sorted) are taken for it.
    const long long parts = direct ? a.slots : (a.slots < a.m ? a.slots : a.m) / 2 + 1;
    const long long full = a.m / (16 * s.mt) + parts, tiles = full < a.m ? full : a.m;
    const long long most = 2LL * sm_count() / tiles, want = most > 1 ? most : 1;
    const int groups = kWarps / s.mt;
    auto cut_up = [&](int n, int grain, int* shares, int* span) {
        const long long units = (n + grain - 1) / grain;
        const long long parts = units < want ? units : want;
        const long long each = (units + parts - 1) / parts;
        *span = (int)(each * grain);
        *shares = (int)((units + each - 1) / each);
    };
    cut_up(a.k, 32 * groups, &s.shares, &s.k_span);
    cut_up(a.n, kWarpCols * groups, &s.col_shares, &s.col_span);
    return s;
}

template <class Kern>
cudaError_t launch_grid(bool early, Kern kern, dim3 grid, int smem, cudaStream_t stream, const LowRankArgs& a, void* ws,
                        const Shape& shape) {
    if (smem > 47 * 1024) {  // with the static arrays past the 48 KiB that need no attribute
        const cudaError_t e = ensure_smem_attr(kern, (size_t)smem);
        if (e != cudaSuccess) return e;
    }
    return launch_kernel(early, kern, grid, dim3(kThreads), (size_t)smem, stream, a, ws, shape);
}

bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <class TX, class TW, int kMT>
cudaError_t launch_shrink(const LowRankArgs& a, void* ws, const Shape& shape, unsigned tiles, cudaStream_t stream) {
    const bool vec = a.k % 8 == 0 && on16(a.x) && a.ldx * sizeof(TX) % 16 == 0 && on16(a.a);
    const int smem = kWarps * 16 * pass_width(a.max_rank) * (int)sizeof(float);
    const dim3 grid(tiles, (unsigned)shape.shares);
    return vec ? launch_grid(true, shrink_kernel<TX, TW, true, kMT>, grid, smem, stream, a, ws, shape)
               : launch_grid(false, shrink_kernel<TX, TW, false, kMT>, grid, smem, stream, a, ws, shape);
}

template <class TW, int kMT>
cudaError_t launch_expand(const LowRankArgs& a, void* ws, const Shape& shape, unsigned tiles, cudaStream_t stream) {
    const bool vb = a.max_rank % 8 == 0 && on16(a.b);
    const bool vy = a.n % 4 == 0 && on16(a.y) && a.ldy % 4 == 0;
    const int smem = 3 * 16 * kMT * part_pitch(a.max_rank) + (int)sizeof(float) * kThreads * kWarpCols / 2;
    const dim3 grid(tiles, (unsigned)shape.col_shares);
    if (vb && vy) return launch_grid(true, expand_kernel<TW, true, true, kMT>, grid, smem, stream, a, ws, shape);
    if (vb) return launch_grid(true, expand_kernel<TW, true, false, kMT>, grid, smem, stream, a, ws, shape);
    if (vy) return launch_grid(true, expand_kernel<TW, false, true, kMT>, grid, smem, stream, a, ws, shape);
    return launch_grid(true, expand_kernel<TW, false, false, kMT>, grid, smem, stream, a, ws, shape);
}

template <class TX, class TW>
cudaError_t launch(const LowRankArgs& a, void* workspace, cudaStream_t stream) {
    const Shape shape = shape_of(a);
    cudaError_t e;
    if (a.m <= kDirectRows) {
        e = launch_shrink<TX, TW, 1>(a, workspace, shape, (unsigned)a.m, stream);
        return e != cudaSuccess ? e : launch_expand<TW, 1>(a, workspace, shape, (unsigned)a.m, stream);
    }
    const Workspace ws = workspace_at(workspace, (size_t)a.m, (size_t)a.slots, shape.shares, a.max_rank, shape.mt);
    const unsigned tiles = (unsigned)max_tiles((size_t)a.m, (size_t)a.slots, 16 * shape.mt);
    e = launch_pdl_kernel(plan_rows_kernel, dim3(1), dim3(kPlanThreads), (size_t)a.slots * sizeof(int), stream, a.ids,
                          (int)a.m, a.slots, 16 * shape.mt, ws);
    if (e == cudaSuccess) e = launch_shrink<TX, TW, kSortedTiles>(a, workspace, shape, tiles, stream);
    return e != cudaSuccess ? e : launch_expand<TW, kSortedTiles>(a, workspace, shape, tiles, stream);
}

template <class TX>
cudaError_t launch_x(const LowRankArgs& a, int w_dtype, void* ws, cudaStream_t stream) {
    return w_dtype == ZQ_DTYPE_F16 ? launch<TX, __half>(a, ws, stream) : launch<TX, __nv_bfloat16>(a, ws, stream);
}

}  // namespace

size_t low_rank_workspace_bytes(const LowRankArgs& a) {
    const Shape s = shape_of(a);
    const size_t m = (size_t)a.m, slots = (size_t)a.slots;
    size_t b = h_bytes(m, s.shares, a.max_rank);
    if (a.m > kDirectRows) b += 256 + max_tiles(m, slots, 16 * s.mt) * sizeof(Tile) + 2 * m * sizeof(int);
    return align256(b);
}

cudaError_t launch_add_low_rank(const LowRankArgs& a, int x_dtype, int w_dtype, void* workspace, cudaStream_t stream) {
    if (x_dtype == ZQ_DTYPE_F32) return launch_x<float>(a, w_dtype, workspace, stream);
    if (x_dtype == ZQ_DTYPE_F16) return launch_x<__half>(a, w_dtype, workspace, stream);
    return launch_x<__nv_bfloat16>(a, w_dtype, workspace, stream);
}

}  // namespace zq

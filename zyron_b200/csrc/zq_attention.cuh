// zq_attention.cuh -- what the attention kernels share: where unfinished sums
// lie, and how they are joined.
#pragma once

#include "zq_elem.cuh"
#include "zq_paged.cuh"

namespace zq {
namespace attn {

// Sums are kept as the unscaled output row, with the maximum (base 2) that its
// weights are relative to and their sum.
struct Cut;
struct Workspace {
    // Of the kernel of few rows and of the other: parts of cut items, [block][2][rows][width]
    // and [block][2][width / 4][rows][4] (a thread a row there), their statistics
    // [block][2][rows][2], and by block the item that its first unit cuts.
    float* part_sums[2];
    float* part_stats[2];
    Cut* cuts[2];
    float* row_sums[2];    // with a prefix: own and prefix sums of every row, [rows][heads][dim]
    float* row_stats[2];   // [rows][heads][2]
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

// ---- plans ----------------------------------------------------------------------
//
// A plan deals the call's work out to the blocks of one kernel.  Work is counted
// in units; every block takes `share` consecutive ones.  Items (a tile of a
// request's rows of one kv head) follow one another, and a place inside an item
// stands for a border between its key tiles (cut()).
struct Item {
    Request r;
    int b;           // request, -1: the prefix
    int head;        // kv head
    int tile;        // tile of rows
    long long start, end;  // units
    int key_tiles;
};

// Requests of at most a.few_rows rows of a kv head: one item a head, units of 64
// keys, at least one, so that rows that see no key are written too.
struct FewPlan {
    static constexpr int kKeys = 64;
    const AttentionArgs& a;
    int group, prefix_rows;

    __device__ __forceinline__ Request get(int b) const {
        return b >= 0 ? load_request(a.batch, b) : Request{0, prefix_rows, a.prefix_length};
    }
    __device__ __forceinline__ int key_tiles(const Request& r) const { return r.length > 0 ? (r.length - 1) / kKeys + 1 : 1; }
    __device__ __forceinline__ long long cost(const Request& r) const {
        return r.rows > 0 && (long long)r.rows * group <= a.few_rows ? (long long)a.batch.kv_heads * key_tiles(r) : 0;
    }
    __device__ __forceinline__ Item item(int b, const Request& r, long long before, long long unit) const {
        const int n = key_tiles(r);
        const int head = (int)((unit - before) / n);
        const long long start = before + (long long)head * n;
        return Item{r, b, head, 0, start, start + n, n};
    }
    // The first item of a request that has some, and the one behind an item of the
    // same request.
    __device__ __forceinline__ Item first(int b, const Request& r, long long unit) const {
        const int n = key_tiles(r);
        return Item{r, b, 0, 0, unit, unit + n, n};
    }
    __device__ __forceinline__ bool advance(Item& it) const {
        if (++it.head == a.batch.kv_heads) return false;
        it.start = it.end;
        it.end += it.key_tiles;
        return true;
    }
    __device__ static __forceinline__ int cut(long long start, long long end, int, long long unit) {
        return (int)(min(max(unit, start), end) - start);
    }
};

// The other requests: tiles of `tokens` tokens, units of a key.  A causal tile
// sees the more keys the later it comes, so tile t counts base + step t units
// (one key tile's worth more than its keys: what an item costs besides), and a
// border is the key tile that lies as far along.
struct ManyPlan {
    static constexpr int kKeys = 128;
    const AttentionArgs& a;
    int group, prefix_rows;
    int tokens;

    __device__ __forceinline__ Request get(int b) const {
        return b >= 0 ? load_request(a.batch, b) : Request{0, prefix_rows, a.prefix_length};
    }
    __device__ __forceinline__ bool causal(int b) const { return b >= 0 && a.causal; }
    __device__ __forceinline__ int tiles(const Request& r) const { return (r.rows + tokens - 1) / tokens; }
    __device__ __forceinline__ long long base(int b, const Request& r) const {
        return (causal(b) ? (long long)max(r.length - r.rows, 0) + tokens : r.length) + kKeys;
    }
    __device__ __forceinline__ long long until(long long base, long long step, long long tile) const {
        return tile * base + step * (tile * (tile - 1) / 2);
    }
    __device__ __forceinline__ long long cost_of(int b, const Request& r) const {
        if ((long long)r.rows * group <= a.few_rows || r.rows <= 0) return 0;
        return a.batch.kv_heads * until(base(b, r), causal(b) ? tokens : 0, tiles(r));
    }
    __device__ __forceinline__ Item item(int b, const Request& r, long long before, long long unit) const {
        const long long base_ = base(b, r), step = causal(b) ? tokens : 0;
        const int n = tiles(r);
        const long long each = until(base_, step, n);
        const int head = (int)((unit - before) / each);
        const long long at = unit - before - head * each;
        int lo = 0, hi = n;  // the last tile that starts at or before `at`
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (until(base_, step, mid) <= at)
                lo = mid;
            else
                hi = mid;
        }
        const long long start = before + head * each + until(base_, step, lo);
        return Item{r, b, head, lo, start, start + base_ + step * lo, key_tiles(b, r, lo)};
    }
    __device__ __forceinline__ int key_tiles(int b, const Request& r, int tile) const {
        int keys = r.length;
        if (causal(b)) keys = min(keys, max(r.length - r.rows + (int)min((long long)r.rows, (tile + 1LL) * tokens), 0));
        return keys > 0 ? (keys - 1) / kKeys + 1 : 1;
    }
    __device__ __forceinline__ Item first(int b, const Request& r, long long unit) const {
        return Item{r, b, 0, 0, unit, unit + base(b, r), key_tiles(b, r, 0)};
    }
    __device__ __forceinline__ bool advance(Item& it) const {
        if ((it.tile + 1LL) * tokens < it.r.rows) {
            ++it.tile;
        } else {
            if (++it.head == a.batch.kv_heads) return false;
            it.tile = 0;
        }
        it.start = it.end;
        it.end += base(it.b, it.r) + (causal(it.b) ? (long long)tokens * it.tile : 0);
        it.key_tiles = key_tiles(it.b, it.r, it.tile);
        return true;
    }
    __device__ static __forceinline__ int cut(long long start, long long end, int key_tiles, long long unit) {
        return (int)((min(max(unit, start), end) - start) * key_tiles / (end - start));
    }
};
__device__ __forceinline__ long long cost_of(const FewPlan& plan, int, const Request& r) { return plan.cost(r); }
__device__ __forceinline__ long long cost_of(const ManyPlan& plan, int b, const Request& r) { return plan.cost_of(b, r); }

// What the join needs to know of an item that the border in front of a block's
// first unit cuts; rows 0: none, or an earlier border cuts it too.
struct alignas(16) Cut {
    long long start, end, share;
    int rows;       // of the item
    int first_row;  // of the request
    int row0;       // the item's first, among the request's rows of the kv head
    int head, key_tiles, prefix;
};

struct Found {
    long long share;   // units a block
    long long total;   // units of the call
    long long before;  // units before request b
    int b;             // the request that holds the block's first unit
};

// Block `g` of `blocks`: its share and where it begins, by a scan of the whole
// block (kThreads threads) over the requests.  `scratch` is kThreads / 32 + 2
// words of 64 bits.
template <int kThreads, class Plan>
__device__ Found find_block(const Plan& plan, long long g, int blocks, long long* scratch) {
    constexpr int kWarps = kThreads / 32;
    const int n = plan.a.batch.requests;
    const int each = (n + kThreads - 1) / kThreads;
    const int first = min(threadIdx.x * each, (unsigned)n), last = min(first + each, n);
    long long mine = 0;
    for (int b = first; b < last; ++b) mine += cost_of(plan, b, plan.get(b));
    const long long head = plan.prefix_rows ? cost_of(plan, -1, plan.get(-1)) : 0;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += v;
    }
    if (lane == 31) scratch[warp] = sum;
    __syncthreads();
    long long total = head, before = head + sum - mine;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) before += scratch[w];
        total += scratch[w];
    }
    const long long share = (total + blocks - 1) / blocks;
    const long long unit = g * share;
    if (unit < head) {
        if (threadIdx.x == 0) scratch[kWarps] = 0, scratch[kWarps + 1] = -1;
    } else if (unit >= before && unit < before + mine) {
        int b = first;
        long long c = cost_of(plan, b, plan.get(b));
        while (unit >= before + c) {
            before += c;
            ++b;
            c = cost_of(plan, b, plan.get(b));
        }
        scratch[kWarps] = before;
        scratch[kWarps + 1] = b;
    }
    __syncthreads();
    return Found{share, total, scratch[kWarps], (int)scratch[kWarps + 1]};  // before and b: if unit < total
}

// A block's way through its items: found once, then step by step, without a
// division but at the borders that cut an item (a search and 64-bit divisions an
// item took 12 us a part).
template <class Plan>
struct Cursor {
    const Plan& plan;
    long long unit, last;  // the block's units
    // the current part
    Item it;
    int first_tile, end_tile;
    bool whole;
    int slot;

    __device__ __forceinline__ Cursor(const Plan& p, const Found& f, long long g)
        : plan(p), unit(g * f.share), last(min(f.total, (g + 1) * f.share)), begin(unit) {
        if (unit < last) it = plan.item(f.b, plan.get(f.b), f.before, unit);
    }
    // The next part with key tiles of its own; false at the end.
    __device__ __forceinline__ bool next() {
        while (unit < last) {
            if (unit >= it.end && !plan.advance(it)) {
                int b = it.b;
                Request r;
                do r = plan.get(++b);
                while (cost_of(plan, b, r) == 0);
                it = plan.first(b, r, unit);
            }
            const long long to = min(it.end, last);
            first_tile = unit == it.start ? 0 : Plan::cut(it.start, it.end, it.key_tiles, unit);
            end_tile = to == it.end ? it.key_tiles : Plan::cut(it.start, it.end, it.key_tiles, to);
            unit = to;
            if (first_tile < end_tile) {
                whole = first_tile == 0 && end_tile == it.key_tiles;
                slot = it.start <= begin ? 0 : 1;
                return true;
            }
        }
        return false;
    }

    // The cut that block g's own first border makes (before the first next()).
    __device__ __forceinline__ Cut cut(long long share, long long g, int tile_rows) const {
        Cut c{};
        if (unit < last && it.start < unit && it.start >= (g - 1) * share) {
            c = Cut{it.start, it.end, share, 0, it.r.first, it.tile * tile_rows, it.head, it.key_tiles, it.b < 0};
            c.rows = (int)min((long long)tile_rows, (long long)it.r.rows * plan.group - c.row0);
        }
        return c;
    }

  private:
    long long begin;
};

// Four elements of a part.
__device__ __forceinline__ void put_part(float* sums, float* stats, long long row, int width, int d, const float (&v)[4],
                                         float most, float total) {
    *reinterpret_cast<float4*>(sums + row * width + d) = make_float4(v[0], v[1], v[2], v[3]);
    if (d == 0) *reinterpret_cast<float2*>(stats + 2 * row) = make_float2(most, total);
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

// Sums of several parts of a row, in a fixed order.
struct Joined {
    float most = -INFINITY, total = 0.0f, v[4] = {0.0f, 0.0f, 0.0f, 0.0f};

    __device__ __forceinline__ void add(const float2& stats, const float4& x) {
        const float now = fmaxf(most, stats.x);
        const float ref = now == -INFINITY ? 0.0f : now;
        const float keep = exp2_approx(most - ref), weight = exp2_approx(stats.x - ref);
        most = now;
        total = total * keep + stats.y * weight;
        v[0] = v[0] * keep + x.x * weight;
        v[1] = v[1] * keep + x.y * weight;
        v[2] = v[2] * keep + x.z * weight;
        v[3] = v[3] * keep + x.w * weight;
    }
};

// Joins the parts of the item that border g (in front of block g's first unit)
// cuts: rows [from, from + kSliceRows) of it.  kRows, kWidth: a part's; kByRow: its
// rows lie side by side (the kernel of many rows).  `parts` has room for the
// numbers of all parts.
constexpr int kSliceRows = 32;
template <class T, class Plan, int kRows, int kWidth, bool kByRow, int kThreads>
__device__ void join_item(const AttentionArgs& a, const Workspace& ws, int kind, int g, int from, int* parts) {
    const PagedBatch& p = a.batch;
    const int group = a.heads / p.kv_heads;
    Cut c;
#pragma unroll
    for (int i = 0; i < (int)(sizeof(Cut) / 16); ++i) {
        const uint4 w = load_l2(reinterpret_cast<const uint4*>(ws.cuts[kind] + g) + i);
        memcpy(reinterpret_cast<char*>(&c) + 16 * i, &w, 16);
    }
    if (from >= c.rows) return;
    // Blocks g - 1 .. hold parts of it; those without key tiles wrote none, and an
    // item that one block holds alone is finished.
    __shared__ int count;
    if (threadIdx.x < 32) {
        const int lane = threadIdx.x, h1 = (int)((c.end - 1) / c.share);
        int n = 0;
        for (int h0 = g - 1; h0 <= h1; h0 += 32) {
            const int h = h0 + lane;
            const bool has = h <= h1 && Plan::cut(c.start, c.end, c.key_tiles, h * c.share) <
                                            Plan::cut(c.start, c.end, c.key_tiles, (h + 1) * c.share);
            const unsigned m = __ballot_sync(0xffffffffu, has);
            // the first block's part may lie in its second slot
            if (has) parts[n + __popc(m & ((1u << lane) - 1u))] = 2 * h + (h == g - 1 && h * c.share < c.start ? 1 : 0);
            n += __popc(m);
        }
        if (lane == 0) count = n;
    }
    __syncthreads();
    const int n = count;
    if (n < 2) return;
    const int rows = min(c.rows - from, kSliceRows);
    for (int i = threadIdx.x; i < kSliceRows * (kWidth / 4); i += kThreads) {
        const int in = kByRow ? i % kSliceRows : i / (kWidth / 4);
        const int d = (kByRow ? i / kSliceRows : i % (kWidth / 4)) * 4, row = from + in;
        if (d >= p.dim || in >= rows) continue;
        Joined j;
        for (int k0 = 0; k0 < n; k0 += 4) {
            float2 stats[4];
            float4 sums[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {  // four parts' loads under way at once
                stats[k] = make_float2(-INFINITY, 0.0f);
                sums[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (k0 + k < n) {
                    const long long part = parts[k0 + k];
                    const long long at = kByRow ? (part * (kWidth / 4) + d / 4) * kRows + row
                                                : (part * kRows + row) * (kWidth / 4) + d / 4;
                    stats[k] = load_l2(reinterpret_cast<const float2*>(ws.part_stats[kind]) + part * kRows + row);
                    sums[k] = load_l2(reinterpret_cast<const float4*>(ws.part_sums[kind]) + at);
                }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) j.add(stats[k], sums[k]);
        }
        const int token = (c.row0 + row) / group, head = c.head * group + (c.row0 + row) % group;
        put_row<T>(a, ws, c.prefix, c.first_row + token, head, d, j.v, j.most, j.total);
    }
}

// The kernel of the requests with more than a.few_rows rows a kv head
// (zq_attention_sm100.cu).
constexpr int kManyRows = 256;  // rows of an item: two tiles of 128
cudaError_t launch_attend_many(const AttentionArgs& a, int dtype, const Workspace& ws, int blocks, cudaStream_t stream);

}  // namespace attn
}  // namespace zq

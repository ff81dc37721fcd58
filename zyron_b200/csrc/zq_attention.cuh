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
    // Of the kernel of few rows and of the other: parts of cut items, [worker][2][rows][width]
    // and [worker][2][width / 4][rows][4] (a thread a row there), their statistics
    // [worker][2][rows][2], and by worker the item that its first unit cuts.
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

// Weights are taken relative to a reference 2^kLift below the row's largest score:
// fp16 ends at 2^-24, so weights relative to the largest itself lose digits from
// 2^-14 down and are gone at e^-18, which counts where one key takes nearly all
// weight and has no value; fp16's upper end has room for 2^15.  bf16 has the
// exponents of fp32.  The reference is rounded up, so that no weight is above
// 2^kLift however large the scores are.
template <class T>
constexpr float kLift = kIsHalf<T> ? 15.0f : 0.0f;

__device__ __forceinline__ float exp2_approx(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

// Two fp32 values as packed pairs of 16-bit parts whose sum they are: to 2^-17 of
// the value for bf16, to 2^-22 for fp16, but not below 2^-25, half its smallest step.
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
// A plan deals the call's work out to the workers of one kernel: its warps (few
// rows) or blocks (many).  Work is counted in units; every worker takes `share`
// consecutive ones.  Items (a tile of a
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

// What the join needs to know of an item that the border in front of a worker's
// first unit cuts; rows 0: none, or an earlier border cuts it too, or one worker
// holds all its key tiles and has finished it.
struct alignas(16) Cut {
    long long start, end, share;
    int rows;       // of the item
    int first_row;  // of the request
    int row0;       // the item's first, among the request's rows of the kv head
    int head, key_tiles, prefix;
};

// Requests of at most a.few_rows rows of a kv head: one item a head.  A unit is 16
// keys, at least one, so that rows that see no key are written too; kItem more stand
// for what an item takes besides (with none, 51 items of 6 keys took 41 us, four a
// worker).
struct FewPlan {
    static constexpr int kKeys = 16;
    static constexpr int kItem = 3;
    static constexpr int kTeam = 4;  // warps of a block, which leave one part of an item that all of them are inside
    const AttentionArgs& a;
    int group, prefix_rows;

    __device__ __forceinline__ Request get(int b) const {
        return b >= 0 ? load_request(a.batch, b) : Request{0, prefix_rows, a.prefix_length};
    }
    __device__ __forceinline__ int key_tiles(const Request& r) const { return r.length > 0 ? (r.length - 1) / kKeys + 1 : 1; }
    __device__ __forceinline__ long long cost(const Request& r) const {
        return r.rows > 0 && (long long)r.rows * group <= a.few_rows ? (long long)a.batch.kv_heads * (key_tiles(r) + kItem) : 0;
    }
    __device__ __forceinline__ Item item(int b, const Request& r, long long before, long long unit) const {
        const int n = key_tiles(r);
        const int head = (int)((unit - before) / (n + kItem));
        const long long start = before + (long long)head * (n + kItem);
        return Item{r, b, head, 0, start, start + n + kItem, n};
    }
    // The first item of a request that has some, and the one behind an item of the
    // same request.
    __device__ __forceinline__ Item first(int b, const Request& r, long long unit) const {
        const int n = key_tiles(r);
        return Item{r, b, 0, 0, unit, unit + n + kItem, n};
    }
    __device__ __forceinline__ bool advance(Item& it) const {
        if (++it.head == a.batch.kv_heads) return false;
        it.start = it.end;
        it.end += it.key_tiles + kItem;
        return true;
    }
    // The extra units come first: a border inside them is in front of the keys.
    __device__ static __forceinline__ int cut(long long start, long long end, int, long long unit) {
        return (int)max(min(max(unit, start), end) - start - kItem, 0LL);
    }
    __device__ static __forceinline__ bool team_inside(long long start, long long end, long long share, int worker) {
        const long long first = worker / kTeam * kTeam * share;
        return start <= first && first + kTeam * share <= end;
    }
    // Whether worker h (of those that the item reaches) left a part of it.
    __device__ static __forceinline__ bool holds(const Cut& c, int h) {
        return cut(c.start, c.end, c.key_tiles, h * c.share) < cut(c.start, c.end, c.key_tiles, (h + 1) * c.share) &&
               (h % kTeam == 0 || !team_inside(c.start, c.end, c.share, h));
    }
};

// The other requests: tiles of `tokens` tokens, units of a key.  A causal tile
// sees the more keys the later it comes, so tile t counts base + step t units,
// and a border is the key tile that lies as far along.  kItem units more than its
// keys stand for what an item costs besides (prompts of 1000 to 2600 tokens: none
// 261 us, one key tile's worth 251, two 233, three 226, four 229, five 232).
struct ManyPlan {
    static constexpr int kKeys = 128;
    static constexpr int kItem = 3 * kKeys;
    const AttentionArgs& a;
    int group, prefix_rows;
    int tokens;

    __device__ __forceinline__ Request get(int b) const {
        return b >= 0 ? load_request(a.batch, b) : Request{0, prefix_rows, a.prefix_length};
    }
    __device__ __forceinline__ bool causal(int b) const { return b >= 0 && a.causal; }
    __device__ __forceinline__ int tiles(const Request& r) const { return (r.rows + tokens - 1) / tokens; }
    __device__ __forceinline__ long long base(int b, const Request& r) const {
        return (causal(b) ? (long long)max(r.length - r.rows, 0) + tokens : r.length) + kItem;
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
        const long long n = (min(max(unit, start), end) - start) * key_tiles;
        if ((n | (end - start)) >> 32 == 0) return (int)((uint32_t)n / (uint32_t)(end - start));  // a fifth of the time
        return (int)(n / (end - start));
    }
    __device__ static __forceinline__ bool holds(const Cut& c, int h) {
        return cut(c.start, c.end, c.key_tiles, h * c.share) < cut(c.start, c.end, c.key_tiles, (h + 1) * c.share);
    }
};
__device__ __forceinline__ long long cost_of(const FewPlan& plan, int, const Request& r) { return plan.cost(r); }
__device__ __forceinline__ long long cost_of(const ManyPlan& plan, int b, const Request& r) { return plan.cost_of(b, r); }

struct Found {
    long long share;   // units a worker
    long long total;   // units of the call
    long long before;  // units before request b
    int b;             // the request that holds the worker's first unit
};

// Workers g0 .. g0 + kFinds - 1 of `workers` (a worker is a warp or a block): their
// share, `least` units or more, and where they begin, by a scan of the whole block
// (kThreads threads) over the requests; for worker g0 + which.  `scratch` is
// kThreads / 32 + 2 kFinds words of 64 bits.
template <int kThreads, int kFinds, class Plan>
__device__ Found find_workers(const Plan& plan, long long g0, int which, int workers, int least, long long* scratch) {
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
    const long long even = (total + workers - 1) / workers, share = even > least ? even : least;
    long long* found = scratch + kWarps;
    int b = first;
    long long end = before;  // units up to request b
#pragma unroll 1
    for (int f = 0; f < kFinds; ++f) {
        const long long unit = (g0 + f) * share;
        if (unit < head) {
            if (threadIdx.x == 0) found[2 * f] = 0, found[2 * f + 1] = -1;
        } else if (unit >= before && unit < before + mine) {
            // one request a thread up to kThreads: nothing is read again
            long long c = each == 1 ? mine : cost_of(plan, b, plan.get(b));
            while (unit >= end + c) {
                end += c;
                ++b;
                c = cost_of(plan, b, plan.get(b));
            }
            found[2 * f] = end;
            found[2 * f + 1] = b;
        }
    }
    __syncthreads();
    return Found{share, total, found[2 * which], (int)found[2 * which + 1]};  // before and b: if its unit < total
}

// A worker's way through its items: found once, then step by step, without a
// division but at the borders that cut an item (a search and 64-bit divisions an
// item took 12 us a part).
template <class Plan>
struct Cursor {
    const Plan& plan;
    long long unit, last;  // the worker's units
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

    // The cut that worker g's own first border makes (before the first next()).
    __device__ __forceinline__ Cut cut(long long share, long long g, int tile_rows) const {
        Cut c{};
        if (unit < last && it.start < unit && it.start >= (g - 1) * share) {
            c = Cut{it.start, it.end, share, 0, it.r.first, it.tile * tile_rows, it.head, it.key_tiles, it.b < 0};
            int holders = 0;
            for (long long h = g - 1; holders < 2 && h * share < it.end; ++h) holders += Plan::holds(c, (int)h);
            if (holders == 2) c.rows = (int)min((long long)tile_rows, (long long)it.r.rows * plan.group - c.row0);
        }
        return c;
    }

  private:
    long long begin;
};

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

__device__ __forceinline__ Cut load_cut(const Workspace& ws, int kind, int g) {
    Cut c;
#pragma unroll
    for (int i = 0; i < (int)(sizeof(Cut) / 16); ++i) {
        const uint4 w = load_l2(reinterpret_cast<const uint4*>(ws.cuts[kind] + g) + i);
        memcpy(reinterpret_cast<char*>(&c) + 16 * i, &w, 16);
    }
    return c;
}

// The parts of the item that border g (in front of worker g's first unit) cuts,
// kDeep slots a call (-1: none), by the whole warp.
template <class Plan, int kDeep, class F>
__device__ __forceinline__ void each_parts(const Cut& c, int g, F f) {
    const int lane = threadIdx.x & 31, last = (int)((c.end - 1) / c.share);
    const bool second = (g - 1) * c.share < c.start;  // the first worker's part lies in its second slot
    for (int h0 = g - 1; h0 <= last; h0 += 32) {
        unsigned m = __ballot_sync(0xffffffffu, h0 + lane <= last && Plan::holds(c, h0 + lane));
        while (m) {
            long long slots[kDeep];
#pragma unroll
            for (int k = 0; k < kDeep; ++k) {
                const int h = h0 + __ffs(m) - 1;
                slots[k] = m ? 2LL * h + (h == g - 1 && second ? 1 : 0) : -1;
                m &= m - 1;
            }
            f(slots);
        }
    }
}

// Joins kSteps rows, kBetween apart, of a split item: a lane four elements of each,
// the loads of kDeep parts under way at once.  place(slot, row) is where a row of a
// part lies: its index in the statistics and in the sums.
template <class T, class Plan, int kSteps, int kBetween, int kDeep, class F>
__device__ __forceinline__ void join_rows(const AttentionArgs& a, const Workspace& ws, const Cut& c, int kind, int g,
                                          int row, int d, F place) {
    const int group = a.heads / a.batch.kv_heads;
    Joined j[kSteps];
    each_parts<Plan, kDeep>(c, g, [&](const long long (&slots)[kDeep]) {
        float2 stats[kDeep][kSteps];
        float4 x[kDeep][kSteps];
#pragma unroll
        for (int k = 0; k < kDeep; ++k)
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                stats[k][s] = make_float2(-INFINITY, 0.0f);
                x[k][s] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (slots[k] < 0 || row + s * kBetween >= c.rows || d >= a.batch.dim) continue;
                long long stats_at, sums_at;
                place(slots[k], row + s * kBetween, stats_at, sums_at);
                stats[k][s] = load_l2(reinterpret_cast<const float2*>(ws.part_stats[kind]) + stats_at);
                x[k][s] = load_l2(reinterpret_cast<const float4*>(ws.part_sums[kind]) + sums_at);
            }
#pragma unroll
        for (int k = 0; k < kDeep; ++k)
#pragma unroll
            for (int s = 0; s < kSteps; ++s) j[s].add(stats[k][s], x[k][s]);
    });
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
        const int in = row + s * kBetween;
        if (in < c.rows && d < a.batch.dim)
            put_row<T>(a, ws, c.prefix, c.first_row + (c.row0 + in) / group, c.head * group + (c.row0 + in) % group, d,
                       j[s].v, j[s].most, j[s].total);
    }
}

// The kernel of the requests with more than a.few_rows rows a kv head
// (zq_attention_sm100.cu).
constexpr int kManyRows = 256;  // rows of an item: two tiles of 128
cudaError_t launch_attend_many(const AttentionArgs& a, int dtype, const Workspace& ws, int blocks, cudaStream_t stream);

}  // namespace attn
}  // namespace zq

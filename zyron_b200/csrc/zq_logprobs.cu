// zq_logprobs.cu -- log probabilities of given tokens, with the entropy and
// the most likely alternatives, over rows of logits (zq_token_logprobs).
//
// One pass over a row, in base 2.  With L = log2(e) in fp32 and a reference
// logit r, every thread sums over its logits
//   a = fl(fl(x - r) L),   S = sum 2^a,   T = sum 2^a a
// and two such sums of references r1, r2 join as
//   r = max(r1, r2),  d_i = (r_i - r) L,  f_i = 2^d_i,
//   S = f1 S1 + f2 S2,  T = f1 (T1 + d1 S1) + f2 (T2 + d2 S2).
// Then  log p(t) = x_t - r - ln S  and  H = ln S - ln 2 T / S.  The reference is
// one of the logits and is subtracted before anything is rounded, so its own a
// is 0 whatever its size: fma(x, L, -fl(r L)), one instruction less a pair,
// leaves fl(r L)'s rounding there, which passes 128 from |r| of about 4e9 on
// (1024 x 150001 bf16, 8 alternatives: 68.5 us, that way 67.5).  No log
// probability comes out above 0: where r is the largest logit, S is at least
// 1; where it is not, S holds r's own 1 beside the largest's at most 2^8.
//
// The reference need not be the maximum: a warp takes the largest of its
// first logits and moves it only when one exceeds it by 2^8, so the sums
// hardly ever rescale and stay far inside fp32's range.  S and T are then of
// the size of the row's largest terms, and log2 S and T / S at most 8 apart
// from their values at the maximum: their difference loses 2^-21 at worst.
//
// Logits below kLow (the lowest values of the type) and above kHigh, where a
// would overflow, count in slow sums of their own with the exact maximum as
// reference.  Beside any logit in between those below vanish, and beside any
// above all others do.
//
// Alternatives: 64-bit keys (value in an order-preserving coding, then the
// complement of the index) make equal values go to the lower index, and no two
// keys are equal.  In the pass over the row a thread only keeps its largest
// value of each of kParts parts.  k threads have a value at least as large as
// the k-th largest of the threads' maxima (or a cheaper lower bound of it), so
// the k largest lie in the parts of threads whose maximum reaches it: about k.
// The loads of those are read again, mostly from L2, and the keys that beat the
// bar wait in the warp's queue in shared memory; 32 at a time are sorted across
// the lanes and merged into the warp's list of 32, one a lane in order, whose
// k-th is the new bar.  At last the block counts for each key left the keys
// above it.
//
// Bound: one read of the logits; 16 exponentials a clock and SM come next (at
// 16-bit logits 0.7 of the read's time).  A row is split over the CTAs of a
// cluster when there are few rows; their sums and lists meet in the first
// CTA's shared memory.
#include <cooperative_groups.h>

#include <cfloat>
#include <type_traits>

#include "zq_common.cuh"
#include "zq_elem.cuh"
#include "zq_kernels.h"

namespace zq {

namespace {

namespace cg = cooperative_groups;

// 16-byte packs that a thread loads ahead, as a power of 2: 4; with fp32 rows in
// blocks of 4 warps 8 (2048 x 32003, one alternative: 48 us against 53 us when it
// was chosen; at 16 bits it gains nothing, 1024 x 150001 with 8 alternatives: 76
// us against 73 us).
template <class T, int kWarps>
constexpr int kLogUnroll = sizeof(T) == 4 && kWarps == 4 ? 3 : 2;
constexpr int kMaxSplit = 8;  // CTAs of a row
constexpr int kStage = 128;   // packs that a warp looks at again at a time
constexpr int kAhead = 1;     // rounds from a load to its prefetch
// Parts of a thread's loads that keep a maximum each.  A block of 4 warps has
// long parts, which a second look reads whole (1024 x 150001 bf16: 8 alternatives
// 71 us with 8 parts, 75 us with 4; 20 alternatives 76 and 84); with 8 warps the
// registers are short (48 x 131072, 20 alternatives: 17.7 us with 8, 15.4 with 4).
template <int kWarps>
constexpr int kParts = kWarps == 4 ? 8 : 4;
constexpr float kLog2E = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kHeadroom = 8.0f;
// 2^kFloor is 0 in fp32; exponents are cut off there where they are multiplied
// by their power: 0 * -inf would be NaN.
constexpr float kFloor = -300.0f;
constexpr uint32_t kAll = 0xffffffffu;

// Logits from kLow on count in the fast sums, where all below kClamp are taken
// as kClamp: more than 150 below any reference, so their powers are 0.
template <class T>
constexpr float kLow = -1.0e37f;
template <>
constexpr float kLow<__half> = -65000.0f;
template <class T>
constexpr float kHigh = 1.0e38f;
template <>
constexpr float kHigh<__half> = INFINITY;
template <class T>
constexpr float kClamp = -1.0e38f;
template <>
constexpr float kClamp<__half> = -65504.0f;

// 2^v; results below 2^-126 are 0.
__device__ __forceinline__ float ex2(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

// Two fp32 values in one register pair, and arithmetic on both at once.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// Fetches packs [from, from + n) of p, as far as `end`, into L2.
__device__ __forceinline__ void prefetch(const uint4* p, int from, int n, int end) {
    if (from >= end) return;
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p + from), "r"(min(n, end - from) * 16) : "memory");
}

// max(v, lo) that keeps NaN.
__device__ __forceinline__ float max_nan(float v, float lo) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "f"(lo));
    return r;
}

// 16 bytes of logits: values 2i and 2i + 1 as a pair.
template <class T>
__device__ __forceinline__ uint64_t two_of(const uint4& raw, int i);
template <>
__device__ __forceinline__ uint64_t two_of<float>(const uint4& raw, int i) {
    return i == 0 ? pair(__uint_as_float(raw.x), __uint_as_float(raw.y))
                  : pair(__uint_as_float(raw.z), __uint_as_float(raw.w));
}
__device__ __forceinline__ uint32_t word_of(const uint4& raw, int i) {
    return i == 0 ? raw.x : i == 1 ? raw.y : i == 2 ? raw.z : raw.w;
}
template <>
__device__ __forceinline__ uint64_t two_of<__nv_bfloat16>(const uint4& raw, int i) {
    const uint32_t w = word_of(raw, i);
    return pair(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
template <>
__device__ __forceinline__ uint64_t two_of<__half>(const uint4& raw, int i) {
    const uint32_t w = word_of(raw, i);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    return pair(f.x, f.y);
}

// The largest of n packs' values (NaN passed over).
template <class T, int n>
__device__ __forceinline__ float most_of(const uint4 (&v)[n]) {
    if constexpr (sizeof(T) == 4) {
        float m = -INFINITY;
#pragma unroll
        for (int i = 0; i < n; ++i)
            m = fmaxf(m, fmaxf(fmaxf(__uint_as_float(v[i].x), __uint_as_float(v[i].y)),
                               fmaxf(__uint_as_float(v[i].z), __uint_as_float(v[i].w))));
        return m;
    } else {
        using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
        T2 m;
#pragma unroll
        for (int i = 0; i < n; ++i) {
            T2 h[4];
            memcpy(h, &v[i], 16);
            const T2 k = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
            m = i == 0 ? k : __hmax2(m, k);
        }
        // -inf where all are NaN
        return fmaxf(fmaxf(to_float(m.x), to_float(m.y)), -INFINITY);
    }
}

// ---- sums ------------------------------------------------------------------

// Sums against reference logit r: fast ones in base 2, slow ones in base e (r =
// the maximum).  None: s = t = 0 at the lowest reference.
struct Sums {
    float r, s, t;
};
__device__ __forceinline__ Sums no_sums() { return Sums{-FLT_MAX, 0.0f, 0.0f}; }

template <bool kBase2>
__device__ __forceinline__ Sums join(const Sums& a, const Sums& b) {
    Sums o;
    o.r = fmaxf(a.r, b.r);
    const float unit = kBase2 ? kLog2E : 1.0f;
    const float da = fmaxf((a.r - o.r) * unit, kFloor), db = fmaxf((b.r - o.r) * unit, kFloor);
    const float fa = ex2(kBase2 ? da : da * kLog2E), fb = ex2(kBase2 ? db : db * kLog2E);
    o.s = a.s * fa + b.s * fb;
    o.t = fa * (a.t + da * a.s) + fb * (b.t + db * b.s);
    return o;
}

template <bool kBase2>
__device__ __forceinline__ Sums warp_join(Sums v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        Sums u;
        u.r = __shfl_xor_sync(kAll, v.r, o);
        u.s = __shfl_xor_sync(kAll, v.s, o);
        u.t = __shfl_xor_sync(kAll, v.t, o);
        v = join<kBase2>(v, u);
    }
    return v;
}

__device__ __forceinline__ void take_slow(Sums& a, float x) {
    if (x > a.r) {
        const float d = fmaxf(a.r - x, kFloor);
        const float f = ex2(d * kLog2E);
        a.t = f * (a.t + d * a.s);
        a.s *= f;
        a.r = x;
    }
    const float d = x - a.r;
    const float e = ex2(d * kLog2E);
    a.s += e;
    a.t = fmaf(e, fmaxf(d, kFloor), a.t);
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kAll, v, o));
    return v;
}

// ---- the largest -------------------------------------------------------------

// Order-preserving: a < b as floats gives order(a) < order(b); -0 and +0 are
// equal; NaN is above everything.  Never 0, which marks an empty place.
__device__ __forceinline__ uint32_t order(float v) {
    if (isnan(v)) return 0xFFFFFFFFu;
    const uint32_t b = __float_as_uint(v + 0.0f);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float order_value(uint32_t o) {
    return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}
__device__ __forceinline__ uint64_t make_key(float v, uint32_t index) {
    return (uint64_t)order(v) << 32 | (uint32_t)~index;
}

// Sorts one value a lane, the smallest in lane 0.
template <class K>
__device__ __forceinline__ K sort_lanes(K v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int size = 2; size <= 32; size *= 2)
#pragma unroll
        for (int step = size / 2; step > 0; step /= 2) {
            const K u = __shfl_xor_sync(kAll, v, step);
            const bool low = ((lane & step) == 0) == ((lane & size) == 0 || size == 32);
            v = low == (u < v) ? u : v;
        }
    return v;
}

struct TopList {
    uint64_t key = 0;  // lane i: the i-th largest
    uint64_t bar = 0;  // a key has to exceed it to enter
    int waiting = 0;   // keys in the warp's queue
};

// Merges one key a lane (0: none) into the list.  With the list falling and
// the keys rising over the lanes, the larger of each lane's two are the 32
// largest of both; they rise and fall once and are put in order.
__device__ __forceinline__ void merge(TopList& l, uint64_t key, int k) {
    const int lane = threadIdx.x & 31;
    key = sort_lanes(key);
    uint64_t v = key > l.key ? key : l.key;
#pragma unroll
    for (int step = 16; step > 0; step /= 2) {
        const uint64_t u = __shfl_xor_sync(kAll, v, step);
        v = ((lane & step) == 0) == (u > v) ? u : v;
    }
    l.key = v;
    l.bar = max(l.bar, __shfl_sync(kAll, v, k - 1));
}

// Queues the lanes' keys that beat the bar.
__device__ __forceinline__ void offer(TopList& l, uint64_t* queue, uint64_t key, int k) {
    const int lane = threadIdx.x & 31;
    const bool in = key > l.bar;
    const uint32_t votes = __ballot_sync(kAll, in);
    if (in) queue[l.waiting + __popc(votes & ((1u << lane) - 1))] = key;
    l.waiting += __popc(votes);
    if (l.waiting >= 32) {
        __syncwarp();
        const uint64_t first = queue[lane], rest = queue[32 + lane];
        __syncwarp();
        l.waiting -= 32;
        if (lane < l.waiting) queue[lane] = rest;
        merge(l, first, k);
    }
}

// The k largest of n distinct keys in order to out[0, k), by counting for each
// key those above it.  Every thread of the block calls it; the keys are 16-byte
// aligned, those up to the next multiple of 8 are 0.
__device__ __forceinline__ void select_top(const uint64_t* keys, int n, int k, uint64_t* out) {
    for (int j = threadIdx.x; j < n; j += blockDim.x) {
        const uint64_t mine = keys[j];
        int above = 0;
        for (int i = 0; i < n; i += 8) {
            ulonglong2 o[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) o[u] = reinterpret_cast<const ulonglong2*>(keys + i)[u];
#pragma unroll
            for (int u = 0; u < 4; ++u) above += (o[u].x > mine) + (o[u].y > mine);
        }
        if (mine != 0 && above < k) out[above] = mine;
    }
}

// ---- the kernel --------------------------------------------------------------


template <int kWarps>
struct Shared {
    Sums fast[kWarps], slow[kWarps];
    Sums cta_fast[kMaxSplit], cta_slow[kMaxSplit];  // first CTA: every CTA's
    Sums row_fast, row_slow;
    uint64_t queue[kWarps][64];
    uint4 stage[kWarps][kStage];        // packs looked at again, and where they are from
    int stage_at[kWarps][kStage];
    uint8_t part[kWarps][kParts<kWarps> * 32];  // parts to look at again: part * 32 + lane
    alignas(16) uint64_t keys[kWarps * kTopMax + 8];
    uint64_t best[kTopMax];             // this CTA's largest
    alignas(16) uint64_t gathered[kMaxSplit * kTopMax + 8];  // first CTA: every CTA's
    uint64_t top[kTopMax];
    uint32_t kth, jth;
    int kept;
};

template <class T>
struct Warp {
    Sums slow = no_sums();
    uint64_t s = 0, t = 0;  // fast sums, two of each
    float ref = -FLT_MAX;   // r
    bool quick = false;     // whether logits go to the fast sums
    bool masked = false;    // whether a logit was below kClamp

    // The warp's maximum `most` of logits to come is too far above the
    // reference: it becomes the reference, if it may.
    __device__ __forceinline__ void look(float most) {
        quick = most >= kLow<T> && most <= kHigh<T>;
        if (!quick) return;
        const float d = fmaxf((ref - most) * kLog2E, kFloor);
        const float f = ex2(d);
        const uint64_t f2 = pair(f, f), d2 = pair(d, d);
        t = fma2(f2, fma2(d2, s, t), 0);
        s = fma2(f2, s, 0);
        ref = most;
    }
    // Whether a lane's maximum asks for a look.  Past one above kHigh, or
    // before one from kLow on, the reference stays and every such maximum does.
    __device__ __forceinline__ bool far(float most) const { return most - ref > kHeadroom * kLn2; }
    __device__ __forceinline__ void add(uint64_t x) {
        const uint64_t a = mul2(add2(x, pair(-ref, -ref)), pair(kLog2E, kLog2E));
        const float2 p = unpair(a);
        const uint64_t e = pair(ex2(p.x), ex2(p.y));
        s = add2(s, e);
        t = fma2(e, a, t);
    }
    // A lane's loads (padded with -inf if not whole).  A logit of -inf makes T NaN (0 * -inf): the warp then
    // takes these and all later loads with their values cut off at kClamp.
    template <int n>
    __device__ __forceinline__ void take(const uint4 (&v)[n], bool whole) {
        constexpr int kPairs = kElemsPer16<T> / 2;
        if (whole && quick && !masked) {
            const uint64_t s0 = s, t0 = t;
#pragma unroll
            for (int u = 0; u < n; ++u)
#pragma unroll
                for (int j = 0; j < kPairs; ++j) add(two_of<T>(v[u], j));
            const float2 f = unpair(t);
            if (!__any_sync(kAll, isnan(f.x + f.y))) return;
            masked = true;
            s = s0;
            t = t0;
        }
        if (quick) {
#pragma unroll
            for (int u = 0; u < n; ++u)
#pragma unroll
                for (int j = 0; j < kPairs; ++j) {
                    const float2 f = unpair(two_of<T>(v[u], j));
                    add(pair(max_nan(f.x, kClamp<T>), max_nan(f.y, kClamp<T>)));
                }
            return;
        }
#pragma unroll
        for (int u = 0; u < n; ++u)
#pragma unroll
            for (int j = 0; j < kPairs; ++j) {
                const float2 f = unpair(two_of<T>(v[u], j));
                take_slow(slow, f.x);
                take_slow(slow, f.y);
            }
    }
    __device__ __forceinline__ Sums fast() const {
        const float2 s2 = unpair(s), t2 = unpair(t);
        return Sums{ref, s2.x + s2.y, t2.x + t2.y};
    }
};

// Rounds of a thread's loads ahead that make one of its kParts parts; with 8
// warps a power of 2, which saves a division's registers.
template <int kWarps>
__device__ __forceinline__ int part_rounds(int packs, int per_round) {
    const int rounds = (packs + per_round - 1) / per_round;
    const int each = max(1, (rounds + kParts<kWarps> - 1) / kParts<kWarps>);
    return kWarps == 8 ? 1 << (32 - __clz(each - 1)) : each;
}

// The sums, and the thread's largest value (NaN passed over) of each part, over
// the packs [p0, p1) of a row's body: a warp takes kUnroll packs a lane at a
// time, every lane all packs of its place in the block.
template <class T, int kWarps>
__device__ __forceinline__ void pass(Warp<T>& w, const uint4* body, int p0, int p1, int per_part, float (&largest)[kParts<kWarps>]) {
    constexpr int kN = kElemsPer16<T>;
    constexpr int kUnroll = 1 << kLogUnroll<T, kWarps>;
    constexpr int kThreads = kWarps * 32;
    constexpr int kRound = kThreads * kUnroll;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int i = 0; i < kParts<kWarps>; ++i) largest[i] = -INFINITY;
    int part = 0, left = per_part;
    for (int p = p0 + warp * 32; p < p1; p += kRound) {
        if (threadIdx.x == 0) prefetch(body + p, kAhead * kRound, kRound, p1 - p);
        const bool whole = p + kRound - kThreads + 32 <= p1;
        uint4 v[kUnroll];
        if (whole) {
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) v[u] = load_l2_once(body + p + u * kThreads + lane);
        } else {
            Pack<T, kN> none;
#pragma unroll
            for (int j = 0; j < kN; ++j) none.e[j] = from_float<T>(-INFINITY);
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                const int q = p + u * kThreads + lane;
                if (q < p1)
                    v[u] = load_l2_once(body + q);
                else
                    memcpy(&v[u], &none, 16);
            }
        }
        const float most = most_of<T>(v);
        if (__any_sync(kAll, w.far(most))) w.look(warp_max(most));
        w.take(v, whole);
#pragma unroll
        for (int i = 0; i < kParts<kWarps>; ++i)
            if (part == i) largest[i] = fmaxf(largest[i], most);
        if (--left == 0) {
            left = per_part;
            ++part;
        }
    }
}

// The keys of the same packs that may be among the block's k largest, into the
// warps' lists and queues.
template <class T, int kWarps>
__device__ __forceinline__ void find_top(TopList& top, Shared<kWarps>& sh, const Warp<T>& w,
                                         const float (&largest)[kParts<kWarps>], const uint4* body, int p0, int p1, int per_part,
                                         int head, int k) {
    constexpr int kN = kElemsPer16<T>;
    constexpr int kThreads = kWarps * 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // A lower bound of the k-th largest: a warp's k-th largest maximum, or the
    // least of all warps' j-th, warps * j >= k.
    float most = largest[0];
#pragma unroll
    for (int i = 1; i < kParts<kWarps>; ++i) most = fmaxf(most, largest[i]);
    const uint32_t sorted = sort_lanes(order(most));
    if (lane == 32 - k) atomicMax(&sh.kth, sorted);
    if (lane == 32 - (k + kWarps - 1) / kWarps) atomicMin(&sh.jth, sorted);
    __syncthreads();
    const uint32_t least = max(sh.kth, sh.jth);
    if (least > order(-INFINITY)) top.bar = ((uint64_t)least << 32) - 1;
    // The parts with a value that may beat it.  A NaN shows in the sums.
    const int first = p0 + warp * 32;
    const float2 s2 = unpair(w.s);
    const bool nan = __any_sync(kAll, isnan(s2.x + s2.y + w.slow.s));
    int parts = 0;
#pragma unroll
    for (int i = 0; i < kParts<kWarps>; ++i) {
        const uint32_t hits = __ballot_sync(kAll, nan || order(largest[i]) >= least);
        if (hits >> lane & 1) sh.part[warp][parts + __popc(hits & ((1u << lane) - 1))] = (uint8_t)(i * 32 + lane);
        parts += __popc(hits);
    }
    __syncwarp();
    // All their packs, as many at a time as the stage holds.
    const int each = per_part << kLogUnroll<T, kWarps>;
    const int n = parts * each;
    for (int i0 = 0; i0 < n; i0 += kStage) {
        int at[kStage / 32];
#pragma unroll
        for (int u = 0; u < kStage / 32; ++u) {
            const int i = i0 + u * 32 + lane;
            at[u] = p1;
            if (i < n) {
                const int entry = kWarps == 8 ? i >> (31 - __clz(each)) : i / each, what = sh.part[warp][entry];
                const long long pack = (long long)(what >> 5) * each + (i - entry * each);
                if (pack * kThreads < p1 - first - (what & 31)) at[u] = first + (what & 31) + (int)pack * kThreads;
            }
            if (at[u] < p1)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(&sh.stage[warp][u * 32 + lane])),
                             "l"(body + at[u])
                             : "memory");
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll
        for (int u = 0; u < kStage / 32; ++u) sh.stage_at[warp][u * 32 + lane] = at[u];
        __syncwarp();
#pragma unroll 1
        for (int u = 0; u < kStage && i0 + u < n; u += 32) {
            const int q = sh.stage_at[warp][u + lane];
            uint64_t most_key = 0;  // the largest key that the pack may hold
            if (q < p1) {
                const uint4 v[1] = {sh.stage[warp][u + lane]};
                most_key = nan ? ~0ull : make_key(most_of<T>(v), (uint32_t)(head + q * kN));
            }
            // one pack at a time, a value a lane
            for (uint32_t packs = __ballot_sync(kAll, most_key > top.bar); packs; packs &= packs - 1) {
                const int src = __ffs(packs) - 1;
                const int from = __shfl_sync(kAll, q, src);
                uint64_t key = 0;
                if (lane < kN)
                    key = make_key(to_float(reinterpret_cast<const T*>(&sh.stage[warp][u + src])[lane]),
                                   (uint32_t)(head + from * kN + lane));
                offer(top, sh.queue[warp], key, k);
            }
        }
        __syncwarp();
    }
}

// Blocks an SM: 8 of 4 warps; 4 of 8 warps, since 5 leave too few registers (48 x
// 131072 bf16, 20 alternatives: 15.1 us against 17.4 us with 5, spilling; 300 x
// 100000, where the fifth would hold the last blocks, 27.6 us against 24.7 us).
template <class T, bool kTop, int kWarps>
__global__ void __launch_bounds__(kWarps * 32, kWarps == 8 ? 4 : 8) token_logprobs_kernel(const LogprobArgs a, int split) {
    cg::cluster_group cluster = cg::this_cluster();
    if (split > 1) cluster.barrier_arrive();
    pdl_launch_dependents();
    pdl_wait_primary();
    constexpr int kN = kElemsPer16<T>;
    constexpr int kThreads = kWarps * 32;
    __shared__ Shared<kWarps> sh;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long row = blockIdx.x / split;
    const int part = blockIdx.x % split;
    const T* x = static_cast<const T*>(a.logits) + row * a.ld;
    if (kTop) {
        if (threadIdx.x == 0) {
            sh.kept = 0;
            sh.kth = 0;
            sh.jth = 0xFFFFFFFFu;
        }
        for (int i = threadIdx.x; i < kWarps * kTopMax + 8; i += kThreads) sh.keys[i] = 0;
        if (threadIdx.x < 8) sh.gathered[split * a.top_k + threadIdx.x] = 0;
        __syncthreads();
    }
    Warp<T> w;
    TopList top;

    // The row in 16-byte packs from the first aligned element on; the elements
    // before and behind them go one by one to the first CTA's first warp.
    const int head = min((int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / (int)sizeof(T), a.vocab);
    const int packs = (a.vocab - head) / kN;
    const uint4* body = reinterpret_cast<const uint4*>(x + head);
    const int p0 = (int)((long long)packs * part / split), p1 = (int)((long long)packs * (part + 1) / split);
    const int per_part = part_rounds<kWarps>(p1 - p0, kThreads << kLogUnroll<T, kWarps>);
    float largest[kParts<kWarps>];
    pass<T, kWarps>(w, body, p0, p1, per_part, largest);
    if (kTop) find_top<T, kWarps>(top, sh, w, largest, body, p0, p1, per_part, head, a.top_k);
    if (part == 0 && warp == 0) {
        const int tail = head + packs * kN;
        const int loose = head + (a.vocab - tail);  // at most 2 (kN - 1) < 32
        const int i = lane < head ? lane : tail + lane - head;
        const float f = lane < loose ? to_float(load_l2_once(x + i)) : -INFINITY;
        const float m = warp_max(f);
        if (w.far(m)) w.look(m);
        if (w.quick)
            w.add(pair(max_nan(f, kClamp<T>), kClamp<T>));
        else
            take_slow(w.slow, f);
        if (kTop) offer(top, sh.queue[0], lane < loose ? make_key(f, (uint32_t)i) : 0, a.top_k);
    }

    // ---- the block's sums and largest ----
    Sums fast = warp_join<true>(w.fast()), slow = no_sums();
    if (__any_sync(kAll, w.slow.s != 0.0f)) slow = warp_join<false>(w.slow);
    if (lane == 0) {
        sh.fast[warp] = fast;
        sh.slow[warp] = slow;
    }
    if (kTop) {
        // a warp's keys: its queue's, or with a list the list's k largest
        __syncwarp();
        uint64_t key = lane < top.waiting ? sh.queue[warp][lane] : 0;
        if (__any_sync(kAll, top.key != 0)) {
            if (top.waiting) merge(top, key, a.top_k);
            key = lane < a.top_k ? top.key : 0;
        }
        const uint32_t votes = __ballot_sync(kAll, key != 0);
        int at = 0;
        if (lane == 0 && votes) at = atomicAdd(&sh.kept, __popc(votes));
        at = __shfl_sync(kAll, at, 0);
        if (key != 0) sh.keys[at + __popc(votes & ((1u << lane) - 1))] = key;
        if (threadIdx.x < kTopMax) sh.best[threadIdx.x] = 0;
    }
    __syncthreads();
    if (warp == 0) {
        fast = warp_join<true>(lane < kWarps ? sh.fast[lane] : no_sums());
        slow = warp_join<false>(lane < kWarps ? sh.slow[lane] : no_sums());
    }
    if (kTop) {
        select_top(sh.keys, sh.kept, a.top_k, sh.best);
        __syncthreads();
    }

    // ---- the row's ----
    if (split > 1) {
        cluster.barrier_wait();  // the first CTA runs: its shared memory may be written
        Shared<kWarps>* to = cluster.map_shared_rank(&sh, 0);
        if (threadIdx.x == 0) {
            to->cta_fast[part] = fast;
            to->cta_slow[part] = slow;
        }
        if (kTop && (int)threadIdx.x < a.top_k) to->gathered[part * a.top_k + threadIdx.x] = sh.best[threadIdx.x];
        cluster.sync();
        if (part != 0) return;
        if (warp == 0) {
            fast = warp_join<true>(lane < split ? sh.cta_fast[lane] : no_sums());
            slow = warp_join<false>(lane < split ? sh.cta_slow[lane] : no_sums());
        }
        if (kTop) select_top(sh.gathered, split * a.top_k, a.top_k, sh.top);
    }
    if (threadIdx.x == 0) {
        sh.row_fast = fast;
        sh.row_slow = slow;
    }
    __syncthreads();
    // Fast sums where any logit is in their range, with the slow ones brought
    // to them; else the slow sums alone.  A row with no token allowed has neither:
    // every log probability is -inf and the entropy 0.
    Sums r = sh.row_slow;
    float unit = 1.0f, log_s = 0.0f, mean = 0.0f;
    if (r.r > kHigh<T>) {
        r.s += 0.0f * sh.row_fast.s;  // NaN where that is
    } else if (!(sh.row_fast.s == 0.0f)) {
        const Sums s2 = {r.r, r.s, r.t * kLog2E};
        r = r.s == 0.0f ? sh.row_fast : join<true>(sh.row_fast, s2);
        unit = kLn2;
    }
    if (!(r.s == 0.0f)) {
        log_s = logf(r.s);
        mean = unit * (r.t / r.s);
    }
    if (threadIdx.x == 0 && a.entropy) {
        const float h = log_s - mean;
        a.entropy[row] = h < 0.0f ? 0.0f : h;  // the two terms' roundings
    }
    auto log_p = [&](float v) { return v - r.r - log_s; };
    for (long long i = threadIdx.x; i < a.n_targets; i += kThreads) {
        const long long t = load_l2_once(reinterpret_cast<const long long*>(a.targets) + row * a.n_targets + i);
        float lp = 0.0f;  // no token asked for
        if (t >= a.vocab)
            lp = __uint_as_float(0x7FC00000u);
        else if (t >= 0)
            lp = log_p(to_float(load_l2_once(x + t)));
        a.logprobs[row * a.n_targets + i] = lp;
    }
    if (kTop && (int)threadIdx.x < a.top_k) {
        const uint64_t key = (split > 1 ? sh.top : sh.best)[threadIdx.x];
        a.top_logprobs[row * a.top_k + threadIdx.x] = log_p(order_value((uint32_t)(key >> 32)));
        a.top_ids[row * a.top_k + threadIdx.x] = (long long)(uint32_t)~(uint32_t)key;
    }
}

template <class T, bool kTop, int kWarps>
cudaError_t launch(const LogprobArgs& a, int split, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.m * split));
    cfg.blockDim = dim3(kWarps * 32);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)split;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, kTop, kWarps>, a, split);
}

template <class T, bool kTop>
cudaError_t launch_rows(const LogprobArgs& a, cudaStream_t stream) {
    // Many rows: a block of 4 warps each, 6 rows an SM or more keep enough
    // loads in flight and more rows are past their ends at any time (1024 x
    // 150001 bf16, 8 alternatives, both with 4 parts: 78 us against 86 us with
    // 8 warps; 600 x 100000: 46 us against 36 us).  The same where one round of 4 warps holds
    // a row (600 x 2000 bf16: 9.4 us against 11.9 us).
    const int sms = sm_count();
    const long long packs = a.vocab / kElemsPer16<T>;
    if (a.m >= 6LL * sms || packs <= 128 << kLogUnroll<T, 4>) return launch<T, kTop, 4>(a, 1, stream);
    // Else CTAs of 8 warps, 4 an SM, none with less than a round: with 8 an SM
    // the steps behind the pass cost more than the shorter passes save
    // (300 x 100000 bf16, 8 alternatives: 24 us against 31 us when it was
    // chosen).
    int split = 1;
    while (split < kMaxSplit && a.m * split < 4LL * sms && packs >= 2LL * split * 256 << kLogUnroll<T, 8>) split *= 2;
    return launch<T, kTop, 8>(a, split, stream);
}

template <class T>
cudaError_t launch_type(const LogprobArgs& a, cudaStream_t stream) {
    return a.top_k ? launch_rows<T, true>(a, stream) : launch_rows<T, false>(a, stream);
}

}  // namespace

cudaError_t launch_token_logprobs(const LogprobArgs& a, int dtype, cudaStream_t stream) {
    if (dtype == ZQ_DTYPE_F32) return launch_type<float>(a, stream);
    if (dtype == ZQ_DTYPE_F16) return launch_type<__half>(a, stream);
    return launch_type<__nv_bfloat16>(a, stream);
}

}  // namespace zq

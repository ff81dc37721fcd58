// zq_logprobs.cu -- log probabilities of given tokens, with the entropy and
// the most likely alternatives, over rows of logits (zq_token_logprobs).
//
// One pass over a row.  Every thread keeps a running maximum m and, against
// it, S = sum exp(x - m) and T = sum exp(x - m) (x - m) in fp32; two such
// triples join as
//   M = max(m1, m2),  f_i = exp(m_i - M),
//   S = f1 S1 + f2 S2,  T = f1 (T1 + (m1 - M) S1) + f2 (T2 + (m2 - M) S2).
// Then  log p(t) = (x_t - M) - log S  and  H = log S - T / S.  T <= 0, so the
// entropy's two terms never cancel.
//
// Alternatives: every warp keeps its kTopMax largest values, one a lane in
// order, as 64-bit keys (value in an order-preserving coding, then the
// complement of the index), so equal values go to the lower index and no two
// keys are equal.  A value enters only if its key beats the k-th of the
// warp's list and the best k-th of the block's warps.
//
// Bound: one read of the logits.  A row is split over the CTAs of a cluster
// when there are few rows; their triples and lists meet in the first CTA's
// shared memory.
#include <cooperative_groups.h>

#include <cfloat>

#include "zq_common.cuh"
#include "zq_elem.cuh"
#include "zq_kernels.h"

namespace zq {

namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr float kLog2E = 1.4426950408889634f;
// exp(kFloor) is 0 in fp32.  Differences are clamped to it where they are
// multiplied by their exponential: 0 * -inf would be NaN.
constexpr float kFloor = -200.0f;

struct Stats {
    float m, s, t;
};
__device__ __forceinline__ Stats no_stats() { return Stats{-FLT_MAX, 0.0f, 0.0f}; }

// 2^v; results below 2^-126 are 0.
__device__ __forceinline__ float ex2(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

__device__ __forceinline__ Stats join(const Stats& a, const Stats& b) {
    Stats r;
    r.m = fmaxf(a.m, b.m);
    const float da = fmaxf(a.m - r.m, kFloor), db = fmaxf(b.m - r.m, kFloor);
    const float fa = ex2(da * kLog2E), fb = ex2(db * kLog2E);
    r.s = a.s * fa + b.s * fb;
    r.t = fa * (a.t + da * a.s) + fb * (b.t + db * b.s);
    return r;
}

__device__ __forceinline__ Stats warp_join(Stats v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        Stats u;
        u.m = __shfl_xor_sync(0xffffffffu, v.m, o);
        u.s = __shfl_xor_sync(0xffffffffu, v.s, o);
        u.t = __shfl_xor_sync(0xffffffffu, v.t, o);
        v = join(v, u);
    }
    return v;
}

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

// A warp's list: lane i holds the i-th largest key, `bar` what a key has to
// exceed to enter.
struct TopList {
    uint64_t key = 0;
    uint64_t bar = 0;
    float bar_value = -INFINITY;  // the value of `bar`
};

__device__ __forceinline__ void raise_bar(TopList& l, uint64_t bar) {
    if (bar > l.bar) {
        l.bar = bar;
        l.bar_value = order_value((uint32_t)(bar >> 32));
    }
}

// Takes the lanes' keys that beat the bar, one after the other.
__device__ __forceinline__ void offer(TopList& l, uint64_t key, int k) {
    const int lane = threadIdx.x & 31;
    uint32_t votes = __ballot_sync(0xffffffffu, key > l.bar);
    while (votes) {
        const int src = __ffs(votes) - 1;
        const uint64_t c = __shfl_sync(0xffffffffu, key, src);
        const int at = __popc(__ballot_sync(0xffffffffu, l.key > c));
        const uint64_t up = __shfl_up_sync(0xffffffffu, l.key, 1);
        if (lane == at) l.key = c;
        if (lane > at) l.key = up;
        raise_bar(l, __shfl_sync(0xffffffffu, l.key, k - 1));
        if (lane == src) key = 0;
        votes = __ballot_sync(0xffffffffu, key > l.bar);
    }
}

// The k largest of n distinct keys (0: empty place) in `keys`, in order, to
// out[0, k).  Every thread of the block calls it; n <= kThreads.
__device__ __forceinline__ void select_top(const uint64_t* keys, int n, int k, uint64_t* out) {
    if ((int)threadIdx.x < n) {
        const uint64_t mine = keys[threadIdx.x];
        int above = 0;
        for (int i = 0; i < n; ++i) above += keys[i] > mine;
        if (mine != 0 && above < k) out[above] = mine;
    }
}

// Adds kBatch logits, `most` their maximum.
template <int kBatch>
__device__ __forceinline__ void take(Stats& st, const float (&v)[kBatch], float most) {
    if (most > st.m) {
        const float d = fmaxf(st.m - most, kFloor);
        const float f = ex2(d * kLog2E);
        st.t = f * (st.t + d * st.s);
        st.s *= f;
        st.m = most;
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
        const float d = v[i] - st.m;
        const float e = ex2(d * kLog2E);
        st.s += e;
        st.t = fmaf(e, fmaxf(d, kFloor), st.t);
    }
}

struct Shared {
    Stats part[kWarps];
    uint64_t keys[kWarps * kTopMax];
    uint64_t best[kTopMax];           // this CTA's k largest
    uint64_t gathered[8 * kTopMax];   // CTA 0: every CTA's
    uint64_t final_keys[kTopMax];
    Stats cta[8];                     // CTA 0: every CTA's
    unsigned long long bar;           // the largest k-th key of the warps
    Stats row;
};

template <class T, bool kTop>
__global__ void __launch_bounds__(kThreads) token_logprobs_kernel(const LogprobArgs a, int split) {
    cg::cluster_group cluster = cg::this_cluster();
    if (split > 1) cluster.barrier_arrive();
    pdl_launch_dependents();
    pdl_wait_primary();
    constexpr int kN = kElemsPer16<T>;
    constexpr int kUnroll = 4;
    __shared__ Shared sh;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long row = blockIdx.x / split;
    const int part = blockIdx.x % split;
    const T* x = static_cast<const T*>(a.logits) + row * a.ld;
    if (kTop) {
        if (threadIdx.x == 0) sh.bar = 0;
        if (threadIdx.x < kTopMax) sh.best[threadIdx.x] = 0;
        __syncthreads();
    }
    Stats st = no_stats();
    TopList top;

    // The row in 16-byte packs from the first aligned element on; the elements
    // before and behind them go one by one to the first CTA's threads.
    const int head = min((int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / (int)sizeof(T), a.vocab);
    const int packs = (a.vocab - head) / kN;
    const Pack<T, kN>* body = reinterpret_cast<const Pack<T, kN>*>(x + head);
    const int p0 = (int)((long long)packs * part / split), p1 = (int)((long long)packs * (part + 1) / split);

    for (int p = p0 + warp * 32; p < p1; p += kThreads * kUnroll) {
        Pack<T, kN> v[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int q = p + u * kThreads + lane;
            if (q < p1) {
                const uint4 w = ld_stream_u4(body + q);
                memcpy(&v[u], &w, 16);
            } else {
#pragma unroll
                for (int j = 0; j < kN; ++j) v[u].e[j] = from_float<T>(-INFINITY);
            }
        }
        if (kTop) raise_bar(top, *(volatile unsigned long long*)&sh.bar);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            float f[kN];
            float most = -INFINITY;
#pragma unroll
            for (int j = 0; j < kN; ++j) {
                f[j] = to_float(v[u].e[j]);
                most = fmaxf(most, f[j]);
            }
            take(st, f, most);
            if (kTop) {
                const int q = p + u * kThreads + lane;
                // S is NaN from the first NaN on, which the maximum passes over
                if (__any_sync(0xffffffffu, q < p1 && (most >= top.bar_value || isnan(st.s)))) {
                    const uint64_t before = top.bar;
#pragma unroll
                    for (int j = 0; j < kN; ++j)
                        offer(top, q < p1 ? make_key(f[j], (uint32_t)(head + q * kN + j)) : 0, a.top_k);
                    if (top.bar > before && lane == 0) atomicMax(&sh.bar, (unsigned long long)top.bar);
                }
            }
        }
    }
    if (part == 0) {
        const int tail = head + packs * kN;
        const int loose = head + (a.vocab - tail);
        // up to 2 * (kN - 1) < 32 elements
        if (warp == 0) {
            const int i = lane < head ? lane : tail + lane - head;
            float f[1] = {lane < loose ? to_float(x[i]) : -INFINITY};
            take(st, f, f[0]);
            if (kTop) offer(top, lane < loose ? make_key(f[0], (uint32_t)i) : 0, a.top_k);
        }
    }

    st = warp_join(st);
    if (lane == 0) sh.part[warp] = st;
    if (kTop && lane < a.top_k) sh.keys[warp * a.top_k + lane] = top.key;
    __syncthreads();
    if (warp == 0) {
        st = lane < kWarps ? sh.part[lane] : no_stats();
        st = warp_join(st);
    }
    if (kTop) {
        select_top(sh.keys, kWarps * a.top_k, a.top_k, sh.best);
        __syncthreads();
    }
    if (split > 1) {
        cluster.barrier_wait();  // the first CTA runs: its shared memory may be written
        Shared* first = cluster.map_shared_rank(&sh, 0);
        if (threadIdx.x == 0) first->cta[part] = st;
        if (kTop && (int)threadIdx.x < a.top_k) first->gathered[part * a.top_k + threadIdx.x] = sh.best[threadIdx.x];
        cluster.sync();
        if (part != 0) return;
        if (warp == 0) {
            st = lane < split ? sh.cta[lane] : no_stats();
            st = warp_join(st);
        }
        if (kTop) select_top(sh.gathered, split * a.top_k, a.top_k, sh.final_keys);
    }
    if (threadIdx.x == 0) sh.row = st;
    __syncthreads();
    const Stats r = sh.row;
    // A row with no token allowed has S = 0: every log probability is -inf
    // and the entropy 0.
    const bool empty = r.s == 0.0f;
    const float log_s = empty ? 0.0f : logf(r.s);
    if (threadIdx.x == 0 && a.entropy) a.entropy[row] = empty ? 0.0f : log_s - r.t / r.s;
    for (long long i = threadIdx.x; i < a.n_targets; i += kThreads) {
        const long long t = a.targets[row * a.n_targets + i];
        float lp = 0.0f;  // no token asked for
        if (t >= a.vocab)
            lp = __uint_as_float(0x7FC00000u);
        else if (t >= 0)
            lp = (to_float(x[t]) - r.m) - log_s;
        a.logprobs[row * a.n_targets + i] = lp;
    }
    if (kTop && (int)threadIdx.x < a.top_k) {
        const uint64_t key = (split > 1 ? sh.final_keys : sh.best)[threadIdx.x];
        a.top_logprobs[row * a.top_k + threadIdx.x] = (order_value((uint32_t)(key >> 32)) - r.m) - log_s;
        a.top_ids[row * a.top_k + threadIdx.x] = (long long)(uint32_t)~(uint32_t)key;
    }
}

template <class T, bool kTop>
cudaError_t launch(const LogprobArgs& a, cudaStream_t stream) {
    // Enough CTAs to fill the SMs several times over, none with less than
    // one full round of its threads' loads.
    int split = 1;
    const long long per_cta = (long long)kThreads * 4 * kElemsPer16<T>;
    while (split < 8 && a.m * split < 8LL * sm_count() && a.vocab >= 2 * split * per_cta) split *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.m * split));
    cfg.blockDim = dim3(kThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)split;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, kTop>, a, split);
}

template <class T>
cudaError_t launch_type(const LogprobArgs& a, cudaStream_t stream) {
    return a.top_k ? launch<T, true>(a, stream) : launch<T, false>(a, stream);
}

}  // namespace

cudaError_t launch_token_logprobs(const LogprobArgs& a, int dtype, cudaStream_t stream) {
    if (dtype == ZQ_DTYPE_F32) return launch_type<float>(a, stream);
    if (dtype == ZQ_DTYPE_F16) return launch_type<__half>(a, stream);
    return launch_type<__nv_bfloat16>(a, stream);
}

}  // namespace zq

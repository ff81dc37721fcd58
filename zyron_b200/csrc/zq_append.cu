// zq_append.cu -- new tokens' queries and keys rotated by their position, keys
// and values written into a paged cache (zq_append_kv).
//
//   angle = (position + offset) * inv_freq[p],   p < rotated / 2
//   (a, b) -> (a cos - b sin, a sin + b cos)
//
// over the pairs (2p, 2p + 1) where interleaved, (p, p + rotated / 2) otherwise;
// elements behind `rotated` pass as they are.  The arithmetic is fp32, rounded
// once to the cache's type.
//
// An angle of a far position loses its fraction in fp32, so it is formed and
// reduced to [-pi/4, pi/4] in 64 bits; the sine and cosine of what is left are
// fp32 Taylor polynomials (terms behind x^9 and x^10 are below 2e-9 there).
// That is done once a token and pair and shared by all heads.
//
// Bound: one read of q, k and v and one write of the same elements in 16 bits:
// memory bandwidth for prompts, latency for single tokens.  The way to a row's place
// (its request, length and page, one load after the other, then angles in 64 bits)
// takes 2 us, during which a block's first loads are under way already.  A block a
// row or two paid that in seven waves; now the blocks that the SMs hold share the
// rows out and find up to 16 rows' places at once.  8074 bf16 rows of 32 + 8 + 8 heads
// of 128: 42 us, 4.7 TB/s (two rows a block: 53 us); 96 rows 3.6 us, one 2.6.
#include "zq_elem.cuh"
#include "zq_paged.cuh"

namespace zq {

namespace {

// Many rows: blocks of up to 128 threads, eight an SM (five of 192 43.1 us, and no
// registers are left for two rows under way), 16 rows at a time (eight 45 us).
constexpr int kAppendThreads = 128;
constexpr int kAppendBlocks = 8;
constexpr int kAppendChunk = 16;
// Few: a block a row, as many threads as it has units up to this.
constexpr int kRowThreads = 384;
constexpr int kMaxPairs = 64;  // dim <= 128

// sin and cos of a, reduced by multiples of pi/2 in 64 bits.
__device__ __forceinline__ float2 sin_cos(double a) {
    const double n = rint(a * 0.63661977236758134308);
    double r = fma(-n, 1.57079632679489661923, a);
    r = fma(-n, 6.12323399573676588613e-17, r);  // the part of pi/2 that its double leaves out
    const float x = (float)r, s = x * x;
    // Taylor: sin x = x (1 - s/3! + s^2/5! - ...), cos x = 1 - s/2! + s^2/4! - ...
    float sn = fmaf(s, 2.7557319e-6f, -1.9841270e-4f);
    sn = fmaf(s, sn, 8.3333333e-3f);
    sn = fmaf(s, sn, -1.6666667e-1f);
    sn = fmaf(x * s, sn, x);
    float cs = fmaf(s, -2.7557319e-7f, 2.4801587e-5f);
    cs = fmaf(s, cs, -1.3888889e-3f);
    cs = fmaf(s, cs, 4.1666667e-2f);
    cs = fmaf(s, cs, -0.5f);
    cs = fmaf(s, cs, 1.0f);
    const int quadrant = (int)(long long)fma(-4.0, floor(n * 0.25), n);  // n mod 4
    if (quadrant & 1) {
        const float t = sn;
        sn = cs;
        cs = -t;
    }
    if (quadrant & 2) {
        sn = -sn;
        cs = -cs;
    }
    return make_float2(sn, cs);
}

// N elements as they lie in memory.
template <class T, int N>
struct Raw {
    static constexpr int kEach = N * sizeof(T) >= 16 ? kElemsPer16<T> : 1;
    Pack<T, kEach> w[N / kEach];

    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (int i = 0; i < N / kEach; ++i) w[i] = load_l2_once(reinterpret_cast<const Pack<T, kEach>*>(p) + i);
    }
    __device__ __forceinline__ void get(float (&v)[N]) const {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = to_float(w[i / kEach].e[i % kEach]);
    }
};
template <class C, int N>
__device__ __forceinline__ void store_elems(C* p, const float (&v)[N]) {
    Pack<C, N> w;
#pragma unroll
    for (int i = 0; i < N; ++i) w.e[i] = from_float<C>(v[i]);
    *reinterpret_cast<Pack<C, N>*>(p) = w;
}

// A unit of work: kPairs pairs of one head, as two runs of kPairs elements at i0 and
// i1 (interleaved pairs lie in one run of twice as many).  kPairs is 8 where
// everything lies on 16-byte borders, 1 otherwise.
template <int kPairs>
__device__ __forceinline__ void rotate(float (&x)[kPairs], float (&y)[kPairs], const float2* turn, bool interleaved) {
    if (!interleaved) {
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
            const float2 e = turn[j];
            const float r = x[j] * e.y - y[j] * e.x;
            y[j] = x[j] * e.x + y[j] * e.y;
            x[j] = r;
        }
    } else if constexpr (kPairs == 1) {
        const float2 e = turn[0];
        const float r = x[0] * e.y - y[0] * e.x;
        y[0] = x[0] * e.x + y[0] * e.y;
        x[0] = r;
    } else {
        // pairs lie side by side: of x first, then of y
#pragma unroll
        for (int j = 0; j < kPairs / 2; ++j) {
            const float2 e = turn[j], s = turn[kPairs / 2 + j];
            const float r = x[2 * j] * e.y - x[2 * j + 1] * e.x;
            x[2 * j + 1] = x[2 * j] * e.x + x[2 * j + 1] * e.y;
            x[2 * j] = r;
            const float q = y[2 * j] * s.y - y[2 * j + 1] * s.x;
            y[2 * j + 1] = y[2 * j] * s.x + y[2 * j + 1] * s.y;
            y[2 * j] = q;
        }
    }
}

// A block takes `share` rows, at most kChunk at a time: their requests and pages are
// found side by side, a lane a row, then their angles; a thread takes the same unit
// of one row after the other, the next row's loads under way.
template <class T, class C, int kPairs, int kChunk>
__global__ void __launch_bounds__(kChunk == 1 ? kRowThreads : kAppendThreads, kChunk == 1 ? 2 : kAppendBlocks) append_kernel(const AppendArgs a, int share) {
    static_assert(kChunk <= 32, "a lane a row");
    __shared__ float2 turns[kChunk][kMaxPairs];
    __shared__ long long places[2][kChunk];  // of the key and the value in the caches, -1: not written
    __shared__ long long positions[kChunk];
    const PagedBatch& p = a.batch;
    const int dim = p.dim, half = a.rotated / 2;
    const int per_head = dim / (2 * kPairs);
    const int heads = a.q ? a.heads : 0;
    const int units = (heads + 2 * p.kv_heads) * per_head;
    const int last = (int)min((blockIdx.x + 1LL) * share, (long long)p.rows);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_launch_dependents();
    pdl_wait_primary();

    for (int t0 = blockIdx.x * share; t0 < last; t0 += kChunk) {
        const int live = min(kChunk, last - t0);
        Raw<T, kPairs> raw[2];
        int head = 0, i0 = 0, apart = 0;
        const T* src = nullptr;
        long long ld = 0;
        const auto load = [&](int t) {
            const T* from = src + t * ld;
            raw[0].load(from);
            raw[1].load(from + apart);
        };
        const auto enter = [&](int u) {
            head = u / per_head;
            const int pair = (u - head * per_head) * kPairs;
            const bool side = a.interleaved || pair >= half;
            i0 = side ? 2 * pair : pair;
            apart = side ? kPairs : half;
            const bool q = head < heads, k = head < heads + p.kv_heads;
            ld = q ? a.ldq : k ? a.ldk : a.ldv;
            src = static_cast<const T*>(q ? a.q : k ? a.k : a.v) + t0 * ld +
                  (long long)(head - (q ? 0 : k ? heads : heads + p.kv_heads)) * dim + i0;
            load(0);
        };
        int u = threadIdx.x;
        if (u < units) enter(u);

        if (warp == 0) {
            const int t = t0 + min(lane, live - 1);
            const int b = kChunk == 1 ? request_of_row(p, t) : request_of_lane(p, t0, t0 + live - 1, t);
            long long k_at = -1, v_at = -1, position = 0;
            if (b >= 0) {
                const Request r = load_request(p, b);
                position = (long long)r.length - r.rows + (t - r.first);
                if (position >= 0) {
                    const int page = page_of(p, b, (int)(position / p.page));
                    const long long in = position % p.page * dim;
                    if (page >= 0) {
                        k_at = page * p.ld_k_page + in;
                        v_at = page * p.ld_v_page + in;
                    }
                }
            }
            if (lane < live) {
                places[0][lane] = b < 0 ? -2 : k_at;
                places[1][lane] = v_at;
                positions[lane] = position;
            }
        }
        if constexpr (kChunk == 1)
            __syncwarp();
        else
            __syncthreads();
        for (int w = warp; w < live; w += blockDim.x >> 5) {
            const double at = (double)(positions[w] + a.offset);
            for (int i = lane; i < half; i += 32) turns[w][i] = sin_cos(at * load_l2(a.inv_freq + i));
        }
        __syncthreads();

        while (u < units) {
            const bool is_q = head < heads, is_v = head >= heads + p.kv_heads;
            const bool turned = !is_v && (a.interleaved ? i0 / 2 : i0) < half;
            C* base = is_q ? static_cast<C*>(a.q_out) + ((long long)t0 * heads + head) * dim + i0
                           : static_cast<C*>(is_v ? a.v_cache : a.k_cache) +
                                 (long long)(head - heads - (is_v ? p.kv_heads : 0)) * p.page * dim + i0;
            const float2* turn = turns[0] + (a.interleaved ? i0 / 2 : i0);
#pragma unroll 1
            for (int t = 0; t < live; ++t, turn += kMaxPairs) {
                float x[kPairs], y[kPairs];
                raw[0].get(x);
                raw[1].get(y);
                if (t + 1 < live) load(t + 1);
                if (turned) rotate<kPairs>(x, y, turn, a.interleaved);
                const long long at = is_q ? (places[0][t] == -2 ? -1 : (long long)t * heads * dim) : places[is_v][t];
                if (at >= 0) {
                    store_elems(base + at, x);
                    store_elems(base + at + apart, y);
                }
            }
            u += blockDim.x;
            if (u < units) enter(u);
        }
        if constexpr (kChunk > 1) __syncthreads();  // the tables have been read
    }
}

template <class T, class C>
cudaError_t launch_append_t(const AppendArgs& a, cudaStream_t stream) {
    const int dim = a.batch.dim;
    const auto on = [](const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; };
    const size_t grain = 16 / sizeof(T);
    const bool wide = dim % 16 == 0 && a.rotated % 16 == 0 && on(a.q, 16) && on(a.k, 16) && on(a.v, 16) &&
                      on(a.k_cache, 16) && on(a.v_cache, 16) && on(a.q_out, 16) &&
                      (!a.q || a.ldq % grain == 0) && a.ldk % grain == 0 && a.ldv % grain == 0 &&
                      a.batch.ld_k_page % 8 == 0 && a.batch.ld_v_page % 8 == 0;
    const int units = ((a.q ? a.heads : 0) + 2 * a.batch.kv_heads) * (dim / (wide ? 16 : 2));
    const auto threads_of = [&](int limit) {
        const int rounds = (units + limit - 1) / limit;
        return ((units + rounds - 1) / rounds + 31) / 32 * 32;
    };
    int threads = threads_of(kRowThreads);
    if (a.batch.rows <= sm_count() * 2) {
        const auto kernel = wide ? append_kernel<T, C, 8, 1> : append_kernel<T, C, 1, 1>;
        return launch_pdl_kernel(kernel, dim3(a.batch.rows), dim3(threads), 0, stream, a, 1);
    }
    threads = threads_of(kAppendThreads);
    const int most = sm_count() * (kAppendBlocks * kAppendThreads / threads);
    const int share = (a.batch.rows + most - 1) / most;
    const auto kernel = wide ? append_kernel<T, C, 8, kAppendChunk> : append_kernel<T, C, 1, kAppendChunk>;
    return launch_pdl_kernel(kernel, dim3((a.batch.rows + share - 1) / share), dim3(threads), 0, stream, a, share);
}

template <class T>
cudaError_t launch_append_c(const AppendArgs& a, int cache_dtype, cudaStream_t stream) {
    return cache_dtype == ZQ_DTYPE_F16 ? launch_append_t<T, __half>(a, stream)
                                       : launch_append_t<T, __nv_bfloat16>(a, stream);
}

}  // namespace

cudaError_t launch_append_kv(const AppendArgs& a, int dtype, int cache_dtype, cudaStream_t stream) {
    if (dtype == ZQ_DTYPE_F32) return launch_append_c<float>(a, cache_dtype, stream);
    if (dtype == ZQ_DTYPE_F16) return launch_append_c<__half>(a, cache_dtype, stream);
    return launch_append_c<__nv_bfloat16>(a, cache_dtype, stream);
}

}  // namespace zq

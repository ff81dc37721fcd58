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
// memory bandwidth for prompts, latency for single tokens.  A block takes a few
// tokens; its threads' loads are under way before the row's request, page and
// angles are known.
#include "zq_elem.cuh"
#include "zq_paged.cuh"

namespace zq {

namespace {

constexpr int kAppendThreads = 256;
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

template <class T, int N>
__device__ __forceinline__ void load_elems(const T* p, float (&v)[N]) {
    if constexpr (N * sizeof(T) >= 16) {
        constexpr int kEach = kElemsPer16<T>;
#pragma unroll
        for (int i = 0; i < N / kEach; ++i) {
            const Pack<T, kEach> w = load_l2_once(reinterpret_cast<const Pack<T, kEach>*>(p) + i);
#pragma unroll
            for (int j = 0; j < kEach; ++j) v[i * kEach + j] = to_float(w.e[j]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = to_float(load_l2_once(p + i));
    }
}
template <class C, int N>
__device__ __forceinline__ void store_elems(C* p, const float (&v)[N]) {
    Pack<C, N> w;
#pragma unroll
    for (int i = 0; i < N; ++i) w.e[i] = from_float<C>(v[i]);
    *reinterpret_cast<Pack<C, N>*>(p) = w;
}

// A unit of work: kPairs pairs of one head of one token, as two runs of kPairs
// elements at i0 and i1 (interleaved pairs lie in one run of twice as many).
// kPairs is 8 where everything lies on 16-byte borders, 1 otherwise.
template <class T, class C, int kPairs>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const AppendArgs a, int tokens) {
    __shared__ float2 turn[8][kMaxPairs];
    __shared__ long long place[2][8];  // of the key and the value in the caches, -1: not written
    const PagedBatch& p = a.batch;
    const int dim = p.dim, half = a.rotated / 2;
    const int per_head = dim / (2 * kPairs);
    const int heads = a.q ? a.heads : 0;
    const int per_token = (heads + 2 * p.kv_heads) * per_head;
    const int t0 = blockIdx.x * tokens;
    const int live = min(tokens, p.rows - t0);
    pdl_launch_dependents();
    pdl_wait_primary();

    const auto fetch = [&](int u, float (&x)[kPairs], float (&y)[kPairs], int& token, int& head, int& i0, int& i1) {
        token = u / per_token;
        const int in = u - token * per_token;
        head = in / per_head;
        const int pair = (in - head * per_head) * kPairs;
        if (a.interleaved || pair >= half) {
            i0 = 2 * pair;
            i1 = 2 * pair + kPairs;
        } else {
            i0 = pair;
            i1 = pair + half;
        }
        const long long t = t0 + token;
        const T* src = head < heads ? static_cast<const T*>(a.q) + t * a.ldq + (long long)head * dim
                       : head < heads + p.kv_heads
                           ? static_cast<const T*>(a.k) + t * a.ldk + (long long)(head - heads) * dim
                           : static_cast<const T*>(a.v) + t * a.ldv + (long long)(head - heads - p.kv_heads) * dim;
        load_elems(src + i0, x);
        load_elems(src + i1, y);
    };

    float x[kPairs], y[kPairs];
    int token = 0, head = 0, i0 = 0, i1 = 0;
    int u = threadIdx.x;
    if (u < live * per_token) fetch(u, x, y, token, head, i0, i1);

    // A warp finds a token's request, page and angles.
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (warp < live) {
        const int t = t0 + warp;
        const int b = request_of_row(p, t);
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
        if (lane == 0) {
            place[0][warp] = b < 0 ? -2 : k_at;
            place[1][warp] = v_at;
        }
        for (int i = lane; i < half; i += 32)
            turn[warp][i] = sin_cos((double)(position + a.offset) * load_l2(a.inv_freq + i));
    }
    __syncthreads();

    while (u < live * per_token) {
        const bool is_q = head < heads, is_v = head >= heads + p.kv_heads;
        if (!is_v && a.interleaved) {
            // pairs lie side by side: of x first, then of y (a single pair is x, y)
            const int pair = i0 / 2;
            if (pair < half) {
                if constexpr (kPairs == 1) {
                    const float2 t = turn[token][pair];
                    const float r = x[0] * t.y - y[0] * t.x;
                    y[0] = x[0] * t.x + y[0] * t.y;
                    x[0] = r;
                } else {
#pragma unroll
                    for (int j = 0; j < kPairs / 2; ++j) {
                        const float2 t = turn[token][pair + j], s = turn[token][pair + kPairs / 2 + j];
                        const float r = x[2 * j] * t.y - x[2 * j + 1] * t.x;
                        x[2 * j + 1] = x[2 * j] * t.x + x[2 * j + 1] * t.y;
                        x[2 * j] = r;
                        const float q = y[2 * j] * s.y - y[2 * j + 1] * s.x;
                        y[2 * j + 1] = y[2 * j] * s.x + y[2 * j + 1] * s.y;
                        y[2 * j] = q;
                    }
                }
            }
        } else if (!is_v && i0 < half) {
#pragma unroll
            for (int j = 0; j < kPairs; ++j) {
                const float2 t = turn[token][i0 + j];
                const float r = x[j] * t.y - y[j] * t.x;
                y[j] = x[j] * t.x + y[j] * t.y;
                x[j] = r;
            }
        }
        C* dst = nullptr;
        if (is_q) {
            if (place[0][token] != -2)
                dst = static_cast<C*>(a.q_out) + ((long long)(t0 + token) * heads + head) * dim;
        } else {
            const long long at = place[is_v][token];
            const int g = head - heads - (is_v ? p.kv_heads : 0);
            if (at >= 0) dst = static_cast<C*>(is_v ? a.v_cache : a.k_cache) + at + (long long)g * p.page * dim;
        }
        if (dst) {
            store_elems(dst + i0, x);
            store_elems(dst + i1, y);
        }
        u += kAppendThreads;
        if (u < live * per_token) fetch(u, x, y, token, head, i0, i1);
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
    // One token a block until every SM has several, then two.
    const int tokens = a.batch.rows <= 8 * sm_count() ? 1 : 2;
    const dim3 grid((a.batch.rows + tokens - 1) / tokens);
    if (wide) return launch_pdl_kernel(append_kernel<T, C, 8>, grid, dim3(kAppendThreads), 0, stream, a, tokens);
    return launch_pdl_kernel(append_kernel<T, C, 1>, grid, dim3(kAppendThreads), 0, stream, a, tokens);
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

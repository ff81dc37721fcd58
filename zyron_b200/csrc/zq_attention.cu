// zq_attention.cu -- attention of new tokens over a paged cache, a prefix that
// all requests share computed once for all of them (zq_paged_attention).
//
//   s_j = scale * q . k_j,   o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m)
//
// over the prefix's keys and the request's own, of which a causal row at
// position t sees those up to t.  One pass over the keys with a running maximum
// m, sum and output in fp32, in base 2.
//
// Split.  A request's rows of one kv head -- its new tokens times the heads of
// the group, which all read the same keys -- make an item (more than 256 rows:
// several); the shared prefix is one more request whose rows are all the call's
// rows.  Every worker -- a warp here, a block in the other kernel -- takes an equal
// run of the items' keys, whatever the lengths are: it finds its run by a scan over
// the requests, so the plan lives on the device and a captured call follows the
// lengths of its replay.  A run covers whole items and at most two parts of items,
// whose sums it leaves in slots of its own; a second kernel joins the parts of each
// item that a border cuts.  With a prefix, own and prefix results stay in fp32 with
// their maxima and sums, and a third joins the two.
//
// Items of many rows are matrix products for tcgen05 (zq_attention_sm100.cu).
// This file has the kernel of few rows -- single tokens, drafts: a decode batch
// reads its cache once, memory bandwidth.  A warp streams its run of keys, 16 a
// stage, through a ring of cp.async stages of its own, so that no barrier stands
// between the memory and the products, and a warp between two items leaves the
// memory to the others (four warps an item, their sums joined in shared memory:
// 96 requests of 20 to 500 tokens took 44 us, now 24); the products are mma.sync,
// which at 16 rows take 4 of the 22 cycles that a key's bytes take an SM.
// exp(s - m) enters the second product as a sum of two 16-bit parts, so that it is
// not rounded to the cache's type; with fp16 m lies 2^15 below the largest score, and
// the parts hold a weight to 2^-22 of itself or 2^-40 of the largest.  64 requests of 100 to 6000 tokens, 32 heads over
// 8 of 128: 805 MB in 137 us with the join, 5.9 TB/s; one token over 576 keys,
// 12 heads over 4 of 64, 10.6.  (At dim 128 two tiles spill 8 to 16 bytes a thread.)
#include "zq_attention.cuh"

namespace zq {

namespace {

using namespace attn;

constexpr int kWarps = FewPlan::kTeam;
constexpr int kThreads = 32 * kWarps;
constexpr int kSlice = FewPlan::kKeys;  // keys of a stage
constexpr int kLeast = 4;  // units of a worker, at least: all warps of a block inside one item have keys of it
static_assert(kLeast > FewPlan::kItem, "");
constexpr int kBlocksPerSm = 2;
constexpr int kJoinThreads = 256;
constexpr int kMaxManyBlocks = 256;

template <int kD>
constexpr int kStageBytes = kSlice * kD * 2 * 2;  // keys, then values
// Two tiles of q take a stage's room.
template <int kMT>
constexpr int kStages = kMT == 1 ? 3 : 2;
// A warp's ring and its q.
template <int kD, int kMT>
constexpr int kWarpBytes = kStages<kMT> * kStageBytes<kD> + 16 * kMT * kD * 2;

// 16-byte chunk `c` of row `r` of a row-major tile of kD 16-bit elements, chunks
// XOR-swizzled by row so that eight rows of a column of chunks lie in different banks.
template <int kD>
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
    return (uint32_t)(r * kD * 2 + ((c ^ (r & 7)) << 4));
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool live) {
    const int n = live ? 16 : 0;  // 0: the chunk is filled with zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
template <class T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (sizeof(T) == 2 && kIsHalf<T>)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// ---- the kernel -----------------------------------------------------------------

// kMT: 16-row tiles of an item's kRows = 16 kMT rows.
template <class T, int kD, int kMT>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm) attend_few_kernel(const AttentionArgs a, const Workspace ws) {
    constexpr int kRows = 16 * kMT, kS = kStages<kMT>;
    constexpr int kChunks = kD / 8;  // 16-byte chunks of a row
    static_assert(kS * kStageBytes<kD> >= kRows * kD * 4 && kRows * kD * 2 >= kRows * 8, "a warp's sums fit in its ring");
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ long long scratch[kWarps + 2 * kWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint8_t* ring = smem + warp * kWarpBytes<kD, kMT>;
    const uint32_t ring_u = smem_u32(ring);
    uint8_t* q_tile = ring + kS * kStageBytes<kD>;
    const uint32_t q_u = smem_u32(q_tile);
    const PagedBatch& p = a.batch;
    const int group = a.heads / p.kv_heads, dim = p.dim;
    const int worker = blockIdx.x * kWarps + warp;

    pdl_wait_primary();
    pdl_launch_dependents();
    const FewPlan plan{a, group, a.prefix_length > 0 ? live_rows(p) : 0};
    const Found at = find_workers<kThreads, kWarps>(plan, blockIdx.x * kWarps, warp, gridDim.x * kWarps, kLeast, scratch);
    Cursor<FewPlan> way(plan, at, worker);
    if (lane == 0) ws.cuts[0][worker] = way.cut(at.share, worker, kRows);

    while (way.next()) {
        const Request r = way.it.r;
        const int c0 = way.first_tile, c1 = way.end_tile, head0 = way.it.head, item_rows = r.rows * group;
        const bool prefix = way.it.b < 0;
        const int32_t* table = prefix ? a.prefix_pages : p.pages + (long long)way.it.b * p.ld_pages;

        const T* q_src = static_cast<const T*>(a.q);  // where a copy of no bytes points: a cache may have no pages
        // q of the item: row i is token i / group, head i % group of the kv head's.
#pragma unroll
        for (int j = 0; j < kRows * kChunks / 32; ++j) {
            const int i = j * 32 + lane, row = i / kChunks, c = i % kChunks;
            const bool live = row < item_rows && c * 8 < dim;
            const T* src = q_src;
            if (live)
                src += (long long)(r.first + row / group) * a.ldq + (long long)(head0 * group + row % group) * dim + c * 8;
            cp_async16(q_u + chunk_at<kD>(row, c), src, live);
        }
        cp_async_commit();

        // Keys [0, limit) are seen by the thread's rows g and g + 8 of each tile.
        int limit[kMT][2], low = r.length;
#pragma unroll
        for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int row = mt * 16 + e * 8 + (lane >> 2);
                int n = r.length;
                if (!prefix && a.causal) n = min(n, max(r.length - r.rows + row / group + 1, 0));
                limit[mt][e] = n;
                low = min(low, n);
            }
        low = __reduce_min_sync(0xffffffffu, low);

        // Slice i: keys key0 + 16 i ... in two halves of eight, each inside one page.
        // A lane keeps the pages of half a slice; a batch of 16 slices is looked up at
        // a time.
        const int key0 = c0 * kSlice;
        const int slices = key0 < r.length ? min(c1 - c0, (r.length - key0 - 1) / kSlice + 1) : 0;
        int found = -1, offset = 0;
        uint32_t missing = 0;  // two bits a stage: a half on no page of the cache
        const T* kc = static_cast<const T*>(a.k_cache) + (long long)head0 * p.page * dim;
        const T* vc = static_cast<const T*>(a.v_cache) + (long long)head0 * p.page * dim;
        const auto issue = [&](int i) {
            if (i < slices) {
                if ((i & 15) == 0) {
                    const int key = key0 + (i + (lane >> 1)) * kSlice + (lane & 1) * 8;
                    found = -1;
                    if (key < r.length) {
                        const int index = key / p.page;
                        offset = (key - index * p.page) * dim;
                        const int id = load_l2(table + index);
                        found = id >= 0 && id < p.cache_pages ? id : -1;
                    }
                }
                const int stage = i % kS;
                const uint32_t dst = ring_u + stage * kStageBytes<kD>;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int from = (i & 15) * 2 + half;
                    const int page = __shfl_sync(0xffffffffu, found, from);
                    const int off = __shfl_sync(0xffffffffu, offset, from);
                    const int keys = r.length - (key0 + i * kSlice + half * 8);  // valid keys of this half
                    missing &= ~(1u << (2 * stage + half));
                    if (page < 0 && keys > 0) missing |= 1u << (2 * stage + half);
                    const T* ks = kc + page * p.ld_k_page + off;
                    const T* vs = vc + page * p.ld_v_page + off;
#pragma unroll
                    for (int j = 0; j < 8 * kChunks / 32; ++j) {
                        const int row = (j * 32 + lane) / kChunks, c = (j * 32 + lane) % kChunks;
                        const bool live = page >= 0 && row < keys && c * 8 < dim;
                        const uint32_t to = chunk_at<kD>(half * 8 + row, c);
                        cp_async16(dst + to, live ? ks + row * dim + c * 8 : q_src, live);
                        cp_async16(dst + kSlice * kD * 2 + to, live ? vs + row * dim + c * 8 : q_src, live);
                    }
                }
            }
            cp_async_commit();
        };
        float o[kMT][kD / 8][4], top[kMT][2], sum[kMT][2];
        // An infinity that a row sees comes out of the products as NaN, since the second part
        // of a weight may be 0 or below.  An item that ends with a NaN is walked through once
        // more, its values multiplied by whole weights, slice by slice.
        for (bool careful = false;; careful = true) {
#pragma unroll
            for (int i = 0; i < kS - 1; ++i) issue(i);
            cp_async_wait<kS - 1>();
            __syncwarp();  // q is there

            // One tile's q stays in registers; two tiles' would not fit beside their sums.
            const auto load_q = [&](int mt, int k, uint32_t (&f)[4]) {
                ldmatrix4(q_u + chunk_at<kD>(mt * 16 + (lane & 15), 2 * k + (lane >> 4)), f);
            };
            uint32_t qf[kMT == 1 ? kD / 16 : 1][4];
            if constexpr (kMT == 1) {
#pragma unroll
                for (int k = 0; k < kD / 16; ++k) load_q(0, k, qf[k]);
            }
#pragma unroll
            for (int mt = 0; mt < kMT; ++mt) {
#pragma unroll
                for (int n = 0; n < kD / 8; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[mt][n][e] = 0.0f;
                top[mt][0] = top[mt][1] = -INFINITY;
                sum[mt][0] = sum[mt][1] = 0.0f;
            }

            for (int i = 0; i < slices; ++i) {
                issue(i + kS - 1);
                cp_async_wait<kS - 1>();
                __syncwarp();
                const int stage = i % kS, key = key0 + i * kSlice;
                const uint32_t k_u = ring_u + stage * kStageBytes<kD>, v_u = k_u + kSlice * kD * 2;
                float s[kMT][2][4];
#pragma unroll
                for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[mt][n][e] = 0.0f;
#pragma unroll
                for (int k = 0; k < kD / 16; ++k) {
                    uint32_t f[4];
                    // lanes 0-7 / 8-15: keys 0-7, low / high half of 16 elements; 16-31: keys 8-15
                    ldmatrix4(k_u + chunk_at<kD>((lane & 7) + (lane >> 4) * 8, 2 * k + ((lane >> 3) & 1)), f);
#pragma unroll
                    for (int mt = 0; mt < kMT; ++mt) {
                        if constexpr (kMT > 1) load_q(mt, k, qf[0]);
                        mma16816<T>(s[mt][0], qf[kMT == 1 ? k : 0], f[0], f[1]);
                        mma16816<T>(s[mt][1], qf[kMT == 1 ? k : 0], f[2], f[3]);
                    }
                }
                const uint32_t gone = (missing >> (2 * stage)) & 3u;
                const bool masked = key + kSlice > low || gone;
                uint32_t hi[kMT][4], lo[kMT][4];
                float pr[kMT][2][4];
#pragma unroll
                for (int mt = 0; mt < kMT; ++mt) {
                    float most[2] = {-INFINITY, -INFINITY};
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float t = s[mt][n][e] * a.scale_log2;
                            if (masked) {
                                const int j = key + n * 8 + (lane & 3) * 2 + (e & 1);
                                if (j >= limit[mt][e >> 1] || ((gone >> n) & 1)) t = -INFINITY;
                            }
                            s[mt][n][e] = t;
                            most[e >> 1] = fmaxf(most[e >> 1], t);
                        }
                    float ref[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        most[e] = fmaxf(most[e], __shfl_xor_sync(0xffffffffu, most[e], 1));
                        most[e] = fmaxf(most[e], __shfl_xor_sync(0xffffffffu, most[e], 2));
                        if (kLift<T> != 0.0f) most[e] = __fadd_ru(most[e], -kLift<T>);
                        const float now = fmaxf(top[mt][e], most[e]);
                        ref[e] = now == -INFINITY ? 0.0f : now;  // nothing seen yet: every weight is 0
                        const float keep = exp2_approx(top[mt][e] - ref[e]);
                        top[mt][e] = now;
                        if (keep != 1.0f) {
                            sum[mt][e] *= keep;
#pragma unroll
                            for (int n = 0; n < kD / 8; ++n) {
                                o[mt][n][2 * e] *= keep;
                                o[mt][n][2 * e + 1] *= keep;
                            }
                        }
                    }
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            pr[mt][n][e] = exp2_approx(s[mt][n][e] - ref[e >> 1]);
                            sum[mt][e >> 1] += pr[mt][n][e];
                        }
                    // the accumulators' layout is that of the second product's left operand
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            split_pair<T>(pr[mt][n][2 * e], pr[mt][n][2 * e + 1], hi[mt][2 * n + e], lo[mt][2 * n + e]);
                }
                if (careful || (masked && wild_values<T, kD>(v_u, lane))) {
                    // A value that some rows must not see is no number: 0 times it would
                    // reach them through the product.  Each row takes its own keys' alone,
                    // with whole weights.
#pragma unroll 1
                    for (int kk = 0; kk < kSlice; ++kk) {
                        const int n = kk >> 3, from = (lane & ~3) | ((kk & 7) >> 1);
#pragma unroll
                        for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const float w0 = n ? pr[mt][1][2 * e] : pr[mt][0][2 * e];
                                const float w1 = n ? pr[mt][1][2 * e + 1] : pr[mt][0][2 * e + 1];
                                const float w = __shfl_sync(0xffffffffu, kk & 1 ? w1 : w0, from);
                                if (key + kk < limit[mt][e] && !((gone >> n) & 1)) {
#pragma unroll
                                    for (int d = 0; d < kD / 8; ++d) {
                                        const T* v = reinterpret_cast<const T*>(
                                            ring + (v_u - ring_u) + chunk_at<kD>(kk, d) + (lane & 3) * 4);
                                        o[mt][d][2 * e] += w * to_float(v[0]);
                                        o[mt][d][2 * e + 1] += w * to_float(v[1]);
                                    }
                                }
                            }
                    }
                } else {
#pragma unroll
                    for (int d = 0; d < kD / 16; ++d) {
                        uint32_t f[4];
                        // lanes 0-15: keys 0-15 of elements 0-7; 16-31: of elements 8-15
                        ldmatrix4_trans(v_u + chunk_at<kD>(lane & 15, 2 * d + (lane >> 4)), f);
#pragma unroll
                        for (int mt = 0; mt < kMT; ++mt) {
                            mma16816<T>(o[mt][2 * d], hi[mt], f[0], f[1]);
                            mma16816<T>(o[mt][2 * d + 1], hi[mt], f[2], f[3]);
                            mma16816<T>(o[mt][2 * d], lo[mt], f[0], f[1]);
                            mma16816<T>(o[mt][2 * d + 1], lo[mt], f[2], f[3]);
                        }
                    }
                }
                __syncwarp();  // the stage may be written again
            }
            cp_async_wait<0>();
            __syncwarp();
            float off = 0.0f;
#pragma unroll
            for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
                for (int n = 0; n < kD / 8; ++n) off += (o[mt][n][0] + o[mt][n][1]) + (o[mt][n][2] + o[mt][n][3]);
            if (careful || !__any_sync(0xffffffffu, off != off)) break;
        }

        if (FewPlan::team_inside(way.it.start, way.it.end, at.share, worker)) {
            // All the block's warps work on this one item: one part of it, by way of
            // their rings; maxima and sums where q was.
            float* mine = reinterpret_cast<float*>(ring);
            float* stats = reinterpret_cast<float*>(q_tile);
#pragma unroll
            for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int row = mt * 16 + e * 8 + (lane >> 2);
                    float t = sum[mt][e];
                    t += __shfl_xor_sync(0xffffffffu, t, 1);
                    t += __shfl_xor_sync(0xffffffffu, t, 2);
#pragma unroll
                    for (int n = 0; n < kD / 8; ++n)
                        *reinterpret_cast<float2*>(mine + row * kD + n * 8 + (lane & 3) * 2) =
                            make_float2(o[mt][n][2 * e], o[mt][n][2 * e + 1]);
                    if ((lane & 3) == 0) *reinterpret_cast<float2*>(stats + 2 * row) = make_float2(top[mt][e], t);
                }
            __syncthreads();
            const long long part = (long long)blockIdx.x * kWarps * 2 * kRows;
            const long long from = blockIdx.x * kWarps * at.share, to = from + kWarps * at.share;
            const bool all = FewPlan::cut(way.it.start, way.it.end, way.it.key_tiles, from) == 0 &&
                             FewPlan::cut(way.it.start, way.it.end, way.it.key_tiles, to) == way.it.key_tiles;
            for (int i = threadIdx.x; i < item_rows * (kD / 4); i += kThreads) {
                const int row = i / (kD / 4), d = i % (kD / 4) * 4;
                Joined j;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    const float* sums = reinterpret_cast<const float*>(smem + w * kWarpBytes<kD, kMT>);
                    const float* st = reinterpret_cast<const float*>(smem + w * kWarpBytes<kD, kMT> + kS * kStageBytes<kD>);
                    j.add(*reinterpret_cast<const float2*>(st + 2 * row),
                          *reinterpret_cast<const float4*>(sums + row * kD + d));
                }
                if (d >= dim) continue;
                if (all) {
                    put_row<T>(a, ws, prefix, r.first + row / group, head0 * group + row % group, d, j.v, j.most, j.total);
                    continue;
                }
                *reinterpret_cast<float4*>(ws.part_sums[0] + (part + row) * kD + d) =
                    make_float4(j.v[0], j.v[1], j.v[2], j.v[3]);
                if (d == 0) *reinterpret_cast<float2*>(ws.part_stats[0] + 2 * (part + row)) = make_float2(j.most, j.total);
            }
            break;  // it is the one part of each of them
        }

        // Rows g and g + 8 of each tile, two elements of every eight a thread.
        const long long slot = (long long)worker * 2 + way.slot;
#pragma unroll
        for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int row = mt * 16 + e * 8 + (lane >> 2);
                float t = sum[mt][e];
                t += __shfl_xor_sync(0xffffffffu, t, 1);
                t += __shfl_xor_sync(0xffffffffu, t, 2);
                if (row >= item_rows) continue;
                const int token = r.first + row / group, head = head0 * group + row % group;
                if (way.whole && a.prefix_length == 0) {
                    const float norm = t == 0.0f ? 0.0f : 1.0f / t;  // a row that sees no key is zero
                    T* dst = static_cast<T*>(a.out) + (long long)token * a.ld_out + (long long)head * dim;
#pragma unroll
                    for (int n = 0; n < kD / 8; ++n)
                        if (n * 8 < dim) {
                            Pack<T, 2> w{{from_float<T>(t == 0.0f ? 0.0f : o[mt][n][2 * e] * norm),
                                          from_float<T>(t == 0.0f ? 0.0f : o[mt][n][2 * e + 1] * norm)}};
                            *reinterpret_cast<Pack<T, 2>*>(dst + n * 8 + (lane & 3) * 2) = w;
                        }
                } else {
                    const long long at_row = way.whole ? (long long)token * a.heads + head : slot * kRows + row;
                    float* sums = way.whole ? (prefix ? ws.row_sums[1] : ws.row_sums[0]) : ws.part_sums[0];
                    float* stats = way.whole ? (prefix ? ws.row_stats[1] : ws.row_stats[0]) : ws.part_stats[0];
                    float* dst = sums + at_row * (way.whole ? dim : kD);
#pragma unroll
                    for (int n = 0; n < kD / 8; ++n)
                        if (n * 8 < dim)
                            *reinterpret_cast<float2*>(dst + n * 8 + (lane & 3) * 2) =
                                make_float2(o[mt][n][2 * e], o[mt][n][2 * e + 1]);
                    if ((lane & 3) == 0) *reinterpret_cast<float2*>(stats + 2 * at_row) = make_float2(top[mt][e], t);
                }
            }
    }
}

// Joins the items that borders of the kernel of few rows cut: a warp two rows of a
// border, eight parts at a time, the rows behind them further along the grid's y
// (17 drafts of up to 6 tokens 9 us; whole blocks after one another 16; four rows a
// warp: 64 requests' join 16 us against 7).
constexpr int kJoinRows = 2;
template <class T, int kD, int kMT>
__global__ void __launch_bounds__(kJoinThreads) join_few_kernel(const AttentionArgs a, const Workspace ws, int workers) {
    constexpr int kLanes = kD / 4, kTogether = 32 / kLanes;  // lanes of a row, rows at a time
    pdl_launch_dependents();
    pdl_wait_primary();  // before any return: who waits for this kernel counts on the ones before it too
    const int g = blockIdx.x * (kJoinThreads / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (g == 0 || g >= workers) return;
    const Cut c = load_cut(ws, 0, g);
    for (int row0 = blockIdx.y * kJoinRows; row0 < c.rows; row0 += gridDim.y * kJoinRows)
        join_rows<T, FewPlan, kJoinRows / kTogether, kTogether, 8>(
            a, ws, c, 0, g, row0 + lane / kLanes, lane % kLanes * 4,
            [&](long long slot, int row, long long& stats, long long& sums) {
                stats = slot * (16 * kMT) + row;
                sums = stats * kLanes + lane % kLanes;
            });
}

// The same of the kernel of many rows, whose parts lie row beside row.  Few borders
// may cut an item of many parts, or all of them one of two: every block lists the
// split items and takes its turn at their pieces, 8 rows and 8 parts at a time of few
// items, 16 and 2 of many (a 16000 key prefix of 96 rows, 16 items of 10 parts, 20 MB:
// 10 us, by blocks a border 19; prompts, 140 items of 2 parts, 36 MB: 18, was 19).
template <int kD>
constexpr int kJoinBlocks = 4 * 128 / kD;  // an SM
template <class T, int kD>
__global__ void __launch_bounds__(2 * kD, kJoinBlocks<kD>) join_many_kernel(const AttentionArgs a, const Workspace ws, int workers) {
    constexpr int kThreads = 2 * kD;  // a warp four chunks of four columns
    __shared__ int split[kMaxManyBlocks], count;
    pdl_launch_dependents();
    pdl_wait_primary();
    if (threadIdx.x == 0) count = 0;
    __syncthreads();
    for (int g0 = 1; g0 < workers; g0 += kThreads) {
        const int g = g0 + threadIdx.x;
        const bool is = g < workers && load_l2(&ws.cuts[1][g].rows) > 0;
        // in order, the same in every block
        __shared__ int before[kThreads / 32];
        const unsigned m = __ballot_sync(0xffffffffu, is);
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        if (lane == 0) before[warp] = __popc(m);
        __syncthreads();
        int at = count;
        for (int w = 0; w < warp; ++w) at += before[w];
        if (is) split[at + __popc(m & ((1u << lane) - 1u))] = g;
        __syncthreads();
        if (threadIdx.x == kThreads - 1) count = at + __popc(m);
        __syncthreads();
    }
    const int lane = threadIdx.x & 31, chunk = (threadIdx.x >> 5) * 4 + (lane >> 3);
    const auto place = [&](long long slot, int row, long long& stats, long long& sums) {
        stats = slot * kManyRows + row;
        sums = (slot * (kD / 4) + chunk) * kManyRows + row;
    };
    const auto join = [&](auto steps, auto deep) {
        constexpr int kSteps = decltype(steps)::value, kPieces = kManyRows / (8 * kSteps);
        for (int i = blockIdx.x; i < count * kPieces; i += gridDim.x) {
            const int g = split[i / kPieces], row = i % kPieces * 8 * kSteps;
            const Cut c = load_cut(ws, 1, g);
            if (row < c.rows)
                join_rows<T, ManyPlan, kSteps, 8, decltype(deep)::value>(a, ws, c, 1, g, row + (lane & 7), chunk * 4, place);
        }
    };
    if (count * (kManyRows / 8) <= (int)gridDim.x)
        join(std::integral_constant<int, 1>{}, std::integral_constant<int, 8>{});
    else
        join(std::integral_constant<int, 2>{}, std::integral_constant<int, 2>{});
}

// Joins the own and the prefix result of every row that a request owns.
template <class T>
__global__ void __launch_bounds__(256) join_prefix_kernel(const AttentionArgs a, const Workspace ws) {
    const PagedBatch& p = a.batch;
    const int t = blockIdx.x;
    const bool owned = request_of_row(p, t) >= 0;
    pdl_launch_dependents();
    pdl_wait_primary();
    if (!owned) return;
    const int each = p.dim / 4;
    for (int i = threadIdx.x; i < a.heads * each; i += 256) {
        const int head = i / each, d = i % each * 4;
        const long long row = (long long)t * a.heads + head;
        Joined j;
#pragma unroll
        for (int k = 0; k < 2; ++k)
            j.add(load_l2(reinterpret_cast<const float2*>(ws.row_stats[k]) + row),
                  load_l2(reinterpret_cast<const float4*>(ws.row_sums[k] + row * p.dim + d)));
        put_out<T>(a, t, head, d, j.v, j.total);
    }
}

// How a call is launched, from its sizes alone.
struct Shape {
    int few_rows;     // 16 or 32: the rows of the kernel of few rows; 0: it has none
    int few_blocks;
    int few_most;     // rows of its items at most
    int many_blocks;  // 0: no item can have more than few_rows
    int width;
};
Shape shape_of(const AttentionArgs& a) {
    Shape s{};
    const int group = a.heads / a.batch.kv_heads;
    const long long all = (long long)a.batch.rows * group;
    // the most rows of a kv head that an item may have
    const long long most = a.batch.starts || a.prefix_length > 0 ? all : group;
    if (group <= 32) s.few_rows = most <= 16 || (!a.batch.starts && group <= 16) ? 16 : 32;
    s.few_most = (int)std::min<long long>(most, s.few_rows);
    s.few_blocks = s.few_rows ? kBlocksPerSm * sm_count() : 0;
    s.many_blocks = most > s.few_rows ? std::min(sm_count(), kMaxManyBlocks) : 0;
    s.width = a.batch.dim <= 64 ? 64 : 128;
    return s;
}

template <class T, int kD, int kMT>
cudaError_t launch_t(const AttentionArgs& a, int dtype, const Shape& s, const Workspace& ws, cudaStream_t stream) {
    cudaError_t e = cudaSuccess;
    if (s.many_blocks) e = launch_attend_many(a, dtype, ws, s.many_blocks, stream);
    if (e != cudaSuccess) return e;
    if (s.few_blocks) {
        constexpr int smem = kWarps * kWarpBytes<kD, kMT>;
        static_assert(kBlocksPerSm * (smem + 1024 + 256) <= 228 * 1024, "both blocks of an SM");
        e = ensure_smem_attr(attend_few_kernel<T, kD, kMT>, smem);
        if (e != cudaSuccess) return e;
        e = launch_pdl_kernel(attend_few_kernel<T, kD, kMT>, dim3(s.few_blocks), dim3(kThreads), smem, stream, a, ws);
        if (e != cudaSuccess) return e;
    }
    if (s.few_blocks) {
        const int workers = s.few_blocks * kWarps, each = kJoinThreads / 32;
        e = launch_pdl_kernel(join_few_kernel<T, kD, kMT>, dim3((workers + each - 1) / each, std::min(8, (s.few_most + kJoinRows - 1) / kJoinRows)),
                              dim3(kJoinThreads), 0, stream, a, ws, workers);
        if (e != cudaSuccess) return e;
    }
    if (s.many_blocks)
        e = launch_pdl_kernel(join_many_kernel<T, kD>, dim3(kJoinBlocks<kD> * sm_count()), dim3(2 * kD), 0, stream, a, ws, s.many_blocks);
    if (e != cudaSuccess || a.prefix_length == 0) return e;
    return launch_pdl_kernel(join_prefix_kernel<T>, dim3(a.batch.rows), dim3(256), 0, stream, a, ws);
}

template <class T>
cudaError_t launch_d(const AttentionArgs& a, int dtype, const Shape& s, const Workspace& ws, cudaStream_t stream) {
    if (s.width == 64)
        return s.few_rows == 32 ? launch_t<T, 64, 2>(a, dtype, s, ws, stream) : launch_t<T, 64, 1>(a, dtype, s, ws, stream);
    return s.few_rows == 32 ? launch_t<T, 128, 2>(a, dtype, s, ws, stream) : launch_t<T, 128, 1>(a, dtype, s, ws, stream);
}

size_t align256(size_t n) { return (n + 255) / 256 * 256; }

// Lays the workspace out; base null: its size alone.
Workspace layout(const AttentionArgs& a, const Shape& s, uint8_t* base, size_t* bytes) {
    Workspace ws{};
    size_t at = 0;
    const auto take = [&](size_t n) {
        float* p = base ? reinterpret_cast<float*>(base + at) : nullptr;
        at += align256(n * sizeof(float));
        return p;
    };
    const size_t parts[2] = {(size_t)s.few_blocks * kWarps * 2 * s.few_rows, (size_t)s.many_blocks * 2 * kManyRows};
    for (int k = 0; k < 2; ++k) {
        ws.part_sums[k] = take(parts[k] * s.width);
        ws.part_stats[k] = take(parts[k] * 2);
        ws.cuts[k] = reinterpret_cast<Cut*>(take((size_t)(k ? s.many_blocks : s.few_blocks * kWarps) * (sizeof(Cut) / sizeof(float))));
    }
    if (a.prefix_length > 0) {
        const size_t rows = (size_t)a.batch.rows * a.heads;
        for (int k = 0; k < 2; ++k) {
            ws.row_sums[k] = take(rows * a.batch.dim);
            ws.row_stats[k] = take(rows * 2);
        }
    }
    *bytes = at;
    return ws;
}

}  // namespace

size_t attention_workspace_bytes(const AttentionArgs& a) {
    size_t n = 0;
    layout(a, shape_of(a), nullptr, &n);
    return n;
}

cudaError_t launch_paged_attention(const AttentionArgs& args, int dtype, void* workspace, cudaStream_t stream) {
    AttentionArgs a = args;
    const Shape s = shape_of(a);
    a.few_rows = s.few_rows;
    size_t n = 0;
    const Workspace ws = layout(a, s, static_cast<uint8_t*>(workspace), &n);
    return dtype == ZQ_DTYPE_F16 ? launch_d<__half>(a, dtype, s, ws, stream)
                                 : launch_d<__nv_bfloat16>(a, dtype, s, ws, stream);
}

}  // namespace zq

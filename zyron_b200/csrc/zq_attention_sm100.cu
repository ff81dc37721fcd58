// zq_attention_sm100.cu -- attention items of many rows on 5th-generation tensor
// cores: prompts, long drafts, and the shared prefix of a batch, whose rows are
// all the batch's (zq_paged_attention; zq_attention.cu has the formulas and how
// work is split).
//
// A persistent block takes 256 rows of a kv head as two tiles of 128 (new tokens
// times the heads of the group) and walks their key tiles of 128:
//   warp 9       TMA: q once an item, then groups of a key tile and the value tile
//                before it through a ring in shared memory, a box for each run of
//                tokens in a page; tokens that do not exist are boxes outside the
//                tensor, which arrive as zeros.
//   warp 8       issues S_i = Q_i K^T into TMEM, for the two tiles by turns.
//   warp 10      issues O_i += P_i V with P_i read from TMEM.  V is the MN-major
//                operand: rows of the same boxes as K's, nothing is transposed.
//                (A thread takes about 50 cycles to issue an MMA of 64 and as long
//                as eight for a wait and a commit, so one warp for both kept the
//                tensor cores at half their rate.)
//   warps 0-7    a warpgroup a tile, a thread a row: scores from TMEM into registers,
//                running maximum, exp2, P back to TMEM, 16 bits each.
// TMEM holds the two outputs, the two P and one S, which both tiles use by turns:
// a warpgroup takes its scores into registers at once, so the next product starts
// while it works, and finds its next scores there when it is done.  With a place of
// its own for each tile's scores, P over them, a warpgroup waited for P V and Q K^T
// in turn: 4500 cycles for 256 rows x 128 keys (5700 in steps of 64 keys, since an
// MMA of 64 columns takes as long as one of 128), where the softmax takes 2250.
// A row's reference is raised, and its output in TMEM rescaled, only when its
// maximum has grown by more than 2^8 since (fp16: 2^3.9): weights up to 2^8 lose
// nothing in the sums' 32 bits.  P is rounded to the cache's type for the second
// product, half a step of each weight; a second part of it has no room in TMEM, which
// S, P and O fill at dim 128.  The sum is that of the unrounded weights: that of the
// rounded ones halves the error of rows that few keys dominate and leaves others' (2 %
// less on prompts), for 244 us instead of 224 as fp32 additions of 16-bit values, 303
// as a matrix instruction beside tcgen05.  fp16 has no exponents for weights far below
// the largest, so the reference is set 2^12 below that: half a step down to 2^-26 of
// the largest (e^-18), 2^-37 of it below.  A score is multiplied and the reference
// subtracted with one rounding, so the reference's own is in every weight alike: a
// factor of 2^-16 for scores of 2^27, which fp16's exponents still hold.  (Scores
// rounded first cost 11 us.)
//
// Bound: 4 dim operations a (row, key) on the tensor cores against one exponential,
// of which the special function unit makes 16 a cycle and SM: at dim 128 both take
// 2048 cycles for 256 rows x 128 keys.  Measured: about 2900, and four prompts of
// 1000 to 2600 tokens (32 heads over 8, dim 128) 224 us with their joins, the tensor
// cores at 54 % (fp16 247); a 16000 key prefix of 96 rows, fp16, 44.  168 registers a
// thread are what 11 warps get; 40 bytes spill.  Some of the exponentials as a
// polynomial on the fp32 pipe cost more issue slots than they freed (one in eight
// 258 us against 251, one in four 268, every other 296).
//
// A value that is no number must not reach rows that do not see it, and 0 times it
// would.  Tiles that a causal border cuts are searched for one; if there is, the
// warpgroup adds its own weighted values by itself and the MMA is left out.
#include "zq_attention.cuh"
#include "zq_internal.h"
#include "zq_tcgen05.cuh"

#include <numeric>

namespace zq {

namespace {

using namespace attn;

constexpr int kManyThreads = 352;
constexpr int kTile = 128;             // rows of a q tile, keys of a key tile
// TMEM columns: the scores of whichever tile, P (two keys a column), O.
constexpr int kScoreCol = 0, kWeightCol = 128, kOutCol = 256;
constexpr int kHalfBytes = kTile * 128;  // 128 rows x 64 elements, 128-byte swizzled
// How far (base 2) below a new maximum the reference is set, and how far above the
// reference a maximum may grow.  All rounded so that no weight is above 2^kRoom, the
// end of fp16, however large the scores are.
template <class T>
constexpr float kSetBelow = kIsHalf<T> ? 12.0f : 0.0f;
template <class T>
constexpr float kRoom = kIsHalf<T> ? 15.9375f : 8.0f;
constexpr int kBadRing = 8;
constexpr int kPartRing = 4;

// What the producer tells the other warps of a part.
struct Part {
    int first, rows, length;  // of the request
    int token0, head;         // first token of the item, kv head
    int first_tile, end_tile;
    int flags;                // kEnd, kPrefix, kWhole, kSecondSlot
};
enum : int { kEnd = 1, kPrefix = 2, kWhole = 4, kSecondSlot = 8 };

template <int kD>
struct Smem {
    static constexpr int kHalves = kD / 64;
    static constexpr int kTileBytes = kHalves * kHalfBytes;
    static constexpr int kGroupBytes = 2 * kTileBytes;  // keys, then values
    static constexpr int kGroups = kD == 128 ? 2 : 4;
    static constexpr int kRing = 2 * kTileBytes;  // after the two q tiles
    static constexpr int kStage = kRing + kGroups * kGroupBytes;  // 4 KiB a softmax warp
    static constexpr int kBars = kStage + 8 * 4096;
    static constexpr int kTotal = 1024 + kBars + 512;
    static_assert(kTotal + 1024 <= 227 * 1024, "shared memory, with the static part");
};

// Instruction descriptor of tcgen05.mma.kind::f16: A and B both fp16 or both bf16,
// A K-major, fp32 accumulators.
template <class T>
__host__ __device__ constexpr uint32_t idesc_f16(int n, bool b_mn_major) {
    const uint32_t type = kIsHalf<T> ? 0u : 1u;
    return (1u << 4) | (type << 7) | (type << 10) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(kTile >> 4) << 24);
}

// MN-major operand with 128-byte swizzle: 64 elements of the N dimension by 8 of K
// are 1024 bytes; the next 8 of K follow (SBO), the next 64 of N a tile half on (LBO).
__device__ __forceinline__ uint64_t make_mn_desc(uint32_t saddr) {
    uint64_t d = 0;
    d |= (uint64_t)((saddr >> 4) & 0x3FFFu);
    d |= (uint64_t)(kHalfBytes >> 4) << 16;
    d |= (uint64_t)(1024u >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}

// Issued by the one thread with `leads`.  The warp stays together around it, so that
// descriptors are formed in uniform registers, where the instruction wants them: 48
// cycles an instruction, 57 in a branch of one lane.
__device__ __forceinline__ void umma_f16(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                         uint32_t accumulate, bool leads) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 e, %5, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"((uint32_t)leads)
        : "memory");
}
// A from TMEM: two elements a column.
__device__ __forceinline__ void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc,
                                            uint32_t accumulate, bool leads) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 e, %5, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
        "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"((uint32_t)leads)
        : "memory");
}
__device__ __forceinline__ void umma_commit_if(uint64_t* bar, bool leads) {
    asm volatile(
        "{\n\t.reg .pred e;\n\t"
        "setp.ne.b32 e, %1, 0;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
        "r"((uint32_t)leads)
        : "memory");
}

__device__ __forceinline__ void tma_load_4d(void* dst, const void* tmap, uint64_t* bar, int x, int y, int z, int w) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_u32(dst)),
        "l"(tmap), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
        : "memory");
}

__device__ __forceinline__ void tmem_ld_32x32b_x8(uint32_t taddr, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr));
}
__device__ __forceinline__ void tmem_st_32x32b_x8(uint32_t taddr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ void tmem_st_32x32b_x32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t tmem_ld_32x32b_x1(uint32_t taddr) {
    uint32_t r;
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r) : "r"(taddr));
    return r;
}

// Whether any thread of a warpgroup (barrier 1 or 2, 128 threads) says so.
template <int kBarrier>
__device__ __forceinline__ bool any_at(bool v) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 q, %1, 0;\n\t"
        "barrier.cta.red.or.pred p, %2, 128, q;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(r)
        : "r"((uint32_t)v), "n"(kBarrier)
        : "memory");
    return r != 0;
}
__device__ __forceinline__ bool group_any(int wg, bool v) { return wg == 0 ? any_at<1>(v) : any_at<2>(v); }

// Two fp32 values an instruction.
__device__ __forceinline__ uint64_t pack_f32(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ float2 unpack_f32(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add_f32x2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

template <class T>
__device__ __forceinline__ uint32_t pack_pair(float x, float y) {
    Pack<T, 2> p{{from_float<T>(x), from_float<T>(y)}};
    uint32_t r;
    memcpy(&r, &p, 4);
    return r;
}

// Address of 16-byte chunk c of row r of a tile in shared memory.
__device__ __forceinline__ const uint8_t* tile_chunk(const uint8_t* tile, int r, int c) {
    return tile + (c >> 3) * kHalfBytes + r * 128 + (((c & 7) ^ (r & 7)) << 4);
}

// Rows [from, to) of a value tile that hold what a page holds behind a request's
// last token: zeros instead, since 0 times a NaN there would count.  Both
// warpgroups write the same zeros.
template <int kD>
__device__ __forceinline__ void clear_rows(uint8_t* v_tile, int from, int to, int t) {
    for (int i = t; i < (to - from) * (kD / 8); i += 128)
        *reinterpret_cast<uint4*>(const_cast<uint8_t*>(tile_chunk(v_tile, from + i / (kD / 8), i % (kD / 8)))) =
            make_uint4(0, 0, 0, 0);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// Whether rows [from, to) of a value tile hold an infinity or NaN (thread t: row t).
// An exponent of all ones carries into the sign bit when its lowest bit is added.
template <class T, int kD>
__device__ __forceinline__ bool wild_rows(const uint8_t* v_tile, int from, int to, int t) {
    constexpr uint32_t kOnes = kIsHalf<T> ? 0x7C007C00u : 0x7F807F80u, kLowest = kIsHalf<T> ? 0x04000400u : 0x00800080u;
    uint32_t carry = 0;
    if (t >= from && t < to) {
#pragma unroll
        for (int c = 0; c < kD / 8; ++c) {
            const uint4 w = *reinterpret_cast<const uint4*>(tile_chunk(v_tile, t, c));
            carry |= ((w.x & kOnes) + kLowest) | ((w.y & kOnes) + kLowest) | ((w.z & kOnes) + kLowest) |
                     ((w.w & kOnes) + kLowest);
        }
    }
    return (carry & 0x80008000u) != 0;
}

// O += P V of one key tile by the warpgroup itself, every row with the keys that it
// sees alone (`seen` of them, less those of `bad` eighths).
template <class T, int kD>
__device__ __noinline__ void add_own_values(uint32_t o_addr, uint32_t p_addr, const uint8_t* v_tile, int seen, uint32_t bad,
                                            bool first) {
    tmem_st_wait();  // P is there
#pragma unroll 1
    for (int c = 0; c < kD / 32; ++c) {
        uint32_t o[32];
        if (first) {
#pragma unroll
            for (int d = 0; d < 32; ++d) o[d] = 0u;
        } else {
            tmem_ld_32x32b_x32(o_addr + c * 32, o);
            tmem_ld_wait();
        }
#pragma unroll 1
        for (int k = 0; k < kTile; ++k) {
            const uint32_t pair = tmem_ld_32x32b_x1(p_addr + k / 2);
            tmem_ld_wait();
            Pack<T, 2> p;
            memcpy(&p, &pair, 4);
            const bool sees = k < seen && !((bad >> (k >> 3)) & 1);
            const float w = to_float(k & 1 ? p.e[1] : p.e[0]);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                Pack<T, 8> v;
                memcpy(&v, tile_chunk(v_tile, k, c * 4 + q), 16);
#pragma unroll
                for (int d = 0; d < 8; ++d) {
                    const float sum = fmaf(w, to_float(v.e[d]), __uint_as_float(o[8 * q + d]));
                    if (sees) o[8 * q + d] = __float_as_uint(sum);
                }
            }
        }
        tmem_st_32x32b_x32(o_addr + c * 32, o);
        tmem_st_wait();
    }
}

// The waits with their long way out of line: the code of the loops stays small.
__device__ __noinline__ bool wait_long(uint64_t* bar, uint32_t parity, uint32_t* err, uint32_t code) {
    return mbar_wait_bounded(bar, parity, err, code);
}
__device__ __forceinline__ bool wait_bounded(uint64_t* bar, uint32_t parity, uint32_t* err, uint32_t code) {
    return mbar_try_wait(bar, parity) || wait_long(bar, parity, err, code);
}
__device__ __noinline__ void drain_bounded(uint64_t* bar, uint32_t parity, uint32_t* err, uint32_t code) {
    mbar_drain_bounded(bar, parity, err, code);
}

struct Shape {
    int group, tile_tokens;  // tokens of a 128-row tile
    int box;                 // tokens of a page box
    int cache_end;           // a page outside the cache
    int wide_out;            // out takes 16-byte stores
};

template <class T, int kD>
__global__ void __launch_bounds__(kManyThreads, 1)
    attend_many_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                       const __grid_constant__ CUtensorMap tmap_v, const AttentionArgs a, const Workspace ws,
                       const Shape shape, uint32_t* __restrict__ err) {
    using S = Smem<kD>;
    constexpr int kGroups = S::kGroups;
    constexpr uint32_t kTmemCols = 512;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    __shared__ long long scratch[kManyThreads / 32 + 2];
    uint8_t* smem = smem_align1024(smem_raw);
    uint8_t* ring = smem + S::kRing;
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kBars);
    uint64_t* q_full = bars;
    uint64_t* q_empty = bars + 1;
    // by tile, a phase a key tile
    uint64_t* s_full = bars + 2;   // scores are there (MMA)
    uint64_t* p_ready = bars + 4;  // weights are there (the tile's warpgroup)
    uint64_t* o_done = bars + 6;   // the product with the values is done (MMA)
    uint64_t* s_free = bars + 8;   // the scores have been taken (whichever warpgroup's they are)
    uint64_t* mma_done = bars + 9;
    uint64_t* kv_full = bars + 10;
    uint64_t* kv_empty = kv_full + kGroups;
    uint32_t* bad_ring = reinterpret_cast<uint32_t*>(kv_empty + kGroups);  // eighths of a key tile on no page
    volatile uint32_t* own = bad_ring + kBadRing;  // by tile: its warpgroup added the values
    uint32_t* tmem_slot = bad_ring + kBadRing + 2;
    uint64_t* part_full = reinterpret_cast<uint64_t*>(bad_ring + kBadRing + 4);
    uint64_t* part_empty = part_full + kPartRing;
    Part* parts = reinterpret_cast<Part*>(part_empty + kPartRing);
    static_assert((10 + 2 * 4 + 2 * kPartRing) * 8 + (kBadRing + 4) * 4 + kPartRing * sizeof(Part) <= 512, "barriers");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const PagedBatch& p = a.batch;

    if (threadIdx.x == 0) {
        mbar_init(q_full, 1);
        mbar_init(q_empty, 1);
        mbar_init(mma_done, 2);
        mbar_init(s_free, 128);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_ready[i], 128);
            mbar_init(&o_done[i], 1);
        }
        for (int i = 0; i < kPartRing; ++i) {
            mbar_init(&part_full[i], 1);
            mbar_init(&part_empty[i], 10);  // every warp but the producer
        }
        for (int i = 0; i < kGroups; ++i) {
            mbar_init(&kv_full[i], 1);
            mbar_init(&kv_empty[i], 2);  // keys and values taken
        }
        fence_mbar_init();
        tma_prefetch_desc(&tmap_q);
        tma_prefetch_desc(&tmap_k);
        tma_prefetch_desc(&tmap_v);
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(kTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_wait_primary();
    pdl_launch_dependents();

    const ManyPlan plan{a, shape.group, a.prefix_length > 0 ? live_rows(p) : 0, 2 * shape.tile_tokens};
    const Found found = find_workers<kManyThreads, 1>(plan, blockIdx.x, 0, gridDim.x, 1, scratch);
    // Tiles of the item that hold rows.
    const auto q_tiles = [&](const Part& q) { return q.rows - q.token0 > shape.tile_tokens ? 2 : 1; };
    // The block's part number `i`; false: the producer gave up.
    const auto part_at = [&](uint32_t i, Part& q) {
        if (!wait_bounded(&part_full[i % kPartRing], (i / kPartRing) & 1, err, kDevErrTimeoutMma)) return false;
        q = parts[i % kPartRing];
        __syncwarp();
        if (lane == 0) mbar_arrive(&part_empty[i % kPartRing]);
        return true;
    };
    // A part of T key tiles has T + 1 groups: keys of tile k in group k, values in
    // the next; groups are counted over the block's parts.  Who takes the half of a
    // group that is there alone frees the other half too, so that nobody frees a
    // group before it has been filled (which would count for the one before it).
    const auto keys_of = [&](int g) { return ring + g % kGroups * S::kGroupBytes; };
    const auto values_of = [&](int g) { return keys_of(g) + S::kTileBytes; };
    const auto phase_of = [](int g) { return (uint32_t)(g / kGroups) & 1u; };

    if (warp == 9) {
        const uint32_t q_bytes = (uint32_t)(128 * shape.group * shape.tile_tokens);
        const int boxes = kTile / shape.box;  // of a half tile; at most 16
        int n = 0, g = 0;
        uint32_t part = 0;
        bool ok = true, q_issued = false;
        Cursor<ManyPlan> way(plan, found, blockIdx.x);
        if (lane == 0) ws.cuts[1][blockIdx.x] = way.cut(found.share, blockIdx.x, plan.tokens * shape.group);
        while (ok) {
            const bool more = way.next();
            const Request r = way.it.r;
            const bool prefix = way.it.b < 0;
            const int head = way.it.head;
            const Part q{r.first, r.rows, r.length, way.it.tile * 2 * shape.tile_tokens, head, way.first_tile, way.end_tile,
                         more ? (prefix ? kPrefix : 0) | (way.whole ? kWhole : 0) | (way.slot ? kSecondSlot : 0) : kEnd};
            if (part >= kPartRing &&
                !wait_bounded(&part_empty[part % kPartRing], (part / kPartRing - 1) & 1u, err, kDevErrTimeoutProducer))
                break;
            if (lane == 0) {
                parts[part % kPartRing] = q;
                mbar_arrive(&part_full[part % kPartRing]);
            }
            if (!more) break;
            const int32_t* table = prefix ? a.prefix_pages : p.pages + (long long)way.it.b * p.ld_pages;
            const int tiles = q_tiles(q);
            if (!wait_bounded(q_empty, (part & 1) ^ 1u, err, kDevErrTimeoutProducer)) break;
            if (lane == 0) mbar_arrive_expect_tx(q_full, (uint32_t)(tiles * S::kHalves) * q_bytes);
            __syncwarp();
            if (lane < tiles * S::kHalves) {
                const int i = lane / S::kHalves, half = lane % S::kHalves;
                tma_load_3d(smem + i * S::kTileBytes + half * kHalfBytes, &tmap_q, q_full, half * 64, head * shape.group,
                            r.first + q.token0 + i * shape.tile_tokens);
            }
            q_issued = true;
            ++part;
            int id = 0, row = 0, id_before = 0, row_before = 0;
            for (int j = q.first_tile; j <= q.end_tile; ++j, ++g) {
                const bool keys = j < q.end_tile, values = j > q.first_tile;
                id_before = id;
                row_before = row;
                if (keys) {
                    // Lane i looks box i's page up.
                    const int key = j * kTile + lane * shape.box;
                    id = shape.cache_end;
                    row = 0;
                    bool bad = false;
                    if (lane < boxes && key < r.length) {
                        const int index = key / p.page;
                        row = key - index * p.page;
                        const int v = load_l2(table + index);
                        bad = v < 0 || v >= p.cache_pages;
                        if (!bad) id = v;
                    }
                    const uint32_t eighths = bad ? ((1u << (shape.box / 8)) - 1u) << (lane * (shape.box / 8)) : 0u;
                    const uint32_t missing = __reduce_or_sync(0xffffffffu, eighths);
                    if (lane == 0) bad_ring[n % kBadRing] = missing;
                    ++n;
                }
                uint64_t* full = &kv_full[g % kGroups];
                if (!wait_bounded(&kv_empty[g % kGroups], phase_of(g) ^ 1u, err, kDevErrTimeoutProducer)) {
                    ok = false;
                    break;
                }
                if (lane == 0) mbar_arrive_expect_tx(full, (uint32_t)((int)keys + (int)values) * S::kTileBytes);
                __syncwarp();
                const int box = lane / S::kHalves, half = lane % S::kHalves;
                const int at = half * kHalfBytes + box * shape.box * 128;
                const int k_page = __shfl_sync(0xffffffffu, id, box), k_row = __shfl_sync(0xffffffffu, row, box);
                const int v_page = __shfl_sync(0xffffffffu, id_before, box), v_row = __shfl_sync(0xffffffffu, row_before, box);
                if (box < boxes) {
                    if (keys) tma_load_4d(keys_of(g) + at, &tmap_k, full, half * 64, k_row, head, k_page);
                    if (values) tma_load_4d(values_of(g) + at, &tmap_v, full, half * 64, v_row, head, v_page);
                }
            }
        }
        // Every copy lands before the block can exit.
        if (q_issued) drain_bounded(q_full, (part - 1) & 1u, err, kDevErrTimeoutDrain);
        for (int i = max(0, g - kGroups); i < g; ++i)
            drain_bounded(&kv_full[i % kGroups], phase_of(i), err, kDevErrTimeoutDrain);
    } else if (warp == 8) {
        // S = Q_i K^T of each group's keys, once the scores before have been taken.
        constexpr uint32_t idesc = idesc_f16<T>(kTile, false);
        constexpr int kHalf = kHalfBytes >> 4;
        const bool leads = lane == 0;
        const uint64_t q_desc = make_sw128_desc(smem_u32(smem)), k_desc = make_sw128_desc(smem_u32(ring));
        int g = 0;
        uint32_t part = 0, taken = 0;
        bool ok = true;
        Part q;
        while (ok && part_at(part, q) && !(q.flags & kEnd)) {
            const int tiles = q_tiles(q);
            ok = wait_bounded(q_full, part++ & 1, err, kDevErrTimeoutMma);
            for (int j = q.first_tile; j < q.end_tile && ok; ++j, ++g) {
                ok = wait_bounded(&kv_full[g % kGroups], phase_of(g), err, kDevErrTimeoutMma);
                const uint64_t kb = k_desc + (uint32_t)(g % kGroups * S::kGroupBytes >> 4);
                for (int i = 0; i < tiles && ok; ++i) {
                    if (taken > 0) ok = wait_bounded(s_free, (taken - 1) & 1, err, kDevErrTimeoutMma);
                    if (!ok) break;
                    ++taken;
                    tmem_fence_after();
                    const uint64_t qa = q_desc + (uint32_t)(i * S::kTileBytes >> 4);
#pragma unroll
                    for (int k = 0; k < kD / 16; ++k)
                        umma_f16(tmem + kScoreCol, qa + ((k >> 2) * kHalf + (k & 3) * 2),
                                 kb + ((k >> 2) * kHalf + (k & 3) * 2), idesc, k > 0, leads);
                    umma_commit_if(&s_full[i], leads);
                }
                if (!ok) break;
                umma_commit_if(&kv_empty[g % kGroups], leads);
                if (j == q.first_tile) umma_commit_if(&kv_empty[g % kGroups], leads);
            }
            if (!ok) break;
            umma_commit_if(q_empty, leads);
            ++g;  // the part's last group has values alone
        }
        // All MMAs issued by this warp complete before TMEM is freed.
        umma_commit_if(mma_done, leads);
        drain_bounded(mma_done, 0, err, kDevErrTimeoutDrain);
    } else if (warp == 10) {
        // O_i += P_i V of each group's values.
        constexpr uint32_t idesc = idesc_f16<T>(kD, true);
        const bool leads = lane == 0;
        const uint64_t v_desc = make_mn_desc(smem_u32(ring) + S::kTileBytes);
        int g = 0;
        uint32_t part = 0, weights[2] = {0, 0};
        bool ok = true;
        Part q;
        while (ok && part_at(part++, q) && !(q.flags & kEnd)) {
            const int tiles = q_tiles(q);
            ++g;  // the part's first group has keys alone
            for (int j = q.first_tile; j < q.end_tile && ok; ++j, ++g) {
                ok = wait_bounded(&kv_full[g % kGroups], phase_of(g), err, kDevErrTimeoutMma);
                const uint64_t vb = v_desc + (uint32_t)(g % kGroups * S::kGroupBytes >> 4);
                for (int i = 0; i < tiles && ok; ++i) {
                    ok = wait_bounded(&p_ready[i], weights[i]++ & 1, err, kDevErrTimeoutMma);
                    if (!ok) break;
                    tmem_fence_after();
                    if (!own[i]) {
#pragma unroll
                        for (int k = 0; k < kTile / 16; ++k)
                            umma_f16_ts(tmem + kOutCol + i * kD, tmem + kWeightCol + i * (kTile / 2) + k * 8,
                                        vb + k * (2048 >> 4), idesc, j > q.first_tile || k > 0, leads);
                    }
                    umma_commit_if(&o_done[i], leads);
                }
                if (!ok) break;
                umma_commit_if(&kv_empty[g % kGroups], leads);
                if (j == q.end_tile - 1) umma_commit_if(&kv_empty[g % kGroups], leads);
            }
        }
        umma_commit_if(mma_done, leads);
        drain_bounded(mma_done, 0, err, kDevErrTimeoutDrain);
    } else {
        const int wg = warp >> 2, t = threadIdx.x & 127;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t s_addr = tmem + lanes + kScoreCol, p_addr = tmem + lanes + kWeightCol + wg * (kTile / 2),
                       o_addr = tmem + lanes + kOutCol + wg * kD;
        const float scale = a.scale_log2;
        int n = 0, g = 0;
        uint32_t tiles_done = 0, part = 0;
        bool ok = true;
        Part r;
        for (; ok && part_at(part++, r) && !(r.flags & kEnd); ++g) {
            if (wg >= q_tiles(r)) {
                n += r.end_tile - r.first_tile;
                g += r.end_tile - r.first_tile;
                continue;
            }
            const bool causal = !(r.flags & kPrefix) && a.causal;
            const int token0 = r.token0 + wg * shape.tile_tokens;  // of the tile, in the request
            const int token = token0 + t / shape.group, in_group = t % shape.group;
            const bool row_ok = t < shape.tile_tokens * shape.group && token < r.rows;
            const auto limit_of = [&](int tok) {
                return causal ? min(max(r.length - r.rows + tok + 1, 0), r.length) : r.length;
            };
            const int limit = limit_of(row_ok ? token : r.rows - 1), low = limit_of(token0);
            float ref = -INFINITY, sum = 0.0f;
            for (int j = r.first_tile; j < r.end_tile; ++j, ++n, ++g, ++tiles_done) {
                const int key0 = j * kTile;
                const bool first = j == r.first_tile;
                if (!wait_bounded(&s_full[wg], tiles_done & 1, err, kDevErrTimeoutEpilogue)) {
                    ok = false;
                    break;
                }
                tmem_fence_after();
                const uint32_t bad = *(volatile uint32_t*)&bad_ring[n % kBadRing];
                const bool masked = key0 + kTile > low || bad;
                float mul = scale;
                if (bad || !(scale > 0.0f)) {
                    // Key tiles with pages outside the cache, and scales that turn the
                    // order around: scaled and masked in their place first.
#pragma unroll 1
                    for (int c = 0; c < 4; ++c) {
                        uint32_t x[32];
                        tmem_ld_32x32b_x32(s_addr + c * 32, x);
                        tmem_ld_wait();
                        const int seen = limit - key0 - c * 32;
#pragma unroll
                        for (int k = 0; k < 32; ++k) {
                            const bool out = k >= seen || ((bad >> (c * 4 + (k >> 3))) & 1);
                            x[k] = __float_as_uint(out ? -INFINITY : __uint_as_float(x[k]) * scale);
                        }
                        tmem_st_32x32b_x32(s_addr + c * 32, x);
                    }
                    tmem_st_wait();
                    mul = 1.0f;
                }
                // Half of the scores at a time: the first half's largest while the second comes.
                uint32_t s[4][32];
                float m[4];
                const auto largest = [&](int half) {
                    if (masked) {
                        const int seen = limit - key0 - half * 64;
#pragma unroll
                        for (int k = 0; k < 64; ++k)
                            if (k >= seen) s[2 * half + k / 32][k % 32] = __float_as_uint(-INFINITY);
                    }
#pragma unroll
                    for (int k = 0; k < 32; ++k) {
                        const float x = fmaxf(__uint_as_float(s[2 * half][k]), __uint_as_float(s[2 * half + 1][k]));
                        m[k & 3] = half == 0 && k < 4 ? x : fmaxf(m[k & 3], x);
                    }
                };
                tmem_ld_32x32b_x32(s_addr, s[0]);
                tmem_ld_32x32b_x32(s_addr + 32, s[1]);
                tmem_ld_wait();
                tmem_ld_32x32b_x32(s_addr + 64, s[2]);
                tmem_ld_32x32b_x32(s_addr + 96, s[3]);
                largest(0);
                tmem_ld_wait();
                tmem_fence_before();
                mbar_arrive(s_free);
                largest(1);
                const float top = __fmul_ru(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])), mul);
                // The product of the key tile before is in O, and has read its weights.
                if (!first) {
                    if (!wait_bounded(&o_done[wg], (tiles_done - 1) & 1, err, kDevErrTimeoutEpilogue)) {
                        ok = false;
                        break;
                    }
                    tmem_fence_after();
                }
                const bool grown = top > __fadd_rd(ref, kRoom<T>);  // from -inf: by anything
                if (__any_sync(0xffffffffu, grown)) {
                    const float now = grown ? __fadd_ru(top, -kSetBelow<T>) : ref;
                    const float keep = grown ? exp2_approx(ref - now) : 1.0f;
                    ref = now;
                    sum *= keep;
                    if (!first) {
#pragma unroll 1
                        for (int c = 0; c < kD / 8; ++c) {
                            uint32_t o[8];
                            tmem_ld_32x32b_x8(o_addr + c * 8, o);
                            tmem_ld_wait();
#pragma unroll
                            for (int k = 0; k < 8; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * keep);
                            tmem_st_32x32b_x8(o_addr + c * 8, o);
                        }
                    }
                }
                const float from = ref == -INFINITY ? 0.0f : -ref;  // nothing seen yet: every weight is 0
                const uint64_t mul2 = pack_f32(mul, mul), from2 = pack_f32(from, from);
                uint64_t acc[2] = {0, 0};
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    uint32_t w[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const int at = (c & 1) * 16 + 2 * k;
                        const float2 x = unpack_f32(
                            fma_f32x2(pack_f32(__uint_as_float(s[c / 2][at]), __uint_as_float(s[c / 2][at + 1])), mul2, from2));
                        const float u = exp2_approx(x.x), v = exp2_approx(x.y);
                        acc[k & 1] = add_f32x2(acc[k & 1], pack_f32(u, v));
                        w[k] = pack_pair<T>(u, v);
                    }
                    tmem_st_32x32b_x8(p_addr + c * 8, w);
                }
                const float2 both = unpack_f32(add_f32x2(acc[0], acc[1]));
                sum += both.x + both.y;
                bool wild = false;
                if (masked) {
                    // Rows of the value tile: those behind the request's last token in
                    // its box, and those that some row does not see.
                    const int valid = min(kTile, r.length - key0), from_row = max(low - key0, 0);
                    const int clear_to = (valid + shape.box - 1) / shape.box * shape.box;
                    if (valid < clear_to || from_row < valid) {
                        uint8_t* v_tile = values_of(g + 1);
                        if (!wait_bounded(&kv_full[(g + 1) % kGroups], phase_of(g + 1), err, kDevErrTimeoutEpilogue)) {
                            ok = false;
                            break;
                        }
                        if (valid < clear_to) clear_rows<kD>(v_tile, valid, clear_to, t);
                        if (from_row < valid) {
                            wild = group_any(wg, wild_rows<T, kD>(v_tile, from_row, valid, t));
                            if (wild) add_own_values<T, kD>(o_addr, p_addr, v_tile, limit - key0, bad, first);
                        }
                    }
                }
                if (t == 0) own[wg] = wild;
                tmem_st_wait();
                tmem_fence_before();
                mbar_arrive(&p_ready[wg]);
            }
            if (!ok) break;
            if (!wait_bounded(&o_done[wg], (tiles_done - 1) & 1, err, kDevErrTimeoutEpilogue)) break;
            tmem_fence_after();
            const int row = wg * shape.tile_tokens * shape.group + t;  // of the item
            const bool whole = r.flags & kWhole, final = whole && a.prefix_length == 0;
            const int head = r.head * shape.group + in_group;
            const float norm = sum == 0.0f ? 0.0f : 1.0f / sum;  // a row that sees no key is zero
            const long long part_at_row = (long long)blockIdx.x * 2 + (r.flags & kSecondSlot ? 1 : 0);
            if (!whole && row_ok)
                *reinterpret_cast<float2*>(ws.part_stats[1] + 2 * (part_at_row * kManyRows + row)) = make_float2(ref, sum);
            if (final && shape.wide_out) {
                // 64 columns at a time through the warp's staging block, so that eight
                // lanes write 128 bytes of a row (a lane its own row: 32 half sectors a
                // store, 5500 cycles an item).
                uint8_t* stage = smem + S::kStage + warp * 4096;
                const long long mine = row_ok ? (long long)(r.first + token) * a.ld_out + (long long)head * p.dim : -1;
#pragma unroll 1
                for (int c = 0; c < kD / 64; ++c) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t o[32];
                        tmem_ld_32x32b_x32(o_addr + c * 64 + h * 32, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            uint4 w;
                            const auto two = [&](int e) {
                                return pack_pair<T>(sum == 0.0f ? 0.0f : __uint_as_float(o[8 * k + e]) * norm,
                                                    sum == 0.0f ? 0.0f : __uint_as_float(o[8 * k + e + 1]) * norm);
                            };
                            w = make_uint4(two(0), two(2), two(4), two(6));
                            *reinterpret_cast<uint4*>(stage + lane * 128 + (((h * 4 + k) ^ (lane & 7)) << 4)) = w;
                        }
                    }
                    __syncwarp();
                    const int d = c * 64 + (lane & 7) * 8;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int rr = i * 4 + (lane >> 3);
                        const long long to = __shfl_sync(0xffffffffu, mine, rr);
                        const uint4 w = *reinterpret_cast<const uint4*>(stage + rr * 128 + (((lane & 7) ^ (rr & 7)) << 4));
                        if (to >= 0 && d < p.dim) *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + to + d) = w;
                    }
                    __syncwarp();
                }
            } else {
#pragma unroll 1
                for (int c = 0; c < kD / 32; ++c) {
                    uint32_t o[32];
                    tmem_ld_32x32b_x32(o_addr + c * 32, o);
                    tmem_ld_wait();
                    if (row_ok) {
#pragma unroll
                        for (int k = 0; k < 32; k += 4) {
                            const int d = c * 32 + k;
                            const float v[4] = {__uint_as_float(o[k]), __uint_as_float(o[k + 1]), __uint_as_float(o[k + 2]),
                                                __uint_as_float(o[k + 3])};
                            if (d >= p.dim) continue;
                            if (whole)
                                put_row<T>(a, ws, r.flags & kPrefix, r.first + token, head, d, v, ref, sum);
                            else
                                *reinterpret_cast<float4*>(
                                    ws.part_sums[1] + 4 * ((part_at_row * (kD / 4) + d / 4) * kManyRows + row)) =
                                    make_float4(v[0], v[1], v[2], v[3]);
                        }
                    }
                    __syncwarp();
                }
            }
            tmem_fence_before();  // O has been read before the next weights are announced
        }
    }
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    if (warp == 8)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
}

template <class T, int kD>
cudaError_t launch_many_t(const AttentionArgs& a, const Workspace& ws, int blocks, cudaStream_t stream) {
    const PagedBatch& p = a.batch;
    Shape s{};
    s.group = a.heads / p.kv_heads;
    s.tile_tokens = kTile / s.group;
    s.box = (int)std::gcd((long long)p.page, (long long)kTile);
    // A cache without pages: a view of one that no box asks for.
    const int pages = p.cache_pages > 0 ? p.cache_pages : 1;
    s.cache_end = pages;
    s.wide_out = a.ld_out % 8 == 0 && reinterpret_cast<uintptr_t>(a.out) % 16 == 0;
    uint32_t* err = nullptr;
    if (device_error_word(&err) != ZQ_OK) return cudaErrorUnknown;
    const CUtensorMapDataType type =
        kIsHalf<T> ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    CUtensorMap q, k, v;
    const uint64_t q_dims[3] = {(uint64_t)p.dim, (uint64_t)a.heads, (uint64_t)p.rows};
    const uint64_t q_pitch[2] = {(uint64_t)p.dim * 2, (uint64_t)a.ldq * 2};
    const uint32_t q_box[3] = {64, (uint32_t)s.group, (uint32_t)s.tile_tokens};
    const uint64_t c_dims[4] = {(uint64_t)p.dim, (uint64_t)p.page, (uint64_t)p.kv_heads, (uint64_t)pages};
    const uint32_t c_box[4] = {64, (uint32_t)s.box, 1, 1};
    uint64_t c_pitch[3] = {(uint64_t)p.dim * 2, (uint64_t)p.page * p.dim * 2, (uint64_t)p.ld_k_page * 2};
    if (encode_tiled(&q, type, 3, a.q, q_dims, q_pitch, q_box) != ZQ_OK) return cudaErrorInvalidValue;
    if (encode_tiled(&k, type, 4, p.cache_pages > 0 ? a.k_cache : a.q, c_dims, c_pitch, c_box) != ZQ_OK)
        return cudaErrorInvalidValue;
    c_pitch[2] = (uint64_t)p.ld_v_page * 2;
    if (encode_tiled(&v, type, 4, p.cache_pages > 0 ? a.v_cache : a.q, c_dims, c_pitch, c_box) != ZQ_OK)
        return cudaErrorInvalidValue;
    const auto kern = attend_many_kernel<T, kD>;
    const cudaError_t e = ensure_smem_attr(kern, Smem<kD>::kTotal);
    if (e != cudaSuccess) return e;
    return launch_pdl_kernel(kern, dim3(blocks), dim3(kManyThreads), Smem<kD>::kTotal, stream, q, k, v, a, ws, s, err);
}

}  // namespace

namespace attn {

cudaError_t launch_attend_many(const AttentionArgs& a, int dtype, const Workspace& ws, int blocks, cudaStream_t stream) {
    if (dtype == ZQ_DTYPE_F16)
        return a.batch.dim <= 64 ? launch_many_t<__half, 64>(a, ws, blocks, stream)
                                 : launch_many_t<__half, 128>(a, ws, blocks, stream);
    return a.batch.dim <= 64 ? launch_many_t<__nv_bfloat16, 64>(a, ws, blocks, stream)
                             : launch_many_t<__nv_bfloat16, 128>(a, ws, blocks, stream);
}

}  // namespace attn
}  // namespace zq

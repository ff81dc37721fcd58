// zq_rows.cu -- quantized matmul of 5 to 64 activation rows.
//
// Computes, for every activation row m and output column n,
//   acc[m][n] = sum_k q_a[m][k] * q_w[n][k]         (exact int32)
//   y[m][n]   = float(acc) * s_row[m] * s_col[n] (+ bias[n])
// and what else the epilogue asks for (zq_epilogue.cuh).
//
// The weights are read once: their stream is the floor (22.5 MB of INT4 at
// K = 11008, N = 4096 take 3.4 us).  A block takes 16 or 32 columns and its warps
// split K, so that every load of the call is under way within two rounds or so.
// Weights go from memory to registers (a lane 16 bytes of a column, the four lanes
// of a column 64 next to one another), INT4 codes are spread there, and 16 x 8 x 32
// matrix instructions multiply them: which codes meet in an instruction is free as
// long as rows and columns agree, so a lane's codes are used as they lie.  The
// activation codes (2 KB an eighth of a column tile's step) come from L2.  The warps'
// sums meet in shared memory.  Against the weights through shared memory, unpacked
// there for tcgen05 (zq_skinny_sm100.cu: a ring of three stages waits for copy, unpack
// and product in turn): 12 rows, K = 11008, N = 4096, INT4 9.3 us, was 24.1, INT8
// 11.6, was 23.8; 16 rows, K = 4096, N = 11008 11.0 and 13.5, were 30.6 and 30.0.
// More rows are more tiles of 16 that the same weights are multiplied by; against the
// GEMM, whose few tiles stream the weights through a part of the SMs: 32 rows, K =
// 11008, N = 4096 14.0 and 17.7 us, were 37.2 and 29.2.
// The activations are what bounds wide ones (16 rows, K = 8192, N = 28672, INT4: 3.7
// TB/s of weights and as much of codes again, 31.8 us, was 63.7).  A ring of loads
// in registers that is refilled tile by tile costs registers, so warps, and measured
// slower (12.3 us), as did steps dealt out to the warps one by one (9.6).  Some of the
// shapes below are past their registers: 100 bytes a thread spill for INT4 with 33 to 64
// rows and blocks of 16 columns, 36 for INT8 with up to 16 and blocks of 32.
#include "zq_common.cuh"
#include "zq_epilogue.cuh"
#include "zq_kernels.h"

namespace zq {

namespace {

constexpr int kRowsTile = 16;  // activation rows of an MMA
constexpr int kColTile = 8;    // weight columns of an MMA

__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// kRowTiles: tiles of 16 rows.  kTiles: tiles of 8 columns a block.  kDeep: steps of 64 bytes a column that a warp
// has under way.  kBlocks: blocks an SM is to hold.
template <int kType, int kRowTiles, int kWarps, int kTiles, int kDeep, int kBlocks, bool kX16, bool kEpi>
__global__ void __launch_bounds__(32 * kWarps, kBlocks) rows_kernel(const uint8_t* __restrict__ panel, int N, int Kp,
                                                                    const float* __restrict__ col_scale, const int8_t* q,
                                                                    const float* row_scale,
                                                                    const float* __restrict__ bias, float* __restrict__ y,
                                                                    int M, const Epilogue epi) {
    constexpr int kCols = kTiles * kColTile;
    constexpr int kCodes = kType == kInt8 ? 16 : 32;  // of a lane's 16 bytes of weights
    constexpr int kParts = kCodes / 16;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int col0 = blockIdx.x * kCols;
    const int steps = Kp / (4 * kCodes);
    const size_t col_bytes = (size_t)Kp * 16 / kCodes;
    extern __shared__ int sums[];  // [kWarps][rows][kPitch]
    constexpr int kRows = kRowTiles * kRowsTile, kPitch = kCols + 2;
    const uint8_t* column[kTiles];
#pragma unroll
    for (int i = 0; i < kTiles; ++i) column[i] = panel + (size_t)min(col0 + i * kColTile + g, N - 1) * col_bytes + t * 16;
    uint4 w[kDeep][kTiles];
    const auto load = [&](int at) {
#pragma unroll
        for (int d = 0; d < kDeep; ++d)
#pragma unroll
            for (int i = 0; i < kTiles; ++i)
                if (at + d < steps) w[d][i] = ld_stream_u4(column[i] + (size_t)(at + d) * 64);
    };
    load(warp * kDeep);  // weights depend on no kernel before this one
    pdl_wait_primary();
    pdl_launch_dependents();
    int acc[kRowTiles][kTiles][4] = {};
    const int8_t* row = q + (size_t)g * Kp + t * kCodes;
    // Codes of a step: rows g and g + 8 of each tile.
    const auto load_x = [&](int s, uint4 (&x)[kRowTiles][2][kParts]) {
#pragma unroll
        for (int r = 0; r < 2 * kRowTiles; ++r) {
            const uint4* p = reinterpret_cast<const uint4*>(row + (size_t)(8 * r) * Kp + s * (4 * kCodes));
#pragma unroll
            for (int h = 0; h < kParts; ++h) {
                x[r / 2][r & 1][h] = make_uint4(0, 0, 0, 0);
                if (8 * r + g < M && s < steps) x[r / 2][r & 1][h] = load_l2(p + h);
            }
        }
    };
    // One tile of rows has registers for all its steps' codes at once, more have not.
    constexpr int kAhead = kRowTiles == 1 ? kDeep : 1;
    for (int at = warp * kDeep; at < steps; at += kDeep * kWarps) {
        uint4 x[kAhead][kRowTiles][2][kParts];
        if constexpr (kAhead > 1) {
#pragma unroll
            for (int d = 0; d < kDeep; ++d) load_x(at + d, x[d % kAhead]);
        }
#pragma unroll
        for (int d = 0; d < kDeep; ++d) {
            if (at + d >= steps) break;
            if constexpr (kAhead == 1) load_x(at + d, x[0]);
#pragma unroll
            for (int i = 0; i < kTiles; ++i) {
                uint4 v[2];
                if constexpr (kType == kInt8)
                    v[0] = w[d][i];
                else if (kX16)
                    zq_expand_int4x32_x16(w[d][i], v[0], v[1]);
                else
                    zq_expand_int4x32(w[d][i], v[0], v[1]);
#pragma unroll
                for (int r = 0; r < kRowTiles; ++r)
#pragma unroll
                    for (int h = 0; h < kParts; ++h) {
                        const uint4 &lo = x[d % kAhead][r][0][h], &hi = x[d % kAhead][r][1][h];
                        mma_s8(acc[r][i], lo.x, hi.x, lo.y, hi.y, v[h].x, v[h].y);
                        mma_s8(acc[r][i], lo.z, hi.z, lo.w, hi.w, v[h].z, v[h].w);
                    }
            }
        }
        load(at + kDeep * kWarps);
    }
#pragma unroll
    for (int r = 0; r < kRowTiles; ++r)
#pragma unroll
        for (int i = 0; i < kTiles; ++i) {
            int* to = sums + (warp * kRows + r * kRowsTile + g) * kPitch + i * kColTile + 2 * t;
            *reinterpret_cast<int2*>(to) = make_int2(acc[r][i][0], acc[r][i][1]);
            *reinterpret_cast<int2*>(to + 8 * kPitch) = make_int2(acc[r][i][2], acc[r][i][3]);
        }
    __syncthreads();
    // A thread's outputs, up to four at once, so that their loads are under way together.
    constexpr int kThreads = 32 * kWarps, kOutputs = (kRows * kCols + kThreads - 1) / kThreads;
    constexpr int kEach = kOutputs < 4 ? kOutputs : 4;
    for (int i0 = threadIdx.x; i0 < M * kCols; i0 += kEach * kThreads) {
        float v[kEach], sr[kEach], sc[kEach], b[kEach], res[kEach];
        bool live[kEach];
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int i = i0 + e * kThreads, m = i / kCols, n = col0 + i % kCols;
            live[e] = m < M && n < N;
            sr[e] = live[e] ? load_l2(row_scale + m) : 0.0f;
            sc[e] = live[e] ? __ldg(col_scale + n) : 0.0f;
            b[e] = bias && live[e] ? __ldg(bias + n) : 0.0f;
            res[e] = kEpi && epi.residual && live[e] ? epi_residual(epi, (size_t)m * (size_t)epi.ld_residual + n) : 0.0f;
        }
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int i = i0 + e * kThreads, m = min(i / kCols, kRows - 1), c = i % kCols;
            int sum = 0;
#pragma unroll
            for (int k = 0; k < kWarps; ++k) sum += sums[(k * kRows + m) * kPitch + c];
            if (kX16) sum >>= 4;
            v[e] = bias ? zq_epilogue_bias(sum, sr[e], sc[e], b[e]) : zq_epilogue(sum, sr[e], sc[e]);
        }
        if constexpr (kEpi) {
            epi_activate(epi.activation, v);
            if (epi.residual) {
#pragma unroll
                for (int e = 0; e < kEach; ++e) v[e] += res[e];
            }
        }
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int i = i0 + e * kThreads;
            const size_t at = (size_t)(i / kCols) * N + col0 + i % kCols;
            if (!live[e]) continue;
            if constexpr (kEpi)
                epi_store(epi, y, at, v[e]);
            else
                y[at] = v[e];
        }
    }
}

template <int kType, int kRowTiles, int kWarps, int kTiles, int kDeep, int kBlocks, bool kX16>
cudaError_t launch_t(const GemvArgs& a, cudaStream_t stream) {
    const auto kernel = a.epi.on ? rows_kernel<kType, kRowTiles, kWarps, kTiles, kDeep, kBlocks, kX16, true>
                                 : rows_kernel<kType, kRowTiles, kWarps, kTiles, kDeep, kBlocks, kX16, false>;
    constexpr int cols = kTiles * kColTile, smem = kWarps * kRowTiles * kRowsTile * (cols + 2) * 4;
    const cudaError_t e = ensure_smem_attr(kernel, smem);
    if (e != cudaSuccess) return e;
    return launch_pdl_kernel(kernel, dim3((a.N + cols - 1) / cols), dim3(32 * kWarps), smem, stream, a.panel, a.N, a.Kp,
                             a.col_scale, a.q, a.row_scale, a.bias, a.y, a.M, a.epi);
}

// Blocks of 16 columns while blocks of 32 would leave SMs without a second one, of 32
// above, which read the activations half as often.  16 rows (INT4, K = 4096): N = 4096
// 5.2 us against 6.9, N = 8192 8.9 against 7.8, N = 11008 12.0 against 11.0; INT8 N =
// 6144 9.4 against 9.5, N = 8192 10.7 against 10.3.  The longer the columns of INT8 the
// more a block of 32 waits for its own loads (its warps have one step under way), so up
// to two waves of blocks of 16 go first there (5 rows, calls): K = 8192, N = 8192 19.8
// us against 21.4, K = 32768, N = 4736 33.3 against 61.1 (16 rows 35.1 and 61.9), N =
// 9472 59.4 and 81.0; K = 4096, N = 8192 13.0 and 13.2 (14.4 and 13.8).
// 32 rows: INT4 N = 4096 6.7 against 7.4, N = 11008 16.5 against 15.2.  64 rows go to
// blocks of 32 sooner, from one for two SMs on: N = 1024 (K = 1024) 3.8 against 5.6, N =
// 4096 (K = 4096) 11.7 against 10.4.
bool narrow(int N) { return N < 32 * sm_count(); }
bool narrow16(int type, int N, int Kp) {
    return N <= 32 * sm_count() || (type == kInt8 && Kp > 4096 && N <= 64 * sm_count());
}
template <int kType, bool kX16>
cudaError_t launch_columns(const GemvArgs& a, cudaStream_t stream) {
    if (a.M > 2 * kRowsTile)
        return a.N < 16 * sm_count() ? launch_t<kType, 4, 8, 2, 2, 2, kX16>(a, stream)
                                     : launch_t<kType, 4, 8, 4, 2, 1, kX16>(a, stream);
    if (a.M > kRowsTile)
        return narrow(a.N) ? launch_t<kType, 2, 8, 2, 2, 2, kX16>(a, stream)
                           : launch_t<kType, 2, 8, 4, 2, 2, kX16>(a, stream);
    return narrow16(kType, a.N, a.Kp) ? launch_t<kType, 1, 16, 2, 2, 2, kX16>(a, stream)
                                      : launch_t<kType, 1, 8, 4, 1, 4, kX16>(a, stream);
}

}  // namespace

// Up to 16 rows always.  More rows read more codes a block of columns, so the GEMM's
// tiles win once there are enough of them.  32 rows: INT8 K = 4096, N = 4096 8.7 us
// against the GEMM's 15.3, N = 11008 20.7 against 24.0, K = 8192, N = 28672 71 against
// 55; INT4 6.7 against 18.7, 15.2 against 29.9, 48 against 62.  64 rows: INT8 N = 4096
// 11.9 against 15.4, N = 11008 31 against 24; INT4 10.4 against 18.7, 27 against 30 (one
// rule for both types: INT4 would win up to there by a tenth).
bool rows_kernel_wins(int type, int M, int N) {
    if (M <= kRowsTile) return true;
    if (M <= 2 * kRowsTile) return type == kInt4 || N < 96 * sm_count();
    return M <= 4 * kRowsTile && narrow(N);
}

cudaError_t launch_rows(const GemvArgs& a, cudaStream_t stream) {
    if (a.M < 1 || a.M > 4 * kRowsTile) return cudaErrorInvalidValue;
    if (a.type == kInt8) return launch_columns<kInt8, false>(a, stream);
    return int4_x16_fits(a.Kp) ? launch_columns<kInt4, true>(a, stream) : launch_columns<kInt4, false>(a, stream);
}

}  // namespace zq

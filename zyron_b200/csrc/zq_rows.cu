// zq_rows.cu -- quantized matmul of 5 to 16 activation rows.
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
// The activations are what bounds wide ones (16 rows, K = 8192, N = 28672, INT4: 3.7
// TB/s of weights and as much of codes again, 31.8 us, was 63.7).  A ring of loads
// in registers that is refilled tile by tile costs registers, so warps, and measured
// slower (12.3 us), as did steps dealt out to the warps one by one (9.6).
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

// kTiles: tiles of 8 columns a block.  kDeep: steps of 64 bytes a column that a warp
// has under way.  kBlocks: blocks an SM is to hold.
template <int kType, int kWarps, int kTiles, int kDeep, int kBlocks, bool kX16, bool kEpi>
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
    __shared__ int sums[kWarps][kRowsTile][kCols + 2];
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
    int acc[kTiles][4];
#pragma unroll
    for (int i = 0; i < kTiles; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0;
    const bool low = g < M, high = g + 8 < M;
    const int8_t* row = q + (size_t)g * Kp + t * kCodes;
    for (int at = warp * kDeep; at < steps; at += kDeep * kWarps) {
        uint4 x[kDeep][2][kParts] = {};
#pragma unroll
        for (int d = 0; d < kDeep; ++d)
#pragma unroll
            for (int h = 0; h < kParts; ++h) {
                const int8_t* p = row + (at + d) * (4 * kCodes);
                if (low && at + d < steps) x[d][0][h] = load_l2(reinterpret_cast<const uint4*>(p) + h);
                if (high && at + d < steps) x[d][1][h] = load_l2(reinterpret_cast<const uint4*>(p + (size_t)8 * Kp) + h);
            }
#pragma unroll
        for (int d = 0; d < kDeep; ++d) {
            if (at + d >= steps) break;
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
                for (int h = 0; h < kParts; ++h) {
                    mma_s8(acc[i], x[d][0][h].x, x[d][1][h].x, x[d][0][h].y, x[d][1][h].y, v[h].x, v[h].y);
                    mma_s8(acc[i], x[d][0][h].z, x[d][1][h].z, x[d][0][h].w, x[d][1][h].w, v[h].z, v[h].w);
                }
            }
        }
        load(at + kDeep * kWarps);
    }
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
        const int c = i * kColTile + 2 * t;
        *reinterpret_cast<int2*>(&sums[warp][g][c]) = make_int2(acc[i][0], acc[i][1]);
        *reinterpret_cast<int2*>(&sums[warp][g + 8][c]) = make_int2(acc[i][2], acc[i][3]);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < M * kCols; i += 32 * kWarps) {
        const int m = i / kCols, c = i % kCols, n = col0 + c;
        if (n >= N) continue;
        int sum = 0;
#pragma unroll
        for (int k = 0; k < kWarps; ++k) sum += sums[k][m][c];
        if (kX16) sum >>= 4;
        const float sr = load_l2(row_scale + m), sc = __ldg(col_scale + n);
        const float v = bias ? zq_epilogue_bias(sum, sr, sc, __ldg(bias + n)) : zq_epilogue(sum, sr, sc);
        if constexpr (kEpi)
            epi_finish(epi, y, N, m, n, v);
        else
            y[(size_t)m * N + n] = v;
    }
}

template <int kType, int kWarps, int kTiles, int kDeep, int kBlocks, bool kX16>
cudaError_t launch_t(const GemvArgs& a, cudaStream_t stream) {
    const auto kernel = a.epi.on ? rows_kernel<kType, kWarps, kTiles, kDeep, kBlocks, kX16, true>
                                 : rows_kernel<kType, kWarps, kTiles, kDeep, kBlocks, kX16, false>;
    constexpr int cols = kTiles * kColTile;
    return launch_pdl_kernel(kernel, dim3((a.N + cols - 1) / cols), dim3(32 * kWarps), 0, stream, a.panel, a.N, a.Kp,
                             a.col_scale, a.q, a.row_scale, a.bias, a.y, a.M, a.epi);
}

// Blocks of 16 columns and 16 warps while blocks of 32 would leave SMs without one;
// of 32 columns and 8 warps above, which read the activations half as often (16 rows,
// INT4, K = 4096: N = 4096 5.2 us against 6.9, N = 5120 7.2 against 7.1, N = 8192 8.9
// against 7.8, N = 11008 12.0 against 11.0; K = 8192, N = 28672 42.6 against 31.8;
// INT8 N = 6144 9.4 against 9.5, N = 8192 10.7 against 10.3).
template <int kType, bool kX16>
cudaError_t launch_columns(const GemvArgs& a, cudaStream_t stream) {
    return a.N < 32 * sm_count() ? launch_t<kType, 16, 2, 2, 2, kX16>(a, stream)
                                     : launch_t<kType, 8, 4, 1, 4, kX16>(a, stream);
}

}  // namespace

cudaError_t launch_rows(const GemvArgs& a, cudaStream_t stream) {
    if (a.M < 1 || a.M > kRowsTile) return cudaErrorInvalidValue;
    if (a.type == kInt8) return launch_columns<kInt8, false>(a, stream);
    return int4_x16_fits(a.Kp) ? launch_columns<kInt4, true>(a, stream) : launch_columns<kInt4, false>(a, stream);
}

}  // namespace zq

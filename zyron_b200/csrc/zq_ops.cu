// zq_ops.cu -- C ABI of the operators around the quantized matmul
// (zq_rms_norm_quantize, zq_add_low_rank, zq_token_logprobs): argument checks
// and launches.
#include "zq.h"
#include "zq_internal.h"
#include "zq_kernels.h"

#include <cmath>
#include <cstdio>
#include <limits>

namespace {

constexpr size_t kIntMax = (size_t)std::numeric_limits<int>::max();

// Rows of an adapter call: their 32-bit indices pass the last by up to two
// rounds of the sorting block.
constexpr size_t kMaxRows = kIntMax - 4096;

zq_status invalid(const char* msg) { return zq::set_error(ZQ_ERR_INVALID_ARGUMENT, msg); }

cudaStream_t as_stream(void* s) { return s ? static_cast<cudaStream_t>(s) : cudaStreamPerThread; }

size_t dtype_bytes(int dtype) {
    return dtype == ZQ_DTYPE_F32 ? 4 : dtype == ZQ_DTYPE_F16 || dtype == ZQ_DTYPE_BF16 ? 2 : 0;
}

bool aligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

// Rows of `pitch` elements of `size` bytes whose byte offsets fit in 63 bits.
bool offsets_fit(size_t rows, size_t pitch, size_t size) {
    return pitch <= kIntMax * 64 && (rows == 0 || pitch <= (std::numeric_limits<size_t>::max() >> 1) / size / rows);
}

}  // namespace

extern "C" {

zq_status zq_rms_norm_quantize(const void* x, int dtype, size_t m, size_t k, size_t ldx, const void* residual,
                               size_t ld_residual, const float* weight, double eps, int reciprocal,
                               void* residual_out, size_t ld_residual_out, void* normed, size_t ld_normed, int8_t* q,
                               size_t ldq, float* row_scale, void* stream) {
    const size_t size = dtype_bytes(dtype);
    if (size == 0) return invalid("zyron_b200: unsupported element type");
    if (k == 0) return invalid("zyron_b200: k must be > 0");
    if (!(eps >= 0.0) || !std::isfinite(eps)) return invalid("zyron_b200: eps must be finite and >= 0");
    if ((residual == nullptr) != (residual_out == nullptr))
        return invalid("zyron_b200: residual and residual_out go together");
    if (ldx < k || ldq < k || (residual && (ld_residual < k || ld_residual_out < k)) || (normed && ld_normed < k))
        return invalid("zyron_b200: a row pitch is smaller than k");
    if (m == 0) return ZQ_OK;
    if (!x || !q || !row_scale) return invalid("zyron_b200: null pointer");
    if (m > kIntMax || k > kIntMax - 4096 || ldq > kIntMax)
        return zq::set_error(ZQ_ERR_OVERFLOW, "zyron_b200: dimension exceeds 2^31-1");
    if (!offsets_fit(m, ldx, size) || (residual && (!offsets_fit(m, ld_residual, size) || !offsets_fit(m, ld_residual_out, size))) ||
        (normed && !offsets_fit(m, ld_normed, size)))
        return zq::set_error(ZQ_ERR_OVERFLOW, "zyron_b200: matrix size overflow");
    if (!aligned(x, size) || !aligned(residual, size) || !aligned(residual_out, size) || !aligned(normed, size) ||
        !aligned(weight, 4) || !aligned(row_scale, 4))
        return invalid("zyron_b200: a pointer is not aligned to its element type");
    zq::NormArgs a{};
    a.x = x;
    a.residual = residual;
    a.weight = weight;
    a.residual_out = residual_out;
    a.normed = normed;
    a.q = q;
    a.row_scale = row_scale;
    a.ldx = (long long)ldx;
    a.ld_residual = (long long)ld_residual;
    a.ld_residual_out = (long long)ld_residual_out;
    a.ld_normed = (long long)ld_normed;
    a.ldq = (long long)ldq;
    a.m = (long long)m;
    a.k = (int)k;
    a.eps = eps;
    a.reciprocal = reciprocal != 0;
    const cudaError_t e = zq::launch_rms_norm_quantize(a, dtype, as_stream(stream));
    return e == cudaSuccess ? ZQ_OK : zq::cuda_error(e, "rms_norm_quantize");
}

size_t zq_add_low_rank_workspace_bytes(size_t m, size_t k, size_t n, size_t slots, size_t max_rank) {
    if (m == 0 || m > kMaxRows || k == 0 || k > kIntMax / 2 || n == 0 || n > kIntMax / 2 || slots == 0 ||
        slots > ZQ_LOW_RANK_MAX_SLOTS || max_rank == 0 || max_rank > ZQ_LOW_RANK_MAX)
        return 0;
    zq::LowRankArgs r{};
    r.m = (long long)m;
    r.k = (int)k;
    r.n = (int)n;
    r.slots = (int)slots;
    r.max_rank = (int)max_rank;
    return zq::low_rank_workspace_bytes(r);
}

zq_status zq_add_low_rank(float* y, size_t ldy, const void* x, int x_dtype, size_t ldx, size_t m, size_t k, size_t n,
                          const void* a, const void* b, int w_dtype, size_t slots, size_t max_rank,
                          const int32_t* ids, const float* scales, const int32_t* ranks, void* workspace,
                          size_t workspace_bytes, void* stream) {
    const size_t size = dtype_bytes(x_dtype);
    if (size == 0) return invalid("zyron_b200: unsupported element type");
    if (w_dtype != ZQ_DTYPE_F16 && w_dtype != ZQ_DTYPE_BF16)
        return invalid("zyron_b200: adapter weights must be fp16 or bf16");
    if (k == 0 || n == 0) return invalid("zyron_b200: k and n must be > 0");
    if (slots == 0 || max_rank == 0) return invalid("zyron_b200: slots and max_rank must be > 0");
    if (slots > ZQ_LOW_RANK_MAX_SLOTS || max_rank > ZQ_LOW_RANK_MAX) {
        char buf[128];
        std::snprintf(buf, sizeof buf, "zyron_b200: at most %d adapter slots of rank %d (got %zu of %zu)",
                      ZQ_LOW_RANK_MAX_SLOTS, ZQ_LOW_RANK_MAX, slots, max_rank);
        return invalid(buf);
    }
    if (ldy < n || ldx < k) return invalid("zyron_b200: a row pitch is smaller than its row");
    if (m == 0) return ZQ_OK;
    if (!y || !x || !a || !b || !ids) return invalid("zyron_b200: null pointer");
    if (m > kMaxRows || k > kIntMax / 2 || n > kIntMax / 2)
        return zq::set_error(ZQ_ERR_OVERFLOW, "zyron_b200: dimension too large");
    if (!offsets_fit(m, ldx, size) || !offsets_fit(m, ldy, 4))
        return zq::set_error(ZQ_ERR_OVERFLOW, "zyron_b200: matrix size overflow");
    if (!aligned(y, 4) || !aligned(x, size) || !aligned(a, 2) || !aligned(b, 2) || !aligned(ids, 4) ||
        !aligned(scales, 4) || !aligned(ranks, 4))
        return invalid("zyron_b200: a pointer is not aligned to its element type");
    const size_t need = zq_add_low_rank_workspace_bytes(m, k, n, slots, max_rank);
    if (!workspace || workspace_bytes < need) {
        char buf[128];
        std::snprintf(buf, sizeof buf, "zyron_b200: workspace too small (%zu < %zu bytes)", workspace_bytes, need);
        return invalid(buf);
    }
    if (!aligned(workspace, 256)) return invalid("zyron_b200: workspace must be 256-byte aligned");
    zq::LowRankArgs r{};
    r.y = y;
    r.x = x;
    r.a = a;
    r.b = b;
    r.ids = ids;
    r.scales = scales;
    r.ranks = ranks;
    r.ldy = (long long)ldy;
    r.ldx = (long long)ldx;
    r.m = (long long)m;
    r.k = (int)k;
    r.n = (int)n;
    r.slots = (int)slots;
    r.max_rank = (int)max_rank;
    const cudaError_t e = zq::launch_add_low_rank(r, x_dtype, w_dtype, workspace, as_stream(stream));
    return e == cudaSuccess ? ZQ_OK : zq::cuda_error(e, "add_low_rank");
}

zq_status zq_token_logprobs(const void* logits, int dtype, size_t m, size_t vocab, size_t ld, const int64_t* targets,
                            size_t n_targets, size_t top_k, float* logprobs, float* entropy, float* top_logprobs,
                            int64_t* top_ids, void* stream) {
    const size_t size = dtype_bytes(dtype);
    if (size == 0) return invalid("zyron_b200: unsupported element type");
    if (vocab == 0) return invalid("zyron_b200: vocab must be > 0");
    if (top_k > vocab || top_k > ZQ_LOGPROBS_MAX_TOP) {
        char buf[128];
        std::snprintf(buf, sizeof buf, "zyron_b200: top_k must be at most %d and at most vocab (got %zu)",
                      ZQ_LOGPROBS_MAX_TOP, top_k);
        return invalid(buf);
    }
    if (ld < vocab) return invalid("zyron_b200: a row pitch is smaller than vocab");
    if (m == 0) return ZQ_OK;
    if (!logits || (n_targets && (!targets || !logprobs)) || (top_k && (!top_logprobs || !top_ids)))
        return invalid("zyron_b200: null pointer");
    if (m > kIntMax || vocab > kIntMax - 4096)
        return zq::set_error(ZQ_ERR_OVERFLOW, "zyron_b200: dimension exceeds 2^31-1");
    if (!offsets_fit(m, ld, size) || !offsets_fit(m, n_targets, 8))
        return zq::set_error(ZQ_ERR_OVERFLOW, "zyron_b200: matrix size overflow");
    if (!aligned(logits, size) || !aligned(targets, 8) || !aligned(logprobs, 4) || !aligned(entropy, 4) ||
        !aligned(top_logprobs, 4) || !aligned(top_ids, 8))
        return invalid("zyron_b200: a pointer is not aligned to its element type");
    zq::LogprobArgs r{};
    r.logits = logits;
    r.ld = (long long)ld;
    r.m = (long long)m;
    r.vocab = (int)vocab;
    r.targets = targets;
    r.n_targets = (long long)n_targets;
    r.top_k = (int)top_k;
    r.logprobs = logprobs;
    r.entropy = entropy;
    r.top_logprobs = top_logprobs;
    r.top_ids = top_ids;
    const cudaError_t e = zq::launch_token_logprobs(r, dtype, as_stream(stream));
    return e == cudaSuccess ? ZQ_OK : zq::cuda_error(e, "token_logprobs");
}

}  // extern "C"

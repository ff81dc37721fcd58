"""Operators of a language model's step around the quantized matmul.

* ``rms_norm_quantize``: the root-mean-square norm that adds the residual
  first and leaves the int8 codes and row scales that ``matmul_codes``
  multiplies (``zq_rms_norm_quantize``).
* ``matmul_codes``: ``matmul`` on activations that are codes already
  (``zq_matmul_codes``).
* ``add_low_rank``: the low-rank adapters of many requests added onto a shared
  projection's output (``zq_add_low_rank``); ``QuantizedLinear.forward`` takes
  them as ``adapters``.
* ``token_logprobs``: log probabilities of given tokens, the entropy and the
  most likely alternatives over a head's logits (``zq_token_logprobs``).
* ``append_kv`` and ``paged_attention``: the paged key/value cache of a batch,
  its new tokens rotated and stored, and attention over it with a prefix that
  the requests share (``zq_append_kv``, ``zq_paged_attention``).

All take and return torch CUDA tensors, run on ``stream`` (default: the
device's current stream) without synchronising, allocate their outputs and
workspaces on that stream, and can be captured into CUDA graphs.  They compute
no gradients.  The arithmetic is documented at the C entry points in
include/zq.h.
"""
from __future__ import annotations

import ctypes as C
import typing

from . import _lib
from ._lib import check, lib
from .quantization import QuantizedMatrix, _context

if typing.TYPE_CHECKING:
    from torch import Tensor

torch = None  # the module, from the first call on
_DTYPES = {}  # torch type -> ZQ_DTYPE_*
_MAX_TOP = 32  # ZQ_LOGPROBS_MAX_TOP


def _setup():
    global torch
    import torch as module

    _DTYPES.update({module.float32: 1, module.float16: 2, module.bfloat16: 3})
    torch = module


def _bad(msg):
    return _lib.ZQInvalidArgument("zyron_b200: " + msg)


def _dtype(t, name):
    d = _DTYPES.get(t.dtype)
    if d is None:
        raise _bad(f"{name} must be float32, float16 or bfloat16")
    return d


def _device(first, names, *others):
    """The CUDA device index that all tensors (or None) are on; `names` are
    the others'."""
    index = first.get_device()
    if index < 0:
        raise _bad("tensors must be on a CUDA device")
    for i, t in enumerate(others):
        if t is not None and t.get_device() != index:
            raise _bad(f"{names.split()[i]} is on {t.device}, not on {first.device}")
    return index


def _empty(shape, dtype, device):
    """A new contiguous tensor.  Strides given make the cheapest allocating
    call: at small sizes a call's time is its host time."""
    if len(shape) == 1:
        return torch.empty_strided(shape, (1,), dtype=dtype, device=device)
    if len(shape) == 2:
        return torch.empty_strided(shape, (shape[1] or 1, 1), dtype=dtype, device=device)
    return torch.empty(shape, dtype=dtype, device=device)


def _rows(t, name):
    """`t` as rows: (2-D tensor with contiguous rows, row pitch)."""
    if t.dim() < 1:
        raise _bad(f"{name} rank must be >= 1")
    k = t.shape[-1]
    if t.dim() != 2:
        t = t.reshape(-1, k) if k else t.reshape(0, 0)
    if t.is_contiguous():
        return t, k
    if (t.stride(1) != 1 and k > 1) or (t.shape[0] > 1 and t.stride(0) < k):
        return t.contiguous(), k
    return t, (t.stride(0) if t.shape[0] > 1 else k)


def _out_rows(t, name, shape, dtype):
    """An output given by the caller as rows; never copied."""
    if t.shape != shape or t.dtype != dtype:
        raise _bad(f"{name} must have shape {tuple(shape)} and type {dtype}")
    k = shape[-1]
    if t.is_contiguous():
        return (t if t.dim() == 2 else t.view(-1, k)), k
    if t.dim() != 2:
        raise _bad(f"{name} must be contiguous or rank 2")
    if (k > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < k):
        raise _bad(f"{name} must have contiguous rows that do not overlap")
    return t, (t.stride(0) if t.shape[0] > 1 else k)


def _apart(out, ld_out, t, ld, name, what="residual_out", same=True):
    """Refuses rows `out` that overlap the rows `t`, otherwise than by being
    them where `same` allows that."""
    at, pitch, at_t, pitch_t = out.data_ptr(), ld_out * out.element_size(), t.data_ptr(), ld * t.element_size()
    (m, k), width, width_t = out.shape, out.shape[1] * out.element_size(), t.shape[-1] * t.element_size()
    if m == 0 or same and at == at_t and pitch == pitch_t:
        return
    if at + (m - 1) * pitch + width <= at_t or at_t + (t.shape[0] - 1) * pitch_t + width_t <= at:
        return
    # columns of one wider buffer
    if pitch != pitch_t or not width_t <= (at - at_t) % pitch <= pitch - width:
        raise _bad(f"{what} overlaps {name}")


def _ptr(t):
    return None if t is None else t.data_ptr()


class NormQuantized(typing.NamedTuple):
    """What ``rms_norm_quantize`` returns."""

    codes: Tensor  # int8 [..., k]; rows lie 128-aligned, ready for matmul_codes
    row_scale: Tensor  # fp32 [...]
    residual: Tensor | None  # x + residual
    normed: Tensor | None  # the normed rows in x's type


def rms_norm_quantize(x, weight=None, residual=None, eps=1e-5, residual_out=None, normed=False, reciprocal=False, stream=None):
    """Adds ``residual`` to ``x`` [..., k], norms the rows by their root mean
    square, scales them by ``weight`` (fp32 [k]) and quantizes them as
    ``quantize_rows`` does, bit for bit.

    ``x`` and ``residual`` share a type (float32, float16 or bfloat16); the
    sum is rounded to it, and the norm reads the rounded sum.  The sum goes to
    ``residual_out`` (a new tensor when None; may be ``residual`` or ``x``
    itself, and overlap neither of them otherwise).
    ``normed=True`` also returns the normed rows, e.g. for adapters.
    ``reciprocal=True`` takes the row scale as max|v| times fp32's 1/127, as
    torch computes absmax / 127.0 on a GPU, instead of the quotient: a last bit
    apart in some rows, for codes equal to such a quantizer's."""
    if torch is None:
        _setup()
    dtype = _dtype(x, "x")
    index = _device(x, "weight residual residual_out", weight, residual, residual_out)
    shape = x.shape
    lead, k = shape[:-1], shape[-1] if len(shape) else 0
    if residual is not None:
        if residual.shape != shape or residual.dtype != x.dtype:
            raise _bad("residual must have x's shape and type")
    elif residual_out is not None:
        raise _bad("residual and residual_out go together")
    if weight is not None and (weight.dtype != torch.float32 or weight.shape != (k,) or not weight.is_contiguous()):
        raise _bad("weight must be contiguous float32 of x's last dimension")
    context, ptr = _context(index, stream)
    with context:
        xr, ldx = _rows(x, "x")
        m = xr.shape[0]
        device = x.device
        rr = so = n = None
        ldr = lds = 0
        if residual is not None:
            rr, ldr = _rows(residual, "residual")
            if residual_out is None:
                so = residual_out = _empty(shape, x.dtype, device)
                lds = k
            else:
                so, lds = _out_rows(residual_out, "residual_out", shape, x.dtype)
                _apart(so, lds, xr, ldx, "x")
                _apart(so, lds, rr, ldr, "residual")
                if weight is not None:
                    _apart(so, lds, weight.view(1, k), k, "weight")
        if normed:
            n = _empty(shape, x.dtype, device)
        kp = (k + 127) // 128 * 128
        codes = _empty((m, kp), torch.int8, device)
        scale = _empty(lead, torch.float32, device)
        check(lib().zq_rms_norm_quantize(xr.data_ptr(), dtype, m, k, ldx, _ptr(rr), ldr, _ptr(weight), eps, reciprocal,
                                         _ptr(so), lds, _ptr(n), k, codes.data_ptr(), kp, scale.data_ptr(), ptr))
    if kp != k:
        codes = codes[:, :k]
    if len(shape) != 2:
        codes = codes.unflatten(0, lead) if lead else codes[0]
    return NormQuantized(codes, scale, residual_out, n)


_ACTIVATIONS = {None: 0, "gelu": 1, "silu": 2, "relu": 3}  # ZQ_ACT_*


def _epilogue(shape, index, activation, residual, dtype, out):
    """Checks the epilogue of a matmul with an output of `shape` (a tuple) on
    device `index`; the output's type."""
    if torch is None:
        _setup()
    if activation not in _ACTIVATIONS:
        raise _bad("activation must be None, 'gelu', 'silu' or 'relu'")
    if dtype is None:
        dtype = torch.float32 if residual is None else residual.dtype
    if dtype not in _DTYPES:
        raise _bad("dtype must be float32, float16 or bfloat16")
    if residual is not None:
        if residual.get_device() != index:
            raise _bad(f"residual is on {residual.device}, not on cuda:{index}")
        if residual.shape != shape or residual.dtype != dtype:
            raise _bad(f"residual must have shape {shape} and type {dtype}")
    if out is not None:
        if out.get_device() != index:
            raise _bad(f"out is on {out.device}, not on cuda:{index}")
        if out.shape != shape or out.dtype != dtype or not out.is_contiguous():
            raise _bad(f"out must be contiguous, of shape {shape} and type {dtype}")
    return dtype


def _run_epilogue(weights, x, codes, scale, m, device, bias, shape, activation, residual, dtype, out, ws, ws_bytes, stream):
    """The call that ``_epilogue`` checked, its device and stream current."""
    n, res, ld = shape[-1], None, 0
    if residual is not None:
        if out is None and residual.is_contiguous():
            res, ld = residual.data_ptr(), n
        else:
            rows, ld = _rows(residual, "residual")
            if out is not None:
                _apart(out.view(-1, n), n, rows, ld, "residual", "out")
            residual, res = rows, rows.data_ptr()  # `residual` holds a copy until the call is made
    if out is None:
        out = _empty(shape, dtype, device)
    check(lib().zq_matmul_epilogue(weights.handle, x, codes, scale, m, None if bias is None else bias.data_ptr(),
                                   _ACTIVATIONS[activation], res, ld, out.data_ptr(), _DTYPES[dtype], ws, ws_bytes, stream))
    return out


def matmul_codes(codes, row_scale, weights: QuantizedMatrix, bias=None, out=None, stream=None, activation=None,
                 residual=None, dtype=None):
    """``matmul`` on activations that are quantized already: ``codes`` int8
    [..., K] and ``row_scale`` fp32 [...], as ``rms_norm_quantize`` or
    ``quantize_rows`` leave them.  Codes whose rows are not 128-aligned, as
    those of ``rms_norm_quantize`` are, are copied first.  ``activation``,
    ``residual`` and ``dtype`` are those of ``matmul``."""
    if torch is None:
        _setup()
    if weights is None or weights.empty():
        raise _lib.ZQInvalidArgument("ZYRON quantization: weights are empty")
    k = weights.rows()
    if codes.dim() < 1 or codes.shape[-1] != k:
        raise _lib.ZQInvalidArgument("ZYRON quantization: input/weight dimension mismatch")
    lead = codes.shape[:-1]
    if codes.dtype != torch.int8 or row_scale.dtype != torch.float32 or row_scale.shape != lead:
        raise _bad("codes must be int8 [..., K] and row_scale float32 [...]")
    index = _device(codes, "row_scale bias out", row_scale, bias, out)
    if weights._device != index:
        raise _bad(f"the weights are on cuda:{weights._device}, not on {codes.device}")
    n = weights.cols()
    if bias is not None and (bias.dtype != torch.float32 or bias.shape != (n,) or not bias.is_contiguous()):
        raise _bad("bias must be contiguous float32 of the output's last dimension")
    fused = activation is not None or residual is not None or dtype is not None
    if fused:
        dtype = _epilogue((*lead, n), index, activation, residual, dtype, out)
    elif out is not None and (out.dtype != torch.float32 or tuple(out.shape) != (*lead, n) or not out.is_contiguous()):
        raise _bad("out must be contiguous float32 [..., N]")
    context, ptr = _context(index, stream)
    with context:
        q, pitch = _rows(codes, "codes")
        m = q.shape[0]
        kp = lib().zq_weight_padded_k(weights.handle)
        room = q.untyped_storage().nbytes() - q.storage_offset()
        if m and ((m > 1 and pitch != kp) or q.data_ptr() % 16 or room < m * kp):
            padded = torch.zeros((m, kp), dtype=torch.int8, device=q.device)
            padded[:, :k] = q
            q = padded
        scale = row_scale.contiguous()
        if out is None and not fused:
            out = _empty((*lead, n), torch.float32, q.device)
        need = lib().zq_matmul_workspace_bytes(weights.handle, m)
        ws = _empty((need + 256,), torch.uint8, q.device)
        base = (ws.data_ptr() + 255) & ~255
        if fused:
            return _run_epilogue(weights, None, q.data_ptr(), scale.data_ptr(), m, q.device, bias, (*lead, n), activation,
                                 residual, dtype, out, base, need, ptr)
        check(lib().zq_matmul_codes(weights.handle, q.data_ptr(), scale.data_ptr(), m, _ptr(bias), out.data_ptr(),
                                    base, need, ptr))
    return out


class LowRankAdapters(typing.NamedTuple):
    """A pool of low-rank adapters of one projection [in, out]."""

    a: Tensor  # [slots, max_rank, in], float16 or bfloat16
    b: Tensor  # [slots, out, max_rank], a's type
    scales: Tensor | None = None  # fp32 [slots]; None: ones
    ranks: Tensor | None = None  # int32 [slots]; None: max_rank


def add_low_rank(y, x, a, b, ids, scales=None, ranks=None, stream=None):
    """Adds each row's adapter onto ``y`` in place and returns it:

        y[i] += scales[s] * b[s] @ (a[s] @ x[i]),   s = ids[i]

    ``y`` is fp32 [..., out] (a projection's output), ``x`` [..., in] float32,
    float16 or bfloat16, ``ids`` int32 [...]; ``a``, ``b``, ``scales`` and
    ``ranks`` are the fields of ``LowRankAdapters``.  Rows whose id is not in
    [0, slots) are left as they are; only the first ``ranks[s]`` of an
    adapter's ranks count."""
    return _add_low_rank(_low_rank_call(x, a, b, ids, scales, ranks, stream), y)


def _low_rank_call(x, a, b, ids, scales, ranks, stream):
    """The arguments of an adapter call, checked, but for y, which may not be
    there yet; y's shape comes first."""
    if torch is None:
        _setup()
    xt = _dtype(x, "x")
    wt = _dtype(a, "a")
    index = _device(x, "a b ids scales ranks", a, b, ids, scales, ranks)
    if a.dim() != 3 or b.dim() != 3 or a.dtype != b.dtype:
        raise _bad("a must be [slots, max_rank, in] and b [slots, out, max_rank], of one type")
    slots, max_rank, k = a.shape
    b_slots, n, b_rank = b.shape
    if slots != b_slots or max_rank != b_rank:
        raise _bad("a must be [slots, max_rank, in] and b [slots, out, max_rank], of one type")
    shape = x.shape
    if len(shape) < 1 or shape[-1] != k:
        raise _bad("input/adapter dimension mismatch")
    lead = shape[:-1]
    if not a.is_contiguous() or not b.is_contiguous():
        raise _bad("a and b must be contiguous")
    if ids.dtype != torch.int32 or ids.shape != lead:
        raise _bad("ids must be int32 of x's leading dimensions")
    if scales is not None and (scales.dtype != torch.float32 or scales.shape != (slots,) or not scales.is_contiguous()):
        raise _bad("scales must be contiguous float32 [slots]")
    if ranks is not None and (ranks.dtype != torch.int32 or ranks.shape != (slots,) or not ranks.is_contiguous()):
        raise _bad("ranks must be contiguous int32 [slots]")
    return (*lead, n), x, xt, a, b, wt, ids, scales, ranks, index, _context(index, stream)


def _add_low_rank(call, y):
    shape, x, xt, a, b, wt, ids, scales, ranks, index, (context, ptr) = call
    slots, max_rank, k = a.shape
    n = shape[-1]
    if y.get_device() != index:
        raise _bad(f"y is on {y.device}, not on {x.device}")
    yr, ldy = _out_rows(y, "y", shape, torch.float32)
    with context:
        xr, ldx = _rows(x, "x")
        if not ids.is_contiguous():
            ids = ids.contiguous()
        m = xr.shape[0]
        need = lib().zq_add_low_rank_workspace_bytes(m, k, n, slots, max_rank)
        ws = _empty((need + 256,), torch.uint8, x.device)
        base = (ws.data_ptr() + 255) & ~255
        check(lib().zq_add_low_rank(yr.data_ptr(), ldy, xr.data_ptr(), xt, ldx, m, k, n, a.data_ptr(), b.data_ptr(),
                                    wt, slots, max_rank, ids.data_ptr(), _ptr(scales), _ptr(ranks), base, need, ptr))
    return y


class TokenLogprobs(typing.NamedTuple):
    """What ``token_logprobs`` returns; None where it was not asked for."""

    logprobs: Tensor | None  # fp32, targets' shape
    entropy: Tensor | None  # fp32 [...]
    top_logprobs: Tensor | None  # fp32 [..., top_k]
    top_ids: Tensor | None  # int64 [..., top_k]


def token_logprobs(logits, targets=None, top_k=0, entropy=True, stream=None):
    """Over the rows of ``logits`` [..., vocab] (float32, float16 or
    bfloat16): the log probabilities of ``targets`` (int64, [...] or
    [..., n]), the entropy, and the ``top_k`` most likely tokens, equal logits
    by the lower id.  All in fp32, in nats.

    A negative target asks for nothing and gives 0; one behind the vocabulary
    gives NaN.  -inf logits are tokens that are not allowed; a row that allows
    none has log probabilities of -inf and entropy 0."""
    if torch is None:
        _setup()
    dtype = _dtype(logits, "logits")
    index = _device(logits, "targets", targets)
    shape = logits.shape
    if len(shape) < 1:
        raise _bad("logits rank must be >= 1")
    lead, vocab = shape[:-1], shape[-1]
    n = 0
    if targets is not None:
        if targets.dtype != torch.int64:
            raise _bad("targets must be int64")
        if targets.shape == lead:
            n = 1
        elif targets.dim() == len(shape) and targets.shape[:-1] == lead:
            n = targets.shape[-1]
        else:
            raise _bad("targets must have logits' leading dimensions, and one more at most")
    if top_k < 0:
        raise _bad("top_k must be >= 0")
    if top_k > min(vocab, _MAX_TOP):  # before outputs of that size are allocated
        raise _bad(f"top_k must be at most {_MAX_TOP} and at most vocab (got {top_k})")
    context, ptr = _context(index, stream)
    with context:
        rows, ld = _rows(logits, "logits")
        device = logits.device
        lp = ent = top_lp = top_ids = None
        if targets is not None:
            if not targets.is_contiguous():
                targets = targets.contiguous()
            lp = _empty(targets.shape, torch.float32, device)
        if entropy:
            ent = _empty(lead, torch.float32, device)
        if top_k:
            top_lp = _empty((*lead, top_k), torch.float32, device)
            top_ids = _empty((*lead, top_k), torch.int64, device)
        check(lib().zq_token_logprobs(rows.data_ptr(), dtype, rows.shape[0], vocab, ld, _ptr(targets), n, top_k,
                                      _ptr(lp), _ptr(ent), _ptr(top_lp), _ptr(top_ids), ptr))
    return TokenLogprobs(lp, ent, top_lp, top_ids)


def _heads(t, name, rows, dim, dtype, caches):
    """A [rows, heads, dim] tensor with contiguous heads, beside the caches:
    (tensor, its address, heads, row pitch)."""
    shape = t.shape
    if len(shape) != 3 or shape[0] != rows or shape[2] != dim:
        raise _bad(f"{name} must be [rows, heads, dim] with dim {dim}, and {rows} rows")
    if t.dtype != dtype:
        raise _bad(f"{name} must be {dtype}")
    heads = shape[1]
    ld = width = heads * dim
    if not t.is_contiguous():
        by_row, by_head, by_element = t.stride()
        if by_element != 1 or heads > 1 and by_head != dim or rows > 1 and by_row < width:
            if rows:
                _beside(t.data_ptr(), 1 + (rows - 1) * by_row + (heads - 1) * by_head + (dim - 1) * by_element, t, name, caches)
            t = t.contiguous()
        elif rows > 1:
            ld = by_row
    at = t.data_ptr()
    _beside(at, (rows - 1) * ld + width if rows else 0, t, name, caches)
    return t, at, heads, ld


def _beside(at, elements, t, name, caches):
    """Refuses `elements` of t at `at` that begin before a cache's end and end
    behind its start."""
    end = at + elements * t.element_size()
    for lo, hi in caches:
        if at < hi and lo < end and at < end:
            raise _bad(f"{name} overlaps the caches")


def _paged_batch(rows, k_cache, v_cache, pages, lengths, starts):
    """The checked batch of a call over a paged cache, (kv_heads, page, dim), and
    where the caches begin and end."""
    shape, kind = k_cache.shape, k_cache.dtype
    if len(shape) != 4 or v_cache.shape != shape or v_cache.dtype != kind:
        raise _bad("k_cache and v_cache must be [pages, kv_heads, page, dim], of one shape and type")
    cache_pages, kv_heads, page, dim = shape
    code = _DTYPES.get(kind)
    if code is None or code == 1:
        raise _bad("the cache must be float16 or bfloat16")
    block = kv_heads * page * dim
    k_pitch = v_pitch = block
    if not k_cache.is_contiguous():
        k_pitch = _page_pitch(k_cache, block)
    if not v_cache.is_contiguous():
        v_pitch = _page_pitch(v_cache, block)
    k_at, v_at = k_cache.data_ptr(), v_cache.data_ptr()
    caches = ()
    if cache_pages:
        k_end, v_end = k_at + 2 * ((cache_pages - 1) * k_pitch + block), v_at + 2 * ((cache_pages - 1) * v_pitch + block)
        caches = ((k_at, k_end), (v_at, v_end))
        if k_at < v_end and v_at < k_end:
            # interleaved page by page, or one inside the other
            if k_pitch != v_pitch or not block <= (v_at - k_at) // 2 % k_pitch <= k_pitch - block:
                raise _bad("k_cache and v_cache overlap")
    of_pages, of_lengths = pages.shape, lengths.shape
    if len(of_pages) != 2 or pages.dtype != torch.int32 or lengths.dtype != torch.int32 or len(of_lengths) != 1:
        raise _bad("pages must be int32 [requests, max_pages] and lengths int32 [requests]")
    requests, max_pages = of_pages
    if of_lengths[0] != requests or not lengths.is_contiguous():
        raise _bad("lengths must be contiguous int32 [requests], as many as rows of pages")
    ld_pages = max_pages
    if not pages.is_contiguous():
        by_row, by_page = pages.stride()
        if max_pages > 1 and by_page != 1 or requests > 1 and by_row < max_pages:
            raise _bad("pages must have contiguous rows that do not overlap")
        if requests > 1:
            ld_pages = by_row
    start = None
    if starts is None:
        if requests != rows:
            raise _bad(f"without starts every request has one row: {requests} requests, {rows} rows")
    elif starts.dtype != torch.int32 or starts.shape != (requests + 1,) or not starts.is_contiguous():
        raise _bad("starts must be contiguous int32 [requests + 1]")
    else:
        start = starts.data_ptr()
    batch = _lib.PagedBatchC(start, lengths.data_ptr(), pages.data_ptr(), ld_pages, max_pages, requests, rows, page,
                             cache_pages, kv_heads, dim, k_pitch, v_pitch, code)
    return C.byref(batch), (kv_heads, page, dim), caches, k_at, v_at


def _page_pitch(t, block):
    """Elements from page to page of a cache that is not contiguous as a whole."""
    pages, kv_heads, page, dim = t.shape
    by_page, by_head, by_token, by_element = t.stride()
    if by_element != 1 or by_token != dim or kv_heads > 1 and by_head != page * dim or pages > 1 and by_page < block:
        raise _bad("each page's [kv_heads, page, dim] must be contiguous in the caches")
    return by_page if pages > 1 else block


def append_kv(q, k, v, k_cache, v_cache, pages, lengths, starts=None, inv_freq=None, interleaved=True, offset=0,
              stream=None):
    """Stores new tokens' keys and values in a paged cache and rotates queries
    and keys by position on the way; returns the rotated queries in the cache's
    type (``None`` where ``q`` is).

    ``q`` [rows, heads, dim], ``k`` and ``v`` [rows, kv_heads, dim] share a type
    (float32, float16 or bfloat16) and may be columns of one projection's
    output; the caches are float16 or bfloat16 [pages, kv_heads, page, dim].
    The rows are the requests' new tokens one request after the other, request
    b's from ``starts[b]`` to ``starts[b + 1]`` (None: one row each);
    ``lengths[b]`` counts its cached tokens, the new ones included, and
    ``pages[b]`` (int32 [requests, max_pages]) names the pages that hold them.
    All three are read on the device when the call runs.

    ``inv_freq`` (float64 [rotated / 2], None: no rotation) holds the angle of
    each pair per position, ``interleaved`` says whether pairs are neighbours
    or half a rotation apart, and ``offset`` is the position of a request's
    first own token, such as a shared prefix's length.  Tokens whose page is
    outside the cache are not stored; rows that no request owns are neither
    stored nor written in the result."""
    if torch is None:
        _setup()
    kind = k.dtype
    dtype = _dtype(k, "k")
    index = _device(k, "q v k_cache v_cache pages lengths starts inv_freq", q, v, k_cache, v_cache, pages, lengths, starts,
                    inv_freq)
    shape = k.shape
    if len(shape) != 3 or v.shape != shape or v.dtype != kind:
        raise _bad("k and v must be [rows, kv_heads, dim], of one shape and type")
    rows = shape[0]
    batch, (kv_heads, _, dim), caches, k_at, v_at = _paged_batch(rows, k_cache, v_cache, pages, lengths, starts)
    if shape[1] != kv_heads:
        raise _bad("k and v must have the caches' kv_heads")
    rotated, freq = 0, None
    if inv_freq is not None:
        if inv_freq.dtype != torch.float64 or inv_freq.dim() != 1 or not inv_freq.is_contiguous():
            raise _bad("inv_freq must be contiguous float64 [rotated / 2]")
        rotated = 2 * inv_freq.shape[0]
        if rotated:
            freq = inv_freq.data_ptr()
    if not 0 <= offset <= 1 << 40:
        raise _bad("offset must be in [0, 2^40]")
    context, ptr = _context(index, stream)
    with context:
        k, at_k, _, ldk = _heads(k, "k", rows, dim, kind, caches)
        v, at_v, _, ldv = _heads(v, "v", rows, dim, kind, caches)
        out, at_q, at_out, heads, ldq = None, None, None, 0, 0
        if q is not None:
            q, at_q, heads, ldq = _heads(q, "q", rows, dim, kind, caches)
            out = torch.empty_strided((rows, heads, dim), (heads * dim, dim, 1), dtype=k_cache.dtype, device=k.device)
            at_out = out.data_ptr()
        check(lib().zq_append_kv(batch, at_q, ldq, at_k, ldk, at_v, ldv, dtype, heads, k_at, v_at, at_out, freq, rotated,
                                 interleaved, offset, ptr))
    return out


def paged_attention(q, k_cache, v_cache, pages, lengths, starts=None, prefix_pages=None, prefix_length=0, causal=True,
                    scale=None, out=None, stream=None):
    """Attention of new tokens ``q`` [rows, heads, dim] (the cache's type) over
    a paged cache, as ``append_kv`` leaves it and with its ``pages``,
    ``lengths`` and ``starts``; returns [rows, heads, dim].

    Every row sees the ``prefix_length`` tokens of a prefix that all requests
    share (on ``prefix_pages``, int32), which is computed once for all of them,
    and its request's own tokens, with ``causal`` those up to its own
    position.  ``scale`` is 1 / sqrt(dim) by default.  A row that sees no token,
    or whose scores are all -inf, is zero; rows that no request owns are left as
    ``out`` has them.  Requests (or a prefix) of more than 32 rows of a kv head
    multiply the values by weights rounded to the cache's type."""
    if torch is None:
        _setup()
    index = _device(q, "k_cache v_cache pages lengths starts prefix_pages out", k_cache, v_cache, pages, lengths, starts,
                    prefix_pages, out)
    shape = q.shape
    if len(shape) != 3:
        raise _bad("q must be [rows, heads, dim]")
    rows, heads, _ = shape
    kind = k_cache.dtype
    batch, (kv_heads, page, dim), caches, k_at, v_at = _paged_batch(rows, k_cache, v_cache, pages, lengths, starts)
    if prefix_length < 0:
        raise _bad("prefix_length must be >= 0")
    prefix = None
    if prefix_length:
        if prefix_pages is None or prefix_pages.dtype != torch.int32 or prefix_pages.dim() != 1 or \
                not prefix_pages.is_contiguous() or prefix_pages.shape[0] * page < prefix_length:
            raise _bad("prefix_pages must be contiguous int32 and hold prefix_length tokens")
        prefix = prefix_pages.data_ptr()
    if scale is None:
        scale = dim**-0.5 if dim else 1.0
    if heads == 0 or kv_heads and heads % kv_heads:  # no kv heads: refused by the call itself
        raise _bad("heads must be a multiple of kv_heads")
    context, ptr = _context(index, stream)
    with context:
        q, at_q, _, ldq = _heads(q, "q", rows, dim, kind, ())
        device, width = q.device, heads * dim
        if at_q % 16 or ldq % 8:
            q, ldq = torch.empty((rows, heads, dim), dtype=kind, device=device).copy_(q), width
            at_q = q.data_ptr()
        ld_out = width
        if out is None:
            out = torch.empty_strided((rows, heads, dim), (width, dim, 1), dtype=kind, device=device)
            at_out = out.data_ptr()
        else:
            if out.shape != shape or out.dtype != kind:
                raise _bad(f"out must have shape {tuple(shape)} and type {kind}")
            by_row, by_head, by_element = out.stride()
            if by_element != 1 or (heads > 1 and by_head != dim) or (rows > 1 and by_row < width):
                raise _bad("out must have contiguous rows that do not overlap")
            if rows > 1:
                ld_out = by_row
            at_out = out.data_ptr()
            if rows:
                _beside(at_out, (rows - 1) * ld_out + width, out, "out", caches)
                _apart(out.flatten(1), ld_out, q.flatten(1), ldq, "q", "out", same=False)
        need = lib().zq_paged_attention_workspace_bytes(batch, heads, prefix_length)
        ws = torch.empty_strided((need + 256,), (1,), dtype=torch.uint8, device=device)
        base = (ws.data_ptr() + 255) & ~255
        check(lib().zq_paged_attention(batch, at_q, ldq, heads, k_at, v_at, prefix, prefix_length, causal, scale, at_out,
                                       ld_out, base, need, ptr))
    return out

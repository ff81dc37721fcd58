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

All take and return torch CUDA tensors, run on ``stream`` (default: the
device's current stream) without synchronising, allocate their outputs and
workspaces on that stream, and can be captured into CUDA graphs.  They compute
no gradients.  The arithmetic is documented at the C entry points in
include/zq.h.
"""
from __future__ import annotations

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


def _apart(out, ld_out, t, ld, name):
    """Refuses rows `out` that overlap the rows `t` otherwise than by being them."""
    at, pitch, at_t, pitch_t = out.data_ptr(), ld_out * out.element_size(), t.data_ptr(), ld * t.element_size()
    (m, k), width, width_t = out.shape, out.shape[1] * out.element_size(), t.shape[-1] * t.element_size()
    if m == 0 or at == at_t and pitch == pitch_t:
        return
    if at + (m - 1) * pitch + width <= at_t or at_t + (t.shape[0] - 1) * pitch_t + width_t <= at:
        return
    # columns of one wider buffer
    if pitch != pitch_t or not width_t <= (at - at_t) % pitch <= pitch - width:
        raise _bad(f"residual_out overlaps {name}")


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


def matmul_codes(codes, row_scale, weights: QuantizedMatrix, bias=None, out=None, stream=None):
    """``matmul`` on activations that are quantized already: ``codes`` int8
    [..., K] and ``row_scale`` fp32 [...], as ``rms_norm_quantize`` or
    ``quantize_rows`` leave them.  Codes whose rows are not 128-aligned, as
    those of ``rms_norm_quantize`` are, are copied first."""
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
    if out is not None and (out.dtype != torch.float32 or tuple(out.shape) != (*lead, n) or not out.is_contiguous()):
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
        if out is None:
            out = _empty((*lead, n), torch.float32, q.device)
        need = lib().zq_matmul_workspace_bytes(weights.handle, m)
        ws = _empty((need + 256,), torch.uint8, q.device)
        base = (ws.data_ptr() + 255) & ~255
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

"""The operators around the matmul without a GPU: every refusal of their
entry points happens on the host, before any device work."""
import ctypes as C
import math

import pytest

from zyron_b200 import _lib

P = C.c_void_p(1 << 20)  # never read: every call below is refused or has no rows
BIG = 1 << 40


def refused(rc, message, status=_lib.ZQ_ERR_INVALID_ARGUMENT):
    assert (rc, _lib.lib().zq_last_error().decode()) == (status, "zyron_b200: " + message)


def norm(L, x=P, dtype=1, m=4, k=64, ldx=64, residual=None, ldr=0, weight=P, eps=1e-5, out=None, ldo=0, normed=None,
         ldn=0, q=P, ldq=128, scale=P):
    return L.zq_rms_norm_quantize(x, dtype, m, k, ldx, residual, ldr, weight, eps, 0, out, ldo, normed, ldn, q, ldq,
                                  scale, None)


def test_norm_refusals(native_lib):
    L = native_lib
    assert norm(L, m=0) == _lib.ZQ_OK
    refused(norm(L, dtype=0), "unsupported element type")
    refused(norm(L, dtype=4), "unsupported element type")
    refused(norm(L, k=0), "k must be > 0")
    for eps in (-1e-9, math.nan, math.inf):
        refused(norm(L, eps=eps), "eps must be finite and >= 0")
    refused(norm(L, residual=P, ldr=64), "residual and residual_out go together")
    refused(norm(L, out=P, ldo=64), "residual and residual_out go together")
    for bad in ({"ldx": 63}, {"ldq": 63}, {"residual": P, "ldr": 63, "out": P, "ldo": 64},
                {"residual": P, "ldr": 64, "out": P, "ldo": 63}, {"normed": P, "ldn": 63}):
        refused(norm(L, **bad), "a row pitch is smaller than k")
    for bad in ("x", "q", "scale"):
        refused(norm(L, **{bad: None}), "null pointer")
    refused(norm(L, m=1 << 31), "dimension exceeds 2^31-1", _lib.ZQ_ERR_OVERFLOW)
    refused(norm(L, ldx=BIG), "matrix size overflow", _lib.ZQ_ERR_OVERFLOW)
    refused(norm(L, x=C.c_void_p(2)), "a pointer is not aligned to its element type")
    refused(norm(L, dtype=3, x=C.c_void_p(1)), "a pointer is not aligned to its element type")


def adapters(L, y=P, ldy=32, x=P, dtype=1, ldx=64, m=4, k=64, n=32, a=P, b=P, wtype=3, slots=2, rank=8, ids=P,
             scales=None, ranks=None, ws=None, ws_bytes=0):
    return L.zq_add_low_rank(y, ldy, x, dtype, ldx, m, k, n, a, b, wtype, slots, rank, ids, scales, ranks, ws, ws_bytes,
                             None)


def test_adapter_refusals(native_lib):
    L = native_lib
    assert adapters(L, m=0) == _lib.ZQ_OK
    refused(adapters(L, dtype=7), "unsupported element type")
    for t in (0, 1, 4):
        refused(adapters(L, wtype=t), "adapter weights must be fp16 or bf16")
    refused(adapters(L, k=0), "k and n must be > 0")
    refused(adapters(L, n=0, ldy=0), "k and n must be > 0")
    refused(adapters(L, slots=0), "slots and max_rank must be > 0")
    refused(adapters(L, rank=0), "slots and max_rank must be > 0")
    refused(adapters(L, rank=257), "at most 8192 adapter slots of rank 256 (got 2 of 257)")
    refused(adapters(L, slots=8193), "at most 8192 adapter slots of rank 256 (got 8193 of 8)")
    refused(adapters(L, ldy=31), "a row pitch is smaller than its row")
    refused(adapters(L, ldx=63), "a row pitch is smaller than its row")
    for bad in ("y", "x", "a", "b", "ids"):
        refused(adapters(L, **{bad: None}), "null pointer")
    refused(adapters(L, n=1 << 31, ldy=1 << 31), "dimension too large", _lib.ZQ_ERR_OVERFLOW)
    refused(adapters(L, m=(1 << 31) - 4096), "dimension too large", _lib.ZQ_ERR_OVERFLOW)
    refused(adapters(L, ldx=BIG), "matrix size overflow", _lib.ZQ_ERR_OVERFLOW)
    refused(adapters(L, y=C.c_void_p(2)), "a pointer is not aligned to its element type")
    need = L.zq_add_low_rank_workspace_bytes(5000, 64, 32, 2, 8)
    assert need > 5000 * 4 and need % 256 == 0
    assert L.zq_add_low_rank_workspace_bytes(1, 4096, 4096, 8, 16) > 0
    for none in ((0, 64, 32, 2, 8), (5, 0, 32, 2, 8), (5, 64, 0, 2, 8), (5, 64, 32, 0, 8), (5, 64, 32, 2, 0),
                 (5, 64, 32, 8193, 8), (5, 64, 32, 2, 257), (1 << 31, 64, 32, 2, 8)):
        assert L.zq_add_low_rank_workspace_bytes(*none) == 0
    refused(adapters(L, m=5000), f"workspace too small (0 < {need} bytes)")
    refused(adapters(L, m=5000, ws=P, ws_bytes=need - 1), f"workspace too small ({need - 1} < {need} bytes)")
    refused(adapters(L, m=5000, ws=C.c_void_p((1 << 20) + 64), ws_bytes=need), "workspace must be 256-byte aligned")


def logprobs(L, x=P, dtype=1, m=4, vocab=100, ld=100, targets=P, n=1, top=0, lp=P, ent=None, top_lp=None, top_ids=None):
    return L.zq_token_logprobs(x, dtype, m, vocab, ld, targets, n, top, lp, ent, top_lp, top_ids, None)


def test_logprob_refusals(native_lib):
    L = native_lib
    assert logprobs(L, m=0) == _lib.ZQ_OK
    refused(logprobs(L, dtype=-1), "unsupported element type")
    refused(logprobs(L, vocab=0), "vocab must be > 0")
    refused(logprobs(L, top=33), "top_k must be at most 32 and at most vocab (got 33)")
    refused(logprobs(L, vocab=5, top=6), "top_k must be at most 32 and at most vocab (got 6)")
    refused(logprobs(L, ld=99), "a row pitch is smaller than vocab")
    for bad in ({"x": None}, {"targets": None}, {"lp": None}, {"top": 2, "top_lp": P}, {"top": 2, "top_ids": P}):
        refused(logprobs(L, **bad), "null pointer")
    refused(logprobs(L, m=1 << 31), "dimension exceeds 2^31-1", _lib.ZQ_ERR_OVERFLOW)
    refused(logprobs(L, targets=C.c_void_p((1 << 20) + 4)), "a pointer is not aligned to its element type")


def test_python_refusals(native_lib):
    """The checks that come before the device is asked for anything."""
    import torch

    import zyron_b200 as zb

    x = torch.zeros(2, 8)
    with pytest.raises(ValueError, match="tensors must be on a CUDA device"):
        zb.rms_norm_quantize(x)
    with pytest.raises(ValueError, match="x must be float32, float16 or bfloat16"):
        zb.rms_norm_quantize(x.double())
    with pytest.raises(ValueError, match="tensors must be on a CUDA device"):
        zb.add_low_rank(x, x, x.bfloat16(), x.bfloat16(), x)
    with pytest.raises(ValueError, match="tensors must be on a CUDA device"):
        zb.token_logprobs(x)
    with pytest.raises(ValueError, match="input must be on a CUDA device"):
        zb.quantize_rows(x)
    with pytest.raises(ValueError, match="weights are empty"):
        zb.matmul_codes(x, x, zb.QuantizedMatrix())

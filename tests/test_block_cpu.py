"""The matmul's epilogue, append_kv and paged_attention without a GPU: every
refusal of their entry points happens on the host, before any device work."""
import ctypes as C
import math

import pytest

from zyron_b200 import _lib

P = C.c_void_p(1 << 20)  # never read: every call below is refused or has no rows
BIG = 1 << 40


def refused(rc, message, status=_lib.ZQ_ERR_INVALID_ARGUMENT):
    assert (rc, _lib.lib().zq_last_error().decode()) == (status, "zyron_b200: " + message)


def batch(starts=None, lengths=P, pages=P, ld_pages=4, max_pages=4, requests=2, rows=2, page=16, cache_pages=9, kv=2, dim=64,
          k_page=2048, v_page=2048, cache=3):
    return C.byref(_lib.PagedBatchC(starts, lengths, pages, ld_pages, max_pages, requests, rows, page, cache_pages, kv, dim,
                                    k_page, v_page, cache))


def append(L, b=None, q=P, ldq=256, k=P, ldk=128, v=P, ldv=128, dtype=3, heads=4, kc=P, vc=P, out=P, inv=None, rotated=0,
           interleaved=1, offset=0, **of_batch):
    return L.zq_append_kv(batch(**of_batch) if b is None else b, q, ldq, k, ldk, v, ldv, dtype, heads, kc, vc, out, inv,
                          rotated, interleaved, offset, None)


def attention(L, q=P, ldq=256, heads=4, kc=P, vc=P, prefix=None, n_prefix=0, scale=0.1, out=C.c_void_p(1 << 24), ldo=256,
              ws=None, ws_bytes=0, **of_batch):
    return L.zq_paged_attention(batch(**of_batch), q, ldq, heads, kc, vc, prefix, n_prefix, 1, scale, out, ldo, ws, ws_bytes,
                                None)


BATCHES = [({"cache": 1}, "the cache must be fp16 or bf16"), ({"dim": 0}, "dim must be a multiple of 8 and at most 128"),
           ({"dim": 60}, "dim must be a multiple of 8 and at most 128"),
           ({"dim": 136}, "dim must be a multiple of 8 and at most 128"),
           ({"page": 0}, "page must be a multiple of 8 and at most 2^20"),
           ({"page": 12}, "page must be a multiple of 8 and at most 2^20"),
           ({"page": (1 << 20) + 8}, "page must be a multiple of 8 and at most 2^20"),
           ({"kv": 0}, "kv_heads must be in [1, 65535]"), ({"ld_pages": 3}, "a row pitch is smaller than its row"),
           ({"requests": 3}, "without starts every request has one row"),
           ({"k_page": 2047}, "a page pitch is smaller than its page"), ({"v_page": 2047}, "a page pitch is smaller than its page")]


@pytest.mark.parametrize("call", [append, attention])
def test_batch_refusals(native_lib, call):
    L = native_lib
    for bad, message in BATCHES:
        refused(call(L, **bad), message)
    for bad in ({"rows": 1 << 31, "requests": 1 << 31}, {"starts": P, "requests": 1 << 31}, {"max_pages": 1 << 31, "ld_pages": 1 << 31},
                {"cache_pages": 1 << 31}):
        refused(call(L, **bad), "dimension too large", _lib.ZQ_ERR_OVERFLOW)
    for bad in ({"k_page": BIG}, {"v_page": BIG}):
        refused(call(L, **bad), "matrix size overflow", _lib.ZQ_ERR_OVERFLOW)
    for bad in ("lengths", "pages", "kc", "vc", "q"):
        refused(call(L, **{bad: None}), "q and q_out go together" if bad == "q" and call is append else "null pointer")
    refused(call(L, starts=C.c_void_p(2)), "a pointer is not aligned to its element type")
    for heads in (0, 3):
        refused(call(L, heads=heads, ldq=1 << 20), "heads must be a multiple of kv_heads")
    refused(call(L, heads=258, ldq=1 << 20), "at most 128 query heads a kv head")
    refused(call(L, ldq=255), "a row pitch is smaller than its row")
    refused(call(L, ldq=BIG), "matrix size overflow", _lib.ZQ_ERR_OVERFLOW)
    assert call(L, rows=0, requests=0) == _lib.ZQ_OK
    assert call(L, rows=5, requests=0, starts=P) == _lib.ZQ_OK
    assert call(L, rows=0, starts=P) == _lib.ZQ_OK


def test_append_refusals(native_lib):
    L = native_lib
    refused(L.zq_append_kv(None, P, 256, P, 128, P, 128, 3, 4, P, P, P, None, 0, 1, 0, None), "null pointer")
    refused(append(L, dtype=0), "unsupported element type")
    refused(append(L, out=None), "q and q_out go together")
    for rotated in (3, 66):
        refused(append(L, inv=P, rotated=rotated), "rotated must be even and at most dim")
    refused(append(L, inv=P), "rotated and inv_freq go together")
    refused(append(L, rotated=8), "rotated and inv_freq go together")
    for offset in (-1, BIG + 1):
        refused(append(L, offset=offset), "offset must be in [0, 2^40]")
    for bad in ({"ldk": 127}, {"ldv": 127}):
        refused(append(L, b=batch(), **bad), "a row pitch is smaller than its row")
    for bad in ("k", "v"):
        refused(append(L, **{bad: None}), "null pointer")
    for bad in ({"k": C.c_void_p(1)}, {"q": C.c_void_p(1)}, {"inv": C.c_void_p(4), "rotated": 8}, {"kc": C.c_void_p(1)}):
        refused(append(L, **bad), "a pointer is not aligned to its element type")
    assert append(L, q=None, out=None, heads=0, rows=0, requests=0) == _lib.ZQ_OK


def test_attention_refusals(native_lib):
    L = native_lib
    for scale in (math.inf, math.nan):
        refused(attention(L, scale=scale), "scale must be finite")
    refused(attention(L, ldo=255), "a row pitch is smaller than its row")
    refused(attention(L, ldq=260), "ldq must be a multiple of 8, ld_out of 4")
    refused(attention(L, ldo=258), "ldq must be a multiple of 8, ld_out of 4")
    refused(attention(L, k_page=2052), "page pitches must be multiples of 8")
    refused(attention(L, n_prefix=1 << 31, prefix=P), "dimension too large", _lib.ZQ_ERR_OVERFLOW)
    refused(attention(L, n_prefix=1), "null pointer")
    refused(attention(L, out=None), "null pointer")
    for bad in ({"q": C.c_void_p(8)}, {"kc": C.c_void_p(8)}, {"out": C.c_void_p(4)}, {"prefix": C.c_void_p(2), "n_prefix": 1}):
        refused(attention(L, **bad), "q and the caches must be 16-byte aligned, out 8-byte")
    need = L.zq_paged_attention_workspace_bytes(batch(), 4, 0)
    assert need > 0 and need % 256 == 0
    assert L.zq_paged_attention_workspace_bytes(batch(), 4, 100) > need
    for bad in (batch(dim=12), batch(page=0)):
        assert L.zq_paged_attention_workspace_bytes(bad, 4, 0) == 0
    assert L.zq_paged_attention_workspace_bytes(batch(), 3, 0) == 0
    assert L.zq_paged_attention_workspace_bytes(batch(), 4, 1 << 31) == 0
    refused(attention(L), f"workspace too small (0 < {need} bytes)")
    refused(attention(L, ws=P, ws_bytes=need - 1), f"workspace too small ({need - 1} < {need} bytes)")
    refused(attention(L, ws=C.c_void_p((1 << 20) + 128), ws_bytes=need), "workspace must be 256-byte aligned")


def test_epilogue_refusals(native_lib):
    """No weight exists without a GPU; what needs none is checked here."""
    L = native_lib
    rc = L.zq_matmul_epilogue(None, P, None, None, 4, None, 1, None, 0, P, 1, None, 0, None)
    assert (rc, L.zq_last_error().decode()) == (_lib.ZQ_ERR_INVALID_ARGUMENT, "ZYRON quantization: weights are empty")

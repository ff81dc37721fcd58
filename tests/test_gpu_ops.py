"""The operators around the matmul against plain implementations in 64 bits:
rms_norm_quantize (bit for bit), add_low_rank and token_logprobs (within
bounds counted from their roundings), and a step that runs them together."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

DTYPES = ["float32", "float16", "bfloat16"]


@pytest.fixture(scope="module")
def zb(cuda):
    import zyron_b200

    return zyron_b200


@pytest.fixture(scope="module")
def torch(cuda):
    import torch

    return torch


def randn(torch, seed, *shape):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g)


def same_bits(torch, got, want, what):
    """Equal values, NaN equal to NaN."""
    got, want = got.cpu(), want.cpu()
    assert got.shape == want.shape and got.dtype == want.dtype, (what, got.shape, want.shape, got.dtype, want.dtype)
    if got.is_floating_point():
        bad = ~((got == want) | (got.isnan() & want.isnan()))
    else:
        bad = got != want
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} differ, first at {bad.nonzero()[0].tolist()}"


# ---- norm -----------------------------------------------------------------------

def norm_oracle(torch, x, residual, weight, eps, reciprocal=False):
    """The definition on the CPU.  Squares of fp32 values are exact in 64
    bits; the sum's rounding there cannot move the fp32 reciprocal root except
    within 1e-15 of a rounding border."""
    s = x.float()
    total = None
    if residual is not None:
        total = (s + residual.float()).to(x.dtype)
        s = total.float()
    mean = s.double().square().sum(-1, keepdim=True) / s.shape[-1]
    r = (1.0 / torch.sqrt(mean + eps)).float()
    v = s * r * (1.0 if weight is None else weight)
    absmax = torch.nan_to_num(v.abs(), nan=0.0, posinf=math.inf).amax(-1, keepdim=True)
    quotient = absmax * torch.tensor(1.0 / 127.0) if reciprocal else absmax / torch.tensor(127.0)
    scale = torch.where(absmax > 0, quotient, torch.ones_like(absmax))
    q = v / scale
    codes = torch.sign(q) * torch.floor(q.double().abs() + 0.5)
    codes = torch.where(q.isnan(), -127.0, codes.clamp(-127, 127))
    codes = torch.where(torch.isinf(scale), 0.0, codes)
    return codes.to(torch.int8), scale[..., 0], total, v.to(x.dtype)


def norm_case(torch, m, k, dtype, residual, pitch=0, seed=0):
    x = randn(torch, 7 * m + k + seed, m, k + pitch).to(getattr(torch, dtype))[:, :k]
    r = (randn(torch, 11 * m + k + seed, m, k + pitch) * 3).to(x.dtype)[:, :k] if residual else None
    w = 1 + 0.2 * randn(torch, k, k)
    if m > 1:
        x[1] = 0
        if residual:
            r[1] = 0
    if k > 5:
        w[5] = 0.0
        x[-1, 3] = 40.0
    return x, r, w


NORM_SIZES = [(1, 1), (1, 4096), (2, 7), (3, 31), (5, 32), (9, 33), (8, 256), (7, 257), (17, 768), (3, 1000),
              (2, 1024), (3, 1025), (4, 2048), (5, 2050), (2, 4099), (3, 8192), (2, 8200), (2, 16384), (1, 20001),
              (2, 32768), (2, 32776), (1, 65537), (300, 64)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k", NORM_SIZES)
def test_norm_bits(zb, torch, m, k, dtype):
    for residual, pitch, normed in ((True, 0, True), (False, 0, False), (True, 8, False), (False, 3, True), (True, 5, True)):
        x, r, w = norm_case(torch, m, k, dtype, residual, pitch)
        codes, scale, total, v = norm_oracle(torch, x, r, w, 1e-5)
        dev = lambda t: None if t is None else torch.empty(t.shape[0], k + pitch, dtype=t.dtype, device="cuda")[:, :k].copy_(t)  # noqa: E731
        got = zb.rms_norm_quantize(dev(x), w.cuda(), residual=dev(r), eps=1e-5, normed=normed)
        same_bits(torch, got.row_scale, scale, "row_scale")
        same_bits(torch, got.codes, codes, "codes")
        if residual:
            same_bits(torch, got.residual, total, "residual")
        else:
            assert got.residual is None
        if normed:
            same_bits(torch, got.normed, v, "normed")
        else:
            assert got.normed is None
        # the padding that matmul_codes multiplies is zero
        kp = (k + 127) // 128 * 128
        pad = torch.as_strided(got.codes, (m, kp), (kp, 1))[:, k:]
        assert not pad.any()


@pytest.mark.parametrize("m,k", [(3, 40), (4, 4096), (2, 70000)])
def test_norm_codes_are_quantize_rows(zb, torch, m, k):
    x, r, w = norm_case(torch, m, k, "float32", True)
    got = zb.rms_norm_quantize(x.cuda(), w.cuda(), residual=r.cuda(), normed=True)
    codes, scale = zb.quantize_rows(got.normed)
    same_bits(torch, got.codes, codes, "codes")
    same_bits(torch, got.row_scale, scale, "row_scale")


@pytest.mark.parametrize("m,k,dtype", [(700, 512, "float32"), (300, 1001, "bfloat16"), (4, 40000, "float16")])
def test_norm_reciprocal_scale(zb, torch, m, k, dtype):
    x, r, w = norm_case(torch, m, k, dtype, True)
    codes, scale, _, _ = norm_oracle(torch, x, r, w, 1e-5, reciprocal=True)
    got = zb.rms_norm_quantize(x.cuda(), w.cuda(), residual=r.cuda(), reciprocal=True)
    same_bits(torch, got.row_scale, scale, "row_scale")
    same_bits(torch, got.codes, codes, "codes")
    other = zb.rms_norm_quantize(x.cuda(), w.cuda(), residual=r.cuda()).row_scale
    assert m < 10 or (other != got.row_scale).any()  # the two rules differ in some rows
    assert ((other - got.row_scale).abs() <= 2.0**-23 * other).all()


@pytest.mark.parametrize("k", [24, 4099, 40000])
def test_norm_extremes(zb, torch, k):
    """Zero rows with and without eps, values whose squares leave fp32's
    range, denormals, infinities and NaN, one row each."""
    x = randn(torch, k, 8, k)
    x[0] = 0
    x[1] *= 1e30
    x[2] *= 1e-30
    x[3] = 0
    x[3, 0] = 1e-40
    x[4, 5] = math.inf
    x[5, 6] = math.nan
    x[6, 7] = -math.inf
    for eps in (1e-5, 0.0):
        codes, scale, _, v = norm_oracle(torch, x, None, None, eps)
        got = zb.rms_norm_quantize(x.cuda(), eps=eps, normed=True)
        same_bits(torch, got.normed, v, "normed")
        same_bits(torch, got.row_scale, scale, "row_scale")
        same_bits(torch, got.codes, codes, "codes")


@pytest.mark.parametrize("k", [8192, 70000])
def test_norm_longest_code_rows(zb, torch, k):
    """Padding up to the largest row pitch of the codes, where a 32-bit count of it would wrap."""
    from zyron_b200 import _lib

    ldq = 2**31 - 1
    x = randn(torch, k, 1, k)
    xd = x.cuda()
    q = torch.full((ldq + 1,), 7, dtype=torch.int8, device="cuda")
    scale = torch.empty(1, device="cuda")
    _lib.check(_lib.lib().zq_rms_norm_quantize(xd.data_ptr(), 1, 1, k, k, None, 0, None, 1e-5, 0, None, 0, None, 0,
                                               q.data_ptr(), ldq, scale.data_ptr(), torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    codes, want, _, _ = norm_oracle(torch, x, None, None, 1e-5)
    same_bits(torch, q[:k], codes[0], "codes")
    same_bits(torch, scale, want, "row_scale")
    assert not q[k:ldq].any() and q[ldq] == 7


def test_norm_in_place_and_shapes(zb, torch):
    x, r, w = norm_case(torch, 6, 320, "bfloat16", True)
    codes, scale, total, v = norm_oracle(torch, x, r, w, 1e-6)
    xd, rd = x.cuda().view(2, 3, 320), r.cuda().view(2, 3, 320)
    got = zb.rms_norm_quantize(xd, w.cuda(), residual=rd, eps=1e-6, residual_out=rd, normed=True)
    assert got.residual.data_ptr() == rd.data_ptr()
    assert got.codes.shape == (2, 3, 320) and got.row_scale.shape == (2, 3)
    same_bits(torch, rd.view(6, 320), total, "residual in place")
    same_bits(torch, got.codes.reshape(6, 320), codes, "codes")
    same_bits(torch, got.normed.view(6, 320), v, "normed")
    # x's own buffer takes the sum as well, and x may be its own residual
    xd = x.cuda()
    again = zb.rms_norm_quantize(xd, w.cuda(), residual=r.cuda(), eps=1e-6, residual_out=xd)
    same_bits(torch, xd, total, "residual into x")
    same_bits(torch, again.codes, codes, "codes, residual into x")
    twice = zb.rms_norm_quantize(x.cuda(), w.cuda(), residual=x.cuda(), eps=1e-6)
    same_bits(torch, twice.codes, norm_oracle(torch, x, x, w, 1e-6)[0], "x twice")
    xd = x.cuda().view(2, 3, 320)
    one = zb.rms_norm_quantize(x[0].cuda(), w.cuda(), eps=1e-6)  # a vector
    assert one.codes.shape == (320,) and one.row_scale.shape == ()
    none = zb.rms_norm_quantize(xd[:0], w.cuda())
    assert none.codes.shape == (0, 3, 320) and none.row_scale.shape == (0, 3)
    # rows in a transposed order are copied, not misread
    t = x.t().contiguous().t()
    same_bits(torch, zb.rms_norm_quantize(t.cuda(), w.cuda()).codes, norm_oracle(torch, x, None, w, 1e-5)[0], "copied")


def test_norm_refusals_on_device(zb, torch):
    x = torch.zeros(4, 64, device="cuda")
    w = torch.ones(64, device="cuda")
    with pytest.raises(ValueError, match="weight must be contiguous float32"):
        zb.rms_norm_quantize(x, w.half())
    with pytest.raises(ValueError, match="weight must be contiguous float32"):
        zb.rms_norm_quantize(x, torch.ones(63, device="cuda"))
    with pytest.raises(ValueError, match="residual must have x's shape and type"):
        zb.rms_norm_quantize(x, w, residual=x.half())
    with pytest.raises(ValueError, match="residual is on cpu"):
        zb.rms_norm_quantize(x, w, residual=x.cpu())
    with pytest.raises(ValueError, match="go together"):
        zb.rms_norm_quantize(x, w, residual_out=x)
    with pytest.raises(ValueError, match="do not overlap"):
        zb.rms_norm_quantize(x, w, residual=x, residual_out=x[0].expand(4, 64))
    with pytest.raises(ValueError, match="eps must be finite"):
        zb.rms_norm_quantize(x, w, eps=-1.0)


def test_norm_overlaps(zb, torch):
    """residual_out may be x, residual, or columns beside them; any other overlap is refused."""
    x, r, w = (t.cuda() for t in norm_case(torch, 6, 64, "float32", True))
    want = norm_oracle(torch, x.cpu(), r.cpu(), w.cpu(), 1e-5)
    wide = torch.zeros(6, 200, device="cuda")
    for into in (lambda: wide[:, 64:128], lambda: wide[:, 136:]):
        wide[:, :64], wide[:, 64:128] = x, r
        got = zb.rms_norm_quantize(wide[:, :64], w, residual=wide[:, 64:128], residual_out=into())
        same_bits(torch, got.codes, want[0], "codes")
        same_bits(torch, into(), want[2], "sum")
        same_bits(torch, wide[:, :64], x, "x")
    flat = torch.zeros(6 * 64 + 64, device="cuda")
    shifted = [flat[i : i + 6 * 64].view(6, 64) for i in (0, 1, 64)]
    square = torch.zeros(64, 64, device="cuda")
    for xx, rr, out, match in ((wide[:, :64], r, wide[:, 1:65], "overlaps x"), (x, wide[:, 64:128], wide[:, 60:124], "overlaps residual"),
                               (shifted[0], r, shifted[1], "overlaps x"), (x, shifted[2], shifted[0], "overlaps residual"),
                               (x, wide[1:, :64].repeat(2, 1)[:6], wide.view(12, 100)[:6, :64], None),
                               (wide[:, :64], r, wide.view(12, 100)[:6, :64], "overlaps x")):
        if match is None:
            zb.rms_norm_quantize(xx, w, residual=rr, residual_out=out)
            continue
        with pytest.raises(ValueError, match=match):
            zb.rms_norm_quantize(xx, w, residual=rr, residual_out=out)
    with pytest.raises(ValueError, match="overlaps weight"):
        zb.rms_norm_quantize(x, square[3], residual=r, residual_out=square[:6])


# ---- matmul_codes -----------------------------------------------------------------

@pytest.mark.parametrize("qtype", [1, 2])
@pytest.mark.parametrize("m,k,n", [(1, 768, 256), (1, 100, 30), (3, 100, 65), (9, 512, 130), (40, 1000, 96)])
def test_matmul_codes_equals_matmul(zb, torch, m, k, n, qtype):
    w = zb.quantize((randn(torch, n, k, n) * 0.02).cuda(), zb.Type(qtype))
    bias = randn(torch, n + 1, n).cuda()
    x = randn(torch, m, m, k).cuda()
    r = zb.rms_norm_quantize(x, normed=True)
    want = zb.matmul(r.normed, w, bias=bias)
    same_bits(torch, zb.matmul_codes(r.codes, r.row_scale, w, bias=bias), want, "padded rows")
    same_bits(torch, zb.matmul_codes(r.codes.contiguous(), r.row_scale, w, bias=bias), want, "dense rows")
    out = torch.empty_like(want)
    assert zb.matmul_codes(*zb.quantize_rows(r.normed), w, out=out) is out
    same_bits(torch, out, zb.matmul(r.normed, w), "without bias")


# ---- adapters -----------------------------------------------------------------------

def adapter_oracle(torch, y, x, a, b, ids, scales, ranks):
    """In 64 bits, with the bound that the kernel's roundings allow: one of
    2^-23 (the tensor cores may cut off) for each of the 16 products and the
    carry of the MMAs that a sum goes through, at most all of k's, one for each
    partial sum of A x, at most 16 or one for 32 of k, and half of one each for
    the scaling and for the sum with y.  Products of parts are exact."""
    y64, x64 = y.double().clone(), x.double()
    tol = y64.abs() * 2.0**-24
    parts = {"float32": 3, "float16": 2, "bfloat16": 1}[str(x.dtype).split(".")[1]] * (2 if a.dtype == torch.float16 else 1)
    k, rank = a.shape[2], a.shape[1]
    steps_a = -(-k // 32) * 2 * parts * 17 + max(16, -(-k // 32))
    steps_b = -(-rank // 32) * 2 * 3 * (2 if a.dtype == torch.float16 else 1) * 17
    for i, s in enumerate(ids.tolist()):
        if not 0 <= s < a.shape[0]:
            tol[i] = 0
            continue
        r = rank if ranks is None else max(0, min(rank, int(ranks[s])))
        if r == 0:
            tol[i] = 0
            continue
        A, B = a[s, :r].double(), b[s, :, :r].double()
        f = 1.0 if scales is None else float(scales[s])
        d = f * (B @ (A @ x64[i]))
        reach = abs(f) * (B.abs() @ (A.abs() @ x64[i].abs()))
        tol[i] = (y64[i].abs() + (y64[i] + d).abs() + reach) * 2.0**-24 + reach * (steps_a + steps_b + 2) * 2.0**-23
        y64[i] += d
    return y64, tol


def adapter_case(torch, m, k, n, slots, rank, dtype, wdtype, layout="mixed", ragged=True, seed=0):
    w = getattr(torch, wdtype)
    x = randn(torch, seed + m + k, m, k).to(getattr(torch, dtype))
    y = randn(torch, seed + n, m, n)
    a = (randn(torch, seed + 1, slots, rank, k) * k**-0.5).to(w)
    b = (randn(torch, seed + 2, slots, n, rank) * rank**-0.5).to(w)
    g = torch.Generator().manual_seed(seed + 3)
    scales = torch.rand(slots, generator=g) * 2 - 0.5
    ranks = torch.randint(0, rank + 1, (slots,), generator=g, dtype=torch.int32) if ragged else None
    if layout == "one":
        ids = torch.zeros(m, dtype=torch.int64)
    else:
        ids = torch.randint(-1, slots, (m,), generator=g)
        if layout == "sorted":
            ids = ids.sort().values
    return y, x, a, b, ids.to(torch.int32), scales, ranks


def check_adapters(torch, zb, y, x, a, b, ids, scales, ranks, **kw):
    want, tol = adapter_oracle(torch, y, x, a, b, ids, scales, ranks)
    up = lambda t: None if t is None else t.cuda()  # noqa: E731
    yd = y.cuda()
    got = zb.add_low_rank(yd, up(x), up(a), up(b), up(ids), scales=up(scales), ranks=up(ranks), **kw)
    assert got is yd
    off = (yd.cpu().double() - want).abs()
    assert (off <= tol).all(), f"{int((off > tol).sum())} outputs off, most {float((off / (tol + 1e-300)).max()):.3g} of the bound"
    return yd


ADAPTER_SIZES = [
    # m, k, n, slots, rank
    (1, 1, 1, 1, 1), (1, 4096, 4096, 3, 16), (2, 33, 5, 2, 7), (3, 64, 32, 8, 8), (5, 100, 30, 2, 12),
    (16, 256, 64, 1, 16), (17, 256, 68, 2, 24), (31, 136, 40, 4, 64), (33, 1000, 1003, 5, 13), (64, 512, 768, 48, 32),
    (40, 2056, 130, 3, 65), (20, 320, 100, 2, 128), (10, 264, 72, 3, 200), (9, 200, 36, 2, 256), (255, 40, 24, 7, 4),
    (256, 72, 20, 300, 8), (257, 72, 20, 300, 8), (300, 64, 48, 2, 16), (1100, 48, 33, 40, 10), (2500, 24, 12, 1, 3),
    (700, 16, 8, 8192, 2),
]


@pytest.mark.parametrize("dtype,wdtype", [("float32", "bfloat16"), ("float32", "float16"), ("bfloat16", "bfloat16"),
                                          ("float16", "bfloat16"), ("float16", "float16")])
@pytest.mark.parametrize("m,k,n,slots,rank", ADAPTER_SIZES)
def test_adapters(zb, torch, m, k, n, slots, rank, dtype, wdtype):
    for layout, ragged in (("mixed", True), ("sorted", False), ("one", False)):
        check_adapters(torch, zb, *adapter_case(torch, m, k, n, slots, rank, dtype, wdtype, layout, ragged))


WDTYPES = ["bfloat16", "float16"]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("wdtype", WDTYPES)
@pytest.mark.parametrize("m,k,n,slots,rank", [(3, 96, 40, 2, 5), (40, 1000, 33, 3, 70), (300, 4096, 64, 3, 16),
                                              (270, 333, 130, 2, 256)])
def test_adapters_exact_products(zb, torch, m, k, n, slots, rank, dtype, wdtype):
    """Sums that fp32 holds exactly, whatever the order, bit for bit: every
    element's own bits through both products, and whole numbers whose sums of
    absolute values stay below 2^24.  A part of a value that is lost shows."""
    t, w = getattr(torch, dtype), getattr(torch, wdtype)
    g = torch.Generator().manual_seed(m + k)
    ids = torch.randint(-1, slots, (m,), generator=g, dtype=torch.int32)
    live = ids >= 0

    def run(y, x, a, b, scales=None):
        yd = y.cuda()
        zb.add_low_rank(yd, x.to(t).cuda(), a.to(w).cuda(), b.to(w).cuda(), ids.cuda(),
                        scales=None if scales is None else scales.cuda())
        return yd

    # one element and one rank an output, weights and scales powers of two
    x = randn(torch, k, m, k).to(t).float()
    a, b = torch.zeros(slots, rank, k), torch.zeros(slots, n, rank)
    col = torch.randint(0, k, (slots, rank), generator=g)
    a.scatter_(2, col[:, :, None], 2.0 ** torch.randint(-3, 4, (slots, rank, 1), generator=g))
    pick = torch.randint(0, rank, (slots, n), generator=g)
    b.scatter_(2, pick[:, :, None], -(2.0 ** torch.randint(-3, 4, (slots, n, 1), generator=g)))
    scales = 2.0 ** torch.arange(slots).float()
    s = ids.clamp(min=0).long()
    h = x.gather(1, col[s]) * a.gather(2, col[:, :, None])[s, :, 0]
    want = scales[s][:, None] * h.gather(1, pick[s]) * b.gather(2, pick[:, :, None])[s, :, 0]
    same_bits(torch, run(torch.zeros(m, n), x, a, b, scales), torch.where(live[:, None], want, 0.0), "single products")

    # whole numbers
    xlimit = {"float32": 1 << 24, "float16": 1 << 11, "bfloat16": 1 << 8}[dtype]
    wlimit = {"float16": (1 << 11) - 1, "bfloat16": 1 << 8}[wdtype]
    for amax, a_n, xmax, bmax, b_n in ((1, 8, 1 << 19, 1, 2), (wlimit, 8, 1 << 9, 1, 1), (1, 4, 1 << 10, wlimit, 1)):
        xmax = min(xmax, xlimit)

        def whole(shape, most):
            return torch.randint(-most, most + 1, shape, generator=g).double()

        x = whole((m, k), xmax)
        a, b = torch.zeros(slots, rank, k).double(), torch.zeros(slots, n, rank).double()
        a.scatter_(2, torch.randint(0, k, (slots, rank, a_n), generator=g), whole((slots, rank, a_n), amax))
        b.scatter_(2, torch.randint(0, rank, (slots, n, b_n), generator=g), whole((slots, n, b_n), bmax))
        y = whole((m, n), 1 << 21)
        h = torch.einsum("mk,mrk->mr", x, a[s])
        want = y + live[:, None] * torch.einsum("mr,mnr->mn", h, b[s])
        assert want.abs().max() < 1 << 24
        same_bits(torch, run(y.float(), x, a, b), want.float(), f"whole numbers to {xmax}, {amax}, {bmax}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("wdtype", WDTYPES)
def test_adapters_long_sums_lose_no_more(zb, torch, dtype, wdtype):
    """Tensor cores cut sums off, so a chain of products of one sign loses the
    more the longer it is.  A sum that is one chain of 24 products shows what a
    chain loses; longer sums of the same values are rounded sums of such chains
    and lose the same share, within a quarter for the spread and half a last
    place for each of the additions."""
    t, w = getattr(torch, dtype), getattr(torch, wdtype)
    parts = {"float32": 3, "float16": 2, "bfloat16": 1}
    wparts = 2 if wdtype == "float16" else 1
    g = torch.Generator(device="cuda").manual_seed(5)

    def draw(*shape):
        return torch.rand(*shape, generator=g, device="cuda") + 0.1

    def loss(m, x, a, b):
        ids = torch.zeros(m, dtype=torch.int32, device="cuda")
        got = zb.add_low_rank(torch.zeros(m, b.shape[1], device="cuda"), x, a, b, ids).double()
        want = x.double() @ a[0].double().T @ b[0].double().T
        return float(((got - want).square().mean() / want.square().mean()).sqrt())

    # A x of one block of four warps a tile, each a quarter of k in chunks of 32; B picks a rank
    m, n = 5000, 64
    pick = torch.eye(n, device="cuda").to(w)[None]
    one = 4 * 32 * (12 // (parts[dtype] * wparts))
    short, long = (loss(m, draw(m, k).to(t), draw(1, n, k).to(w), pick) for k in (one, 8 * one))
    assert long <= 1.25 * short + 8 * 2.0**-25, (short * 2**24, long * 2**24)
    # B h, h the elements of x as they are, over all ranks
    one = 32 * (12 // (3 * wparts))
    short, long = (loss(m, draw(m, r).to(t), torch.eye(r, device="cuda").to(w)[None], draw(1, n, r).to(w))
                   for r in (one, 256))
    assert long <= 1.25 * short + 4 * 2.0**-25, (short * 2**24, long * 2**24)


@pytest.mark.parametrize("m", [6, 300])
def test_adapters_leave_other_rows(zb, torch, m):
    """Rows without an adapter keep their bits, whatever they hold, and what
    no row's adapter covers is not read into any result: NaN in unused slots,
    in ranks past an adapter's own, and in rows of x that have no adapter."""
    y, x, a, b, ids, scales, ranks = adapter_case(torch, m, 72, 44, 4, 16, "float32", "bfloat16")
    ids = torch.where(ids == 3, torch.tensor(-1, dtype=torch.int32), ids)
    ids[0], ids[2], ids[4] = 5, -(2**31), 2**31 - 1  # no such slots
    ranks = torch.tensor([9, 16, 0, 5], dtype=torch.int32)
    a[3], b[3] = math.nan, math.nan
    for s, r in enumerate(ranks.tolist()):
        a[s, r:], b[s, :, r:] = math.nan, math.nan
    none = (ids < 0) | (ids > 3) | (ids == 2)
    x[none] = math.nan
    y[0, 0] = math.nan
    want, tol = adapter_oracle(torch, y, torch.nan_to_num(x), torch.nan_to_num(a), torch.nan_to_num(b), ids, scales, ranks)
    yd = y.cuda()
    zb.add_low_rank(yd, x.cuda(), a.cuda(), b.cuda(), ids.cuda(), scales=scales.cuda(), ranks=ranks.cuda())
    same_bits(torch, yd[none.cuda()], y[none], "rows without an adapter")
    off = (yd.cpu().double() - want).abs()[~none]
    assert (off <= tol[~none]).all()
    # ranks outside [0, max_rank] are clamped
    clamped = y.cuda()
    zb.add_low_rank(clamped, x.cuda(), a[:2].contiguous().cuda(), b[:2].contiguous().cuda(), ids.cuda(),
                    ranks=torch.tensor([-4, 16], dtype=torch.int32).cuda())
    same_bits(torch, clamped[(ids == 0).cuda()], y[ids == 0], "rank below zero")


def test_adapters_infinities(zb, torch):
    """An infinite or NaN input, or an A x past fp32's range, leaves its own
    row's outputs infinite or NaN and no other's."""
    y, x, a, b, ids, _, _ = adapter_case(torch, 20, 64, 32, 2, 8, "float32", "float16", "one", False)
    a, b = a.abs() + 0.1, b.abs() + 0.1
    x[1, 7], x[2, 9], x[3] = math.inf, math.nan, -3.0e38
    yd = y.cuda()
    zb.add_low_rank(yd, x.cuda(), a.cuda(), b.cuda(), ids.cuda())
    got = yd.cpu()
    assert not got[1:4].isfinite().any() and got[2].isnan().all()
    want, tol = adapter_oracle(torch, y, torch.nan_to_num(x, posinf=1.0), a, b, ids, None, None)
    rest = [i for i in range(20) if i not in (1, 2, 3)]
    assert ((got.double() - want).abs() <= tol)[rest].all()


@pytest.mark.parametrize("wdtype", WDTYPES)
@pytest.mark.parametrize("m,rank", [(6, 8), (6, 13), (300, 40)])
def test_adapters_infinite_weights(zb, torch, m, rank, wdtype):
    """An infinite or NaN element of B reaches its column, one of A its
    adapter's rows, and neither any other adapter's."""
    y, x, a, b, ids, _, _ = adapter_case(torch, m, 64, 40, 3, rank, "float32", wdtype, "mixed", False)
    ids[:3] = torch.arange(3, dtype=torch.int32)
    a, b = a.abs() + 0.1, b.abs() + 0.1
    x = x.abs() + 0.1
    want, tol = adapter_oracle(torch, y, x, a, b, ids, None, None)
    for bad in (math.inf, math.nan):
        a2, b2 = a.clone(), b.clone()
        b2[0, 7, rank - 1], b2[0, 33, 0] = bad, -bad
        a2[1, rank - 1, 5] = bad
        got = zb.add_low_rank(y.cuda(), x.cuda(), a2.cuda(), b2.cuda(), ids.cuda()).cpu()
        hit = torch.zeros(m, 40, dtype=torch.bool)
        hit[ids == 0, 7] = hit[ids == 0, 33] = True
        hit[ids == 1] = True
        assert not got[hit].isfinite().any()
        assert ((got.double() - want).abs() <= tol)[~hit].all()


def test_matmul_codes_without_rows(zb, torch):
    w = zb.quantize(torch.ones(100, 30, device="cuda"))
    h = zb.rms_norm_quantize(torch.ones(2, 0, 100, device="cuda"))
    assert zb.matmul_codes(h.codes, h.row_scale, w).shape == (2, 0, 30)
    one = zb.rms_norm_quantize(randn(torch, 1, 100).cuda(), normed=True)  # a vector
    same_bits(torch, zb.matmul_codes(one.codes, one.row_scale, w), zb.matmul(one.normed[None], w)[0], "a vector")


@pytest.mark.parametrize("m", [200, 600])
def test_adapters_rows_do_not_depend_on_others(zb, torch, m):
    """A row's bits are the same twice, with the rows in another order, and
    with other values and adapters in the other rows."""
    y, x, a, b, ids, scales, ranks = adapter_case(torch, m, 200, 100, 3, 24, "float32", "bfloat16", "mixed", False)
    y, x, a, b, ids, scales = (t.cuda() for t in (y, x, a, b, ids, scales))
    every = zb.add_low_rank(y.clone(), x, a, b, ids, scales=scales)
    same_bits(torch, zb.add_low_rank(y.clone(), x, a, b, ids, scales=scales), every, "twice")
    order = torch.randperm(m, generator=torch.Generator().manual_seed(2)).cuda()
    moved = zb.add_low_rank(y[order], x[order], a, b, ids[order], scales=scales)
    same_bits(torch, moved, every[order], "in another order")
    x2, ids2 = x * 3 + 1, (ids + 2) % 3
    keep = torch.arange(m, device="cuda") % 7 == 3
    x2[keep], ids2[keep] = x[keep], ids[keep]
    part = zb.add_low_rank(y.clone(), x2, a, b, ids2.int(), scales=scales)
    same_bits(torch, part[keep], every[keep], "among others")


@pytest.mark.parametrize("m", [5, 400])
def test_adapters_strides(zb, torch, m):
    y, x, a, b, ids, scales, ranks = adapter_case(torch, m, 48, 40, 3, 8, "float16", "float16")
    want = check_adapters(torch, zb, y, x, a, b, ids, scales, ranks)
    for pad, start in ((4, 0), (3, 1), (8, 4)):
        wide_y = torch.full((m, 40 + pad + start), 9.0, device="cuda")
        wide_x = torch.zeros(m, 48 + pad + start, dtype=x.dtype, device="cuda")
        yv, xv = wide_y[:, start : start + 40], wide_x[:, start : start + 48]
        yv.copy_(y)
        xv.copy_(x)
        zb.add_low_rank(yv, xv, a.cuda(), b.cuda(), ids.cuda(), scales=scales.cuda(), ranks=ranks.cuda())
        same_bits(torch, yv, want, f"pitch +{pad}")
        assert (wide_y[:, :start] == 9).all() and (wide_y[:, start + 40 :] == 9).all()
    y3 = y.view(1, m, 40).cuda()
    zb.add_low_rank(y3, x.view(1, m, 48).cuda(), a.cuda(), b.cuda(), ids.view(1, m).cuda(), scales=scales.cuda(),
                    ranks=ranks.cuda())
    same_bits(torch, y3[0], want, "three dimensions")


@pytest.mark.parametrize("m", [5, 300])
def test_adapters_subnormal_outputs(zb, torch, m):
    """Subnormal y, sums and additions count as zeros, wherever y lies; rows
    without an adapter keep theirs."""
    n, k = 40, 16
    tiny = 2.0**-126
    a = torch.zeros(2, 1, k).bfloat16()
    b = torch.ones(2, n, 1).bfloat16()
    a[0, 0, 0] = 1.0
    x = torch.zeros(m, k)
    y = torch.full((m, n), tiny / 8)
    x[1, 0], y[1] = -tiny, 1.5 * tiny     # a normal sum's terms
    x[2, 0], y[2] = tiny / 4, tiny        # a subnormal addition
    x[3, 0], y[3] = 2.0**-100, tiny / 2   # beside a normal one
    ids = torch.zeros(m, dtype=torch.int32)
    ids[4:] = -1
    want = y.clone()
    want[0], want[1], want[2], want[3] = 0.0, 0.0, tiny, 2.0**-100
    for start in (0, 1):
        wide = torch.zeros(m, n + start, device="cuda")
        got = wide[:, start:]
        got.copy_(y)
        zb.add_low_rank(got, x.cuda(), a.cuda(), b.cuda(), ids.cuda())
        same_bits(torch, got.abs(), want, f"y at {start}")


def test_adapters_linear_forward(zb, torch):
    w = randn(torch, 1, 96, 80) * 0.05
    lin = zb.QuantizedLinear(w.cuda(), randn(torch, 2, 80))
    y, x, a, b, ids, scales, ranks = adapter_case(torch, 12, 96, 80, 3, 8, "float32", "bfloat16")
    pool = zb.LowRankAdapters(a.cuda(), b.cuda(), scales.cuda(), ranks.cuda())
    base = lin(x.cuda())
    want = zb.add_low_rank(base.clone(), x.cuda(), a.cuda(), b.cuda(), ids.cuda(), scales=scales.cuda(), ranks=ranks.cuda())
    same_bits(torch, lin(x.cuda(), adapters=pool, adapter_ids=ids.cuda()), want, "forward with adapters")
    same_bits(torch, lin(x.cuda()), base, "forward without")
    with pytest.raises(ValueError, match="go together"):
        lin(x.cuda(), adapters=pool)
    with pytest.raises(ValueError, match="need a CUDA tensor"):
        lin(x.numpy(), adapters=pool, adapter_ids=ids.cuda())


def test_adapters_refusals_on_device(zb, torch):
    y, x, a, b, ids, scales, ranks = [t.cuda() for t in adapter_case(torch, 4, 32, 16, 2, 8, "float32", "bfloat16")]
    for bad, match in ((dict(y=y.half()), "y must have shape"), (dict(y=y[:, :8]), "y must have shape"),
                       (dict(y=y[0].expand(4, 16)), "do not overlap"), (dict(x=x[:, :31]), "dimension mismatch"),
                       (dict(a=a.float()), "of one type"), (dict(a=a.transpose(1, 2)), "must be \\[slots"),
                       (dict(b=b.transpose(1, 2).contiguous().transpose(1, 2)), "must be contiguous"),
                       (dict(ids=ids.long()), "ids must be int32"), (dict(ids=ids[:3]), "ids must be int32"),
                       (dict(scales=scales[:1]), "scales must be"), (dict(ranks=ranks.long()), "ranks must be"),
                       (dict(ids=ids.cpu()), "ids is on cpu")):
        kw = {"y": y, "x": x, "a": a, "b": b, "ids": ids, **bad}
        with pytest.raises(ValueError, match=match):
            zb.add_low_rank(**kw)
    lin = zb.QuantizedLinear(torch.zeros(32, 16, device="cuda"))
    pool = zb.LowRankAdapters(a, b)
    assert lin(x[:0], adapters=pool, adapter_ids=ids[:0]).shape == (0, 16)
    with pytest.raises(ValueError, match="dimension mismatch"):
        lin(x, adapters=zb.LowRankAdapters(a[:, :, :31].contiguous(), b), adapter_ids=ids)
    empty = zb.add_low_rank(y[:0], x[:0], a, b, ids[:0])
    assert empty.shape == (0, 16)


def test_linear_refusals_on_device(zb, torch):
    """Nothing is launched for a call that is refused: out keeps what it holds."""
    y, x, a, b, ids, _, _ = [t.cuda() for t in adapter_case(torch, 4, 32, 16, 2, 8, "float32", "bfloat16")]
    lin = zb.QuantizedLinear(torch.ones(32, 16, device="cuda"))
    out = torch.full((4, 16), 7.0, device="cuda")
    for pool, bad_ids, match in (((a, b), ids.long(), "ids must be int32"), ((a, b), ids[:2], "ids must be int32"),
                                 ((a[:, :, :31].contiguous(), b), ids, "dimension mismatch"),
                                 ((a, b[:, :15].contiguous()), ids, "output/adapter dimension mismatch"),
                                 ((a, b.half()), ids, "of one type"), ((a, b.cpu()), ids, "b is on cpu")):
        with pytest.raises(ValueError, match=match):
            lin(x, out=out, adapters=zb.LowRankAdapters(*pool), adapter_ids=bad_ids)
    w = lin.weight()
    for bad in (out.half(), out[:3], out.cpu(), torch.empty(4, 32, device="cuda")[:, :16], torch.empty(4, 17, device="cuda")):
        with pytest.raises(ValueError, match="out must be contiguous float32"):
            zb.matmul(x, w, out=bad)
    bias = torch.zeros(16, device="cuda")
    for bad in (bias.cpu(), bias.half(), bias[:15], torch.zeros(32, device="cuda")[::2]):
        with pytest.raises(ValueError, match="bias must be contiguous float32"):
            zb.matmul(x, w, bias=bad, out=out)
    for bad in (x.half(), x[0]):
        with pytest.raises(ValueError, match="input must be float32"):
            zb.quantize_rows(bad)
    torch.cuda.synchronize()
    assert (out == 7).all()
    assert zb.matmul(x, w, bias=bias, out=out).data_ptr() == out.data_ptr()
    assert zb.matmul(x.view(2, 2, 32), w, out=out).shape == (2, 2, 16)  # out by its number of elements


# ---- log probabilities ------------------------------------------------------------

def logprob_oracle(torch, x, targets, k):
    """In 64 bits.  The tolerances count roundings: a thread adds at most
    n = ceil(vocab / 256) + 64 exponentials one after the other and the joins
    add 32 more; an exponential is within 2^-22, and its argument's rounding
    weighs at most |d| exp(d) 2^-23 < 2^-24."""
    x = x.double()
    most = x.amax(-1, keepdim=True)
    empty = most == -math.inf
    d = x - torch.where(empty, 0.0, most)
    e = torch.exp(d)
    s = e.sum(-1, keepdim=True)
    log_s = torch.where(empty, 0.0, torch.log(s))
    lp = d - log_s
    ent = torch.where(empty[:, 0], 0.0, (log_s - torch.where(e > 0, e * d, 0.0).sum(-1, keepdim=True) / s)[:, 0])
    n = -(-x.shape[1] // 256) + 64 + 32 + 8
    base = n * 2.0**-24
    picked = None if targets is None else torch.where(
        targets < 0, 0.0, torch.where(targets >= x.shape[1], math.nan, lp.gather(1, targets.clamp(0, x.shape[1] - 1))))
    # order by value (NaN first), then by index
    key = torch.nan_to_num(x, nan=math.inf, posinf=1e300, neginf=-math.inf)
    ids = torch.argsort(key, dim=-1, descending=True, stable=True)[:, :k]
    return picked, ent, lp.gather(1, ids), ids, base


def close(torch, got, want, base, what):
    got = got.cpu().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    # want's rounding to fp32 is infinite for a difference past fp32's range
    same = (got == want.float()) | (got.isnan() & want.isnan())
    off = torch.where(same, torch.zeros_like(want), (got - want).abs())
    tol = base * (1 + want.abs()) + 3 * 2.0**-24 * want.abs()
    bad = ~(same | (off <= tol))
    assert not bad.any(), f"{what}: {int(bad.sum())} off, most {float((off / tol).max()):.3g} of the bound"


def check_logprobs(zb, torch, x, targets, k):
    lp, ent, top, ids, base = logprob_oracle(torch, x.cpu(), targets, k)
    got = zb.token_logprobs(x, None if targets is None else targets.cuda(), top_k=k)
    if targets is not None:
        close(torch, got.logprobs, lp, base, "logprobs")
    close(torch, got.entropy, ent, base, "entropy")
    if k:
        same_bits(torch, got.top_ids, ids, "top_ids")
        close(torch, got.top_logprobs, top, base, "top_logprobs")
    else:
        assert got.top_ids is None and got.top_logprobs is None
    return got


LOGPROB_SIZES = [(1, 1), (1, 2), (2, 7), (3, 16), (1, 33), (5, 100), (4, 1000), (2, 1023), (1, 4096), (7, 5003),
                 (1, 16384), (3, 32003), (1, 100001), (2, 131072), (400, 300), (1300, 8200)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,vocab", LOGPROB_SIZES)
def test_logprobs(zb, torch, m, vocab, dtype):
    g = torch.Generator().manual_seed(m + vocab)
    targets = torch.randint(-1, vocab, (m, 3), generator=g)
    for k, pitch, spread in ((0, 0, 2.0), (1, 3, 0.3), (5, 8, 4.0), (32, 1, 2.0)):
        k = min(k, vocab)
        x = torch.zeros(m, vocab + pitch, dtype=getattr(torch, dtype), device="cuda")[:, :vocab]
        x.copy_(randn(torch, m + k, m, vocab) * spread)
        check_logprobs(zb, torch, x, targets, k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,vocab", [(9, 70), (9, 5003), (9, 40000), (700, 257)])
def test_logprobs_masks_and_extremes(zb, torch, m, vocab, dtype):
    t = getattr(torch, dtype)
    low = torch.finfo(t).min
    x = randn(torch, vocab, m, vocab).to(t)
    x[0] = -math.inf                        # nothing allowed
    x[1] = low                              # all at the lowest value: uniform
    x[2, 1:] = low                          # one token and the lowest value
    x[3] = -math.inf
    x[3, vocab // 2] = -5.0                 # one token allowed
    x[4] = 1.5                              # all equal: ties go to the lowest ids
    x[5, 3] = math.inf
    x[6, 9] = math.nan
    x[6, 20] = math.nan
    x[7] = torch.finfo(t).max
    x[7, ::2] = low
    x[8, ::3] = -math.inf
    x[8, 1] = 0.0
    x[8, 4] = -0.0                          # equal to +0: the lower id first
    targets = torch.arange(m).view(m, 1) % vocab
    targets = torch.cat([targets, torch.full((m, 1), vocab // 2), torch.full((m, 1), -100), torch.full((m, 1), vocab),
                         torch.full((m, 1), 2**62)], 1)
    for k in (1, 7, 32):
        check_logprobs(zb, torch, x.cuda(), targets, k)


@pytest.mark.parametrize("vocab", [300, 20000])
def test_logprobs_orders(zb, torch, vocab):
    """Rising rows take every logit into the lists, falling ones the first;
    many equal values fill them with the lowest ids."""
    up = torch.arange(vocab, dtype=torch.float32) / vocab
    x = torch.stack([up, -up, (torch.arange(vocab) % 5).float(), (torch.arange(vocab) % 5 == 3).float() * 1e-3])
    check_logprobs(zb, torch, x.cuda(), torch.zeros(4, 1, dtype=torch.int64), 32)


@pytest.mark.parametrize("m,vocab", [(9, 70), (9, 40000), (300, 17000), (900, 9001)])
@pytest.mark.parametrize("dtype,far", [("float32", (1e4, 1e9, 1e10, 1e12, 1e30)), ("bfloat16", (1e4, 1e9, 1e10, 1e12, 1e30)),
                                       ("float16", (1e4, 6e4))])
def test_logprobs_finite_masks_and_far_maxima(zb, torch, m, vocab, dtype, far):
    """Masks of a finite value anywhere in the type's range, over whole rows,
    whole shares of a row and single tokens, and maxima as far above the rest."""
    t = getattr(torch, dtype)
    targets = torch.arange(m).view(m, 1) % vocab
    targets = torch.cat([targets, torch.full((m, 1), vocab // 2), torch.full((m, 1), vocab - 1)], 1)
    base = randn(torch, vocab, m, vocab)
    for c in far:
        x = base.clone()
        few = randn(torch, 1, vocab) > 2.0
        few[vocab // 3] = True
        for i in range(0, m - 8, 9):
            x[i] = -c                                # every token masked
            x[i + 1, ~few] = -c                      # most
            x[i + 2, : vocab * 6 // 10] = -c         # the first ones
            x[i + 3, vocab * 4 // 10 :] = -c         # the last ones
            x[i + 4, :-1] = -c                       # all but the last
            x[i + 5, vocab // 5] = c                 # one far above
            x[i + 6, vocab // 3] = x[i + 6, -1] = c  # two
            x[i + 7] = c                             # all
            x[i + 8, ::2], x[i + 8, 1::2] = -c, c
        check_logprobs(zb, torch, x.to(t).cuda(), targets, 3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,vocab", [(3000, 64), (1000, 3000), (40, 70000)])
def test_logprobs_are_not_positive(zb, torch, m, vocab, dtype):
    """Probabilities near 1, where the roundings of a log probability are larger than itself."""
    likely = torch.arange(m) * 37 % vocab
    g = torch.Generator().manual_seed(3)
    x = randn(torch, vocab, m, vocab) - 40 * torch.rand(m, 1, generator=g)
    x[torch.arange(m), likely] = 60 * torch.rand(m, generator=g)
    got = check_logprobs(zb, torch, x.to(getattr(torch, dtype)).cuda(), likely[:, None], 4)
    assert (got.logprobs <= 0).all() and (got.top_logprobs <= 0).all()


def test_logprobs_shapes_and_views(zb, torch):
    x = randn(torch, 3, 2, 3, 1000)
    t = torch.randint(0, 1000, (2, 3), generator=torch.Generator().manual_seed(1))
    got = zb.token_logprobs(x.cuda(), t.cuda(), top_k=4)
    assert got.logprobs.shape == (2, 3) and got.top_ids.shape == (2, 3, 4) and got.entropy.shape == (2, 3)
    flat = zb.token_logprobs(x.view(6, 1000).cuda(), t.view(6, 1).cuda(), top_k=4)
    same_bits(torch, got.logprobs.view(6), flat.logprobs[:, 0], "targets of the rows' shape")
    same_bits(torch, got.top_ids.view(6, 4), flat.top_ids, "top_ids")
    one = zb.token_logprobs(x[0, 0].cuda(), t[0, 0].cuda(), entropy=False)
    assert one.logprobs.shape == () and one.entropy is None and one.top_ids is None
    same_bits(torch, one.logprobs, got.logprobs[0, 0], "a vector")
    only = zb.token_logprobs(x.cuda())
    assert only.logprobs is None
    same_bits(torch, only.entropy, got.entropy, "entropy alone")
    none = zb.token_logprobs(x[:0].cuda(), t[:0].cuda(), top_k=2)
    assert none.logprobs.shape == (0, 3) and none.top_ids.shape == (0, 3, 2)
    cols = x.view(6, 1000).t().contiguous().cuda().t()  # strided rows are copied
    same_bits(torch, zb.token_logprobs(cols).entropy, flat.entropy, "transposed")


def test_logprobs_refusals_on_device(zb, torch):
    x = torch.zeros(4, 10, device="cuda")
    t = torch.zeros(4, dtype=torch.int64, device="cuda")
    for kw, match in ((dict(targets=t.int()), "targets must be int64"), (dict(targets=t[:3]), "leading dimensions"),
                      (dict(targets=t.cpu()), "targets is on cpu"), (dict(top_k=11), "at most vocab"),
                      (dict(top_k=-1), "top_k must be >= 0"), (dict(top_k=33), "at most 32")):
        with pytest.raises(ValueError, match=match):
            zb.token_logprobs(x, **kw)


def test_logprobs_refusals_allocate_nothing(zb, torch):
    x = torch.zeros(4, 10, device="cuda")
    before = torch.cuda.memory_allocated()
    for top_k in (1 << 24, 1 << 40):
        with pytest.raises(ValueError, match="at most 32"):
            zb.token_logprobs(x, top_k=top_k)
    assert torch.cuda.memory_allocated() == before


def test_logprobs_offsets_past_32_bits(zb, torch):
    """The last rows of a buffer of more than 2^32 bytes and 2^31 elements."""
    m, vocab = 3, (1 << 30) // 3 + 12345
    x = torch.zeros(7, vocab, dtype=torch.float16, device="cuda")
    assert x.numel() > 1 << 31
    x[6, vocab - 3] = 9.0
    x[6, 5] = 8.0
    got = zb.token_logprobs(x[4:], torch.full((m, 1), vocab - 3, device="cuda"), top_k=3)
    s = (vocab - 2) + math.exp(9) + math.exp(8)
    assert got.top_ids.tolist() == [[0, 1, 2], [0, 1, 2], [vocab - 3, 5, 0]]
    # n = vocab / (256 * 8) additions in a row at most
    tol = (vocab / 2048 + 200) * 2.0**-24 + 40 * 2.0**-23
    assert abs(float(got.logprobs[2, 0]) - (9 - math.log(s))) < tol
    assert abs(float(got.logprobs[0, 0]) + math.log(vocab)) < tol


# ---- devices -----------------------------------------------------------------------

def test_every_operator_on_a_second_device(zb, torch):
    """After calls on the first device, with sizes that need more shared memory
    than a kernel may have without asking, the first device staying current."""
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    y, x, a, b, ids, scales, ranks = adapter_case(torch, 300, 264, 136, 3, 256, "float32", "bfloat16")
    logits = randn(torch, 1, 5, 5000)
    got = []
    for device in ("cuda:0", "cuda:1"):
        up = lambda *ts: [t.to(device) for t in ts]  # noqa: E731
        yd = zb.add_low_rank(*up(y, x, a, b, ids), scales=scales.to(device), ranks=ranks.to(device))
        n = zb.rms_norm_quantize(x.to(device), normed=True)
        w = zb.quantize((randn(torch, 2, 264, 136) * 0.05).to(device))
        z = zb.matmul_codes(n.codes, n.row_scale, w)
        lp = zb.token_logprobs(logits.to(device), top_k=5)
        got.append([yd, n.codes, n.normed, z, zb.matmul(n.normed, w), lp.entropy, lp.top_ids])
        assert all(t.device == torch.device(device) for t in got[-1])
    torch.cuda.synchronize(1)
    assert torch.cuda.current_device() == 0
    for first, second in zip(*got):
        same_bits(torch, second, first, "second device")


# ---- together ------------------------------------------------------------------------

def make_step(zb, torch, hidden=256, vocab=1000, slots=3, rank=8):
    w1 = zb.quantize((randn(torch, 1, hidden, hidden) * hidden**-0.5).cuda())
    w2 = zb.quantize((randn(torch, 2, hidden, vocab) * hidden**-0.5).cuda(), zb.Type.Int4)
    pool = zb.LowRankAdapters((randn(torch, 3, slots, rank, hidden) * hidden**-0.5).bfloat16().cuda(),
                              randn(torch, 4, slots, hidden, rank).bfloat16().cuda(),
                              torch.tensor([0.5, 1.0, 2.0]).cuda())
    g1, g2 = (1 + 0.1 * randn(torch, s, hidden).cuda() for s in (5, 6))

    def step(x, residual, ids, targets):
        h = zb.rms_norm_quantize(x, g1, residual=residual, normed=True)
        y = zb.matmul_codes(h.codes, h.row_scale, w1)
        zb.add_low_rank(y, h.normed, pool.a, pool.b, ids, scales=pool.scales)
        f = zb.rms_norm_quantize(y, g2, residual=h.residual)
        logits = zb.matmul_codes(f.codes, f.row_scale, w2)
        return logits, zb.token_logprobs(logits, targets, top_k=5)

    return step, (w1, w2, pool, g1, g2)


def step_inputs(torch, m, hidden=256, vocab=1000, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [t.cuda() for t in (randn(torch, seed + 10, m, hidden), randn(torch, seed + 11, m, hidden),
                               torch.randint(-1, 3, (m,), generator=g, dtype=torch.int32),
                               torch.randint(0, vocab, (m,), generator=g))]


@pytest.mark.parametrize("m", [1, 7, 40, 300])
def test_step_together(zb, torch, m):
    """Against the same step with every operator's own oracle on the one
    before's actual output."""
    step, (w1, w2, pool, g1, g2) = make_step(zb, torch)
    x, residual, ids, targets = step_inputs(torch, m)
    logits, lp = step(x, residual, ids, targets)
    codes, scale, total, v = norm_oracle(torch, x.cpu(), residual.cpu(), g1.cpu(), 1e-5)
    y = zb.matmul(v.cuda(), w1)  # quantizes v to the same codes
    want, tol = adapter_oracle(torch, y.cpu(), v, pool.a.cpu(), pool.b.cpu(), ids.cpu(), pool.scales.cpu(), None)
    zb.add_low_rank(y, v.cuda(), pool.a, pool.b, ids, scales=pool.scales)
    assert ((y.cpu().double() - want).abs() <= tol).all()
    v2 = norm_oracle(torch, y.cpu(), total, g2.cpu(), 1e-5)[3]
    same_bits(torch, logits, zb.matmul(v2.cuda(), w2), "logits")
    wlp, went, wtop, wids, base = logprob_oracle(torch, logits.cpu(), targets.cpu()[:, None], 5)
    close(torch, lp.logprobs, wlp[:, 0], base, "logprobs")
    close(torch, lp.entropy, went, base, "entropy")
    same_bits(torch, lp.top_ids, wids, "top_ids")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k", [(6000, 5), (3000, 36), (500, 1001)])
def test_chains_of_calls(zb, torch, m, k, dtype):
    """Calls that follow one another without a pause, each on what the one
    before wrote in place, rows sharing sectors of memory: the same bits as with
    the device waited for after every call."""
    t = getattr(torch, dtype)
    w = (1 + 0.1 * randn(torch, 1, k)).cuda()
    a = (randn(torch, 2, 3, 8, k) * k**-0.5).bfloat16().cuda()
    b = (randn(torch, 3, 3, k, 8) * 8**-0.5).bfloat16().cuda()
    ids = torch.randint(-1, 3, (m,), generator=torch.Generator().manual_seed(4), dtype=torch.int32).cuda()
    W = zb.quantize((randn(torch, 5, k, k) * k**-0.5).cuda())

    def chain(pause):
        r = randn(torch, 6, m, k).to(t).cuda()
        y = randn(torch, 7, m, k).cuda()
        x = r * 2
        for i in range(12):
            h = zb.rms_norm_quantize(x, w, residual=r, residual_out=r, normed=True)
            pause()
            zb.add_low_rank(y, h.normed, a, b, ids)
            pause()
            n = zb.rms_norm_quantize(y, w, residual=y, residual_out=y, normed=True)
            pause()
            zb.add_low_rank(y, y, a, b, ids)  # x may be y: all of it is read before y is added to
            pause()
            z = zb.matmul_codes(n.codes, n.row_scale, W, out=y)
            pause()
            lp = zb.token_logprobs(y, top_k=2)
            pause()
            z = zb.matmul(y, W)
            pause()
            x = zb.rms_norm_quantize(z.to(t) if i % 2 else h.normed, w, residual=r, normed=True).normed
            pause()
        return r, y, z, lp.entropy, lp.top_ids

    want = chain(torch.cuda.synchronize)
    for _ in range(3):
        for got, ref, what in zip(chain(lambda: None), want, ("residual", "y", "matmul", "entropy", "top_ids")):
            same_bits(torch, got, ref, what)


@pytest.mark.parametrize("m", [1, 40, 300])
def test_step_in_graphs_and_streams(zb, torch, m):
    """Two captured graphs of the step, replayed in turn and on two streams at
    once with new inputs, give what the eager calls give."""
    step, _keep = make_step(zb, torch)
    sets = [step_inputs(torch, m, seed=s) for s in (1, 2)]
    graphs, outs = [], []
    for s in sets:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(*s)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(*s))
        graphs.append(graph)
    for new in ((3, 4), (5, 6)):
        fresh = [step_inputs(torch, m, seed=s) for s in new]
        want = [step(*f) for f in fresh]
        for s, f in zip(sets, fresh):
            for a, b in zip(s, f):
                a.copy_(b)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for (logits, lp), (wl, wlp) in zip(outs, want):
            same_bits(torch, logits, wl, "logits")
            for a, b in zip(lp, wlp):
                same_bits(torch, a, b, "log probabilities")


@pytest.mark.parametrize("m", [6, 40, 300])
def test_captured_linears_have_scratch_of_their_own(zb, torch, monkeypatch, m):
    """Two graphs captured on one stream, replayed at once and beside eager calls on that stream."""
    from zyron_b200 import _lib

    scratch = []
    real = _lib.lib()

    class Spy:
        def __getattr__(self, name):
            if name == "zq_matmul":
                return lambda *args: scratch.append(getattr(args[5], "value", args[5])) or real.zq_matmul(*args)
            return getattr(real, name)

    monkeypatch.setattr("zyron_b200.quantization.lib", lambda: Spy())
    lin = zb.QuantizedLinear((randn(torch, 1, 512, 384) * 0.05).cuda())
    _, x, a, b, ids, _, _ = adapter_case(torch, m, 512, 384, 3, 8, "float32", "bfloat16")
    pool = zb.LowRankAdapters(a.cuda(), b.cuda())
    xs, ids = [x.cuda(), x.cuda() * 2 + 1, x.cuda() - 3], ids.cuda()
    want = [lin(v, adapters=pool, adapter_ids=ids) for v in xs]
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        lin(xs[0])
    graphs, outs = [], []
    for v in xs[:2]:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=st):
            outs.append(lin(v, adapters=pool, adapter_ids=ids))
    others = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, other in zip(graphs, others):
            with torch.cuda.stream(other):
                graph.replay()
        with torch.cuda.stream(st):
            outs[2:] = [lin(xs[2], adapters=pool, adapter_ids=ids)]
        torch.cuda.synchronize()
        for got, ref in zip(outs, want):
            same_bits(torch, got, ref, "linear")
    eager, first, second = scratch[3], scratch[4], scratch[5]
    assert len({eager, first, second}) == 3 and set(scratch[6:]) == {eager}


def test_calls_from_threads(zb, torch):
    """Calls from several threads at once, each on a stream of its own."""
    import threading

    step, _keep = make_step(zb, torch)
    sets = [step_inputs(torch, m, seed=20 + i) for i, m in enumerate((3, 40, 300, 17))]
    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    got = [None] * len(sets)

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                got[i] = step(*sets[i])
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(sets))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for (logits, lp), (wl, wlp) in zip(got, want):
        same_bits(torch, logits, wl, "logits")
        for a, b in zip(lp, wlp):
            same_bits(torch, a, b, "log probabilities")


def test_matmul_on_another_stream(zb, torch):
    """matmul, quantize_rows and a linear with adapters on a stream that is not
    the current one: copies of their inputs run there, not behind the current
    stream's work, and their outputs' memory is that stream's."""
    st = torch.cuda.Stream()
    lin = zb.QuantizedLinear((randn(torch, 1, 96, 80) * 0.05).cuda())
    _, x, a, b, ids, scales, ranks = adapter_case(torch, 300, 96, 80, 3, 8, "float32", "bfloat16")
    pool = zb.LowRankAdapters(a.cuda(), b.cuda(), scales.cuda(), ranks.cuda())
    x, ids = x.cuda(), ids.cuda()
    cols = x.t().contiguous().t()  # rows in a transposed order are copied
    want = lin(x, adapters=pool, adapter_ids=ids), zb.matmul(x, lin.weight()), *zb.quantize_rows(x)
    lin(cols, adapters=pool, adapter_ids=ids, stream=st)  # workspaces and memory at hand on both streams
    junk = [torch.full((300, 96), math.nan, device="cuda") for _ in range(8)]
    del junk  # what a copy on the current stream would be made in
    torch.cuda.synchronize()
    torch.cuda._sleep(400_000_000)  # the current stream is busy for about 0.2 s
    got = (lin(cols, adapters=pool, adapter_ids=ids, stream=st), zb.matmul(cols, lin.weight(), stream=st),
           *zb.quantize_rows(cols, stream=st))
    st.synchronize()
    with torch.cuda.stream(st):
        host = [t.cpu() for t in got]
    assert not torch.cuda.current_stream().query()  # nothing above waited for it
    torch.cuda.synchronize()
    for g, w, what in zip(host, want, ("linear with adapters", "matmul", "codes", "row scales")):
        same_bits(torch, g, w, what)
    # given back, the memory does not go to the current stream's next tensor
    at = got[1].data_ptr()
    del got, g
    fresh = [torch.empty_like(want[1]) for _ in range(32)]
    assert at not in [t.data_ptr() for t in fresh]
    if torch.cuda.device_count() > 1:
        with pytest.raises(ValueError, match="the stream is on cuda:1"):
            zb.matmul(x, lin.weight(), stream=torch.cuda.Stream(1))


def test_calls_of_one_step_share_a_stream(zb, torch, monkeypatch):
    """On torch's default stream every call passes the same handle."""
    from zyron_b200 import _lib

    handles = {}
    real = _lib.lib()

    class Spy:
        def __getattr__(self, name):
            f = getattr(real, name)

            def call(*args):
                if name in ("zq_matmul", "zq_matmul_codes", "zq_quantize_rows", "zq_add_low_rank", "zq_rms_norm_quantize"):
                    handles[name] = getattr(args[-1], "value", args[-1])
                return f(*args)

            return call

    for module in ("zyron_b200.quantization.lib", "zyron_b200.ops.lib"):
        monkeypatch.setattr(module, lambda: Spy())
    lin = zb.QuantizedLinear((randn(torch, 1, 96, 80) * 0.05).cuda())
    _, x, a, b, ids, _, _ = adapter_case(torch, 6, 96, 80, 3, 8, "float32", "bfloat16")
    h = zb.rms_norm_quantize(x.cuda(), normed=True)
    lin(h.normed, adapters=zb.LowRankAdapters(a.cuda(), b.cuda()), adapter_ids=ids.cuda())
    zb.matmul_codes(*zb.quantize_rows(h.normed), lin.weight())
    torch.cuda.synchronize()
    assert len(handles) == 5 and len(set(handles.values())) == 1, handles


def test_stream_argument(zb, torch):
    """A call on another stream than the current one, its inputs made there."""
    st = torch.cuda.Stream()
    x, residual, ids, targets = step_inputs(torch, 300)
    pool = make_step(zb, torch)[1][2]
    w = zb.quantize((randn(torch, 1, 256, 64) * 0.05).cuda())
    torch.cuda.synchronize()
    n = zb.rms_norm_quantize(x, residual=residual, normed=True, stream=st)
    z = zb.matmul_codes(n.codes, n.row_scale, w, stream=st)
    with torch.cuda.stream(st):
        y = n.normed * 2
    zb.add_low_rank(y, n.normed, pool.a, pool.b, ids, scales=pool.scales, stream=st)
    lp = zb.token_logprobs(y, targets.clamp(max=255), top_k=3, stream=st)
    torch.cuda.synchronize()
    n2 = zb.rms_norm_quantize(x, residual=residual, normed=True)
    same_bits(torch, n.codes, n2.codes, "codes")
    same_bits(torch, z, zb.matmul_codes(n2.codes, n2.row_scale, w), "matmul_codes")
    y2 = zb.add_low_rank(n2.normed * 2, n2.normed, pool.a, pool.b, ids, scales=pool.scales)
    same_bits(torch, y, y2, "adapters")
    same_bits(torch, lp.top_ids, zb.token_logprobs(y2, top_k=3).top_ids, "top_ids")

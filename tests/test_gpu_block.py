"""The operators that complete a decoder block -- the matmul's epilogue,
append_kv and paged_attention -- against plain implementations in 64 bits,
within bounds counted from their roundings, and a block that runs them
together."""
import math

import pytest

pytestmark = pytest.mark.gpu

DTYPES = ["float32", "float16", "bfloat16"]
CACHES = ["float16", "bfloat16"]


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


def within(torch, got, want, tol, what):
    """NaN where wanted, infinities equal, elsewhere |got - want| <= tol."""
    got = got.double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fine = want.isfinite()
    assert torch.equal(got.isnan(), want.isnan()), f"{what}: NaN in other places"
    other = ~fine & ~want.isnan()
    assert torch.equal(got[other], want[other]), f"{what}: infinities differ"
    off = (got - want).abs() - tol
    bad = fine & ~(off <= 0)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}, " \
        f"{got[bad][0]} for {want[bad][0]} (allowed {tol.expand_as(want)[bad][0]})"


def half_step(torch, dtype, value):
    """Half a step of the type at the value, its smallest step at least."""
    f = torch.finfo(dtype)
    return value.abs() * (f.eps / 2) + f.smallest_normal * f.eps


# ---- the matmul's epilogue --------------------------------------------------------

def activated(torch, v, activation):
    """The activation and |t|, the exponent's size, in 64 bits."""
    if activation == "gelu":
        t = -2.0 * math.sqrt(2.0 / math.pi) * (v + 0.044715 * v**3)
    elif activation == "silu":
        t = -v
    else:
        return (v.clamp(min=0) if activation == "relu" else v), torch.zeros_like(v)
    return v * torch.sigmoid(-t), t.abs()


def epilogue_want(torch, zb, x, w, bias, activation, residual, dtype):
    """(value, tolerance) in 64 bits.  The codes and scales are the library's
    own quantizers' (tested elsewhere, bit for bit)."""
    codes, scale = zb.quantize_rows(x)
    payload = w.dequantize().double().cpu()  # codes times column scales, each product rounded once
    cols = torch.from_numpy(w.scales()).double()
    wcodes = torch.round(payload / cols)
    p = (codes.double().cpu() @ wcodes) * scale.double().cpu()[:, None] * cols
    v = p if bias is None else p + bias.double().cpu()
    a, t = activated(torch, v, activation)
    u = 2.0**-24
    # float(acc), two products and the bias's sum round once each; the slopes of
    # the activations are at most 1.13; expf is off by an ulp, the argument by
    # three roundings, 1 + e by one, the quotient by two ulps
    tol = 1.13 * (3 * u * p.abs() + u * v.abs())
    if activation in ("gelu", "silu"):
        tol = tol + a.abs() * (3 * t + 8) * u + 1e-37
    y = a
    if residual is not None:
        y = a + residual.double().cpu()
        tol = tol + u * y.abs()
    return y, tol + half_step(torch, dtype, y) + (0 if dtype == torch.float32 else tol * 2.0**-8)


EPILOGUE_SIZES = [(1, 256, 512), (2, 130, 77), (3, 40, 1003), (4, 1000, 264), (5, 128, 64), (8, 520, 200), (16, 300, 72),
                  (17, 256, 100), (130, 50, 260), (300, 512, 1000), (700, 130, 8200)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("qtype", ["Int8", "Int4"])
@pytest.mark.parametrize("m,k,n", EPILOGUE_SIZES)
def test_epilogue(zb, torch, m, k, n, qtype, dtype):
    t = getattr(torch, dtype)
    w = zb.quantize((randn(torch, n + k, k, n) * k**-0.5).cuda(), getattr(zb.Type, qtype))
    x = randn(torch, m + k, m, k).cuda()
    b = randn(torch, n, n).cuda()
    wide = (randn(torch, m, m, n + 24) * 2).to(t).cuda()
    for activation, bias, residual in ((None, None, None), ("gelu", b, None), ("gelu", None, wide[:, :n].contiguous()),
                                       ("silu", b, wide[:, 8 : 8 + n]), ("relu", b, wide[:, 3 : 3 + n]),
                                       (None, b, wide[:, :n])):
        want, tol = epilogue_want(torch, zb, x, w, bias, activation, residual, t)
        got = zb.matmul(x, w, bias=bias, activation=activation, residual=residual, dtype=t)
        assert got.dtype == t
        within(torch, got, want, tol, f"{activation} {None if residual is None else residual.stride()}")
    codes, scale = zb.quantize_rows(x)
    again = zb.matmul_codes(codes, scale, w, bias=b, activation="relu", residual=wide[:, 3 : 3 + n], dtype=t)
    first = zb.matmul(x, w, bias=b, activation="relu", residual=wide[:, 3 : 3 + n])
    assert torch.equal(first, again)


@pytest.mark.parametrize("decode", [1, 2])
@pytest.mark.parametrize("m", [1, 2, 4, 7])
def test_epilogue_decode_kernels(zb, torch, m, decode):
    w = zb.quantize((randn(torch, 1, 700, 300) * 0.04).cuda())
    w.set_decode_kernel(decode)
    x, r = randn(torch, 2, m, 700).cuda(), randn(torch, 3, m, 300).bfloat16().cuda()
    want, tol = epilogue_want(torch, zb, x, w, None, "gelu", r, torch.bfloat16)
    within(torch, zb.matmul(x, w, activation="gelu", residual=r), want, tol, f"decode {decode}")


@pytest.mark.parametrize("qtype", ["Int8", "Int4"])
@pytest.mark.parametrize("m,k,n", [(5, 1000, 9), (7, 129, 1003), (8, 4100, 48), (9, 640, 9477), (12, 2048, 9472), (16, 5000, 8)])
def test_five_to_sixteen_rows(zb, torch, m, k, n, qtype):
    """Every decode kernel's integers are exact: the same bits, and the formula's."""
    w = zb.quantize((randn(torch, 1, k, n) * 0.04).cuda(), getattr(zb.Type, qtype))
    x, r = randn(torch, 2, m, k).cuda(), randn(torch, 3, m, n).bfloat16().cuda()
    want, tol = epilogue_want(torch, zb, x, w, None, "silu", r, torch.bfloat16)
    got, plain = zb.matmul(x, w, activation="silu", residual=r), zb.matmul(x, w)
    within(torch, got, want, tol, "rows")
    codes, scale = zb.quantize_rows(x)
    assert torch.equal(zb.matmul_codes(codes, scale, w, activation="silu", residual=r), got)
    w.set_decode_kernel(1)
    assert torch.equal(zb.matmul(x, w), plain) and torch.equal(zb.matmul(x, w, activation="silu", residual=r), got)
    w.set_decode_kernel(0)
    w.set_option(2, 8)  # SMs left out
    assert torch.equal(zb.matmul(x, w), plain)


@pytest.mark.parametrize("qtype", ["Int8", "Int4"])
@pytest.mark.parametrize("m,k,n", [(17, 1000, 9), (31, 700, 4803), (32, 300, 1003), (20, 128, 14300), (33, 700, 100), (50, 129, 2405),
                                   (64, 4100, 4000), (64, 200, 4800), (65, 300, 64)])
def test_rows_up_to_sixty_four(zb, torch, m, k, n, qtype):
    """The kernel of few rows and the GEMM, by columns and type: the same bits, and the formula's."""
    w = zb.quantize((randn(torch, 1, k, n) * 0.04).cuda(), getattr(zb.Type, qtype))
    x, r, b = randn(torch, 2, m, k).cuda(), randn(torch, 3, m, n).bfloat16().cuda(), randn(torch, 4, n).cuda()
    want, tol = epilogue_want(torch, zb, x, w, b, "gelu", r, torch.bfloat16)
    got, plain = zb.matmul(x, w, bias=b, activation="gelu", residual=r), zb.matmul(x, w, bias=b)
    within(torch, got, want, tol, "rows")
    again = r.clone()
    assert torch.equal(zb.matmul(x, w, bias=b, activation="gelu", residual=again, out=again), got)
    w.set_decode_kernel(1)
    assert torch.equal(zb.matmul(x, w, bias=b), plain)


def test_nine_rows_of_a_long_int4_dot(zb, torch):
    """K past 2^17, where sixteen times the dot would pass 32 bits, at extreme codes."""
    k = (1 << 17) + 300
    w = zb.quantize((torch.ones(k, 3) * torch.tensor([1.0, -1.0, 1.0])).cuda(), zb.Type.Int4)
    x = torch.ones(9, k)
    x[4] = -1.0
    want, tol = epilogue_want(torch, zb, x.cuda(), w, None, None, None, torch.float32)
    within(torch, zb.matmul(x.cuda(), w), want, tol, "long dots")


def test_epilogue_plain_is_matmul(zb, torch):
    """float32 without anything else is the plain matmul, bit for bit, at every kernel's size."""
    for m, k, n in EPILOGUE_SIZES:
        w = zb.quantize(randn(torch, 5, k, n).cuda())
        x, b = randn(torch, 6, m, k).cuda(), randn(torch, 7, n).cuda()
        assert torch.equal(zb.matmul(x, w, bias=b, dtype=torch.float32), zb.matmul(x, w, bias=b))


@pytest.mark.parametrize("m", [1, 9, 200])
def test_epilogue_in_place_and_shapes(zb, torch, m):
    w = zb.quantize((randn(torch, 1, 96, 128) * 0.1).cuda())
    x, r = randn(torch, 2, m, 96).cuda(), randn(torch, 3, m, 128).half().cuda()
    want = zb.matmul(x, w, activation="silu", residual=r)
    y = r.clone()
    assert zb.matmul(x, w, activation="silu", residual=y, out=y).data_ptr() == y.data_ptr()
    assert torch.equal(y, want)
    three = zb.matmul(x.view(m, 1, 96), w, activation="silu", residual=r.view(m, 1, 128))
    assert three.shape == (m, 1, 128) and torch.equal(three.view(m, 128), want)
    lin = zb.QuantizedLinear(w)
    assert torch.equal(lin(x, activation="silu", residual=r), want)
    codes, scale = zb.quantize_rows(x)
    out = torch.empty(m, 128, dtype=torch.half, device="cuda")
    assert zb.matmul_codes(codes, scale, w, activation="silu", residual=r, out=out) is out and torch.equal(out, want)
    assert zb.matmul(x[:0], w, activation="gelu").shape == (0, 128)


def test_epilogue_infinities(zb, torch):
    """Overflow to a 16-bit infinity, infinities and NaN of the residual, activations far out."""
    w = zb.quantize(torch.eye(128).cuda())
    x = torch.zeros(20, 128)
    x[:, 0], x[:, 1], x[:, 2] = 1e30, -1e30, 127.0
    x[1] = 0
    x[2] = -200.0
    r = torch.zeros(20, 128, dtype=torch.half)
    r[0, 5], r[0, 6], r[0, 7] = math.inf, -math.inf, math.nan
    for activation in ("gelu", "silu", "relu"):
        y = zb.matmul(x.cuda(), w, activation=activation, residual=r.cuda()).cpu()
        assert y[0, 0] == math.inf and y[0, 1] == 0 and y[0, 5] == math.inf and y[0, 6] == -math.inf and y[0, 7].isnan()
        assert not y[1].any() and not y[2].any()
        assert y.isnan().sum() == 1


def test_epilogue_refusals_on_device(zb, torch):
    w = zb.quantize(randn(torch, 1, 64, 32).cuda())
    x = torch.zeros(4, 64, device="cuda")
    r = torch.zeros(4, 32, device="cuda")
    for call in (lambda **a: zb.matmul(x, w, **a), lambda **a: zb.matmul_codes(*zb.quantize_rows(x), w, **a),
                 lambda **a: zb.QuantizedLinear(w)(x, **a)):
        with pytest.raises(ValueError, match="activation must be"):
            call(activation="tanh")
        with pytest.raises(ValueError, match="dtype must be"):
            call(dtype=torch.float64)
        with pytest.raises(ValueError, match="residual must have shape"):
            call(residual=r[:3])
        with pytest.raises(ValueError, match="residual must have shape"):
            call(residual=r, dtype=torch.half)
        with pytest.raises(ValueError, match="residual is on cpu"):
            call(residual=r.cpu())
        with pytest.raises(ValueError, match="out must be contiguous, of shape"):
            call(residual=r.half(), out=r)
        buf = torch.zeros(4 * 32 + 8, device="cuda")
        with pytest.raises(ValueError, match="out overlaps residual"):
            call(residual=buf[8:].view(4, 32), out=buf[:-8].view(4, 32))
    with pytest.raises(ValueError, match="need a CUDA tensor"):
        zb.matmul(x.cpu().numpy(), w, activation="gelu")
    pool = zb.LowRankAdapters(torch.zeros(1, 4, 64, device="cuda").half(), torch.zeros(1, 32, 4, device="cuda").half())
    ids = torch.zeros(4, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="adapters are added to a float32 output"):
        zb.QuantizedLinear(w)(x, adapters=pool, adapter_ids=ids, activation="gelu")
    with pytest.raises(ValueError, match="adapters are added to a float32 output"):
        zb.QuantizedLinear(w)(x, adapters=pool, adapter_ids=ids, dtype=torch.half)


# ---- a paged cache ------------------------------------------------------------------

class Batch:
    """Requests over a cache whose pages are handed out in no order; everything
    that no request owns is NaN."""

    def __init__(self, torch, seed, new, lengths, page, kv, dim, dtype, prefix=0, interleave=False, spare=2):
        g = torch.Generator().manual_seed(seed)
        self.torch, self.new, self.lens, self.page, self.kv, self.dim, self.prefix = torch, new, lengths, page, kv, dim, prefix
        each = [-(-n // page) for n in lengths]
        shared = -(-prefix // page)
        total = sum(each) + shared + spare
        order = torch.randperm(total, generator=g).to(torch.int32)
        self.width = max(each + [0]) + 1
        self.pages = torch.full((len(lengths), self.width), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(each):
            self.pages[b, :n] = order[at : at + n]
            at += n
        self.prefix_pages = order[at : at + shared].clone()
        both = torch.full((total, 2, kv, page, dim), math.nan)
        self.own = []
        for b, n in enumerate(lengths):
            self.own.append(self._fill(both, self.pages[b], n, g, dtype))
        self.shared = self._fill(both, self.prefix_pages, prefix, g, dtype)
        both = both.to(dtype)
        if interleave:
            dev = both.cuda()
            self.k_cache, self.v_cache = dev[:, 0], dev[:, 1]
        else:
            self.k_cache, self.v_cache = both[:, 0].contiguous().cuda(), both[:, 1].contiguous().cuda()
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        self.rows = starts[-1]
        self.starts_host = starts
        self.starts = torch.tensor(starts, dtype=torch.int32).cuda()
        self.lengths = torch.tensor(lengths, dtype=torch.int32).cuda()
        self.dev_pages = self.pages.cuda()
        self.dev_prefix = self.prefix_pages.cuda()

    def _fill(self, both, table, n, g, dtype):
        """Random keys and values of n tokens, in the cache's type: [2, kv, n, dim] in 64 bits."""
        torch = self.torch
        kv = torch.randn(2, self.kv, n, self.dim, generator=g).to(dtype)
        j = torch.arange(n)
        both[table[j // self.page].long(), :, :, j % self.page] = kv.permute(2, 0, 1, 3).float()
        return kv.double()

    def attention(self, zb, q, **how):
        if self.prefix:
            how = {"prefix_pages": self.dev_prefix, "prefix_length": self.prefix, **how}
        return zb.paged_attention(q, self.k_cache, self.v_cache, self.dev_pages, self.lengths,
                                  **{"starts": self.starts, **how})

    def want(self, q, causal=True, scale=None, gone=()):
        """(output, tolerance) in 64 bits; `gone`: (request, token) pairs that are not in the cache."""
        torch = self.torch
        heads, dim = q.shape[1:]
        group = heads // self.kv
        scale = dim**-0.5 if scale is None else scale
        out, tol = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
        q = q.double().cpu()
        for b, (n, length) in enumerate(zip(self.new, self.lens)):
            if n == 0:
                continue
            rows = slice(self.starts_host[b], self.starts_host[b] + n)
            k = torch.cat([self.shared[0], self.own[b][0]], 1).repeat_interleave(group, 0)  # [heads, keys, dim]
            v = torch.cat([self.shared[1], self.own[b][1]], 1).repeat_interleave(group, 0)
            x = q[rows].transpose(0, 1)  # [heads, n, dim]
            key = torch.arange(self.prefix + length) - self.prefix
            at = length - n + torch.arange(n)
            seen = (key < 0) | (key <= at[:, None]) if causal else torch.ones(n, len(key), dtype=torch.bool)
            for r, j in gone:
                if r == b:
                    seen[:, self.prefix + j] = False
            s = (x @ k.transpose(1, 2)) * scale
            s = torch.where(seen, s, -math.inf)
            most = s.amax(-1, keepdim=True) if s.shape[-1] else torch.full((heads, n, 1), -math.inf).double()
            e = torch.where(seen, torch.exp(s - torch.where(most == -math.inf, 0.0, most)), 0.0)
            total = e.sum(-1, keepdim=True)
            weighted = torch.where(total == 0, 0.0, self._by_row(e, seen, v) / total)
            out[rows] = weighted.transpose(0, 1)
            # Scores: dim / 16 tensor-core steps and two more roundings of at most
            # 2^-22 of sum |q k|, the subtraction 2^-24 of the score's range, the
            # exponential 2^-22; a weight's error counts twice (itself and in the
            # sum).  Weights rounded to the cache's type add half a step of each;
            # sums of the products 2^-22 a step of 16 keys.
            big = (x.abs().nan_to_num(0, 0, 0) @ k.abs().nan_to_num(0, 0, 0).transpose(1, 2)).amax(-1, keepdim=True) \
                if s.shape[-1] else torch.zeros(heads, n, 1).double()
            size = torch.where(v.isfinite(), v, 0.0).abs()
            mean = torch.where(total > 0, torch.einsum("hnk,hkd->hnd", e.nan_to_num(0), size) / total, 0.0).nan_to_num(0)
            delta = (dim / 16 + 4) * 2.0**-22 * big * abs(scale) + 2.0**-21
            steps = (len(key) / 16 + 8) * 2.0**-22
            t = (2 * delta + steps + torch.finfo(self.k_cache.dtype).eps / 2) * mean
            tol[rows] = t.transpose(0, 1)
        return out, tol + half_step(torch, self.k_cache.dtype, out) * (1 + 2.0**-7)

    def _by_row(self, e, seen, v):
        """The weighted sums; values that are no numbers reach only the rows that see them."""
        torch = self.torch
        if v.isfinite().all():
            return torch.einsum("hnk,hkd->hnd", e, v)
        return torch.stack([torch.einsum("hk,hkd->hd", e[:, i, seen[i]], v[:, seen[i]]) for i in range(e.shape[1])], 1)


# ---- append ---------------------------------------------------------------------------

def turned(torch, x, angle, interleaved):
    """x [rows, heads, dim] in 64 bits, angle [rows, rotated / 2]."""
    half = angle.shape[1]
    x = x.clone()
    r = x[..., : 2 * half]
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :half], r[..., half:])
    c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    new = (a * c - b * s, a * s + b * c)
    x[..., : 2 * half] = torch.stack(new, -1).flatten(-2) if interleaved else torch.cat(new, -1)
    return x


def append_case(zb, torch, batch, heads, dtype, rotated, interleaved, offset, cache, one_each=False, with_q=True, qkv=True):
    """Runs append_kv and checks the queries, the stored tokens, and that nothing else changed."""
    t, ct = getattr(torch, dtype), getattr(torch, cache)
    kv, dim, rows = batch.kv, batch.dim, batch.rows
    wide = randn(torch, rows + heads, rows, (heads + 2 * kv) * dim + (0 if qkv else 1)).to(t)
    dev = wide.cuda()
    cut = lambda w, a, n: w[:, a * dim : (a + n) * dim].unflatten(1, (n, dim))  # noqa: E731
    q, k, v = (cut(wide, a, n).double() for a, n in ((0, heads), (heads, kv), (heads + kv, kv)))
    dq, dk, dv = (cut(dev, a, n) for a, n in ((0, heads), (heads, kv), (heads + kv, kv)))
    inv = (10000.0 ** (-torch.arange(rotated // 2, dtype=torch.float64) / max(rotated // 2, 1))) if rotated else None
    kc, vc = batch.k_cache.cpu().double(), batch.v_cache.cpu().double()
    at = torch.zeros(rows, dtype=torch.float64)
    touched = torch.zeros(kc.shape[0], batch.page, dtype=torch.bool)
    stored = []
    for b, (n, length) in enumerate(zip(batch.new, batch.lens)):
        for i in range(n):
            row, p = batch.starts_host[b] + i, length - n + i
            at[row] = p + offset
            page = int(batch.pages[b, p // batch.page]) if p >= 0 else -1
            if 0 <= page < kc.shape[0]:
                stored.append((row, page, p % batch.page))
                touched[page, p % batch.page] = True
    turn = (lambda x: x) if inv is None else (lambda x: turned(torch, x, at[:, None] * inv, interleaved))
    out = zb.append_kv(dq if with_q else None, dk, dv, batch.k_cache, batch.v_cache, batch.dev_pages, batch.lengths,
                       starts=None if one_each else batch.starts, inv_freq=None if inv is None else inv.cuda(),
                       interleaved=interleaved, offset=offset)
    # sine and cosine are off by 2^-23 each (the reduced angle's rounding, and the
    # polynomial's last two), and products and sum round once each
    turn_tol = lambda x: (x.abs().amax(-1, keepdim=True) * 8 * 2.0**-24) if inv is not None else 0 * x  # noqa: E731
    tol = lambda x, w: turn_tol(x) * (1 + 2.0**-7) + half_step(torch, ct, w) * (1 + 2.0**-7)  # noqa: E731
    if with_q:
        want = turn(q)
        assert out.dtype == ct and out.shape == (rows, heads, dim)
        within(torch, out, want, tol(q, want), "q")
    else:
        assert out is None
    ktol, vtol = torch.zeros_like(kc), torch.zeros_like(vc)
    wk = turn(k)
    for row, page, slot in stored:
        kc[page, :, slot], vc[page, :, slot] = wk[row], v[row]
        ktol[page, :, slot], vtol[page, :, slot] = tol(k, wk)[row], half_step(torch, ct, v[row])
    within(torch, batch.k_cache, kc, ktol, "k_cache")
    within(torch, batch.v_cache, vc, vtol, "v_cache")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("heads,kv,dim,rotated,page", [(12, 4, 64, 64, 16), (32, 8, 128, 128, 32), (5, 5, 24, 24, 8),
                                                       (6, 2, 128, 32, 64), (3, 1, 80, 48, 24), (4, 2, 40, 14, 8),
                                                       (2, 1, 8, 0, 16), (130, 2, 64, 2, 128)])
def test_append(zb, torch, heads, kv, dim, rotated, page, cache, dtype):
    for interleaved, qkv, offset in ((True, True, 0), (False, True, 99991), (True, False, 5), (False, False, 0)):
        batch = Batch(torch, dim, [3, 0, 1, 40], [3, 5, 77, 130], page, kv, dim, getattr(torch, cache), interleave=interleaved)
        append_case(zb, torch, batch, heads, dtype, rotated, interleaved, offset, cache, qkv=qkv)
    batch = Batch(torch, dim, [1] * 37, [i * 3 + 1 for i in range(37)], page, kv, dim, getattr(torch, cache))
    append_case(zb, torch, batch, heads, dtype, rotated, True, 3, cache, one_each=True)
    append_case(zb, torch, batch, heads, dtype, rotated, False, 0, cache, with_q=False)


def test_append_many_rows(zb, torch):
    """More rows than blocks of one token, more requests than one round of the search."""
    new = [(i * 7) % 5 for i in range(1500)]
    batch = Batch(torch, 1, new, [n + i % 3 for i, n in enumerate(new)], 8, 1, 16, torch.bfloat16)
    assert batch.rows > 8 * 148
    append_case(zb, torch, batch, 2, "bfloat16", 16, True, 0, "bfloat16")


@pytest.mark.parametrize("offset", [0, 1 << 20, (1 << 24) - 3, (1 << 31) + 7, 1 << 40])
def test_append_far_positions(zb, torch, offset):
    """Angles of far positions: 64 bits lose 2^-53 of the angle, which the bound has beside its own."""
    rows, dim = 64, 128
    batch = Batch(torch, 3, [rows], [rows], 64, 1, dim, torch.float16)
    q = torch.zeros(rows, 1, dim)
    q[..., : dim // 2] = 1.0  # (1, 0) -> (cos, sin)
    inv = 10000.0 ** (-torch.arange(dim // 2, dtype=torch.float64) / (dim // 2))
    z = torch.zeros(rows, 1, dim, device="cuda")
    got = zb.append_kv(q.cuda(), z, z, batch.k_cache, batch.v_cache, batch.dev_pages, batch.lengths, starts=batch.starts,
                       inv_freq=inv.cuda(), interleaved=False, offset=offset)
    angle = (torch.arange(rows, dtype=torch.float64) + offset)[:, None] * inv
    want = torch.cat([torch.cos(angle), torch.sin(angle)], 1)[:, None]
    # the product's rounding is shared with the oracle's own where both round alike; count both
    within(torch, got, want, 2.0**-22 + 2 * angle.abs().max() * 2.0**-53 + half_step(torch, torch.float16, want), "turn")


def test_append_rows_and_pages_left_alone(zb, torch):
    """Padding rows, tokens before position 0, pages outside the cache, lengths behind the table."""
    kv, dim, page = 2, 32, 16
    batch = Batch(torch, 9, [2, 5, 3], [2, 3, 40], page, kv, dim, torch.bfloat16)  # request 1: two rows too many
    batch.pages[2, 2] = 1 << 30
    batch.dev_pages = batch.pages.cuda()
    append_case(zb, torch, batch, 4, "float32", dim, True, 0, "bfloat16")
    # rows behind the last request, and none in front of the first
    batch = Batch(torch, 9, [2, 2], [2, 30], page, kv, dim, torch.bfloat16)
    batch.starts_host = [1, 3, 5]
    starts = torch.tensor(batch.starts_host, dtype=torch.int32).cuda()
    k = randn(torch, 1, 9, kv, dim).bfloat16().cuda()
    before = batch.k_cache.clone()
    out = zb.append_kv(k, k, k, batch.k_cache, batch.v_cache, batch.dev_pages, batch.lengths, starts=starts)
    assert out.shape == k.shape and torch.equal(out[1:5], k[1:5])
    changed = (batch.k_cache != before) & ~(batch.k_cache.isnan() & before.isnan())
    assert int(changed.any(-1).any(1).sum()) == 4
    # a length behind the table is cut to it, a negative one is none
    batch = Batch(torch, 9, [1, 1], [16, 16], page, kv, dim, torch.bfloat16)
    lengths = torch.tensor([1000, -5], dtype=torch.int32).cuda()
    table = batch.dev_pages[:, :1].contiguous()
    other = int(batch.pages[1, 0])
    before = batch.k_cache.clone()
    zb.append_kv(None, k[:2], k[:2], batch.k_cache, batch.v_cache, table, lengths)
    assert torch.equal(batch.k_cache[int(batch.pages[0, 0]), :, 15], k[0])
    assert torch.equal(batch.k_cache[other], before[other])


# ---- attention --------------------------------------------------------------------------

def attention_case(zb, torch, batch, heads, causal=True, scale=None, factor=1.0, **how):
    q = (randn(torch, heads + batch.rows, batch.rows, heads, batch.dim) * factor).to(batch.k_cache.dtype)
    want, tol = batch.want(q, causal, scale)
    got = batch.attention(zb, q.cuda(), causal=causal, scale=scale, **how)
    assert got.dtype == q.dtype
    within(torch, got, want, tol, "attention")
    return q, got


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("heads,kv,dim,page", [(12, 4, 64, 16), (32, 8, 128, 32), (4, 4, 128, 8), (15, 3, 80, 24), (8, 1, 24, 64),
                                               (40, 2, 72, 256), (71, 1, 64, 16), (128, 1, 128, 40), (1, 1, 8, 8)])
def test_attention(zb, torch, heads, kv, dim, page, cache):
    t = getattr(torch, cache)
    for new, lengths in (([1] * 5, [1, 64, 65, 700, 16]), ([1], [3]), ([3, 0, 7, 1], [3, 9, 130, 1]),
                         ([150, 1, 40], [150, 800, 333])):
        for prefix in (0, 37, 300):
            batch = Batch(torch, dim + page, new, lengths, page, kv, dim, t, prefix=prefix, interleave=prefix == 37)
            attention_case(zb, torch, batch, heads)
    batch = Batch(torch, dim, [4, 33], [200, 90], page, kv, dim, t)
    attention_case(zb, torch, batch, heads, causal=False)
    attention_case(zb, torch, batch, heads, scale=-0.3)
    attention_case(zb, torch, batch, heads, scale=0.0)
    batch = Batch(torch, dim, [1] * 9, [90] * 9, page, kv, dim, t, prefix=17)
    attention_case(zb, torch, batch, heads, starts=None, factor=6.0)


@pytest.mark.parametrize("prefix", [0, 130])
def test_attention_many_requests(zb, torch, prefix):
    new = [(i * 5) % 4 for i in range(700)]
    lengths = [n + (i * 37) % 90 for i, n in enumerate(new)]
    batch = Batch(torch, 4, new, lengths, 16, 2, 64, torch.bfloat16, prefix=prefix)
    attention_case(zb, torch, batch, 4)


@pytest.mark.parametrize("new", [1, 5, 200])
def test_attention_long(zb, torch, new):
    """One long request: its keys are split over the whole device."""
    batch = Batch(torch, 5, [new], [20011], 32, 2, 64, torch.float16)
    attention_case(zb, torch, batch, 6)


def test_attention_long_prompts(zb, torch):
    batch = Batch(torch, 6, [1500, 700, 1, 901], [1500, 1900, 64, 901], 64, 2, 128, torch.bfloat16)
    attention_case(zb, torch, batch, 8)
    batch = Batch(torch, 6, [600, 1, 333], [600, 40, 400], 48, 3, 64, torch.bfloat16, prefix=1000)
    attention_case(zb, torch, batch, 9)


@pytest.mark.parametrize("prefix", [0, 40])
def test_attention_rows_that_see_nothing(zb, torch, prefix):
    """No own tokens, more rows than tokens: zeros, or the prefix alone."""
    batch = Batch(torch, 7, [2, 5, 1, 300], [0, 3, 1, 100], 16, 2, 64, torch.bfloat16, prefix=prefix)
    q, got = attention_case(zb, torch, batch, 8)
    if prefix == 0:
        assert not got[:4].any()


@pytest.mark.parametrize("new", [4, 30, 200])
@pytest.mark.parametrize("cache", CACHES)
def test_attention_wild_values_do_not_spread(zb, torch, cache, new):
    """Infinities and NaN in keys and values reach the rows that see them, no others."""
    length = new + 50
    t = getattr(torch, cache)
    batch = Batch(torch, 8, [new, 3], [length, 60], 16, 2, 64, t)
    for token, what, value in ((length - 2, 1, math.nan), (length - 1, 0, math.nan), (length - new // 2, 1, math.inf),
                               (length - new // 2 + 1, 1, -math.inf)):
        page, slot = int(batch.pages[0, token // 16]), token % 16
        (batch.v_cache if what else batch.k_cache)[page, 0, slot, 5] = value
        batch.own[0][what, 0, token, 5] = value
    attention_case(zb, torch, batch, 4)


def test_attention_pages_outside(zb, torch):
    """Tokens on pages outside the cache are not seen, wherever they lie in a tile."""
    page = 24
    for new in (1, 4, 90):
        batch = Batch(torch, 10, [new, 2], [400, 70], page, 2, 80, torch.float16)
        gone = []
        for index, bad in ((1, -1), (7, 1 << 30), (400 // page, batch.k_cache.shape[0])):
            batch.pages[0, index] = bad
            gone += [(0, j) for j in range(index * page, min((index + 1) * page, 400))]
        batch.dev_pages = batch.pages.cuda()
        q = randn(torch, 1, batch.rows, 6, 80).half()
        want, tol = batch.want(q, gone=gone)
        within(torch, batch.attention(zb, q.cuda()), want, tol, f"{new} rows")


@pytest.mark.parametrize("prefix", [0, 50])
def test_attention_layouts(zb, torch, prefix):
    """Rows of a wider buffer, an output of the caller's, padding rows left as they were."""
    batch = Batch(torch, 11, [3, 90], [50, 100], 16, 2, 64, torch.bfloat16, prefix=prefix)
    wide = randn(torch, 1, batch.rows + 7, 8, 64).bfloat16()
    q = torch.zeros(batch.rows + 7, 1000, dtype=torch.bfloat16)
    q[:, 64:576] = wide.flatten(1)
    view = q.cuda()[:, 64:576].unflatten(1, (8, 64))
    out = torch.full((batch.rows + 7, 9, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    got = batch.attention(zb, view, out=out[:, :8])
    want, tol = batch.want(wide[: batch.rows])
    within(torch, got[: batch.rows], want, tol, "strided")
    assert (out[:, 8] == 7).all() and (out[batch.rows :] == 7).all()
    odd = torch.empty(batch.rows * 512 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(batch.rows, 8, 64)
    odd.copy_(wide[: batch.rows])
    assert torch.equal(batch.attention(zb, odd), got[: batch.rows])


def test_attention_determinism(zb, torch):
    batch = Batch(torch, 12, [3, 90, 1], [50, 900, 3000], 16, 2, 128, torch.bfloat16, prefix=200)
    q = randn(torch, 1, batch.rows, 8, 128).bfloat16().cuda()
    first = batch.attention(zb, q)
    for _ in range(3):
        assert torch.equal(batch.attention(zb, q), first)


def test_attention_refusals_on_device(zb, torch):
    batch = Batch(torch, 13, [1, 1], [5, 5], 16, 2, 64, torch.bfloat16)
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device="cuda")
    call = lambda q=q, k=batch.k_cache, v=batch.v_cache, p=batch.dev_pages, n=batch.lengths, **a: \
        zb.paged_attention(q, k, v, p, n, **a)  # noqa: E731
    for bad, message in (({"q": q.half()}, "q must be torch.bfloat16"), ({"q": q[:, :3]}, "multiple of kv_heads"),
                         ({"q": q[:1]}, "without starts every request has one row"),
                         ({"q": q[..., :32]}, "with dim 64"), ({"k": batch.k_cache.float(), "v": batch.v_cache.float()}, "float16 or bfloat16"),
                         ({"v": batch.v_cache[:1]}, "of one shape and type"), ({"v": batch.k_cache}, "overlap"),
                         ({"p": batch.dev_pages.long()}, "pages must be int32"), ({"n": batch.lengths[:1]}, "lengths must be"),
                         ({"starts": batch.starts[:2]}, "starts must be"), ({"prefix_length": 3}, "prefix_pages must be"),
                         ({"prefix_length": 17, "prefix_pages": batch.dev_pages[0, :1].contiguous()}, "hold prefix_length"),
                         ({"prefix_length": -1}, "prefix_length must be"), ({"scale": math.inf}, "scale must be finite"),
                         ({"out": q}, "out overlaps q"), ({"out": q.half()}, "out must have"),
                         ({"out": batch.k_cache[:1].view(2, 16, 64)[:, :4]}, "out overlaps the caches"),
                         ({"p": batch.dev_pages.cpu()}, "pages is on cpu")):
        with pytest.raises(ValueError, match=message):
            call(**bad)
    k = torch.zeros(2, 2, 64, device="cuda")
    app = lambda q=None, k=k, v=k, **a: zb.append_kv(q, k, v, batch.k_cache, batch.v_cache, batch.dev_pages, batch.lengths, **a)  # noqa: E731
    f = torch.ones(33, dtype=torch.float64, device="cuda")
    for bad, message in (({"q": q}, "q must be torch.float32"), ({"k": k.double()}, "k must be float32"), ({"v": k.half()}, "of one shape and type"),
                         ({"inv_freq": f}, "rotated must be even and at most dim"), ({"inv_freq": f.float()}, "inv_freq must be"),
                         ({"offset": -1}, "offset must be"), ({"k": k[:, :1], "v": k[:, :1]}, "caches' kv_heads"),
                         ({"q": k[:, :1]}, "multiple of kv_heads"), ({"offset": 1 << 64}, "offset must be"),
                         ({"k": batch.v_cache[0, :, :2].transpose(0, 1), "v": k.bfloat16()}, "k overlaps the caches"),
                         ({"q": batch.k_cache[0, :, :2].transpose(0, 1), "k": k.bfloat16(), "v": k.bfloat16()}, "q overlaps the caches")):
        with pytest.raises(ValueError, match=message):
            app(**bad)


def test_caches_without_pages(zb, torch):
    """Nothing is stored, nothing seen; queries are rotated all the same."""
    cache = torch.empty(0, 2, 16, 64, dtype=torch.bfloat16, device="cuda")
    pages = torch.zeros(3, 4, dtype=torch.int32, device="cuda")
    lengths = torch.tensor([40, 1, 64], dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, 40, 41, 45], dtype=torch.int32, device="cuda")
    q, k = randn(torch, 1, 45, 4, 64).bfloat16().cuda(), randn(torch, 2, 45, 2, 64).bfloat16().cuda()
    assert torch.equal(zb.append_kv(q, k, k, cache, cache.clone(), pages, lengths, starts), q)
    out = torch.full_like(q, 7)
    zb.paged_attention(q, cache, cache.clone(), pages, lengths, starts, prefix_pages=pages[0], prefix_length=60, out=out)
    assert not out.any()


@pytest.mark.parametrize("rows", [1, 40])
def test_attention_lengths_at_the_end_of_32_bits(zb, torch, rows):
    """2^31 - 1 cached tokens, as far as a table can say: those on a page count, none is read twice."""
    page = 1024
    pages = torch.full((1, 1 << 21), -1, dtype=torch.int32, device="cuda")
    pages[0, 3] = 1
    lengths = torch.tensor([2**31 - 1], dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
    kc, vc = (randn(torch, 3 + i, 2, 1, page, 64).half().cuda() for i in range(2))
    q = randn(torch, 1, rows, 4, 64).half().cuda()
    got = zb.paged_attention(q, kc, vc, pages, lengths, starts)
    short = zb.paged_attention(q, kc, vc, pages[:, 3:4].contiguous(), torch.full_like(lengths, page), starts, causal=False)
    within(torch, got, short.double().cpu(), 2.0**-10 * vc[1].abs().max().double().cpu(), "far lengths")
    k = randn(torch, 9, rows, 1, 64).half().cuda()
    before = kc.clone()
    zb.append_kv(None, k, k, kc, vc, pages, lengths, starts)
    assert torch.equal(kc, before)  # its place is on no page


# ---- streams and graphs ------------------------------------------------------------------

def test_operators_on_other_streams(zb, torch):
    """Calls on two streams at once, and on a stream given by name, give what one alone gives."""
    batch = Batch(torch, 14, [1] * 20 + [200], [300] * 20 + [400], 16, 2, 128, torch.bfloat16, prefix=500)
    q = randn(torch, 1, batch.rows, 8, 128).bfloat16().cuda()
    w = zb.quantize(randn(torch, 2, 256, 512).cuda())
    x = randn(torch, 3, 30, 256).cuda()
    want, y = batch.attention(zb, q), zb.matmul(x, w, activation="gelu", dtype=torch.half)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(5):
        for s in streams:
            got.append((batch.attention(zb, q, stream=s), zb.matmul(x, w, activation="gelu", dtype=torch.half, stream=s)))
    torch.cuda.synchronize()
    for a, b in got:
        assert torch.equal(a, want) and torch.equal(b, y)


def test_captured_calls_follow_the_batch(zb, torch):
    """Two graphs of one batch replayed in turn; lengths, starts and pages are read at the replay."""
    batch = Batch(torch, 15, [2, 1, 3], [40, 90, 33], 16, 2, 64, torch.bfloat16, prefix=20)
    q = randn(torch, 1, batch.rows, 6, 64).bfloat16()
    qd = q.cuda()
    batch.attention(zb, qd)
    torch.cuda.synchronize()
    graphs = []
    for scale in (0.1, 0.2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = batch.attention(zb, qd, scale=scale)
        graphs.append((g, scale, out))
    for lengths in ([40, 90, 33], [30, 60, 10], [0, 17, 3]):
        batch.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
        keep, full = batch.own, batch.lens
        batch.own, batch.lens = [o[:, :, :n] for o, n in zip(batch.own, lengths)], lengths
        for g, scale, out in graphs:
            g.replay()
        for g, scale, out in graphs:
            want, tol = batch.want(q, scale=scale)
            within(torch, out, want, tol, f"replay {lengths}")
        batch.own, batch.lens = keep, full


# ---- a block -----------------------------------------------------------------------------

@pytest.mark.parametrize("new,lengths,prefix", [([1] * 6, [5, 90, 33, 1, 64, 200], 0), ([1, 4, 0, 60], [1, 70, 9, 100], 48)])
def test_decoder_block(zb, torch, new, lengths, prefix):
    """Norm, q|k|v, append, attention, output projection with the residual, norm,
    up with its activation, down with the residual: each step against its
    definition on the library's own inputs of that step, and the whole captured."""
    heads, kv, dim, hidden, inner = 8, 2, 64, 256, 640
    batch = Batch(torch, 16, new, lengths, 16, kv, dim, torch.bfloat16, prefix=prefix)
    rows = batch.rows
    w = {n: zb.quantize((randn(torch, i, *s) * s[0] ** -0.5).cuda()) for i, (n, s) in enumerate(
        {"qkv": (hidden, (heads + 2 * kv) * dim), "out": (heads * dim, hidden), "up": (hidden, inner), "down": (inner, hidden)}.items())}
    norm = [(1 + 0.1 * randn(torch, i, hidden)).cuda() for i in (20, 21)]
    inv = (10000.0 ** (-torch.arange(dim // 2, dtype=torch.float64) / (dim // 2))).cuda()
    x = randn(torch, 30, rows, hidden).bfloat16().cuda()

    def block():
        h = zb.rms_norm_quantize(x, norm[0])
        qkv = zb.matmul_codes(h.codes, h.row_scale, w["qkv"], dtype=torch.bfloat16)
        q, k, v = (t.unflatten(1, (-1, dim)) for t in qkv.split([heads * dim, kv * dim, kv * dim], 1))
        q = zb.append_kv(q, k, v, batch.k_cache, batch.v_cache, batch.dev_pages, batch.lengths, starts=batch.starts,
                         inv_freq=inv, offset=prefix)
        o = batch.attention(zb, q)
        mid = zb.matmul(o.flatten(1).float(), w["out"], residual=x)
        h2 = zb.rms_norm_quantize(mid, norm[1])
        a = zb.matmul_codes(h2.codes, h2.row_scale, w["up"], activation="gelu")
        y = zb.matmul(a, w["down"], residual=mid)
        return qkv, q, o, mid, a, y, h2

    qkv, q, o, mid, a, y, h2 = block()
    # the cache now holds the new tokens: the oracle reads them back from it
    for b, (n, length) in enumerate(zip(new, lengths)):
        for i in range(length - n, length):
            page, slot = int(batch.pages[b, i // 16]), i % 16
            row = batch.starts_host[b] + i - (length - n)
            assert torch.equal(batch.v_cache[page, :, slot], qkv[row, (heads + kv) * dim :].view(kv, dim))
            batch.own[b][0, :, i] = batch.k_cache[page, :, slot].double().cpu()
            batch.own[b][1, :, i] = batch.v_cache[page, :, slot].double().cpu()
    within(torch, o, *batch.want(q.cpu()), "attention")
    within(torch, mid, *epilogue_want(torch, zb, o.flatten(1).float(), w["out"], None, None, x, torch.bfloat16), "out")
    want = zb.matmul_codes(h2.codes, h2.row_scale, w["up"]).double().cpu()
    g, t = activated(torch, want, "gelu")
    within(torch, a, g, g.abs() * (3 * t + 9) * 2.0**-24 + 1e-37, "up")
    within(torch, y, *epilogue_want(torch, zb, a, w["down"], None, None, mid, torch.bfloat16), "down")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        captured = block()
    for t in captured[:6]:
        t.zero_()
    graph.replay()
    for got, want in zip(captured[:6], (qkv, q, o, mid, a, y)):
        assert torch.equal(got, want)


@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 128), (6, 3, 64)])
def test_attention_of_many_prompts_gives_the_same_each_time(zb, torch, heads, kv_heads, dim):
    """Short and long prompts in one call, so that blocks go from parts of many key
    tiles to parts of one and back: right, and the same bits at every call."""
    import random

    rng = random.Random(heads)
    for i in range(6):
        new = [rng.choice([5, 60, 130, 257, 520, 901]) for _ in range(5)]
        lengths = [n + rng.choice([0, 0, 1, 100, 700]) for n in new]
        batch = Batch(torch, 20 + i, new, lengths, 32, kv_heads, dim, torch.bfloat16)
        q = randn(torch, 30 + i, batch.rows, heads, dim).bfloat16()
        want, tol = batch.want(q)
        first = batch.attention(zb, q.cuda())
        within(torch, first, want, tol, f"prompts {new} in {lengths}")
        for _ in range(20):
            assert torch.equal(batch.attention(zb, q.cuda()), first)


@pytest.mark.parametrize("dim,kv_heads,heads", [(64, 1, 4), (128, 1, 3), (80, 2, 10)])
def test_attention_split_over_every_block(zb, torch, dim, kv_heads, heads):
    """One item over all workers: a long cache for one token, for a draft, for a prompt, for a prefix."""
    batch = Batch(torch, 50, [1], [5000], 16, kv_heads, dim, torch.float16)
    attention_case(zb, torch, batch, heads)
    batch = Batch(torch, 51, [5, 1], [3000, 40], 16, kv_heads, dim, torch.bfloat16)
    attention_case(zb, torch, batch, heads)
    batch = Batch(torch, 52, [40], [9000], 32, kv_heads, dim, torch.bfloat16)
    attention_case(zb, torch, batch, heads)
    batch = Batch(torch, 53, [1, 0, 3], [10, 0, 30], 16, kv_heads, dim, torch.float16, prefix=7001)
    attention_case(zb, torch, batch, heads)


@pytest.mark.parametrize("heads,kv,dim,new,cached", [(8, 1, 24, [70, 0, 2000, 1, 17, 0, 0, 13000, 3, 5000], 40),
                                                     (3, 1, 128, [5, 0, 0, 700, 31, 1, 2500], 900)])
def test_append_many_rows(zb, torch, heads, kv, dim, new, cached):
    """Several rows a block, requests that begin and end inside a block's run, some empty."""
    batch = Batch(torch, 60, new, [n + cached * (i % 3) for i, n in enumerate(new)], 64, kv, dim, torch.bfloat16)
    append_case(zb, torch, batch, heads, "bfloat16", 16, False, 3, "bfloat16")

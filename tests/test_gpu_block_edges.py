"""paged_attention, append_kv and the matmul's epilogue where a rounding, an
infinity or a layout can make them wrong: against plain implementations in 64
bits, within bounds counted from their roundings."""
import math

import pytest

from test_gpu_block import CACHES, Batch, append_case, attention_case, half_step, randn, torch, within, zb  # noqa: F401 (torch and zb are fixtures)

pytestmark = pytest.mark.gpu


# ---- the weights of the attention -------------------------------------------------------

def attention64(torch, batch, q, weight_step, causal=True):
    """Output and tolerance in 64 bits, of a batch whose values are finite.  Scores: dim / 16
    tensor-core steps and two more roundings of at most 2^-22 of sum |q k|, the subtraction
    2^-24 of the scores' range, the exponential 2^-22; a weight's error counts twice (itself
    and in the sum).  Weights are off by `weight_step` of themselves beside that, sums of
    products by 2^-22 a step of 16 keys, the output by half a step of its type."""
    heads, dim = q.shape[1:]
    out, tol = (torch.zeros(q.shape, dtype=torch.float64) for _ in range(2))
    x = q.double().cpu()
    for b, (n, length) in enumerate(zip(batch.new, batch.lens)):
        rows = slice(batch.starts_host[b], batch.starts_host[b] + n)
        k, v = (torch.cat([batch.shared[i], batch.own[b][i]], 1).repeat_interleave(heads // batch.kv, 0) for i in (0, 1))
        key, at = torch.arange(batch.prefix + length) - batch.prefix, length - n + torch.arange(n)
        seen = (key < 0) | (key <= at[:, None]) | (not causal)
        mine = x[rows].transpose(0, 1)
        p = torch.softmax(torch.where(seen, mine @ k.transpose(1, 2) * dim**-0.5, -math.inf), -1)
        big = (mine.abs() @ k.abs().transpose(1, 2)).amax(-1, keepdim=True) * dim**-0.5
        delta = (dim / 16 + 4) * 2.0**-22 * big + 2.0**-21
        out[rows] = (p @ v).transpose(0, 1)
        tol[rows] = ((2 * delta + (len(key) / 16 + 8) * 2.0**-22 + weight_step) * (p @ v.abs())).transpose(0, 1)
    return out, tol + half_step(torch, q.dtype, out) * (1 + 2.0**-7)


def put(batch, torch, request, token, key=None, value=None):
    """Sets the key's first element, or the whole value, of a request's own token (None: the prefix's)."""
    own = batch.shared if request is None else batch.own[request]
    table = batch.prefix_pages if request is None else batch.pages[request]
    page, slot = int(table[token // batch.page]), token % batch.page
    if key is not None:
        batch.k_cache[page, :, slot, 0] = key
        own[0][:, token, 0] = batch.k_cache[page, :, slot, 0].double().cpu()
    if value is not None:
        batch.v_cache[page, :, slot] = value
        own[1][:, token] = batch.v_cache[page, :, slot].double().cpu()


def flat(batch, torch, mean):
    """Takes the first element out of all keys and sets the values around `mean`."""
    for cache, own in ((batch.k_cache, 0), (batch.v_cache, 1)):
        if own == 0:
            cache[..., 0] = 0
        else:
            cache += mean
        for side, table, n in [(batch.shared, batch.prefix_pages, batch.prefix)] + \
                [(o, batch.pages[b], batch.lens[b]) for b, o in enumerate(batch.own)]:
            j = torch.arange(n)
            side[own] = cache[table[j // batch.page].long().cuda(), :, (j % batch.page).cuda()].double().cpu().transpose(0, 1)


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("nats", [12, 16, 18])
@pytest.mark.parametrize("new,dim,prefix", [(1, 64, 0), (5, 128, 0), (1, 128, 300), (5, 64, 300), (200, 128, 0),
                                            (200, 64, 0), (200, 128, 300)])
def test_weights_far_below_the_largest(zb, torch, cache, nats, new, dim, prefix):
    """A key that takes nearly all weight and has no value: the output is the sum of weights
    of e^-12 to e^-18, each off by half a step of the cache's type at most."""
    t = getattr(torch, cache)
    batch = Batch(torch, nats, [new, 2], [new + 700, 90], 16, 2, dim, t, prefix=prefix)
    flat(batch, torch, 64.0)
    sink = nats * dim**0.5 / 8
    for place in ([(0, 0), (1, 0)], [(0, 300), (1, 50)], [(None, 17)]):
        if place[0][0] is None and prefix == 0:
            continue
        for request, token in place:
            put(batch, torch, request, token, key=sink, value=0.0)
        q = 0.05 * randn(torch, new, batch.rows, 4, dim)
        q[..., 0] = 8.0
        q = q.to(t)
        want, tol = attention64(torch, batch, q, torch.finfo(t).eps / 2)
        assert (want.abs() < 1).all()  # nothing but the small weights
        within(torch, batch.attention(zb, q.cuda()), want, tol, f"sink at {place}")
        for request, token in place:
            put(batch, torch, request, token, key=0.0)


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("scale", [2.0**-5, 2.0**-6, 2.0**-7, 2.0**-8, 2.0**-9])
@pytest.mark.parametrize("new", [1, 5, 100])
def test_scores_of_many_millions(zb, torch, cache, scale, new):
    """Scores so large (to 2^27) that neighbouring fp32 numbers lie whole powers of two of
    weight apart: the two largest are equal and the output is their values' mean, exactly."""
    t = getattr(torch, cache)
    batch = Batch(torch, 4, [new], [400 + new], 16, 1, 64, t)
    batch.k_cache[..., 1:] = 0
    for token in range(400 + new):  # 59392 twice, all others far below
        put(batch, torch, 0, token, key=59392.0 if token in (17, 300) else 128.0 * (token % 300), value=float(token % 7))
    q = torch.zeros(new, 4, 64, dtype=t)
    q[..., 0] = 59392.0
    got = batch.attention(zb, q.cuda(), scale=scale)
    assert torch.equal(got, torch.full_like(got, (17 % 7 + 300 % 7) / 2))


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("new", [1, 3, 100])
def test_equal_values_come_back(zb, torch, cache, new):
    """Where every key has the value 1, the output is 1.  Few rows: products and sums are off
    by less than a quarter of a step of 16 bits, so 1 is the nearest.  Many: the weights of
    the products are rounded, half a step each, those of the sum are not.  Keys up to 2^7.2
    above the first tile's largest, with weights that are no powers of two."""
    t = getattr(torch, cache)
    dim = 128
    batch = Batch(torch, 2, [new], [500 + new], 32, 2, dim, t)
    flat(batch, torch, 0.0)
    batch.v_cache[:] = 1.0
    batch.k_cache[:] *= 0.01
    for token, nats in ((3, 20), (200, 25), (333, 24), (499, 23.5)):
        put(batch, torch, 0, token, key=nats * dim**0.5 / 8)
    q = 0.01 * randn(torch, new, batch.rows, 8, dim)
    q[..., 0] = torch.linspace(8.0, 6.0, batch.rows * 8).view(batch.rows, 8)
    got = batch.attention(zb, q.to(t).cuda())
    if new * 4 <= 16:
        assert torch.equal(got, torch.ones_like(got))
    else:
        one = torch.ones(got.shape, dtype=torch.float64)
        steps = (600 / 16 + 8) * 2.0**-22
        within(torch, got, one, steps + torch.finfo(t).eps / 2 + half_step(torch, t, one), "ones")


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("new,heads,prefix", [([1] * 9, 4, 0), ([1] * 9, 4, 200), ([3, 4, 1], 8, 0)])
def test_weights_of_few_rows_are_not_rounded(zb, torch, cache, new, heads, prefix):
    """Rows of few-row items alone: the weights' two 16-bit parts hold them to 2^-17.  Values
    of both signs cancel, so that a weight rounded once (half a step each) would show."""
    t = getattr(torch, cache)
    batch = Batch(torch, 31, new, [n + 60 * (i % 3) + 20 for i, n in enumerate(new)], 16, 2, 64, t, prefix=prefix)
    if prefix:  # one row in all: the prefix's item has few rows too
        batch = Batch(torch, 31, [1], [80], 16, 2, 64, t, prefix=prefix)
    q = (0.5 * randn(torch, 5, batch.rows, heads, 64)).to(t)
    want, tol = attention64(torch, batch, q, 2.0**-17)
    within(torch, batch.attention(zb, q.cuda()), want, tol, "few rows")


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("new,lengths,dim,prefix", [([1], [700], 64, 0), ([4], [700], 128, 0), ([1, 6], [90, 641], 64, 0),
                                                    ([2, 1], [500, 65], 128, 200), ([100], [700], 128, 0), ([1] * 3, [3000, 40, 77], 80, 0)])
def test_infinities_that_are_seen(zb, torch, cache, new, lengths, dim, prefix):
    """A lone infinity in the values comes out as it is, wherever it lies among the keys; with the
    opposite one or a NaN beside it in the same element, as NaN."""
    t = getattr(torch, cache)
    batch = Batch(torch, 40, new, lengths, 16, 2, dim, t, prefix=prefix)
    for token, element, value in ((0, 1, math.inf), (11, 2, -math.inf), (33, 3, math.inf), (lengths[0] // 2, 4, -math.inf),
                                  (20, 5, math.inf), (35, 5, math.inf), (5, 6, math.inf), (lengths[0] - 9, 6, -math.inf),
                                  (12, 7, math.nan)):
        page, slot = int(batch.pages[0, token // 16]), token % 16
        batch.v_cache[page, 0, slot, element] = value
        batch.own[0][1, 0, token, element] = value
    if prefix:
        batch.v_cache[int(batch.prefix_pages[6]), 1, 3, 0] = math.inf
        batch.shared[1, 1, 6 * 16 + 3, 0] = math.inf
    q = randn(torch, 3, batch.rows, 8, dim).to(t)
    want, tol = batch.want(q)
    got = batch.attention(zb, q.cuda())
    within(torch, got, want, tol, "seen infinities")
    assert int(got.isinf().sum()) > 0


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("new,prefix", [(1, 0), (5, 0), (100, 0), (1, 30), (100, 30)])
def test_scores_of_minus_infinity(zb, torch, cache, new, prefix):
    """A key whose score is -inf has no weight; a row that has no other is zero, as one that
    sees none.  Scores of +inf are NaN."""
    t = getattr(torch, cache)
    batch = Batch(torch, 80, [new, 3, 2], [200 + new, 50, 40], 16, 1, 64, t, prefix=prefix)
    for request, some in ((0, range(200 + new)), (1, range(0, 50, 2)), (None, range(prefix))):
        for token in some:
            put(batch, torch, request, token, key=-math.inf)
    q = randn(torch, 81, batch.rows, 2, 64)
    q[..., 0] = q[..., 0].abs() + 0.1
    q[-1, :, 0] *= -1.0  # its last request: the prefix's scores are +inf
    q = q.to(t)
    want, tol = batch.want(q)
    got = batch.attention(zb, q.cuda())
    if prefix:
        want[-1] = math.nan
    within(torch, got, want, tol, "minus infinity")
    assert not got[:new].any() and got[new:-1].any()


# ---- refusals -----------------------------------------------------------------------------

@pytest.mark.parametrize("shape,message", [((3, 0, 16, 64), "kv_heads must be in"), ((3, 2, 0, 64), "page must be a multiple of 8"),
                                           ((3, 2, 16, 0), "dim must be a multiple of 8"), ((0, 0, 16, 64), "kv_heads must be in"),
                                           ((3, 0, 0, 0), "must be")])
def test_caches_without_heads_tokens_or_elements(zb, torch, shape, message):
    cache = torch.zeros(shape, dtype=torch.float16, device="cuda")
    pages, lengths = torch.zeros(2, 1, dtype=torch.int32, device="cuda"), torch.ones(2, dtype=torch.int32, device="cuda")
    q, k = (torch.zeros(2, n, shape[3], dtype=torch.float16, device="cuda") for n in (4, shape[1]))
    for call in (lambda: zb.paged_attention(q, cache, cache.clone(), pages, lengths),
                 lambda: zb.append_kv(None, k, k, cache, cache.clone(), pages, lengths)):
        with pytest.raises(zb.ZQInvalidArgument, match=message):
            call()


# ---- many requests --------------------------------------------------------------------------

@pytest.mark.parametrize("requests,most", [(1500, 5), (1100, 2), (2100, 1)])
def test_append_of_many_requests(zb, torch, requests, most):
    """More rows than blocks of one token, more requests (some empty) than two rounds of the
    search for a row's request tell apart."""
    new = [(i * 7) % most if most > 1 else int(i % 9 == 4) for i in range(requests)]
    batch = Batch(torch, 1, new, [n + i % 3 for i, n in enumerate(new)], 8, 1, 16, torch.bfloat16)
    append_case(zb, torch, batch, 2, "bfloat16", 16, True, 0, "bfloat16")


@pytest.mark.parametrize("prefix", [0, 45])
def test_attention_of_many_requests(zb, torch, prefix):
    """The same for the attention, and for the rows' two results with a prefix."""
    new = [(i * 7) % 5 if i % 100 < 60 else 0 for i in range(1500)]
    batch = Batch(torch, 70, new, [n + i % 30 for i, n in enumerate(new)], 8, 1, 32, torch.bfloat16, prefix=prefix)
    attention_case(zb, torch, batch, 4)


# ---- the matmul in place --------------------------------------------------------------------

@pytest.mark.parametrize("qtype", ["Int8", "Int4"])
@pytest.mark.parametrize("m", [1, 2, 3, 4, 5, 16, 40, 300])
def test_matmul_over_its_input(zb, torch, m, qtype):
    """x = x + W x in place: the output lies over the activations, which every block of the
    product needs, and over the residual."""
    k = 2048
    w = zb.quantize((randn(torch, 1, k, k) * 0.02).cuda(), getattr(zb.Type, qtype))
    for activation in (None, "gelu"):
        for _ in range(5):
            x = randn(torch, m, m, k).cuda()
            want = zb.matmul(x, w, activation=activation, residual=x)
            got = zb.matmul(x, w, activation=activation, residual=x, out=x)
            assert got.data_ptr() == x.data_ptr() and torch.equal(got, want)
    # without an epilogue, and over a part of it
    buffer = torch.zeros(m + 1, k, device="cuda")
    for x, y in ((buffer[:m], buffer[:m]), (buffer[:m], buffer[1:]), (buffer[1:], buffer[:m])):
        x.copy_(randn(torch, 9, m, k))
        want = zb.matmul(x, w)
        assert torch.equal(zb.matmul(x, w, out=y), want)
    # a 16-bit output in the front half
    x = randn(torch, 10, m, k).cuda()
    want = zb.matmul(x, w, dtype=torch.half)
    assert torch.equal(zb.matmul(x, w, dtype=torch.half, out=x.view(torch.half).flatten()[: m * k].view(m, k)), want)


@pytest.mark.parametrize("qtype", ["Int8", "Int4"])
@pytest.mark.parametrize("m,k,n", [(5, 4097, 4736), (16, 4097, 4744), (7, 8200, 9472), (16, 5000, 9488), (9, 4096, 4737)])
def test_few_rows_at_borders_of_the_column_rule(zb, torch, m, k, n, qtype):
    """Where blocks of 16 columns end and blocks of 32 begin: the same bits as of the
    tcgen05 kernel."""
    w = zb.quantize((randn(torch, k, k, n) * 0.05).cuda(), getattr(zb.Type, qtype))
    x, b = randn(torch, m, m, k).cuda(), randn(torch, 3, n).cuda()
    got = zb.matmul(x, w, bias=b), zb.matmul(x, w, bias=b, activation="silu", dtype=torch.half)
    w.set_decode_kernel(1)
    assert torch.equal(got[0], zb.matmul(x, w, bias=b))
    assert torch.equal(got[1], zb.matmul(x, w, bias=b, activation="silu", dtype=torch.half))


@pytest.mark.parametrize("m", [1, 9, 70])
@pytest.mark.parametrize("activation", ["gelu", "silu"])
def test_activations_far_below_zero(zb, torch, m, activation):
    """Down to where the exponential's quotient ends (2^-126): numbers to their precision, 0
    or the number below 2^-119, never more."""
    w = zb.quantize(torch.eye(128).cuda())
    x = torch.full((m, 128), -127.0)
    x[:, 1:] = -torch.arange(127.0)  # whole codes of scale 1: -0 to -126
    bias = torch.full((128,), 0.25)
    got = zb.matmul(x.cuda(), w, bias=bias.cuda(), activation=activation).double().cpu()
    v = x.double() * float(w.scales()[0]) * 127 + 0.25
    t = 2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v**3) if activation == "gelu" else v
    want = v * torch.sigmoid(t)
    # the product's and the bias's four roundings, by the activation's slope, and its own
    slope = 1.2 * torch.exp(t).clamp(max=1) * (1 + t.abs())
    slack = want.abs() * (3 * t.abs() + 8) * 2.0**-24 + 4 * 2.0**-24 * v.abs() * slope
    within(torch, got, want, slack + half_step(torch, torch.float32, want) + 2.0**-119, activation)
    assert (got[v <= 0] <= 0).all()


# ---- the activation quantizer ----------------------------------------------------------------

@pytest.mark.parametrize("m", [1, 7, 300, 1300, 5000])
@pytest.mark.parametrize("k", [1, 31, 33, 127, 129, 301, 511, 513, 1003, 1056, 1058, 2050, 2111, 2114, 4097, 4223, 4226, 6001, 8191, 8193])
def test_quantizer_of_rows_off_the_grid(zb, torch, m, k):
    """Odd lengths, and rows of whole words that lie off the 16-byte grid: the codes and
    scales of the same rows with zeros behind them, which lie on it."""
    x = randn(torch, m + k, m, k).cuda() * torch.linspace(0.0, 3.0, m, device="cuda")[:, None]
    x[m // 2, k // 2] = math.nan
    more = -k % 4 + 4
    codes, scale = zb.quantize_rows(torch.nn.functional.pad(x, (0, more)))
    got, got_scale = zb.quantize_rows(x)
    assert torch.equal(got[:, :k], codes[:, :k]) and torch.equal(got_scale, scale)
    whole = torch.nn.functional.pad(x, (0, more))
    apart = torch.empty(whole.numel() + 1, device="cuda")[1:].view_as(whole).copy_(whole)
    got, got_scale = zb.quantize_rows(apart)
    assert torch.equal(got, codes) and torch.equal(got_scale, scale)

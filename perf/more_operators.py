"""Cases of the operators that complete a decoder block over quantized
projections: what they are timed on and compared with.

Three operators of a serving step, between ``rms_norm_quantize`` and the head:

* ``matmul``: the quantized matmul with bias, activation, residual and the
  stored type in its epilogue;
* ``append``: ``append_kv``, new tokens' queries and keys rotated by their
  position, keys and values written into a paged cache;
* ``attention``: ``paged_attention``, attention of the new tokens over that
  cache, with a prefix that all requests share computed once for all of them.

``own = False`` computes the plain forms from elementary torch operations,
``own = True`` makes the library's calls.
"""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
BYTES = {"float32": 4, "float16": 2, "bfloat16": 2}


def listed():
    return [
        # One decoded token through the up projection of the decode benchmark's weight: latency, weights streamed.
        {"name": "matmul token", "op": "matmul", "rows": 1, "in": 4096, "out": 11008, "weights": "int8",
         "bias": True, "activation": "gelu", "residual": False, "dtype": "float32"},
        # A decode batch through a down projection of INT4 weights, onto a 16-bit residual stream.
        {"name": "matmul batch", "op": "matmul", "rows": 12, "in": 11008, "out": 4096, "weights": "int4",
         "bias": False, "activation": "none", "residual": True, "dtype": "bfloat16"},
        # Prompts through the up projection: the epilogue behind a large product.
        {"name": "matmul prompts", "op": "matmul", "rows": 4096, "in": 4096, "out": 11008, "weights": "int8",
         "bias": True, "activation": "gelu", "residual": False, "dtype": "bfloat16"},
        # Odd sizes, every part of the epilogue at once.
        {"name": "matmul odd", "op": "matmul", "rows": 333, "in": 2050, "out": 1003, "weights": "int8",
         "bias": True, "activation": "silu", "residual": True, "dtype": "float32"},
        # One decoded token of the benchmark's language model (12 heads over 4, 64 wide): latency.
        {"name": "append token", "op": "append", "requests": 1, "new_min": 1, "new_max": 1, "context_min": 300, "context_max": 300, "heads": 12,
         "kv_heads": 4, "dim": 64, "rotated": 64, "interleaved": True, "page": 16, "offset": 0,
         "dtype": "float32", "cache": "bfloat16"},
        # A decode batch behind a long shared prefix: far positions.
        {"name": "append batch", "op": "append", "requests": 96, "new_min": 1, "new_max": 1, "context_min": 10, "context_max": 900, "heads": 32,
         "kv_heads": 8, "dim": 128, "rotated": 128, "interleaved": False, "page": 32, "offset": 100000,
         "dtype": "float32", "cache": "float16"},
        # Prompts of several requests at once, some of them continued: bandwidth.
        {"name": "append prompts", "op": "append", "requests": 6, "new_min": 700, "new_max": 2000, "context_min": 0, "context_max": 1000,
         "heads": 32, "kv_heads": 8, "dim": 128, "rotated": 128, "interleaved": False, "page": 64, "offset": 0,
         "dtype": "bfloat16", "cache": "bfloat16"},
        # One decoded token of the benchmark's language model at the end of its context: latency.
        {"name": "attention token", "op": "attention", "requests": 1, "new_min": 1, "new_max": 1, "context_min": 575, "context_max": 575,
         "heads": 12, "kv_heads": 4, "dim": 64, "page": 16, "prefix": 0, "causal": True, "dtype": "bfloat16"},
        # A decode batch of requests of all lengths: the cache is what is read.
        {"name": "attention batch", "op": "attention", "requests": 64, "new_min": 1, "new_max": 1, "context_min": 100, "context_max": 6000,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 32, "prefix": 0, "causal": True, "dtype": "bfloat16"},
        # A decode batch that shares a long prompt, short texts of its own behind it.
        {"name": "attention shared", "op": "attention", "requests": 96, "new_min": 1, "new_max": 1, "context_min": 20, "context_max": 500,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "prefix": 16000, "causal": True, "dtype": "float16"},
        # Prompts of several requests at once, some of them continued: the products are what counts.
        {"name": "attention prompts", "op": "attention", "requests": 4, "new_min": 1000, "new_max": 2600, "context_min": 0, "context_max": 1200,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "prefix": 0, "causal": True, "dtype": "bfloat16"},
        # A few tokens a request (drafts to verify) behind a prefix, with a group, a head and pages that nothing divides.
        {"name": "attention odd", "op": "attention", "requests": 17, "new_min": 0, "new_max": 7, "context_min": 0, "context_max": 700,
         "heads": 15, "kv_heads": 3, "dim": 80, "page": 24, "prefix": 1001, "causal": True, "dtype": "float16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi, grain):
    """Log-uniform, three times in four a multiple of `grain` where it is large enough."""
    v = _log(rng, lo, hi)
    return v // grain * grain if v >= 2 * grain and rng.random() < 0.75 else v


def draw(rng):
    op = rng.choice(["matmul", "append", "attention", "attention"])
    if op == "matmul":
        rows, k, n = _log(rng, 1, 4096), _size(rng, 128, 11008, 64), _size(rng, 128, 11008, 64)
        rows = max(1, min(rows, 4096 * 4096 * 11008 // (k * n)))
        return {"op": op, "rows": rows, "in": k, "out": n, "weights": rng.choice(["int8", "int4"]),
                "bias": rng.random() < 0.5, "activation": rng.choice(["none", "gelu", "silu", "relu"]),
                "residual": rng.random() < 0.5, "dtype": rng.choice(["float32", "bfloat16", "float16"])}
    kv = rng.choice([1, 2, 4, 8, rng.randint(1, 12)])
    heads = kv * rng.choice([1, 2, 4, 8, rng.randint(1, 16)])
    dim = rng.choice([64, 64, 128, 128, 128, 8 * rng.randint(2, 16)])
    page = rng.choice([8, 16, 32, 64, 128, 8 * rng.randint(1, 32)])
    requests = _log(rng, 1, 96)
    if rng.random() < 0.5:
        fewest = newest = 1
    else:
        newest = _log(rng, 2, max(2, 8000 // requests))
        fewest = rng.choice([0, newest // 3, newest])
    if op == "append":
        low = rng.choice([0, 0, 10, 300])
        return {"op": op, "requests": requests, "new_min": fewest, "new_max": newest, "context_min": low,
                "context_max": low + _log(rng, 1, 1000), "heads": heads, "kv_heads": kv, "dim": dim, "rotated": rng.choice([dim, dim, dim // 2 // 2 * 2, 0]),
                "interleaved": rng.random() < 0.5, "page": page, "offset": rng.choice([0, 0, _log(rng, 100, 1000000)]),
                "dtype": rng.choice(["float32", "bfloat16", "float16"]), "cache": rng.choice(["bfloat16", "float16"])}
    most = max(1, min(8000, (1 << 27) // (requests * kv * dim), int(4e10) // (requests * newest * heads * dim)))
    longest = _log(rng, 1, most)
    prefix = rng.choice([0, _log(rng, 1, max(1, min(16000, int(1e11) // (requests * newest * heads * dim))))])
    return {"op": op, "requests": requests, "new_min": fewest, "new_max": newest,
            "context_min": rng.choice([0, longest // 2]), "context_max": longest, "heads": heads, "kv_heads": kv, "dim": dim, "page": page, "prefix": prefix, "causal": rng.random() < 0.8,
            "dtype": rng.choice(["bfloat16", "float16"])}


# ---- inputs ------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _spread(lo, hi, n, salt):
    """n whole numbers all over [lo, hi], in no order."""
    return [lo + int((hi - lo + 1) * (((i + 1) * 0.6180339887 + salt) % 1.0)) for i in range(n)]


def _lengths(case):
    """Each request's new tokens and its own length with them."""
    new = _spread(case["new_min"], case["new_max"], case["requests"], 0.0)
    context = _spread(case["context_min"], case["context_max"], case["requests"], 0.37)
    return new, [n + c for n, c in zip(new, context)]


def _paged(st, case, g):
    """A cache whose pages are handed out in no order: the requests' table, the prefix's pages."""
    new, lengths = _lengths(case)
    page, prefix = case["page"], case.get("prefix", 0)
    each = [-(-n // page) for n in lengths]
    shared = -(-prefix // page)
    total = sum(each) + shared + 3
    order = torch.randperm(total, generator=g, device="cuda", dtype=torch.int64).to(torch.int32)
    width = max(each) + 2  # tables have room to grow; what is behind a request's length is not read
    starts = [0]
    for n in each:
        starts.append(starts[-1] + n)
    at = torch.tensor(starts[:-1], device="cuda")[:, None] + torch.arange(width, device="cuda")
    st["pages"] = torch.where(at < torch.tensor(starts[1:], device="cuda")[:, None], order[at.clamp(max=total - 1)], -1)
    st["prefix_pages"] = order[starts[-1] : starts[-1] + shared].contiguous() if prefix else None
    st["lengths"] = torch.tensor(lengths, device="cuda", dtype=torch.int32)
    ends = [0]
    for n in new:
        ends.append(ends[-1] + n)
    st["starts"] = torch.tensor(ends, device="cuda", dtype=torch.int32)
    # what the program knows of its batch on the host
    st["rows"], st["most_new"], st["used"] = ends[-1], max(new), max(1, max(each))
    st["one_each"] = all(n == 1 for n in new)
    cache = DTYPES[case.get("cache", case["dtype"])]
    shape = (total, case["kv_heads"], page, case["dim"])
    st["k_cache"], st["v_cache"] = _normal(g, *shape).to(cache), _normal(g, *shape).to(cache)


def prepare(case, seed):
    g = _gen(seed)
    st = dict(case)
    if case["op"] == "matmul":
        rows, k, n = case["rows"], case["in"], case["out"]
        w = _normal(g, k, n) * k**-0.5
        limit = 127.0 if case["weights"] == "int8" else 7.0
        top = w.abs().amax(0)
        st["w_scale"] = torch.where(top > 0, top / torch.full_like(top, limit), 1.0)
        st["w_codes"] = _round(w / st["w_scale"]).clamp(-limit, limit).to(torch.int8)
        if own:  # the handle that a program keeps of the same codes
            import zyron_b200 as zb

            st["matrix"] = zb.quantize(w, zb.Type.Int8 if case["weights"] == "int8" else zb.Type.Int4)
        st["x"] = _normal(g, rows, k)
        st["bias_row"] = _normal(g, n) * 0.1 if case["bias"] else None
        st["onto"] = _normal(g, rows, n).to(DTYPES[case["dtype"]]) if case["residual"] else None
        return st
    _paged(st, case, g)
    t, heads, kv, dim = st["rows"], case["heads"], case["kv_heads"], case["dim"]
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "append":
        # one buffer of q | k | v rows, as the projection leaves them
        qkv = _normal(g, t, (heads + 2 * kv) * dim).to(dtype)
        st["q"] = qkv[:, : heads * dim].unflatten(1, (heads, dim))
        st["k"] = qkv[:, heads * dim : (heads + kv) * dim].unflatten(1, (kv, dim))
        st["v"] = qkv[:, (heads + kv) * dim :].unflatten(1, (kv, dim))
        half = case["rotated"] // 2
        st["inv_freq"] = None
        if half:
            st["inv_freq"] = 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    else:
        st["q"] = (_normal(g, t, heads, dim) * 1.5).to(dtype)
    return st


def _round(q):
    """To the nearest whole number, halves away from zero."""
    return torch.sign(q) * torch.floor(q.double().abs() + 0.5).float()


# ---- one pass ------------------------------------------------------------------

def run(st):
    if st["op"] == "matmul":
        return _matmul(st)
    if st["op"] == "append":
        return _append(st)
    return _attention(st)


def _matmul(st):
    x, bias, onto, dtype = st["x"], st["bias_row"], st["onto"], DTYPES[st["dtype"]]
    if own:
        import zyron_b200 as zb

        return zb.matmul(x, st["matrix"], bias=bias, activation=None if st["activation"] == "none" else st["activation"], residual=onto, dtype=dtype)
    top = x.abs().amax(1, keepdim=True)
    scale = torch.where(top > 0, top / torch.full_like(top, 127.0), 1.0)
    codes = _round(x / scale).clamp(-127, 127)
    y = codes @ st["w_codes"].float() * scale * st["w_scale"]
    if bias is not None:
        y = y + bias
    if st["activation"] == "gelu":
        y = y / (1.0 + torch.exp(-2.0 * math.sqrt(2.0 / math.pi) * (y + 0.044715 * y * y * y)))
    elif st["activation"] == "silu":
        y = y / (1.0 + torch.exp(-y))
    elif st["activation"] == "relu":
        y = y.clamp(min=0)
    if onto is not None:
        y = y + onto.float()
    return y.to(dtype)


def _row_of(st):
    """Each row's request and its place among that request's new tokens."""
    t = torch.arange(st["rows"], device="cuda")
    request = torch.searchsorted(st["starts"][1:].long(), t, right=True)
    return request, t - st["starts"].long()[request]


def _turned(x, cos, sin, interleaved):
    half = cos.shape[-1]
    x = x.float()
    if interleaved:
        a, b = x[..., 0 : 2 * half : 2], x[..., 1 : 2 * half : 2]
        r = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half : 2 * half]
        r = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([r, x[..., 2 * half :]], -1)


def _append(st):
    q, k, v, kc, vc = (st[n] for n in ("q", "k", "v", "k_cache", "v_cache"))
    if own:
        import zyron_b200 as zb

        out = zb.append_kv(q, k, v, kc, vc, st["pages"], st["lengths"], starts=None if st["one_each"] else st["starts"],
                           inv_freq=st["inv_freq"], interleaved=st["interleaved"], offset=st["offset"])
        return {"q": out, "k_cache": kc, "v_cache": vc}
    request, place = _row_of(st)
    new = st["starts"][1:] - st["starts"][:-1]
    at = (st["lengths"] - new).long()[request] + place
    q, k = q.float(), k.float()
    if st["inv_freq"] is not None:
        angle = (at + st["offset"])[:, None, None] * st["inv_freq"]
        cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
        q, k = _turned(q, cos, sin, st["interleaved"]), _turned(k, cos, sin, st["interleaved"])
    page = st["pages"][request, at // st["page"]].long()
    kc[page, :, at % st["page"]] = k.to(kc.dtype)
    vc[page, :, at % st["page"]] = v.to(vc.dtype)
    return {"q": q.to(kc.dtype), "k_cache": kc, "v_cache": vc}


def _attention(st):
    q, kc, vc = st["q"], st["k_cache"], st["v_cache"]
    if own:
        import zyron_b200 as zb

        return zb.paged_attention(q, kc, vc, st["pages"], st["lengths"],
                                  starts=None if st["one_each"] else st["starts"], prefix_pages=st["prefix_pages"],
                                  prefix_length=st["prefix"], causal=st["causal"])
    # Requests side by side, padded to the longest: [request, kv head, new token x group, ...].
    n, most, kv, dim = st["requests"], st["most_new"], st["kv_heads"], st["dim"]
    group = st["heads"] // kv
    i = torch.arange(most, device="cuda")
    new = (st["starts"][1:] - st["starts"][:-1]).long()
    rows = (st["starts"][:-1].long()[:, None] + i).clamp(max=max(st["rows"] - 1, 0))
    x = q[rows].float().unflatten(2, (kv, group)).permute(0, 2, 1, 3, 4).reshape(n, kv, most * group, dim)
    x = x * dim**-0.5
    table = st["pages"][:, : st["used"]].long().clamp(min=0)
    k = kc[table].float().permute(0, 2, 1, 3, 4).reshape(n, kv, -1, dim)
    v = vc[table].float().permute(0, 2, 1, 3, 4).reshape(n, kv, -1, dim)
    key = torch.arange(k.shape[2], device="cuda")
    length = st["lengths"].long()[:, None, None]
    last = (length - new[:, None, None] + i[:, None]) if st["causal"] else length - 1
    seen = ((key <= last) & (key < length)).expand(n, most, -1)  # [request, new token, key]
    s = (x @ k.transpose(2, 3)).unflatten(2, (most, group))
    s = torch.where(seen[:, None, :, None], s, -math.inf).flatten(2, 3)
    top = s.amax(-1, keepdim=True)
    if st["prefix"]:
        # all rows of all requests against the prefix at once
        kp = kc[st["prefix_pages"].long()].float().transpose(0, 1).reshape(kv, -1, dim)[:, : st["prefix"]]
        vp = vc[st["prefix_pages"].long()].float().transpose(0, 1).reshape(kv, -1, dim)[:, : st["prefix"]]
        xp = x.transpose(0, 1).reshape(kv, n * most * group, dim)
        sp = xp @ kp.transpose(1, 2)
        top = torch.maximum(top, sp.amax(-1).unflatten(1, (n, -1)).transpose(0, 1)[..., None])
    top = torch.where(top == -math.inf, 0.0, top)
    e = torch.exp(s - top)
    total, out = e.sum(-1, keepdim=True), e @ v
    if st["prefix"]:
        ep = torch.exp(sp - top.transpose(0, 1).reshape(kv, -1, 1))
        total = total + ep.sum(-1).unflatten(1, (n, -1)).transpose(0, 1)[..., None]
        out = out + (ep @ vp).unflatten(1, (n, -1)).transpose(0, 1)
    out = torch.where(total > 0, out / total, 0.0).unflatten(2, (most, group))
    request, place = _row_of(st)
    return out.permute(0, 2, 1, 3, 4)[request, place].flatten(1, 2).to(q.dtype)


# ---- what a pass cannot do without ----------------------------------------------

def work(case):
    if case["op"] == "matmul":
        m, k, n, size = case["rows"], case["in"], case["out"], BYTES[case["dtype"]]
        weights = k * n if case["weights"] == "int8" else k * n // 2
        return {"bytes": 4 * m * k + weights + 4 * n * (1 + case["bias"]) + m * n * size * (1 + case["residual"]),
                "flops": 2 * m * k * n}
    new, lengths = _lengths(case)
    heads, kv, dim, rows = case["heads"], case["kv_heads"], case["dim"], sum(new)
    if case["op"] == "append":
        e = rows * (heads + 2 * kv) * dim
        turned = rows * (heads + kv) * case["rotated"]
        return {"bytes": e * (BYTES[case["dtype"]] + BYTES[case["cache"]]) + 4 * (rows + 2 * case["requests"]),
                "flops": 3 * turned}
    prefix = case["prefix"]
    pairs = 0
    for t, n in zip(new, lengths):
        pairs += t * (prefix + n) - (t * (t - 1) // 2 if case["causal"] else 0)
    keys = sum(n for t, n in zip(new, lengths) if t) + prefix
    return {"bytes": 2 * (2 * rows * heads * dim + 2 * keys * kv * dim), "flops": 4 * pairs * heads * dim}


# ---- the definitions in 64 bits ---------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "matmul":
        x = st["x"]
        scale = x.abs().amax(1)
        scale = torch.where(scale > 0, scale / torch.full_like(scale, 127.0), torch.ones_like(scale))
        # the codes are defined by the quotient in fp32
        ratio = (x / scale[:, None]).double()
        codes = torch.trunc(ratio + 0.5 * torch.sign(ratio))
        y = (codes @ st["w_codes"].double()) * torch.outer(scale.double(), st["w_scale"].double())
        if st["bias_row"] is not None:
            y += st["bias_row"].double()
        if case["activation"] == "gelu":
            inner = math.sqrt(2 / math.pi) * (y + 0.044715 * y.pow(3))
            y = y * torch.sigmoid(2 * inner)
        elif case["activation"] == "silu":
            y = y * torch.sigmoid(y)
        elif case["activation"] == "relu":
            y = torch.where(y < 0, 0.0, y)
        return y if st["onto"] is None else y + st["onto"].double()
    new, lengths = _lengths(case)
    page, kv = case["page"], case["kv_heads"]
    group = case["heads"] // kv
    if case["op"] == "append":
        q, kc, vc = st["q"].double(), st["k_cache"].double(), st["v_cache"].double()
        t = 0
        for b, (n, length) in enumerate(zip(new, lengths)):
            at = torch.arange(length - n, length, device="cuda")
            k = st["k"][t : t + n].double()
            if st["inv_freq"] is not None and n:
                turn = torch.polar(torch.ones(1, device="cuda", dtype=torch.float64),
                                   (at[:, None].double() + case["offset"]) * st["inv_freq"])[:, None]
                for x in (q[t : t + n], k):
                    r = x[..., : case["rotated"]]
                    pairs = r.unflatten(-1, (-1, 2)) if case["interleaved"] else r.unflatten(-1, (2, -1)).transpose(-1, -2)
                    z = torch.view_as_real(torch.complex(pairs[..., 0], pairs[..., 1]) * turn)
                    x[..., : case["rotated"]] = z.flatten(-2) if case["interleaved"] else z.transpose(-1, -2).flatten(-2)
            where = st["pages"][b, at // page].long()
            kc[where, :, at % page] = k
            vc[where, :, at % page] = st["v"][t : t + n].double()
            t += n
        return {"q": q, "k_cache": kc, "v_cache": vc}
    out = torch.zeros_like(st["q"], dtype=torch.float64)
    t = 0
    for b, (n, length) in enumerate(zip(new, lengths)):
        table = st["pages"][b, : -(-length // page)].long()
        for h in range(kv if n else 0):
            k, v = st["k_cache"][table, h].flatten(0, 1)[:length], st["v_cache"][table, h].flatten(0, 1)[:length]
            if case["prefix"]:
                shared = st["prefix_pages"].long()
                k = torch.cat([st["k_cache"][shared, h].flatten(0, 1)[: case["prefix"]], k])
                v = torch.cat([st["v_cache"][shared, h].flatten(0, 1)[: case["prefix"]], v])
            if not len(k):
                continue
            q = st["q"][t : t + n, h * group : (h + 1) * group].double()
            s = torch.einsum("tgd,kd->tgk", q, k.double()) / math.sqrt(case["dim"])
            if case["causal"]:
                behind = torch.ones(n, len(k), device="cuda", dtype=torch.bool).triu(len(k) - n + 1)
                s.masked_fill_(behind[:, None], -math.inf)
            out[t : t + n, h * group : (h + 1) * group] = torch.softmax(s, -1) @ v.double()
        t += n
    return out

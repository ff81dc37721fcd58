"""Cases of the operators around the quantized matmul: what they are timed on
and compared with.

Three operators of a serving step whose projections are ``QuantizedMatrix``
weights:

* ``norm``: ``rms_norm_quantize``, the root-mean-square norm that adds the
  residual first and leaves the int8 codes and row scales that
  ``matmul_codes`` multiplies;
* ``adapters``: ``add_low_rank``, the low-rank adapters of many requests
  added onto a shared projection's fp32 output;
* ``logprobs``: ``token_logprobs``, log probabilities of given tokens with the
  entropy and the most likely alternatives, over a head's logits.

``own = False`` computes the plain forms from elementary torch operations,
``own = True`` makes the library's calls.
"""
import math

import torch

own = False

EPS = 1e-5
DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
BYTES = {"float32": 4, "float16": 2, "bfloat16": 2}


def listed():
    return [
        # One decoded token of a 4096-wide model: latency.
        {"name": "norm token", "op": "norm", "rows": 1, "hidden": 4096, "dtype": "float32", "residual": True,
         "normed": False, "pitch": 0},
        # A decode batch of the 768-wide benchmark model, with the float rows that adapters read.
        {"name": "norm batch", "op": "norm", "rows": 48, "hidden": 768, "dtype": "float16", "residual": True,
         "normed": True, "pitch": 0},
        # A prompt batch as wide as the prefill workload: bandwidth.
        {"name": "norm prompt", "op": "norm", "rows": 8192, "hidden": 8192, "dtype": "bfloat16", "residual": True,
         "normed": False, "pitch": 0},
        # An odd width inside a wider buffer, no residual: rows start on any element.
        {"name": "norm odd", "op": "norm", "rows": 1537, "hidden": 4099, "dtype": "float32", "residual": False,
         "normed": True, "pitch": 6},
        # One request with one adapter, one token: latency.
        {"name": "adapters token", "op": "adapters", "rows": 1, "in": 4096, "out": 4096, "slots": 8, "rank": 16,
         "ragged": False, "dtype": "float32", "wdtype": "bfloat16", "ids": "each", "none": 0.0},
        # A decode batch where most requests have an adapter of their own, of different ranks: the
        # adapters' weights are what is read.
        {"name": "adapters batch", "op": "adapters", "rows": 64, "in": 4096, "out": 11008, "slots": 48, "rank": 32,
         "ragged": True, "dtype": "float32", "wdtype": "bfloat16", "ids": "each", "none": 0.1},
        # Prompts of a dozen requests, one after the other: the output is read and written once.
        {"name": "adapters prompts", "op": "adapters", "rows": 4096, "in": 4096, "out": 4096, "slots": 12, "rank": 64,
         "ragged": False, "dtype": "float32", "wdtype": "bfloat16", "ids": "prompts", "none": 0.0},
        # Rows of few adapters in any order, with sizes that no vector load divides.
        {"name": "adapters odd", "op": "adapters", "rows": 517, "in": 2050, "out": 1003, "slots": 5, "rank": 13,
         "ragged": True, "dtype": "bfloat16", "wdtype": "float16", "ids": "each", "none": 0.25},
        # One decoded token of the benchmark model (vocabulary 16384).
        {"name": "logprobs token", "op": "logprobs", "rows": 1, "vocab": 16384, "dtype": "float32", "top": 5,
         "pitch": 0, "masked": 0.0, "spread": 3.0},
        # A decode batch over a large vocabulary, some requests restricted to few allowed tokens.
        {"name": "logprobs batch", "op": "logprobs", "rows": 48, "vocab": 131072, "dtype": "bfloat16", "top": 20,
         "pitch": 0, "masked": 0.2, "spread": 3.0},
        # Scoring a prompt's own tokens: only the best alternative is kept. Odd vocabulary.
        {"name": "logprobs score", "op": "logprobs", "rows": 2048, "vocab": 32003, "dtype": "float32", "top": 1,
         "pitch": 0, "masked": 0.0, "spread": 4.0},
        # The largest: long prompts over a large odd vocabulary stored at a padded pitch.
        {"name": "logprobs large", "op": "logprobs", "rows": 1024, "vocab": 150001, "dtype": "bfloat16", "top": 8,
         "pitch": 15, "masked": 0.05, "spread": 2.5},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi, grain):
    """Log-uniform, three times in four a multiple of `grain` where it is large enough."""
    v = _log(rng, lo, hi)
    return v // grain * grain if v >= 2 * grain and rng.random() < 0.75 else v


def draw(rng):
    op = rng.choice(["norm", "adapters", "logprobs"])
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    if op == "norm":
        hidden = _size(rng, 64, 16384, 64)
        return {"op": op, "rows": min(_log(rng, 1, 8192), (48 << 20) // hidden), "hidden": hidden, "dtype": dtype,
                "residual": rng.random() < 0.75, "normed": rng.random() < 0.5, "pitch": rng.choice([0, 0, 8, 3])}
    if op == "adapters":
        k, n = _size(rng, 128, 12288, 64), _size(rng, 128, 12288, 64)
        rank = rng.choice([4, 8, 16, 32, 64, 128, rng.randint(1, 100)])
        slots = min(_log(rng, 1, 64), max(1, (96 << 20) // (rank * (k + n))))
        rows = min(_log(rng, 1, 8192), (32 << 20) // (k + n), max(1, int(24e9) // (slots * rank * (k + n))))
        return {"op": op, "rows": max(1, rows), "in": k, "out": n, "slots": slots, "rank": rank,
                "ragged": rng.random() < 0.5, "dtype": dtype, "wdtype": rng.choice(["bfloat16", "float16"]),
                "ids": rng.choice(["each", "prompts"]), "none": rng.choice([0.0, 0.1, 0.4])}
    vocab = _size(rng, 100, 200000, 64)
    return {"op": op, "rows": min(_log(rng, 1, 4096), (128 << 20) // vocab), "vocab": vocab, "dtype": dtype,
            "top": rng.choice([0, 1, 5, 20, rng.randint(2, 32)]), "pitch": rng.choice([0, 0, 16, 7]),
            "masked": rng.choice([0.0, 0.0, 0.3]), "spread": rng.choice([1.0, 3.0, 8.0])}


# ---- inputs ------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _uniform(g, *shape):
    return torch.rand(*shape, generator=g, device="cuda")


def prepare(case, seed):
    g = _gen(seed)
    st = dict(case)
    if case["op"] == "norm":
        rows, hidden, dtype = case["rows"], case["hidden"], DTYPES[case["dtype"]]
        # Hidden states have a few channels far larger than the rest; one row in
        # fifty is a padding row of zeros.
        channel = torch.where(_uniform(g, hidden) < 0.01, 20.0, 1.0)
        live = (_uniform(g, rows, 1) < 0.98) | (torch.arange(rows, device="cuda")[:, None] == 0)
        wide = hidden + case["pitch"]
        st["x"] = (_normal(g, rows, wide) * live).to(dtype)[:, :hidden]
        st["residual"] = None
        if case["residual"]:
            r = torch.zeros(rows, wide, device="cuda")
            r[:, :hidden] = _normal(g, rows, hidden) * channel * live * 2
            st["residual"] = r.to(dtype)[:, :hidden]
        st["weight"] = 1.0 + 0.2 * _normal(g, hidden)
    elif case["op"] == "adapters":
        rows, k, n, slots, rank = (case[v] for v in ("rows", "in", "out", "slots", "rank"))
        w = DTYPES[case["wdtype"]]
        st["x"] = _normal(g, rows, k).to(DTYPES[case["dtype"]])
        st["y"] = _normal(g, rows, n)  # the shared projection's output, which the adapters are added to
        st["a"] = (_normal(g, slots, rank, k) * k**-0.5).to(w)
        st["b"] = (_normal(g, slots, n, rank) * rank**-0.5).to(w)
        st["scales"] = 0.25 + _uniform(g, slots)
        st["ranks"] = None
        if case["ragged"]:
            st["ranks"] = torch.randint(max(1, rank // 4), rank + 1, (slots,), generator=g, device="cuda",
                                        dtype=torch.int32)
        if case["ids"] == "prompts":
            # requests of different lengths, one after the other
            cuts = torch.sort(torch.randint(0, rows, (slots,), generator=g, device="cuda")).values
            request = torch.searchsorted(cuts, torch.arange(rows, device="cuda"), right=True)
            ids = torch.randint(0, slots, (slots + 1,), generator=g, device="cuda")[request]
        else:
            ids = torch.randint(0, slots, (rows,), generator=g, device="cuda")
        if rows > 1:
            ids = torch.where(_uniform(g, rows) < case["none"], -1, ids)
        st["ids"] = ids.to(torch.int32)
    else:
        rows, vocab, dtype = case["rows"], case["vocab"], DTYPES[case["dtype"]]
        logits = torch.zeros(rows, vocab + case["pitch"], dtype=dtype, device="cuda")
        for r0 in range(0, rows, 256):
            r1 = min(rows, r0 + 256)
            part = _normal(g, r1 - r0, vocab) * case["spread"]
            if case["masked"]:
                # a restricted row keeps one token in a hundred
                row = _uniform(g, r1 - r0, 1) < case["masked"]
                part.masked_fill_(row & (_uniform(g, r1 - r0, vocab) < 0.99), -math.inf)
            logits[r0:r1, :vocab] = part.to(dtype)
        st["logits"] = logits[:, :vocab]
        targets = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
        if rows > 1:  # prompt positions whose token is not asked for
            targets = torch.where(_uniform(g, rows) < 0.05, -1, targets)
        st["targets"] = targets
    return st


# ---- one pass ------------------------------------------------------------------

def run(st):
    if st["op"] == "norm":
        return _norm(st)
    if st["op"] == "adapters":
        return _adapters(st)
    return _logprobs(st)


def _norm(st):
    x, residual, weight = st["x"], st["residual"], st["weight"]
    if own:
        import zyron_b200 as zb

        # torch takes absmax / 127.0 as a product with fp32's 1/127
        r = zb.rms_norm_quantize(x, weight, residual=residual, eps=EPS, normed=st["normed"], reciprocal=True)
        return {"codes": r.codes, "row_scale": r.row_scale, "residual": r.residual, "normed": r.normed}
    s = x.float()
    total = None
    if residual is not None:
        total = (s + residual.float()).to(x.dtype)
        s = total.float()
    # The mean of squares in 64 bits: a last-bit difference there would move
    # values across the codes' rounding borders.
    mean = s.double().square().mean(-1, keepdim=True)
    v = s * (1.0 / torch.sqrt(mean + EPS)).float() * weight
    absmax = v.abs().amax(-1, keepdim=True)
    scale = torch.where(absmax > 0, absmax / 127.0, 1.0)
    q = v / scale
    codes = (torch.sign(q) * torch.floor(q.double().abs() + 0.5)).clamp(-127, 127).to(torch.int8)
    return {"codes": codes, "row_scale": scale[:, 0], "residual": total, "normed": v.to(x.dtype) if st["normed"] else None}


def _adapters(st):
    x, y, a, b, ids, scales, ranks = (st[v] for v in ("x", "y", "a", "b", "ids", "scales", "ranks"))
    if own:
        import zyron_b200 as zb

        return zb.add_low_rank(y, x, a, b, ids, scales=scales, ranks=ranks)
    slots, rank, k = a.shape
    # Every row through every adapter, then only its own one's columns kept.
    h = (x.float() @ a.float().reshape(slots * rank, k).T).reshape(-1, slots, rank)
    keep = ids[:, None] == torch.arange(slots, device=x.device)
    h = h * (keep * scales)[:, :, None]
    if ranks is not None:
        h = h * (torch.arange(rank, device=x.device) < ranks[:, None])
    y += h.reshape(-1, slots * rank) @ b.float().transpose(1, 2).reshape(slots * rank, -1)
    return y


def _logprobs(st):
    logits, targets, top = st["logits"], st["targets"], st["top"]
    if own:
        import zyron_b200 as zb

        r = zb.token_logprobs(logits, targets, top_k=top)
        return {"logprobs": r.logprobs, "entropy": r.entropy, "top_logprobs": r.top_logprobs, "top_ids": r.top_ids}
    x = logits.float()
    most = x.amax(-1, keepdim=True)
    empty = most[:, 0] == -math.inf  # no token allowed
    d = x - torch.where(empty[:, None], 0.0, most)
    e = torch.exp(d)
    total = e.sum(-1)
    log_total = torch.log(total)
    mean = torch.where(e > 0, e * d, 0.0).sum(-1) / total
    entropy = torch.where(empty, 0.0, log_total - mean)
    log_total = torch.where(empty, 0.0, log_total)[:, None]
    asked = targets >= 0
    lp = torch.where(asked, (d.gather(1, targets.clamp(min=0)[:, None]) - log_total)[:, 0], 0.0)
    out = {"logprobs": lp, "entropy": entropy, "top_logprobs": None, "top_ids": None}
    if top:
        # Order by value, then by the lower index, in one whole number.
        bits = (x + 0.0).view(torch.int32)
        bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
        key = bits * (1 << 32) + (0x7FFFFFFF - torch.arange(x.shape[1], device=x.device))
        ids = 0x7FFFFFFF - (torch.topk(key, top, dim=-1).values & 0xFFFFFFFF)
        out["top_ids"] = ids
        out["top_logprobs"] = d.gather(1, ids) - log_total
    return out


# ---- what a pass cannot do without ----------------------------------------------

def work(case):
    if case["op"] == "norm":
        e = case["rows"] * case["hidden"]
        parts = 1 + 2 * case["residual"] + case["normed"]
        return {"bytes": e * (BYTES[case["dtype"]] * parts + 1) + 4 * (case["rows"] + case["hidden"]), "flops": 8 * e}
    if case["op"] == "adapters":
        none = case["none"] if case["rows"] > 1 else 0.0
        rows = case["rows"] * (1 - none)
        requests = min(rows, case["slots"] + 1) if case["ids"] == "prompts" else rows
        used = case["slots"] * (1 - (1 - 1 / case["slots"]) ** requests)  # adapters that some row has, on average
        rank = (max(1, case["rank"] // 4) + case["rank"]) / 2 if case["ragged"] else case["rank"]
        both = case["in"] + case["out"]
        return {"bytes": rows * (case["in"] * BYTES[case["dtype"]] + 8 * case["out"]) + 2 * used * rank * both,
                "flops": 2 * rows * rank * both}
    e = case["rows"] * case["vocab"]
    return {"bytes": e * BYTES[case["dtype"]] + case["rows"] * (16 + 12 * case["top"]), "flops": 6 * e}


# ---- the definitions in 64 bits ---------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "norm":
        x = st["x"].double()
        total = None
        if st["residual"] is not None:
            total = x + st["residual"].double()
            x = total.float().to(st["x"].dtype).double()  # the norm reads the sum as it is stored
        v = x / (x.pow(2).mean(1, keepdim=True) + EPS).sqrt() * st["weight"].double()
        scale = v.abs().amax(1) / 127
        return {"codes": None, "row_scale": torch.where(scale > 0, scale, torch.ones_like(scale)), "residual": total,
                "normed": v if case["normed"] else None}
    if case["op"] == "adapters":
        y = st["y"].double()
        for s in range(case["slots"]):
            rows = (st["ids"] == s).nonzero()[:, 0]
            r = case["rank"] if st["ranks"] is None else int(st["ranks"][s])
            h = st["x"][rows].double() @ st["a"][s, :r].double().T
            y[rows] += float(st["scales"][s]) * (h @ st["b"][s, :, :r].double().T)
        return y
    lps, ents, tops = [], [], []
    for r0 in range(0, case["rows"], 128):
        x = st["logits"][r0 : r0 + 128].double()
        t = st["targets"][r0 : r0 + 128]
        norm = torch.logsumexp(x, 1)
        p = torch.exp(x - norm[:, None])
        ents.append(-torch.where(p > 0, p * (x - norm[:, None]), 0.0).sum(1).nan_to_num(0.0))
        ents[-1][norm == -math.inf] = 0.0
        norm = torch.where(norm == -math.inf, 0.0, norm)
        lps.append(torch.where(t < 0, 0.0, x.gather(1, t.clamp(min=0)[:, None])[:, 0] - norm))
        if case["top"]:
            tops.append(torch.topk(x, case["top"], dim=1).values - norm[:, None])
    return {"logprobs": torch.cat(lps), "entropy": torch.cat(ents), "top_ids": None,
            "top_logprobs": torch.cat(tops) if tops else None}

"""The operators of language models in this library and what is measured of them.

A case is a plain dict; ``kind`` says which operator it goes through:

* ``quantize`` - ``tensor.quantize``: rows of floating-point values to 8-bit integers, a scale for each row;
* ``product``  - ``tensor.matmul_int8``: the product of two matrices of 8-bit integers with a scale for each row of
  A (token) and each row of B (output channel), the bias and the ReLU that follow it;
* ``cross``    - ``gdnn.attention``: the queries of a decoder (or of an image) over an encoder's states of another
  length, with grouped heads and the padding of the encoder's batch;
* ``append``   - ``gdnn.paged_append``: new keys and values to their places in a paged cache;
* ``paged``    - ``gdnn.paged_attention``: one new token of every sequence over its paged cache.
"""
import math

import torch

own = False

_TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_BYTES = {"f16": 2, "bf16": 2, "f32": 4}


def listed():
    return [
        # the activations of a few new tokens in front of a quantised layer: what a call costs
        {"name": "quantize_8x4096", "kind": "quantize", "dtype": "bf16", "rows": 8, "cols": 4096},
        # those of a whole prompt, rows of an odd number of values
        {"name": "quantize_8192x11007", "kind": "quantize", "dtype": "f16", "rows": 8192, "cols": 11007},
        # a quantised layer while tokens are generated: the weights are read, little else
        {"name": "product_16x4096x4096", "kind": "product", "dtype": "bf16", "m": 16, "n": 4096, "k": 4096, "bias": False, "relu": False},
        # odd sizes, rows that start on odd addresses
        {"name": "product_1111x1537x777", "kind": "product", "dtype": "f32", "m": 1111, "n": 1537, "k": 777, "bias": True, "relu": True},
        # a quantised layer over a long prompt
        {"name": "product_8192", "kind": "product", "dtype": "bf16", "m": 8192, "n": 8192, "k": 8192, "bias": True, "relu": False},
        # every pixel of a latent image attends to the states of a short text
        {"name": "cross_image_77", "kind": "cross", "dtype": "f16", "batch": 16, "queries": 4096, "keys": 77, "heads": 8, "kv_heads": 8, "size": 64, "padding": "none"},
        # one new token for each sequence over the states of an audio encoder, padded to the batch's longest
        {"name": "cross_token_1500", "kind": "cross", "dtype": "bf16", "batch": 32, "queries": 1, "keys": 1500, "heads": 16, "kv_heads": 16, "size": 64, "padding": "lengths"},
        # long targets over long sources, grouped heads, sources of different lengths
        {"name": "cross_4096x8192", "kind": "cross", "dtype": "bf16", "batch": 2, "queries": 4096, "keys": 8192, "heads": 32, "kv_heads": 8, "size": 128, "padding": "lengths"},
        # the new token of each of 64 sequences goes into the cache
        {"name": "append_64", "kind": "append", "dtype": "bf16", "batch": 64, "tokens": 1, "kv_heads": 8, "size": 128, "page": 16, "longest": 4096},
        # prompts go into the cache
        {"name": "append_16x1024", "kind": "append", "dtype": "f16", "batch": 16, "tokens": 1024, "kv_heads": 8, "size": 128, "page": 64, "longest": 4096},
        # a few short conversations, pages of 16 tokens: what a call costs
        {"name": "paged_4x1000", "kind": "paged", "dtype": "f16", "batch": 4, "heads": 16, "kv_heads": 16, "size": 64, "page": 16, "longest": 1000},
        # a full server: 64 sequences of up to 8192 tokens
        {"name": "paged_64x8192", "kind": "paged", "dtype": "bf16", "batch": 64, "heads": 32, "kv_heads": 8, "size": 128, "page": 16, "longest": 8192},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """Log-uniform; half of them a multiple of 16, the rest whatever comes, odd ones among them."""
    v = _log(rng, lo, hi)
    return max(16, v // 16 * 16) if rng.random() < 0.5 else v


def draw(rng):
    kind = rng.choice(("quantize", "product", "product", "cross", "cross", "append", "paged", "paged"))
    if kind == "quantize":
        while True:
            c = {"kind": kind, "dtype": rng.choice(("f16", "bf16", "f32")), "rows": _log(rng, 1, 16384), "cols": _size(rng, 32, 16384)}
            if work(c)["bytes"] <= 2.5e8:
                return c
    if kind == "product":
        while True:
            c = {"kind": kind, "dtype": rng.choice(("f16", "bf16", "f32")), "m": _log(rng, 1, 8192), "n": _size(rng, 32, 16384),
                 "k": _size(rng, 32, 16384), "bias": rng.random() < 0.5, "relu": rng.random() < 0.3}
            if work(c)["flops"] <= 5.5e11:
                return c
    if kind == "cross":
        while True:
            kv = rng.choice((1, 2, 4, 5, 8, 12, 16))
            c = {"kind": kind, "dtype": rng.choice(("f16", "bf16")), "batch": _log(rng, 1, 32), "queries": _log(rng, 1, 4096),
                 "keys": _log(rng, 1, 16384), "heads": kv * rng.choice((1, 1, 2, 4)), "kv_heads": kv,
                 "size": rng.choice((40, 64, 64, 80, 96, 128, 128)), "padding": rng.choice(("none", "lengths", "lengths", "mask"))}
            if c["batch"] * c["heads"] * c["queries"] * c["keys"] <= 1e9 and work(c)["bytes"] <= 1e9:
                return c
    while True:
        kv = rng.choice((1, 2, 4, 8, 16))
        c = {"kind": kind, "dtype": rng.choice(("f16", "bf16")), "batch": _log(rng, 1, 128), "kv_heads": kv, "size": rng.choice((64, 80, 128, 128)),
             "page": rng.choice((8, 16, 16, 24, 32, 64, 128)), "longest": _log(rng, 16, 65536)}
        if kind == "append":
            c["tokens"] = min(c["longest"], _log(rng, 1, 1024))
        else:
            c["heads"] = kv * rng.choice((1, 2, 4, 8))
        if c["batch"] * c["longest"] * kv * c["size"] <= 5e8:
            return c


# ------------------------------------------------------------------------------------------------


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, shape, dtype, scale=1.0):
    return torch.randn(shape, generator=g, device="cuda").mul_(scale).to(_TYPES[dtype])


def _int8(g, shape):
    """Whole numbers as a row's quantisation gives them: normally distributed, none beyond +-127."""
    return torch.randn(shape, generator=g, device="cuda").mul_(32).round_().clamp_(-127, 127).to(torch.int8)


def _lengths(g, batch, longest):
    """Between an eighth of the longest and the longest; one sequence has the longest."""
    n = torch.randint(max(1, longest // 8), longest + 1, (batch,), generator=g, device="cuda", dtype=torch.int32)
    n[batch // 2] = longest
    return n


def _cache(g, c):
    """An allocator's pages after some time of use: a sequence's pages lie anywhere, spare ones between them."""
    per = -(-c["longest"] // c["page"])
    pages = c["batch"] * per + 8
    table = torch.randperm(pages, generator=g, device="cuda")[:c["batch"] * per].to(torch.int32).view(c["batch"], per)
    shape = (pages, c["page"], c["kv_heads"], c["size"])
    return table, _randn(g, shape, c["dtype"]), _randn(g, shape, c["dtype"])


def prepare(case, seed):
    c, g = case, _generator(seed)
    s = {"case": c}
    if c["kind"] == "quantize":
        # activations: some channels far larger than the others, tokens of different sizes
        x = torch.randn((c["rows"], c["cols"]), generator=g, device="cuda")
        x *= torch.exp(torch.randn((1, c["cols"]), generator=g, device="cuda")) * torch.exp(torch.randn((c["rows"], 1), generator=g, device="cuda"))
        s["x"] = x.to(_TYPES[c["dtype"]])
        s["q"] = torch.empty((c["rows"], c["cols"]), dtype=torch.int8, device="cuda")
        s["scales"] = torch.empty(c["rows"], device="cuda")
    elif c["kind"] == "product":
        s["a"], s["b"] = _int8(g, (c["m"], c["k"])), _int8(g, (c["n"], c["k"]))
        s["a_scales"] = 0.01 + 0.04 * torch.rand(c["m"], generator=g, device="cuda")
        s["b_scales"] = (0.5 + torch.rand(c["n"], generator=g, device="cuda")) / (32 * math.sqrt(c["k"]))
        s["bias"] = _randn(g, (c["n"],), c["dtype"], 0.1) if c["bias"] else None
        s["y"] = torch.empty((c["m"], c["n"]), dtype=_TYPES[c["dtype"]], device="cuda")
    elif c["kind"] == "cross":
        # one projection gives the encoder's keys and values, next to each other
        s["q"] = _randn(g, (c["batch"], c["queries"], c["heads"], c["size"]), c["dtype"], 1.5)
        s["k"], s["v"] = _randn(g, (c["batch"], c["keys"], 2, c["kv_heads"], c["size"]), c["dtype"]).unbind(2)
        s["y"] = torch.empty_like(s["q"])
        s["lengths"] = _lengths(g, c["batch"], c["keys"]) if c["padding"] == "lengths" else None
        s["mask"] = torch.rand((c["batch"], c["keys"]), generator=g, device="cuda") < 0.8 if c["padding"] == "mask" else None
    else:
        s["table"], s["k_pages"], s["v_pages"] = _cache(g, c)
        if c["kind"] == "append":
            t = c["batch"] * c["tokens"]
            s["k"], s["v"] = (_randn(g, (t, c["kv_heads"], c["size"]), c["dtype"]) for _ in range(2))
            first = torch.randint(0, c["longest"] - c["tokens"] + 1, (c["batch"], 1), generator=g, device="cuda")
            s["positions"] = (first + torch.arange(c["tokens"], device="cuda")).to(torch.int32).view(-1)
            s["sequences"] = torch.arange(c["batch"], dtype=torch.int32, device="cuda").repeat_interleave(c["tokens"])
        else:
            s["q"] = _randn(g, (c["batch"], c["heads"], c["size"]), c["dtype"], 1.5)
            s["y"] = torch.empty_like(s["q"])
            s["lengths"] = _lengths(g, c["batch"], c["longest"])
    return s


# ------------------------------------------------------------------------------------------------
# the operators in their plain form


def _quantize(s):
    x = s["x"].float()
    largest = x.abs().amax(1, keepdim=True)
    scales = (largest.double() / 127).float().clamp_min_(2.0 ** -126)
    # the quotients in 64 bits: in 32 some of those next to the middle of two whole numbers land on it
    return torch.round(x.double() / scales.double()).to(torch.int8), scales.view(-1)


def _product(s):
    y = s["a"].float() @ s["b"].float().t()  # sums of whole numbers
    y = y * s["b_scales"] * s["a_scales"].unsqueeze(1)
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if s["case"]["relu"]:
        y = y.clamp_min(0)
    return y.to(s["y"].dtype)


def _attend(q, k, v, keep):
    """q (batch, kv_heads, rows, size), k and v (batch, kv_heads, keys, size) in 32 bits, keep (batch, keys) or None."""
    p = (q @ k.transpose(-1, -2)).mul_(1 / math.sqrt(q.shape[-1]))
    if keep is not None:
        p.masked_fill_(~keep[:, None, None], -math.inf)
        v = v.masked_fill(~keep[:, None, :, None], 0)
    p.sub_(p.amax(-1, keepdim=True).clamp_min_(-1e30)).exp_()
    return (p @ v).div_(p.sum(-1, keepdim=True).clamp_min_(1e-30))


def _cross(s):
    b, lq, h, d = s["q"].shape
    kv = s["k"].shape[2]
    q = s["q"].float().transpose(1, 2).reshape(b, kv, h // kv * lq, d)
    k, v = (t.float().transpose(1, 2) for t in (s["k"], s["v"]))
    keep = s["mask"]
    if s["lengths"] is not None:
        keep = torch.arange(k.shape[2], device="cuda") < s["lengths"].unsqueeze(1)
    return _attend(q, k, v, keep).view(b, h, lq, d).transpose(1, 2).to(s["q"].dtype)


def _append(s):
    page = s["case"]["page"]
    pos = s["positions"].long()
    where = s["table"][s["sequences"].long(), pos // page].long()
    s["k_pages"][where, pos % page] = s["k"]
    s["v_pages"][where, pos % page] = s["v"]
    return s["k_pages"], s["v_pages"]


def _paged(s):
    b, h, d = s["q"].shape
    page, kv = s["case"]["page"], s["k_pages"].shape[2]
    pos = torch.arange(s["table"].shape[1] * page, device="cuda")
    where = s["table"][:, pos // page].long()
    k, v = (t[where, pos % page].float().transpose(1, 2) for t in (s["k_pages"], s["v_pages"]))
    keep = pos < s["lengths"].unsqueeze(1)
    return _attend(s["q"].float().view(b, kv, h // kv, d), k, v, keep).view(b, h, d).to(s["q"].dtype)


_PLAIN = {"quantize": _quantize, "product": _product, "cross": _cross, "append": _append, "paged": _paged}


def _own(s):
    from dlf_b200 import gdnn, tensor
    kind = s["case"]["kind"]
    if kind == "quantize":
        return tensor.quantize(s["x"], s["q"], s["scales"])
    if kind == "product":
        return tensor.matmul_int8(s["a"], s["a_scales"], s["b"], s["b_scales"], s["y"], bias=s["bias"],
                                  activation="relu" if s["case"]["relu"] else None)
    if kind == "cross":
        gdnn.attention(s["q"], s["k"], s["v"], s["y"], key_lengths=s["lengths"], key_mask=s["mask"])
        return s["y"]
    if kind == "append":
        gdnn.paged_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["positions"], s["sequences"])
        return s["k_pages"], s["v_pages"]
    gdnn.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lengths"], s["y"])
    return s["y"]


def run(state):
    return _own(state) if own else _PLAIN[state["case"]["kind"]](state)


def work(case):
    c = case
    if c["kind"] == "quantize":
        n = c["rows"] * c["cols"]
        return {"bytes": n * (_BYTES[c["dtype"]] + 1) + 4 * c["rows"], "flops": 4 * n}
    if c["kind"] == "product":
        m, n, k = c["m"], c["n"], c["k"]
        return {"bytes": (m + n) * (k + 4) + m * n * _BYTES[c["dtype"]] + (n * _BYTES[c["dtype"]] if c["bias"] else 0), "flops": 2 * m * n * k}
    row = c["kv_heads"] * c["size"] * 2  # bytes of a token's keys, or values
    if c["kind"] == "append":
        return {"bytes": 4 * c["batch"] * c["tokens"] * row, "flops": 0}
    # sequences between an eighth of the longest and the longest; a mask that keeps four fifths still reads every key
    mean = 0.5625 if c["kind"] == "paged" or c["padding"] == "lengths" else 1.0
    queries = c.get("queries", 1)
    keys = c["batch"] * mean * c.get("keys", c.get("longest"))
    return {"bytes": 2 * keys * row + 4 * c["batch"] * queries * c["heads"] * c["size"], "flops": 4 * keys * queries * c["heads"] * c["size"]}


# ------------------------------------------------------------------------------------------------
# from the definitions, in 64 bits


def _softmax_average(q, k, v, rows):
    """One query of every head against the keys `rows`: sum_j exp(q k_j / sqrt(d) - log sum_i exp(q k_i / sqrt(d))) v_j."""
    heads, d = q.shape[-2:]
    k, v = (t[rows].double() for t in (k, v))
    group = heads // k.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    if k.shape[0]:
        for head in range(heads):
            logits = torch.einsum("qd,kd->qk", q[:, head].double(), k[:, head // group]) / math.sqrt(d)
            out[:, head] = torch.exp(logits - torch.logsumexp(logits, 1, keepdim=True)) @ v[:, head // group]
    return out


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] == "quantize":
        # the scale is a 32-bit number by definition: 1/127 of the row's largest magnitude, rounded once
        scales = (s["x"].double().abs().max(1).values / 127.0).to(torch.float32)
        return None, torch.maximum(scales, torch.full_like(scales, 2.0 ** -126)).double()
    if c["kind"] == "product":
        y = torch.einsum("mk,nk->mn", s["a"].double(), s["b"].double())  # below 2^53: exact
        y = torch.einsum("mn,m,n->mn", y, s["a_scales"].double(), s["b_scales"].double())
        y = y if s["bias"] is None else s["bias"].double() + y
        return torch.where(y > 0, y, torch.zeros_like(y)) if c["relu"] else y
    if c["kind"] == "append":
        token = s["table"].long()[s["sequences"].long(), s["positions"].long() // c["page"]] * c["page"] + s["positions"].long() % c["page"]
        return tuple(t.double().flatten(0, 1).index_copy(0, token, new.double()).view(t.shape)
                     for t, new in ((s["k_pages"], s["k"]), (s["v_pages"], s["v"])))
    out = []
    for i in range(c["batch"]):
        if c["kind"] == "cross":
            n = c["keys"] if s["lengths"] is None else int(s["lengths"][i])
            rows = torch.arange(n, device="cuda") if s["mask"] is None else s["mask"][i].nonzero().view(-1)
            out.append(_softmax_average(s["q"][i], s["k"][i], s["v"][i], rows))
        else:
            rows = torch.arange(int(s["lengths"][i]), device="cuda")
            at = s["table"][i].long()[rows // c["page"]] * c["page"] + rows % c["page"]
            k, v = (t.flatten(0, 1) for t in (s["k_pages"], s["v_pages"]))
            out.append(_softmax_average(s["q"][i].unsqueeze(0), k, v, at)[0])
    return torch.stack(out)

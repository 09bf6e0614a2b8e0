"""The operators of a decode layer held in 4 bits as cases that can be timed and checked.

Projections whose weights are E2M1 codes with a power-of-two scale for each 32 along K; a key/value cache held the same
way (groups of 32 along the head), with the store of new tokens, the read of a cached prefix, and the attention that reads
it in place; and the two norms around a block (after its output, and before the next one) with the gate and the scale of
its residual between them. Widths are those of the 8B Llama layer that the benchmark and the decode step use (hidden 4096,
32 query and 8 key/value heads of 128, intermediate 14336) or generic ones around them.

A pass over decode weights or a small cache goes through several layers', as a decode step does, so that they come from
HBM.
"""

from __future__ import annotations

import math

import torch

own = False

EPS = 1e-5
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
GROUP = 32  # values that share a scale


def listed():
    return [
        # One token's QKV projection with its bias, eight layers' weights: the smallest product of a decode loop.
        {"name": "token_qkv", "op": "linear", "rows": 1, "n": 6144, "k": 4096, "layers": 8, "dtype": "bf16",
         "bias": "fp32", "act": "none", "add": "none"},
        # 13 sequences through the gate and up projections with SwiGLU, two layers' weights.
        {"name": "batch_gate_up", "op": "linear", "rows": 13, "n": 28672, "k": 4096, "layers": 2, "dtype": "fp16",
         "bias": "none", "act": "swiglu", "add": "none"},
        # An odd number of sequences through a layer of odd widths with everything in its epilogue.
        {"name": "odd_gelu", "op": "linear", "rows": 29, "n": 5003, "k": 2051, "layers": 4, "dtype": "fp16",
         "bias": "fp16", "act": "gelu", "add": "fp32"},
        # A short prompt (or many sequences) through the down projection with the residual: the matrix cores.
        {"name": "prompt_down", "op": "linear", "rows": 384, "n": 4096, "k": 14336, "layers": 2, "dtype": "bf16",
         "bias": "none", "act": "none", "add": "bf16"},
        # One token between two blocks: latency and launch.
        {"name": "token_norm", "op": "norm", "rows": 1, "n": 4096, "dtype": "fp16", "wdtype": "fp16", "gate": "none",
         "scale": 1.0, "view": False},
        # A long prompt (or a batch of them) between two blocks with a gate a channel: streaming.
        {"name": "prompt_norm", "op": "norm", "rows": 8192, "n": 4096, "dtype": "bf16", "wdtype": "bf16",
         "gate": "channel", "scale": 0.5, "view": False},
        # 8 sequences append a token each to caches of pages, and their short prefixes are read.
        {"name": "token_store", "op": "store", "batch": 8, "new": 1, "ctx": 130, "heads": 8, "dim": 128, "page": 64,
         "ragged": 0.5, "dtype": "fp16", "layers": 1},
        # A chunk of 4 prompts is appended and the prefixes are read for its attention: streaming.
        {"name": "prompt_store", "op": "store", "batch": 4, "new": 2048, "ctx": 8192, "heads": 8, "dim": 128,
         "page": 256, "ragged": 0.0, "dtype": "bf16", "layers": 1},
        # One sequence of a thousand tokens, one new token, eight layers' caches: latency.
        {"name": "token_attend", "op": "attend", "batch": 1, "new": 1, "ctx": 1000, "heads": 8, "group": 4, "dim": 128,
         "page": 0, "ragged": 0.0, "dtype": "fp16", "layers": 8},
        # Five drafted tokens of seven sequences, odd heads, pages that end inside a tile.
        {"name": "draft_attend", "op": "attend", "batch": 7, "new": 5, "ctx": 3001, "heads": 3, "group": 5, "dim": 64,
         "page": 24, "ragged": 0.9, "dtype": "bf16", "layers": 4},
        # 32 sequences of different lengths in pages of 64: the ordinary step of a server.
        {"name": "batch_attend", "op": "attend", "batch": 32, "new": 1, "ctx": 8192, "heads": 8, "group": 4, "dim": 128,
         "page": 64, "ragged": 0.75, "dtype": "bf16", "layers": 1},
        # One long sequence: the cache split over the card.
        {"name": "long_attend", "op": "attend", "batch": 1, "new": 1, "ctx": 131072, "heads": 8, "group": 4, "dim": 128,
         "page": 256, "ragged": 0.0, "dtype": "fp16", "layers": 1},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "norm", "store", "attend", "attend"])
    dtype = rng.choice(["fp16", "bf16"])
    if op == "linear":
        act = rng.choice(["none", "none", "relu", "silu", "gelu", "gelu_tanh", "swiglu"])
        n, k = _log(rng, 256, 28672), _log(rng, 256, 14336)
        n = n // 2 * 2 if act == "swiglu" else n | 1 if rng.random() < 0.2 else max(16, n // 16 * 16)
        k = k | 1 if rng.random() < 0.2 else max(32, k // 32 * 32)
        rows = _log(rng, 1, 32) if rng.random() < 0.7 else _log(rng, 33, 384)
        layers = max(1, min(4, 200_000_000 // (n * k)))
        rows = max(1, min(rows, 45_000_000_000 // (layers * n * k)))
        return {"op": op, "rows": rows, "n": n, "k": k, "layers": layers, "dtype": dtype,
                "bias": rng.choice(["none", dtype, "fp32"]), "act": act, "add": rng.choice(["none", dtype, "fp32"])}
    if op == "norm":
        n = _log(rng, 64, 20000)
        n = n | 1 if rng.random() < 0.25 else max(8, n // 8 * 8)
        return {"op": op, "rows": _log(rng, 1, max(2, min(8192, 30_000_000 // n))), "n": n, "dtype": dtype,
                "wdtype": rng.choice([dtype, "fp32"]), "gate": rng.choice(["none", "channel", "row", "full"]),
                "scale": rng.choice([1.0, 0.22]), "view": rng.random() < 0.3}
    dim, page = rng.choice([64, 96, 128, 192, 256]), rng.choice([0, 16, 24, 64, 100, 256])
    heads = rng.choice([1, 2, 3, 4, 8, 16])
    if op == "store":
        ctx = _log(rng, 1, 8192)
        batch = _log(rng, 1, max(1.01, min(64, 30_000_000 // (ctx * heads * dim))))
        return {"op": op, "batch": batch, "new": min(ctx, _log(rng, 1, 2048)), "ctx": ctx, "heads": heads, "dim": dim,
                "page": page, "ragged": rng.choice([0.0, 0.5, 0.95]), "dtype": dtype, "layers": 1}
    ctx = _log(rng, 1, 32768)
    batch = _log(rng, 1, max(1.01, min(64, 120_000_000 // (ctx * heads * dim))))
    return {"op": op, "batch": batch, "new": min(ctx, _log(rng, 1, 16) if rng.random() < 0.4 else 1), "ctx": ctx,
            "heads": heads, "group": rng.choice([1, 2, 4, 5, 8, 16]), "dim": dim, "page": page,
            "ragged": rng.choice([0.0, 0.5, 0.95]), "dtype": dtype, "layers": 1}


# ------------------------------------------------------------------ inputs


def _rnd(g, *shape, dtype=torch.float32, scale=1.0, mean=0.0):
    t = torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)
    return t.mul_(scale).add_(mean).to(dtype)


def _codes(v):
    """E2M1 codes (one a byte) of float32 values ``[..., 32 q]`` and their groups' scales as exponent bytes: the smallest
    power of two that the group's largest magnitude is less than 7 of, values rounded to the nearest, ties to the even
    code, 6 at most."""
    g = v.reshape(*v.shape[:-1], -1, GROUP)
    top = g.abs().amax(dim=-1)
    byte = ((top.view(torch.int32) + 0x200000) >> 23) - 2
    byte = torch.where(top > 0, byte.clamp(1, 254), 127)
    a = g.abs() * ((254 - byte) << 23).view(torch.float32)[..., None]
    code = ((a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code = code + 8 * (g.view(torch.int32) < 0)
    return code.to(torch.uint8).reshape(v.shape), byte.to(torch.uint8)


def _packed(v):
    """Codes two a byte, the first in the low half, and the scales."""
    code, byte = _codes(v.float())
    return code[..., 0::2] | (code[..., 1::2] << 4), byte.view(torch.float8_e8m0fnu)


def _lengths(case):
    """Tokens of each sequence, the new ones among them: the longest, and down to a share `ragged` less."""
    ctx = case["ctx"]
    return [max(1, ctx - int(ctx * case["ragged"] * ((b * 0.618034) % 1.0))) for b in range(case["batch"])]


def _blank(case):
    """An empty cache's tensors (codes and scales of keys and values) and the table of pages: pages of the pool in an
    order of the seed's, or, without pages, a sequence's own row."""
    b, h, d, page = case["batch"], case["heads"], case["dim"], case["page"] or case["ctx"]
    per = -(-case["ctx"] // page)
    rows = b * per
    z = lambda w: torch.zeros(rows, h, page, w, dtype=torch.uint8, device="cuda")
    s = lambda: torch.full((rows, h, page, d // GROUP), 127, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu)
    return [z(d // 2), s(), z(d // 2), s()], per


def _pages(case, per, g):
    return None if not case["page"] else (torch.randperm(case["batch"] * per, generator=g, device="cuda")
                                          .to(torch.int32).reshape(case["batch"], per))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    op, dt = case["op"], DTYPES[case["dtype"]]
    s = {"op": op, "dtype": dt}
    if op == "norm":
        m, n, w = case["rows"], case["n"], DTYPES[case["wdtype"]]
        # a block's output and a residual stream with a few large channels, rows of different sizes
        x = _rnd(g, m, n + (64 if case["view"] else 0)) * (0.2 + torch.rand(m, 1, generator=g, device="cuda"))
        r = _rnd(g, m, n) * (1.0 + 2.0 * torch.rand(m, 1, generator=g, device="cuda"))
        r[:, :: max(1, n // 5)] *= 8.0
        s.update(x=x.to(dt)[:, :n], r=r.to(dt), post=_rnd(g, n, dtype=w, scale=0.1, mean=1.0),
                 w=_rnd(g, n, dtype=w, scale=0.1, mean=1.0), scale=case["scale"])
        shape = {"none": None, "channel": (n,), "row": (m, 1), "full": (m, n)}[case["gate"]]
        s["gate"] = None if shape is None else _rnd(g, *shape, dtype=dt, scale=0.3, mean=0.7)
        return s
    if op == "linear":
        m, n, k = case["rows"], case["n"], case["k"]
        kp = -(-k // GROUP) * GROUP
        s.update(x=_rnd(g, m, k, dtype=dt), act=case["act"], layers=[])
        for _ in range(case["layers"]):
            w = _rnd(g, n, kp, scale=k ** -0.5)
            w[:, k:] = 0.0
            s["layers"].append((*_packed(w), None if case["bias"] == "none"
                                else _rnd(g, n, dtype=DTYPES[case["bias"]], scale=0.5)))
        nout = n // 2 if case["act"] == "swiglu" else n
        s["add"] = None if case["add"] == "none" else _rnd(g, m, nout, dtype=DTYPES[case["add"]])
        return s
    b, h, d, new = case["batch"], case["heads"], case["dim"], case["new"]
    s["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
    # keys with a few large channels, as they have them
    loud = 1.0 + 3.0 * (torch.rand(h, 1, d, generator=g, device="cuda") < 0.05)
    s["caches"], s["count"] = [], case["ctx"]
    for _ in range(case["layers"]):
        cache, per = _blank(case)
        rows, page = cache[0].shape[0], cache[0].shape[2]
        step = max(1, 64_000_000 // (h * page * d))
        for at in range(0, rows, step):  # some pages at a time, so that inputs fit
            some = min(rows, at + step) - at
            for i, mul in ((0, loud), (2, 1.0)):
                c, e = _packed(_rnd(g, some, h, page, d) * mul)
                cache[i][at:at + some] = c
                cache[i + 1].view(torch.uint8)[at:at + some] = e.view(torch.uint8)
        s["caches"].append((cache, _pages(case, per, g)))
    if op == "store":
        s["k"], s["v"] = (_rnd(g, b, new, h, d) * loud.squeeze(1)).to(dt), _rnd(g, b, new, h, d, dtype=dt)
    else:
        s["q"] = _rnd(g, b, new, h * case["group"], d, dtype=dt)
    return s


# ------------------------------------------------------------------ passes

_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def _values(codes, scale):
    """float32 values of packed codes and their scales."""
    table = torch.tensor(_VALUES, device=codes.device)
    v = torch.stack((table[(codes & 15).int()], table[(codes >> 4).int()]), dim=-1)
    v = v.reshape(*codes.shape[:-1], -1, GROUP) * (scale.view(torch.uint8).int() << 23).view(torch.float32)[..., None]
    return v.reshape(*codes.shape[:-1], -1)


def _act(v, name):
    if name == "relu":
        return v.clamp_min(0)
    if name == "silu":
        return v / (1 + torch.exp(-v))
    if name == "gelu":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v * v * v)))
    if name == "swiglu":
        gate, up = v.chunk(2, dim=-1)
        return gate / (1 + torch.exp(-gate)) * up
    return v


def _laid_out(t, pages, count):
    """A cache tensor as its sequences see it, ``[B, heads, count, width]``."""
    if pages is not None:
        b, per = pages.shape
        t = t[pages.long()].transpose(1, 2).reshape(b, t.shape[1], per * t.shape[2], t.shape[3])
    return t[:, :, :count]


def _plain_store(s, cache, pages):
    b, new, h, d = s["k"].shape
    page = cache[0].shape[2]
    at = s["lengths"].long()[:, None] - new + torch.arange(new, device="cuda")
    seq = torch.arange(b, device="cuda")[:, None].expand_as(at)
    live = at >= 0
    seq, pos = seq[live], at[live]
    row = seq if pages is None else pages[seq, pos // page].long()
    for t, i in ((s["k"], 0), (s["v"], 2)):
        codes, scale = _packed(t)
        cache[i][row, :, pos % page] = codes[live]
        cache[i + 1].view(torch.uint8)[row, :, pos % page] = scale.view(torch.uint8)[live]
    seen = torch.arange(s["count"], device="cuda") < s["lengths"][:, None]
    out = []
    for i in (0, 2):
        v = _values(_laid_out(cache[i], pages, s["count"]),
                    _laid_out(cache[i + 1].view(torch.uint8), pages, s["count"])).transpose(1, 2)
        out.append(torch.where(seen[:, :, None, None], v, 0.0).to(s["dtype"]))
    return out


def _plain_attend(s, cache, pages):
    q = s["q"].float()
    b, new, hq, d = q.shape
    h = cache[0].shape[1]
    count = s["count"]
    k, v = (_values(_laid_out(cache[i], pages, count), _laid_out(cache[i + 1].view(torch.uint8), pages, count))
            for i in (0, 2))
    q = q.reshape(b, new, h, hq // h, d).permute(0, 2, 1, 3, 4).reshape(b, h, new * (hq // h), d)
    p = torch.matmul(q, k.transpose(2, 3).contiguous()) * d ** -0.5
    last = s["lengths"][:, None] - new + torch.arange(new, device="cuda")  # the last position that a query sees
    seen = torch.arange(count, device="cuda") <= last[..., None]
    seen = seen.repeat_interleave(hq // h, dim=1)[:, None]
    p = p.masked_fill(~seen, -math.inf)
    e = torch.where(seen, torch.exp(p - p.amax(dim=-1, keepdim=True)), 0.0)
    y = torch.matmul(e, v) / e.sum(dim=-1, keepdim=True)
    y = torch.where(seen.any(dim=-1, keepdim=True), y, 0.0)
    return y.reshape(b, h, new, hq // h, d).permute(0, 2, 1, 3, 4).reshape(b, new, hq, d).to(s["dtype"])


def _plain(s):
    if s["op"] == "norm":
        x, r = s["x"].float(), s["r"].float()
        t = x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPS) * s["post"].float() * s["scale"]
        t = r + (t if s["gate"] is None else t * s["gate"].float())
        y = t * torch.rsqrt((t * t).mean(dim=-1, keepdim=True) + EPS) * s["w"].float()
        return y.to(s["dtype"]), t.to(s["dtype"])
    if s["op"] == "linear":
        x, out = s["x"].float(), []
        for codes, scale, bias in s["layers"]:
            v = x @ _values(codes, scale)[:, : x.shape[1]].t()
            v = _act(v if bias is None else v + bias.float(), s["act"])
            out.append((v if s["add"] is None else v + s["add"].float()).to(s["dtype"]))
        return out
    form = _plain_store if s["op"] == "store" else _plain_attend
    return [form(s, cache, pages) for cache, pages in s["caches"]]


def _own(s):
    import fused_decode as fd

    if s["op"] == "norm":
        return fd.norm_add_norm(s["x"], s["r"], s["post"], s["w"], EPS, gate=s["gate"], residual_scale=s["scale"])
    if s["op"] == "linear":
        act = None if s["act"] == "none" else s["act"]
        return [fd.linear_fp4(s["x"], codes, scale, bias, activation=act, row_add=s["add"])
                for codes, scale, bias in s["layers"]]
    out = []
    for cache, pages in s["caches"]:
        cache = fd.KvCacheFp4(*cache)
        if s["op"] == "store":
            fd.append_kv_fp4(cache, s["k"], s["v"], s["lengths"], pages)
            out.append(list(fd.read_kv_fp4(cache, s["lengths"], s["count"], pages, dtype=s["dtype"])))
        else:
            out.append(fd.attend_kv_fp4(s["q"], cache, s["lengths"], pages))
    return out


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------ what a pass cannot do without


_SIZE = {"none": 0, "fp16": 2, "bf16": 2, "fp32": 4}


def work(case):
    if case["op"] == "norm":
        m, n = case["rows"], case["n"]
        gate = 2 * {"none": 0, "channel": n, "row": m, "full": m * n}[case["gate"]]
        return {"bytes": 8 * m * n + 2 * n * _SIZE[case["wdtype"]] + gate, "flops": 12 * m * n}
    if case["op"] == "linear":
        m, n, k, layers = case["rows"], case["n"], case["k"], case["layers"]
        nout, groups = n // 2 if case["act"] == "swiglu" else n, -(-k // GROUP)
        per = n * (17 * groups + _SIZE[case["bias"]]) + 2 * m * nout
        return {"bytes": layers * per + 2 * m * k + m * nout * _SIZE[case["add"]], "flops": layers * 2 * m * n * k}
    b, h, d, new, layers = case["batch"], case["heads"], case["dim"], case["new"], case["layers"]
    row = 2 * h * (d // 2 + d // GROUP)  # a token's keys and values in the cache
    tokens = sum(_lengths(case))
    if case["op"] == "store":
        return {"bytes": layers * (4 * b * new * h * d + b * new * row + tokens * row + 4 * b * case["ctx"] * h * d),
                "flops": layers * 4 * h * d * (b * new + tokens)}
    q = b * new * h * case["group"] * d
    return {"bytes": layers * (tokens * row + 4 * q), "flops": layers * 4 * new * h * case["group"] * d * tokens}


# ------------------------------------------------------------------ the definition in float64


def exact(case, seed):
    """The values in float64 (16-bit outputs before their rounding). What the cache holds is rounded by definition: the
    nearest multiple of the group's scale among the sixteen, found here by their distances."""
    s = prepare(case, seed)
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device="cuda")

    def held(codes, scale):
        n = torch.stack([codes % 16, codes // 16], dim=-1).flatten(-2).long()
        v = torch.where(n < 8, 1.0, -1.0).double() * grid[n % 8]
        return v * torch.exp2(scale.view(torch.uint8).double() - 127.0).repeat_interleave(GROUP, dim=-1)

    if case["op"] == "norm":
        x, t = s["x"].double(), s["r"].double()
        z = s["post"].double() * x / torch.sqrt(x.square().sum(dim=-1, keepdim=True) / case["n"] + EPS)
        t = t + case["scale"] * (z if s["gate"] is None else s["gate"].double() * z)
        return s["w"].double() * t / torch.sqrt(t.square().sum(dim=-1, keepdim=True) / case["n"] + EPS), t
    if case["op"] == "linear":
        out = []
        for codes, scale, bias in s["layers"]:
            v = s["x"].double() @ held(codes, scale)[:, : case["k"]].t()
            if bias is not None:
                v = v + bias.double()
            kind = case["act"]
            if kind == "relu":
                v = torch.where(v > 0, v, 0.0)
            elif kind == "silu":
                v = v * torch.sigmoid(v)
            elif kind == "gelu":
                v = v * 0.5 * torch.special.erfc(-v / math.sqrt(2.0))
            elif kind == "gelu_tanh":
                v = v * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (v + 0.044715 * v ** 3))
            elif kind == "swiglu":
                v = v[:, : case["n"] // 2] * torch.sigmoid(v[:, : case["n"] // 2]) * v[:, case["n"] // 2:]
            out.append(v if s["add"] is None else v + s["add"].double())
        return out

    def rows(t, pages, b, length):
        """What sequence b's first `length` positions hold, [heads, length, width]."""
        if pages is None:
            return t[b][:, :length]
        page = t.shape[2]
        ids = pages[b, : -(-length // page)].tolist()
        return torch.cat([t[i] for i in ids], dim=1)[:, :length]

    lengths, new, d = _lengths(case), case["new"], case["dim"]
    outs = []
    for cache, pages in s["caches"]:
        raw = [t.view(torch.uint8) for t in cache]
        if case["op"] == "store":
            pair = []
            for i, t in ((0, s["k"]), (2, s["v"])):
                y = torch.zeros(case["batch"], case["ctx"], case["heads"], d, dtype=torch.float64, device="cuda")
                for b, length in enumerate(lengths):
                    y[b, :length] = held(rows(raw[i], pages, b, length), rows(raw[i + 1], pages, b, length)).transpose(0, 1)
                    x = t[b, max(0, new - length):].double().unflatten(-1, (-1, GROUP))
                    top = x.abs().amax(dim=-1, keepdim=True)
                    unit = torch.exp2(torch.floor(torch.log2((top / 7.0).clamp_min(2.0 ** -127))) + 1.0).clamp_min(2.0 ** -126)
                    a = x.abs() / unit
                    near = (a[..., None] - grid).abs()
                    tied = near == near.amin(dim=-1, keepdim=True)  # one or two neighbours: the even one of two
                    pick = torch.where(tied & (torch.arange(8, device="cuda") % 2 == 0), 2, tied.int()).argmax(dim=-1)
                    y[b, max(0, length - new): length] = (torch.sign(x) * grid[pick] * unit).flatten(-2)
                pair.append(y)
            outs.append(pair)
            continue
        y = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        for b, length in enumerate(lengths):
            k, v = (held(rows(raw[i], pages, b, length), rows(raw[i + 1], pages, b, length)) for i in (0, 2))
            for j in range(new):
                to = length - new + j + 1
                if to <= 0:
                    continue
                q = s["q"][b, j].double().unflatten(0, (case["heads"], case["group"]))
                p = torch.softmax(q @ k[:, :to].transpose(1, 2) / math.sqrt(d), dim=-1)
                y[b, j] = (p @ v[:, :to]).flatten(0, 1)
        outs.append(y)
    return outs

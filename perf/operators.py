"""The operators with 8-bit activations as cases that can be timed and checked.

Rows are quantised to E4M3 codes with a float32 scale each (alone, after an RMSNorm, or after the residual's addition and
an RMSNorm), and codes are multiplied by E4M3 weights with the bias, an activation and the residual in the product's
epilogue. Widths are those of the 8B Llama layer that the benchmark and the decode step use (hidden 4096, 32 query and 8
key/value heads of 128, intermediate 14336) or generic ones around them.

A pass over decode weights goes through several layers' weights, as a decode step does, so that they come from HBM.
"""

from __future__ import annotations

import math

import torch

own = False

EPS = 1e-5
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0
SMALLEST = 2.0 ** -126  # a scale is a normal float32


def listed():
    return [
        # One token's norm before a projection: the smallest call of a decode loop, latency and launch.
        {"name": "token_norm", "op": "rms", "rows": 1, "n": 4096, "dtype": "fp16", "wdtype": "fp16", "view": False},
        # A batch of prompts, an odd number of rows of an odd width, with a float32 norm weight.
        {"name": "ragged_norm", "op": "rms", "rows": 1111, "n": 5001, "dtype": "bf16", "wdtype": "fp32", "view": False},
        # 16 sequences' residual addition and norm, the input the left part of a wider buffer.
        {"name": "batch_add_norm", "op": "add_rms", "rows": 16, "n": 4096, "dtype": "bf16", "wdtype": "bf16",
         "view": True},
        # The same over a long prompt (or a batch of them): streaming.
        {"name": "prompt_add_norm", "op": "add_rms", "rows": 8192, "n": 4096, "dtype": "bf16", "wdtype": "bf16",
         "view": False},
        # The attention output of 8 sequences before its projection.
        {"name": "batch_quantize", "op": "quantize", "rows": 8, "n": 4096, "dtype": "fp16", "view": False},
        # The middle of a prompt's MLP before the down projection.
        {"name": "prompt_quantize", "op": "quantize", "rows": 2048, "n": 14336, "dtype": "bf16", "view": False},
        # One token's QKV projection with its bias, eight layers' weights.
        {"name": "token_qkv", "op": "linear", "rows": 1, "n": 6144, "k": 4096, "layers": 8, "dtype": "fp16",
         "bias": "fp32", "act": "none", "add": "none"},
        # 13 sequences through the gate and up projections with SwiGLU, two layers' weights.
        {"name": "batch_gate_up", "op": "linear", "rows": 13, "n": 28672, "k": 4096, "layers": 2, "dtype": "bf16",
         "bias": "none", "act": "swiglu", "add": "none"},
        # A short prompt (or many sequences) through the down projection with the residual, two layers' weights.
        {"name": "short_down", "op": "linear", "rows": 120, "n": 4096, "k": 14336, "layers": 2, "dtype": "bf16",
         "bias": "none", "act": "none", "add": "bf16"},
        # An odd number of tokens through a layer of odd widths with everything in its epilogue.
        {"name": "odd_gelu", "op": "linear", "rows": 777, "n": 5003, "k": 2051, "layers": 1, "dtype": "fp16",
         "bias": "fp16", "act": "gelu", "add": "fp32"},
        # A prompt's attention output projection with the residual.
        {"name": "prompt_out", "op": "linear", "rows": 2048, "n": 4096, "k": 4096, "layers": 1, "dtype": "fp16",
         "bias": "none", "act": "none", "add": "fp16"},
        # A long prompt through the gate and up projections with SwiGLU: the matrix cores.
        {"name": "prompt_gate_up", "op": "linear", "rows": 8192, "n": 28672, "k": 4096, "layers": 1, "dtype": "bf16",
         "bias": "none", "act": "swiglu", "add": "none"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rms", "add_rms", "quantize", "linear", "linear", "linear"])
    dtype = rng.choice(["fp16", "bf16"])
    if op != "linear":
        n = _log(rng, 64, 20000)
        n = n | 1 if rng.random() < 0.25 else max(8, n // 8 * 8)
        case = {"op": op, "rows": _log(rng, 1, max(2, min(8192, 33_000_000 // n))), "n": n, "dtype": dtype,
                "view": rng.random() < 0.3}
        if op != "quantize":
            case["wdtype"] = rng.choice([dtype, "fp32"])
        return case
    act = rng.choice(["none", "none", "relu", "silu", "gelu", "gelu_tanh", "swiglu"])
    n, k = _log(rng, 256, 28672), _log(rng, 256, 14336)
    n = n // 2 * 2 if act == "swiglu" else n | 1 if rng.random() < 0.2 else max(16, n // 16 * 16)
    k = k | 1 if rng.random() < 0.2 else max(16, k // 16 * 16)
    rows = _log(rng, 1, 64) if rng.random() < 0.5 else _log(rng, 65, 4096)
    return {"op": "linear", "rows": rows, "n": n, "k": k, "layers": max(1, min(8, 200_000_000 // (n * k))) if rows <= 64 else 1,
            "dtype": dtype, "bias": rng.choice(["none", dtype, "fp32"]), "act": act,
            "add": rng.choice(["none", dtype, "fp32"])}


# ------------------------------------------------------------------ inputs


def _rnd(g, *shape, dtype=torch.float32, scale=1.0, mean=0.0):
    t = torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)
    return t.mul_(scale).add_(mean).to(dtype)


def _quantised(y):
    """E4M3 codes of float32 rows and a float32 scale for each: the row's largest magnitude at the largest code."""
    a = y.abs().amax(dim=-1)
    scale = torch.where(a > 0, (a * (1.0 / E4M3_MAX)).clamp_min(SMALLEST), torch.ones_like(a))
    return (y / scale[..., None]).to(E4M3), scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    m, n, dt = case["rows"], case["n"], DTYPES[case["dtype"]]
    s = {"op": case["op"], "dtype": dt}
    if case["op"] != "linear":
        # rows of different sizes, with a few large channels, as hidden states have them
        x = _rnd(g, m, n + (64 if case["view"] else 0)) * (1.0 + 2.0 * torch.rand(m, 1, generator=g, device="cuda"))
        x[:, :: max(1, n // 5)] *= 8.0
        s["x"] = x.to(dt)[:, :n]
        if case["op"] == "add_rms":
            s["r"] = _rnd(g, m, n, dtype=dt)
        if case["op"] != "quantize":
            s["w"] = _rnd(g, n, dtype=DTYPES[case["wdtype"]], scale=0.1, mean=1.0)
        return s
    k = case["k"]
    s["x"], s["xs"] = _quantised(_rnd(g, m, k))
    nout = n // 2 if case["act"] == "swiglu" else n
    s["act"] = case["act"]
    s["layers"] = []
    for _ in range(case["layers"]):
        w, ws = _quantised(_rnd(g, n, k, scale=k ** -0.5))
        bias = None if case["bias"] == "none" else _rnd(g, n, dtype=DTYPES[case["bias"]], scale=0.5)
        s["layers"].append((w, ws, bias))
    s["add"] = None if case["add"] == "none" else _rnd(g, m, nout, dtype=DTYPES[case["add"]])
    return s


# ------------------------------------------------------------------ passes


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


def _plain(s):
    if s["op"] == "quantize":
        return _quantised(s["x"].float())
    if s["op"] != "linear":
        x = s["x"].float()
        t = x + s["r"].float() if s["op"] == "add_rms" else x
        y = t * torch.rsqrt((t * t).mean(dim=-1, keepdim=True) + EPS) * s["w"].float()
        return (*_quantised(y), t.to(s["dtype"])) if s["op"] == "add_rms" else _quantised(y)
    x, out = s["x"].float(), []
    for w, ws, bias in s["layers"]:
        v = (x @ w.float().t()) * s["xs"][:, None] * ws
        v = _act(v if bias is None else v + bias.float(), s["act"])
        out.append((v if s["add"] is None else v + s["add"].float()).to(s["dtype"]))
    return out


def _own(s):
    import fused_decode as fd

    if s["op"] == "quantize":
        return fd.quantize_rows_fp8(s["x"])
    if s["op"] == "rms":
        return fd.rms_norm_fp8(s["x"], s["w"], EPS)
    if s["op"] == "add_rms":
        return fd.add_rms_norm_fp8(s["x"], s["r"], s["w"], EPS)
    act = None if s["act"] == "none" else s["act"]
    return [fd.linear_w8a8(s["x"], s["xs"], w, ws, bias, activation=act, row_add=s["add"], dtype=s["dtype"])
            for w, ws, bias in s["layers"]]


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------ what a pass cannot do without


_SIZE = {"none": 0, "fp16": 2, "bf16": 2, "fp32": 4}


def work(case):
    m, n = case["rows"], case["n"]
    if case["op"] == "quantize":
        return {"bytes": m * (3 * n + 4), "flops": 3 * m * n}
    if case["op"] == "rms":
        return {"bytes": m * (3 * n + 4) + n * _SIZE[case["wdtype"]], "flops": 7 * m * n}
    if case["op"] == "add_rms":
        return {"bytes": m * (7 * n + 4) + n * _SIZE[case["wdtype"]], "flops": 8 * m * n}
    k, layers = case["k"], case["layers"]
    nout = n // 2 if case["act"] == "swiglu" else n
    per = n * (k + 4 + _SIZE[case["bias"]]) + 2 * m * nout
    return {"bytes": layers * per + m * (k + 4) + m * nout * _SIZE[case["add"]], "flops": layers * 2 * m * n * k}


# ------------------------------------------------------------------ the definition in float64


def exact(case, seed):
    """The values in float64, codes and 16-bit outputs before their rounding."""
    s = prepare(case, seed)

    def rows(y):
        top = y.abs().max(dim=-1).values
        scale = torch.where(top == 0, 1.0, torch.maximum(top / E4M3_MAX, torch.full_like(top, SMALLEST)))
        return y / scale.unsqueeze(-1), scale

    if s["op"] == "quantize":
        return rows(s["x"].double())
    if s["op"] != "linear":
        t = s["x"].double()
        if s["op"] == "add_rms":
            t = t + s["r"].double()
        y = s["w"].double() * t / torch.sqrt(t.square().sum(dim=-1, keepdim=True) / case["n"] + EPS)
        return (*rows(y), t) if s["op"] == "add_rms" else rows(y)
    a = s["x"].double() * s["xs"].double().unsqueeze(-1)
    out = []
    for w, ws, bias in s["layers"]:
        v = a @ (w.double() * ws.double().unsqueeze(-1)).t()
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

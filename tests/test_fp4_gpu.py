"""linear_fp4 against float64.

Of activations that are small integers, with any codes and scales of 2^-2 to 2, every product and sum is a multiple of
2^-3 below 2^21 and exact in float32 in any order, and so is what a product without an activation returns before its one
rounding. Of any activations, the products of a float16 one's two parts make up to 2 K float32 additions, off by at most
2 K * 2^-23 of the sum of magnitudes s (2^-23 covers an addition that truncates, and the parts' magnitudes are below 1.01
of the number's), bias and row_add by 2^-23 each: below (2.1 K + 8) * 2^-23 * (s + |bias| + |row_add|) before the output's
rounding (half a step: 2^-11 relative for float16, 2^-8 for bfloat16, or half of float16's smallest number). The activations
here have slopes of at most 1.2 (SwiGLU, silu(g) u: 1.2 |u| and |g|), and their own float32 evaluation is off by at most
64 steps of 2^-24 of their argument and result."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF_STEP = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
BOTH = [torch.float16, torch.bfloat16]
E8M0 = torch.float8_e8m0fnu
GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rnd(*shape, seed, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=gen(seed)) * scale).to(dtype).to(DEV)


def random_codes(n, k, seed, lo=-2, hi=1):
    """Any codes and scales of 2^lo .. 2^hi, garbage past K among them."""
    g = -(-k // 32)
    codes = torch.randint(0, 256, (n, 16 * g), generator=gen(seed), dtype=torch.uint8)
    scale = torch.randint(127 + lo, 128 + hi, (n, g), generator=gen(seed + 1), dtype=torch.uint8)
    return codes.to(DEV), scale.to(DEV).view(E8M0)


def weights64(codes, scale, k):
    """Written apart from the package's dequantiser."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(1).long().cpu()
    v = GRID[c & 7] * (1 - 2 * (c >> 3))
    s = torch.exp2(scale.view(torch.uint8).cpu().double() - 127).repeat_interleave(32, 1)
    return (v * s)[:, :k].to(DEV)


def ints(*shape, seed, dtype, most=2):
    return torch.randint(-most, most + 1, shape, generator=gen(seed)).to(dtype).to(DEV)


SIZES = [(1, 1, 1), (1, 16, 128), (1, 33, 4096), (1, 300, 100), (2, 130, 272), (2, 64, 14336), (3, 4, 16), (4, 2049, 512),
         (5, 40, 131), (7, 257, 1008), (13, 96, 2064), (16, 640, 512), (16, 100, 8192), (17, 128, 640), (20, 100, 2051),
         (31, 200, 144), (32, 1000, 1024), (33, 48, 96), (64, 127, 256), (65, 129, 128), (70, 140, 1023), (100, 384, 400),
         (128, 128, 8192), (129, 260, 160), (257, 255, 384), (300, 515, 48), (513, 769, 272), (9, 24, 15), (12, 9, 33),
         (1, 5000, 31), (8, 5003, 2051),
         (5, 20, 3), (20, 33, 7), (6, 40, 8), (30, 21, 9)]


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_products_of_small_integers_are_exact(m, n, k, dtype):
    import fused_decode as fd

    x, (codes, scale) = ints(m, k, seed=m, dtype=dtype), random_codes(n, k, n)
    v = x.double() @ weights64(codes, scale, k).t()
    assert torch.equal(fd.linear_fp4(x, codes, scale), v.to(dtype))
    bias, add = ints(n, seed=3, dtype=torch.float32, most=8), ints(m, n, seed=4, dtype=dtype, most=8)
    want = (v + bias.double() + add.double()).to(dtype)
    assert torch.equal(fd.linear_fp4(x, codes, scale, bias, row_add=add), want)
    out = add.clone()
    assert fd.linear_fp4(x, codes, scale, bias, row_add=out, out=out) is out and torch.equal(out, want)
    want = (v + bias.double()).clamp_min(0).to(dtype)
    assert torch.equal(fd.linear_fp4(x, codes, scale, bias, activation="relu"), want)


def act64(v, name):
    if name == "silu":
        return v * torch.sigmoid(v)
    if name == "gelu":
        return 0.5 * v * torch.special.erfc(-v / math.sqrt(2))
    if name == "gelu_tanh":
        return v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v**3))
    return v.clamp_min(0) if name == "relu" else v


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("m,n,k", [(1, 66, 4096), (1, 514, 777), (2, 48, 96), (6, 130, 1000), (16, 258, 2048), (29, 70, 999),
                                   (60, 200, 640), (200, 322, 1030)])
@pytest.mark.parametrize("name", [None, "relu", "silu", "gelu", "gelu_tanh", "swiglu"])
def test_any_activations(m, n, k, dtype, name):
    import fused_decode as fd

    x = rnd(m, k, seed=m + k, dtype=dtype)
    w = rnd(n, k, seed=n, scale=k**-0.5)
    codes, scale = fd.quantize_fp4(w)
    nout = n // 2 if name == "swiglu" else n
    bias, add = rnd(n, seed=5, dtype=dtype, scale=0.5), rnd(m, nout, seed=6)
    w64 = weights64(codes, scale, k)
    v = x.double() @ w64.t() + bias.double()
    err = (2.1 * k + 8) * 2.0**-23 * (x.double().abs() @ w64.abs().t() + bias.double().abs())
    if name == "swiglu":
        g, u, eg, eu = v[:, :nout], v[:, nout:], err[:, :nout], err[:, nout:]
        want = g * torch.sigmoid(g) * u
        err = 1.2 * (u.abs() + eu) * eg + g.abs() * eu + 2.0**-18 * (want.abs() + g.abs())
    else:
        want = act64(v, name)
        err = 1.2 * err + (2.0**-18 * (want.abs() + v.abs()) if name else 0)
    want = want + add.double()
    err = err + 2.0**-23 * (want.abs() + add.double().abs())
    y = fd.linear_fp4(x, codes, scale, bias, activation=name, row_add=add)
    assert y.dtype == dtype
    assert bool(((y.double() - want).abs() <= err + HALF_STEP[dtype] * (want.abs() + err) + 2.0**-25).all())


@pytest.mark.parametrize("m", [1, 2, 9, 24, 70])
def test_float16_keeps_its_eleven_bits(m):
    """Odd integers up to 2047, subnormal numbers and the largest ones: their two bfloat16 parts add up to them."""
    import fused_decode as fd

    k, n = 64, 40
    codes, scale = random_codes(n, k, 1, lo=0, hi=0)
    x = (torch.randint(-1024, 1024, (m, k), generator=gen(2)) * 2 + 1).to(torch.float16).to(DEV)
    w = weights64(codes, scale, k)
    for unit in (1.0, 2.0**-24, 2.0**-14):
        v = (x.double() * unit).to(torch.float16).double() @ w.t()
        y = fd.linear_fp4((x.double() * unit).to(torch.float16), codes, scale)
        assert torch.equal(y, v.to(torch.float16))
    x = torch.zeros(m, k, dtype=torch.float16, device=DEV)
    x[:, 5] = 65504.0
    codes[:, 2] = 0x10  # position 5: 0.5, position 4: 0
    scale.view(torch.uint8)[:] = 120
    assert torch.equal(fd.linear_fp4(x, codes, scale), torch.full((m, n), 65504 / 256, dtype=torch.float16, device=DEV))


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("m", [1, 3, 20, 40])
def test_scales_of_every_exponent(m, dtype):
    """2^-127 to 2^127, and NaN, beside each other in a row; infinities and NaN among the activations."""
    import fused_decode as fd

    k = 32 * 256
    codes = torch.zeros(256, k // 2, dtype=torch.uint8, device=DEV)
    for row in range(256):  # one value, 1.0, in the group with this scale
        codes[row, row * 16] = 2
    scale = torch.arange(256, dtype=torch.uint8, device=DEV).expand(256, 256).contiguous()
    x = torch.zeros(m, k, dtype=dtype, device=DEV)
    finite = scale.clone()
    finite[:, 255] = 0
    x[:, ::32] = 1.5
    y = fd.linear_fp4(x, codes, finite.view(E8M0))
    want = 1.5 * torch.exp2(torch.arange(255, device=DEV).double() - 127)
    got = y[:, :255].double()
    least = 2.0**-25 if dtype is torch.float16 else 2.0**-126  # what a product of numbers near 2^-126 may lose
    assert bool(((got - want.to(dtype).double()).abs() <= least).logical_or(got == want.to(dtype).double()).all())
    y = fd.linear_fp4(x, codes, scale.view(E8M0))
    assert bool(torch.isnan(y).all())
    plain = torch.full_like(finite, 127).view(E8M0)
    for bad in (float("inf"), float("nan")):
        x[m - 1, 64] = bad
        y = fd.linear_fp4(x, codes, plain)
        assert bool((y[: m - 1] == 1.5).all())
        last = y[m - 1].float()
        last[2] = float("nan")  # 1 times it there, 0 times it in the other rows
        assert bool(torch.isnan(last).all())
        codes[:, 32] = 2
        y = fd.linear_fp4(x, codes, plain)[m - 1].float()
        assert bool((torch.isinf(y) if math.isinf(bad) else torch.isnan(y)).all())
        codes[:, 32] = 0
        codes[2, 32] = 2


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("m", [1, 5, 26, 50])
def test_strides_and_broadcasts(m, dtype):
    import fused_decode as fd

    n, k = 90, 224
    codes, scale = random_codes(n, k, 1)
    w = weights64(codes, scale, k)
    wide = ints(m, k + 9, seed=2, dtype=dtype)
    tall = ints(k, m, seed=3, dtype=dtype)
    for x in (wide[:, :k], wide[:, 9:], wide[:, 1 : k + 1], tall.t()):
        assert torch.equal(fd.linear_fp4(x, codes, scale), (x.double() @ w.t()).to(dtype))
    x = ints(2, m, 3, k, seed=4, dtype=dtype).transpose(0, 2)
    assert torch.equal(fd.linear_fp4(x, codes, scale), (x.double() @ w.t()).to(dtype))
    x = wide[:, :k]
    v = x.double() @ w.t()
    for add in (ints(n, seed=5, dtype=torch.float32), ints(m, 1, seed=6, dtype=dtype), ints(1, n, seed=7, dtype=dtype),
                ints(m, 2 * n, seed=8, dtype=torch.bfloat16)[:, ::2], ints(n, m, seed=9, dtype=torch.float16).t()):
        assert torch.equal(fd.linear_fp4(x, codes, scale, row_add=add), (v + add.double()).to(dtype))
    # codes and scales that are views: wider rows, off alignment, transposed
    spread = torch.zeros(n, k // 2 + 16, dtype=torch.uint8, device=DEV)
    spread[:, : k // 2] = codes
    odd = torch.zeros(n * k // 2 + 3, dtype=torch.uint8, device=DEV)[3:].view(n, k // 2)
    odd.copy_(codes)
    s2 = torch.zeros(n, 11, dtype=torch.uint8, device=DEV)
    s2[:, 4:] = scale.view(torch.uint8)
    bias = ints(2 * n, seed=10, dtype=torch.float32)[::2]
    for c in (spread[:, : k // 2], odd, codes.t().contiguous().t()):
        for s in (scale, s2[:, 4:].view(E8M0), scale.view(torch.uint8).t().contiguous().t().view(E8M0)):
            assert torch.equal(fd.linear_fp4(x, c, s, bias), (v + bias.double()).to(dtype))
    # an output over an operand is written beside it
    if n <= k:
        hold = torch.zeros(m * k, dtype=dtype, device=DEV)
        xin = hold.view(m, k)
        xin.copy_(x)
        out = hold[: m * n].view(m, n)
        assert fd.linear_fp4(xin, codes, scale, out=out) is out and torch.equal(out, v.to(dtype))


@pytest.mark.parametrize("dtype", BOTH)
def test_no_rows_no_columns_no_depth(dtype):
    import fused_decode as fd

    codes, scale = random_codes(6, 64, 1)
    e = lambda *s: torch.empty(s, dtype=dtype, device=DEV)
    assert fd.linear_fp4(e(0, 64), codes, scale).shape == (0, 6)
    assert fd.linear_fp4(e(2, 64), codes[:0], scale[:0]).shape == (2, 0)
    bias, add = ints(6, seed=2, dtype=torch.float32), ints(3, 6, seed=3, dtype=dtype)
    for m in (1, 3, 40):
        y = fd.linear_fp4(e(m, 0), codes[:, :0], scale[:, :0], bias, activation="relu")
        assert torch.equal(y, bias.clamp_min(0).to(dtype).expand(m, 6))
    x = ints(64, seed=4, dtype=dtype)
    assert torch.equal(fd.linear_fp4(x, codes, scale), (x.double() @ weights64(codes, scale, 64).t()).to(dtype))


def test_nan_past_k_and_past_the_last_row_is_not_read():
    """x rows lie in memory that is NaN around them; the last rows end where the memory does."""
    import fused_decode as fd

    for dtype in BOTH:
        for m in (1, 3, 18, 40):
            for k in (33, 100, 128, 1000, 2051):
                codes, scale = random_codes(50, k, k)
                hold = torch.full((m + 2, k + 5), float("nan"), dtype=dtype, device=DEV)
                hold[1:-1, 2:-3] = ints(m, k, seed=m, dtype=dtype)
                x = hold[1:-1, 2:-3]
                want = (x.double() @ weights64(codes, scale, k).t()).to(dtype)
                assert torch.equal(fd.linear_fp4(x, codes, scale), want)


@pytest.mark.parametrize("m,n,k,name", [(1, 6144, 4096, None), (13, 4096, 4096, "swiglu"), (29, 1003, 2051, "gelu"),
                                        (300, 512, 4096, None)])
def test_captured_replayed_and_on_another_stream(m, n, k, name):
    """Two graphs of one signature replayed in turn, and the eager call between them: no workspace is shared."""
    import fused_decode as fd

    if name == "swiglu":
        n *= 2
    weights = [random_codes(n, k, seed) for seed in (1, 2)]
    x = rnd(m, k, seed=3, dtype=torch.float16, scale=0.1)
    want = [fd.linear_fp4(x, *w, activation=name) for w in weights]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = fd.linear_fp4(x, *weights[0], activation=name)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want[0])
    graphs = []
    for w in weights:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = fd.linear_fp4(x, *w, activation=name)
        graphs.append((graph, y))
    for seed in (4, 5, 6):
        x.copy_(rnd(m, k, seed=seed, dtype=torch.float16, scale=0.1))
        for (graph, y), w in zip(graphs, weights):
            graph.replay()
            eager = fd.linear_fp4(x, *w, activation=name)
            torch.cuda.synchronize()
            assert torch.equal(y, eager)


def test_the_quantiser_on_the_gpu_gives_the_cpus_codes():
    import fused_decode as fd

    w = torch.randn(300, 1000, generator=gen(1)) * torch.rand(300, 1, generator=gen(2))
    codes, scale = fd.quantize_fp4(w)
    c, s = fd.quantize_fp4(w.to(DEV))
    assert torch.equal(c.cpu(), codes) and torch.equal(s.cpu().view(torch.uint8), scale.view(torch.uint8))
    assert torch.equal(fd.dequantize_fp4(c, s).cpu(), fd.dequantize_fp4(codes, scale))
    assert torch.equal(fd.dequantize_fp4(c, s, 1000).double(), weights64(c, s, 1000))

"""norm_add_norm against float64.

z's float32 evaluation (a sum of n squares, its root, four products) is off by less than d = (n + 32) * 2^-24 relative, t
by dt = d |z| + 2^-23 (|r| + |z|). The second norm's root is off by d and by what the dt make of the sum of squares,
sum |t| dt / sum t^2 (relative, eps only lowers it), y before its rounding by |w| inv dt + |y| (both of these). Outputs
add half a step of their type, or of its smallest number."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF_STEP = {torch.float16: (2.0**-11, 2.0**-25), torch.bfloat16: (2.0**-8, 2.0**-134)}


def rnd(*shape, seed, dtype=torch.float32, scale=1.0, mean=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale + mean).to(dtype).to(DEV)


def check(got, x, r, pw, w, eps, gate=None, scale=1.0):
    y, stream = got
    n, dtype = x.shape[-1], x.dtype
    x, r, pw, w = (t.double() for t in (x, r, pw, w))
    d = (n + 32) * 2.0**-24
    z = scale * x * pw / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    if gate is not None:
        z = z * gate.double()
    t = r + z
    dt = d * z.abs() + 2.0**-23 * (r.abs() + z.abs())
    inv = 1 / torch.sqrt(t.square().mean(-1, keepdim=True) + eps)
    want = t * inv * w
    off = d + (t.abs() * dt).sum(-1, keepdim=True) / t.square().sum(-1, keepdim=True).clamp_min(1e-300)
    half, least = HALF_STEP[dtype]
    for v, exact, err in ((stream, t, dt), (y, want, w.abs() * inv * dt + want.abs() * off)):
        assert v.dtype == dtype and v.shape == exact.shape
        assert bool(((v.double() - exact).abs() <= err + half * (exact.abs() + err) + least).all())


# lanes of a row change after 128 and 512 elements, vectors of a lane or lanes after 1024, 2048, 4096, 8192, 16384
LENGTHS = [8, 9, 15, 127, 128, 129, 512, 513, 1024, 1025, 2049, 4096, 4097, 8193, 16384, 16385, 32767, 32768]
ODD = [1, 2, 7, 32769, 40001]  # the kernel for any strides


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", LENGTHS + ODD)
def test_rows_of_any_length_and_alignment(dtype, n):
    import fused_decode as fd

    m = 5
    for offset, wdtype in ((0, dtype), (1, torch.float32)):
        buf = rnd(m * (n + 3) + 1, seed=n, dtype=dtype, scale=2.0)
        x = buf[offset : offset + m * (n + 3)].view(m, n + 3)[:, :n]
        r = rnd(m, n, seed=n + 1, dtype=dtype, scale=3.0)
        pw, w = (rnd(n + 1, seed=n + i, dtype=wdtype, scale=0.2, mean=1.0)[offset : offset + n] for i in (2, 3))
        check(fd.norm_add_norm(x, r, pw, w, 1e-5), x, r, pw, w, 1e-5)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [100, 640, 3001, 4096, 9000, 20000])
def test_gates_and_scales(dtype, n):
    import fused_decode as fd

    b, m = 2, 3
    x, r = rnd(b, m, n, seed=1, dtype=dtype), rnd(b, m, n, seed=2, dtype=dtype, scale=2.0)
    pw, w = rnd(n, seed=3, dtype=dtype, mean=1.0), rnd(n, seed=4, dtype=dtype, mean=1.0)
    shapes = [(n,), (m, 1), (b, 1, n), (b, m, n), (1, 1, 1), ()]
    for i, shape in enumerate(shapes):
        for gdtype in (dtype, torch.float32, torch.float16 if dtype is torch.bfloat16 else torch.bfloat16):
            gate = rnd(*shape, seed=5 + i, dtype=gdtype)
            for scale in (1.0, -0.22):
                got = fd.norm_add_norm(x, r, pw, w, 1e-6, gate=gate, residual_scale=scale)
                check(got, x, r, pw, w, 1e-6, gate, scale)
    gate = rnd(2 * n, seed=11, dtype=dtype)[::2]  # strided gate, weights of two types and strides
    pw2, w2 = rnd(n, 2, seed=12, dtype=torch.float32)[:, 1], rnd(n, seed=13, dtype=dtype)
    check(fd.norm_add_norm(x, r, pw2, w2, 1e-6, gate=gate), x, r, pw2, w2, 1e-6, gate)
    check(fd.norm_add_norm(x, r, w2, pw, 1e-6, residual_scale=0.0), x, r, w2, pw, 1e-6, None, 0.0)


@pytest.mark.parametrize("n", [24, 1000, 4096, 17000, 33000])
def test_outputs_over_inputs(n):
    import fused_decode as fd

    x, r = rnd(7, n, seed=1, dtype=torch.bfloat16), rnd(7, n, seed=2, dtype=torch.bfloat16)
    w, pw = rnd(n, seed=3), rnd(n, seed=4)
    want = fd.norm_add_norm(x, r, pw, w, gate=w)
    for out, ro in (("x", "r"), ("r", "x"), (None, "r"), ("r", None), ("x", None), (None, "x")):
        t = {"x": x.clone(), "r": r.clone(), None: None}
        got = fd.norm_add_norm(t["x"], t["r"], pw, w, gate=w, out=t[out], residual_out=t[ro])
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert (out is None or got[0] is t[out]) and (ro is None or got[1] is t[ro])
    # every second element, the others left: another kernel, whose sums have another order
    wide = torch.zeros(7, 2 * n + 2, dtype=torch.bfloat16, device=DEV)
    got = fd.norm_add_norm(x, r, pw, w, gate=w, out=wide[:, : 2 * n : 2])
    assert got[0].data_ptr() == wide.data_ptr() and not wide[:, 1::2].any() and not wide[:, 2 * n :].any()
    check(got, x, r, pw, w, 1e-6, w)


def test_layouts_of_many_dims():
    import fused_decode as fd

    w, pw = rnd(40, seed=1), rnd(40, seed=2)
    for perm in ((0, 1, 2, 3, 4), (3, 2, 1, 0, 4), (1, 0, 3, 2, 4)):
        x = rnd(3, 4, 2, 5, 40, seed=3, dtype=torch.float16).permute(perm)
        r = rnd(*x.shape, seed=4, dtype=torch.float16)
        gate = rnd(*x.shape[2:-1], 1, seed=5)
        check(fd.norm_add_norm(x, r, pw, w, gate=gate), x, r, pw, w, 1e-6, gate)
        y, stream = x.clone(), r.clone()
        fd.norm_add_norm(x, stream, pw, w, out=y, residual_out=stream)
        check((y, stream), x, r, pw, w, 1e-6)
    line = rnd(40, seed=6, dtype=torch.float16)
    check(fd.norm_add_norm(line, line, pw, w), line, line, pw, w, 1e-6)
    assert fd.norm_add_norm(x[:0], r[:0], pw, w)[0].shape == (0, *x.shape[1:])


@pytest.mark.parametrize("n", [64, 700, 4096, 4097, 33001])
def test_rows_whose_squares_leave_float32(n):
    """x or the stream above 1e19 or below 1e-20: the sums are taken again at another scale."""
    import fused_decode as fd

    w, pw = rnd(n, seed=1, mean=1.0), rnd(n, seed=2, mean=1.0)
    unit, other = rnd(6, n, seed=3, dtype=torch.bfloat16), rnd(6, n, seed=4, dtype=torch.bfloat16)
    size = torch.tensor([1.0, 1e30, 1.0, 1e-30, 1e25, 1e-30], device=DEV)[:, None]
    big = (unit * size).to(torch.bfloat16)
    for eps in (0.0, 1e-6):
        check(fd.norm_add_norm(big, other, pw, w, eps), big, other, pw, w, eps)
        for scale in (1.0, 2.0**-100):
            check(fd.norm_add_norm(other, big, pw, w, eps, residual_scale=scale), other, big, pw, w, eps, None, scale)


@pytest.mark.parametrize("n", [50, 4096, 33000])
def test_rows_of_zeros_and_of_no_numbers(n):
    import fused_decode as fd

    x, r = rnd(4, n, seed=1, dtype=torch.float16), rnd(4, n, seed=2, dtype=torch.float16)
    x[0] = 0.0
    r[1], x[1] = 0.0, 0.0
    w = rnd(n, seed=3)
    check(fd.norm_add_norm(x[:2], r[:2], w, w, 1e-5), x[:2], r[:2], w, w, 1e-5)
    for bad in (float("nan"), float("inf")):
        for t in (x, r):
            held = t[2, n // 2].item()
            t[2, n // 2] = bad
            y, stream = fd.norm_add_norm(x, r, w, w, 1e-5)
            assert bool(torch.isnan(y[2, n // 2])) and not bool(torch.isfinite(stream[2, n // 2]))
            check((y[3:], stream[3:]), x[3:], r[3:], w, w, 1e-5)
            t[2, n // 2] = held


def test_captured_replayed_and_on_another_stream():
    import fused_decode as fd

    x, r = rnd(9, 4096, seed=1, dtype=torch.bfloat16), rnd(9, 4096, seed=2, dtype=torch.bfloat16)
    w, pw, gate = rnd(4096, seed=3), rnd(4096, seed=4), rnd(9, 1, seed=5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = fd.norm_add_norm(x, r, pw, w, gate=gate)
    torch.cuda.current_stream().wait_stream(side)
    check(got, x, r, pw, w, 1e-6, gate)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, stream = fd.norm_add_norm(x, r, pw, w, gate=gate)
    for seed in (6, 7, 8):
        x.copy_(rnd(9, 4096, seed=seed, dtype=torch.bfloat16))
        graph.replay()
        want = fd.norm_add_norm(x, r, pw, w, gate=gate)
        torch.cuda.synchronize()
        assert torch.equal(y, want[0]) and torch.equal(stream, want[1])


def test_many_rows():
    import fused_decode as fd

    x, r = rnd(70000, 72, seed=1, dtype=torch.float16), rnd(70000, 72, seed=2, dtype=torch.float16)
    w, pw = rnd(72, seed=3), rnd(72, seed=4)
    check(fd.norm_add_norm(x, r, pw, w), x, r, pw, w, 1e-6)

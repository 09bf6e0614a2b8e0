"""Products with 4-bit weights on the CPU: the quantiser against its definition, what the entry point and the argument
contract refuse, the scratch a product asks for, the fake kernel, and which calls go to the custom op."""

from __future__ import annotations

import contextlib
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

from fused_decode import _lib as L
from fused_decode import fp4, ops
from fused_decode._checks import check

E8M0 = torch.float8_e8m0fnu
# The entry point's checks return before any HIP call; no pointer is read.
nogpu = pytest.mark.skipif(torch.cuda.is_available(), reason="host-only argument checks")
X, W, S, Y, B, R, P = (0x100000 * i for i in range(1, 8))  # far apart
GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


# ------------------------------------------------------------------ codes


def test_values_and_their_midpoints_take_the_nearest_code():
    """Every value, every midpoint (to the even code), and the floats beside them, at several scales."""
    edges = [(a + b) / 2 for a, b in zip(GRID.tolist(), GRID.tolist()[1:])]
    marks = torch.tensor(sorted(GRID.tolist() + edges), dtype=torch.float32)
    v = torch.cat([marks, torch.nextafter(marks, marks * 0 - 1), torch.nextafter(marks, marks * 0 + 9)]).clamp(0, 6)
    v = torch.cat([v, -v, torch.full((6,), 6.0)]).reshape(-1, 32)
    v[:, -1] = 6.0
    for e in (-100, -3, 0, 5, 100):
        codes, scale = fp4.quantize_fp4(v * 2.0**e)
        assert bool((scale.float() == 2.0**e).all())
        got = fp4.dequantize_fp4(codes, scale).double() / 2.0**e
        near = (v.double().abs()[..., None] - GRID).abs()
        best = near.amin(-1, keepdim=True)
        tied = near == best
        pick = torch.where(tied & (torch.arange(8) % 2 == 0), 2, tied.int()).argmax(-1)
        assert torch.equal(got.abs(), GRID[pick]) and bool((torch.signbit(got) == torch.signbit(v)).all())


def test_scales():
    """The smallest power of two that the largest magnitude is less than 7 of."""
    top = torch.tensor([1.0, 3.49, 3.5, 6.0, 6.99, 7.0, 7.01, 2.0**-130, 2.0**-127, 2.0**-149, 0.0, 3.0e38, 3.4e38])
    w = torch.zeros(len(top), 32)
    w[:, 7] = -top
    codes, scale = fp4.quantize_fp4(w)
    s = scale.double().squeeze(1)
    assert s.tolist()[:7] == [0.25, 0.5, 1.0, 1.0, 1.0, 2.0, 2.0] and s[10] == 1.0
    assert bool((s[7:10] == 2.0**-126).all())
    assert bool((top.double()[11:] < 7 * s[11:]).all()) and bool((top.double()[11:] >= 3.5 * s[11:]).all())
    assert not fp4.dequantize_fp4(codes, scale)[10].any()
    for bad in (float("inf"), float("nan")):
        w = torch.ones(1, 64)
        w[0, 3] = bad
        codes, scale = fp4.quantize_fp4(w)
        assert scale.view(torch.uint8).tolist() == [[255, 125]]
        d = fp4.dequantize_fp4(codes, scale)
        assert bool(torch.isnan(d[0, :32]).all()) and bool((d[0, 32:] == 1).all())


@pytest.mark.parametrize("n,k", [(3, 1), (2, 31), (5, 64), (4, 100), (0, 40), (3, 0)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32, torch.float64])
def test_shapes_of_codes(n, k, dtype):
    w = torch.randn(n, k).to(dtype)
    codes, scale = fp4.quantize_fp4(w)
    g = -(-k // 32)
    assert codes.shape == (n, 16 * g) and codes.dtype == torch.uint8 and codes.is_contiguous()
    assert scale.shape == (n, g) and scale.dtype == E8M0
    full = fp4.dequantize_fp4(codes, scale)
    assert full.shape == (n, 32 * g) and not full[:, k:].any()
    d = fp4.dequantize_fp4(codes, scale, k)
    step = scale.double().repeat_interleave(32, 1)[:, :k]
    assert d.shape == (n, k) and bool(((d.double() - w.double()).abs() <= step).all())


def test_the_quantiser_refuses():
    for bad in (torch.zeros(3), torch.zeros(2, 3, 4), [[1.0]]):
        with pytest.raises(ValueError):
            fp4.quantize_fp4(bad)
    with pytest.raises(TypeError):
        fp4.quantize_fp4(torch.zeros(2, 32, dtype=torch.int32))


# ------------------------------------------------------------------ the C entry


def refused(status, code, words):
    return status == code and words in L.lib().fd_last_error()


def linear(y=Y, x=X, w=W, s=S, bias=None, bd=0, act=0, row=None, rd=0, m=40, n=64, k=128, sxm=None, swn=None, ssn=None,
           sb=1, srm=64, srn=1, sym=None, syn=1, scratch=None, size=0, dtype=1):
    g, nout = -(-k // 32), n // 2 if act == 5 else n
    return L.lib().fd_linear_fp4(y, x, w, s, bias, bd, act, row, rd, m, n, k, k if sxm is None else sxm,
                                 16 * g if swn is None else swn, g if ssn is None else ssn, sb, srm, srn,
                                 nout if sym is None else sym, syn, scratch, size, dtype, None)


def scratch(m, n, k, dtype=1):
    out = ctypes.c_int64(-1)
    return L.lib().fd_linear_fp4_scratch(m, n, k, dtype, ctypes.byref(out)), out.value


@nogpu
def test_linear_refuses():
    assert refused(linear(dtype=2), L.FD_EINVAL, b"act_dtype")
    for name in ("m", "n", "k"):
        assert refused(linear(**{name: -1}), L.FD_EINVAL, b"size"), name
        assert refused(linear(**{name: 2**31 - 1}), L.FD_EUNSUPPORTED, b"large"), name
    for name in ("sxm", "swn", "ssn", "sb", "srm", "srn", "sym", "syn"):
        assert refused(linear(**{name: -1}), L.FD_EINVAL, b"stride"), name
    assert refused(linear(act=6), L.FD_EINVAL, b"activation") and refused(linear(act=-1), L.FD_EINVAL, b"activation")
    assert refused(linear(act=5, n=63), L.FD_EINVAL, b"even")
    assert refused(linear(bias=B, bd=9), L.FD_EINVAL, b"bias_dtype")
    assert refused(linear(row=R, rd=-1), L.FD_EINVAL, b"row_dtype")
    for name in ("y", "x", "w", "s"):
        assert refused(linear(**{name: None}), L.FD_EINVAL, b"null"), name
    assert linear(m=0, y=None) == L.FD_OK and linear(n=0, w=None) == L.FD_OK
    assert refused(linear(w=W + 8), L.FD_EUNSUPPORTED, b"aligned")
    assert refused(linear(swn=72), L.FD_EUNSUPPORTED, b"aligned")
    assert refused(linear(scratch=P + 4, size=1 << 20), L.FD_EUNSUPPORTED, b"aligned")
    assert refused(linear(sym=0), L.FD_EINVAL, b"share") and refused(linear(sym=63), L.FD_EINVAL, b"share")


@nogpu
def test_linear_refuses_an_output_over_an_operand():
    """40 x 64 outputs (5120 bytes) of 40 rows of 256 bytes, 64 rows of 64 and 64 of 4."""
    for at, size in ((X, 10240), (W, 4096), (S, 256)):
        for where in (at, at + size - 1, at - 5119):
            assert refused(linear(y=where), L.FD_EUNSUPPORTED, b"overlap")
    assert refused(linear(y=P, bias=P + 5118), L.FD_EUNSUPPORTED, b"overlap")
    assert refused(linear(y=P, row=P + 2, rd=1), L.FD_EUNSUPPORTED, b"overlap")          # one element on
    assert refused(linear(y=P, row=P, rd=2), L.FD_EUNSUPPORTED, b"overlap")              # float32 under 16-bit outputs
    assert refused(linear(y=P, row=P, rd=1, srm=0), L.FD_EUNSUPPORTED, b"overlap")       # one row under all


@nogpu
def test_copied_activations_need_scratch():
    need = lambda status: refused(status, L.FD_EUNSUPPORTED, b"scratch")
    assert need(linear(dtype=0)) and need(linear(k=100)) and need(linear(sxm=130)) and need(linear(x=X + 2))
    assert need(linear(dtype=0, scratch=P, size=40 * 128 * 4 - 1))
    assert need(linear(k=100, scratch=P, size=40 * 128 * 2 - 1))


def test_scratch_sizes():
    assert scratch(-1, 2, 3)[0] == L.FD_EINVAL and scratch(1, 2, 3, 2)[0] == L.FD_EINVAL
    assert L.lib().fd_linear_fp4_scratch(1, 2, 3, 0, None) == L.FD_EINVAL
    for m, n, k in ((0, 64, 128), (40, 0, 128), (40, 64, 0), (2**31, 64, 128)):
        assert scratch(m, n, k) == (L.FD_OK, 0)
    # rows of whole steps, float16 twice; K splits of few tiles: whole [M, N] sums behind them
    for m, n, k, dtype in ((40, 64, 128, 1), (64, 64, 16384, 0), (300, 4096, 1000, 0)):
        status, size = scratch(m, n, k, dtype)
        copies = m * -(-k // 128) * 128 * (2 if dtype else 4)
        assert status == L.FD_OK and size >= copies and (size - copies) % (m * n * 4) == 0


# ------------------------------------------------------------------ the contract and where a call goes


def cuda(*shape, dtype=torch.float16):
    return torch.empty(shape, dtype=dtype, device="cuda")


def test_the_contract():
    with FakeTensorMode():
        good = dict(x=cuda(3, 5, 70), weight=cuda(30, 48, dtype=torch.uint8), scale=cuda(30, 3, dtype=E8M0), bias=None,
                    activation=None, row_add=None)
        given = lambda **other: check("linear_fp4", **{**good, **other})
        given(), given(x=cuda(70, dtype=torch.bfloat16)), given(x=cuda(2, 96))
        given(bias=cuda(30, dtype=torch.float32), activation="swiglu", row_add=cuda(15))
        for wrong in (dict(x=cuda(3, 70, dtype=torch.float32)), dict(x=None), dict(weight=cuda(30, 48)),
                      dict(weight=None), dict(scale=cuda(30, 3, dtype=torch.uint8)), dict(scale=1.0), dict(bias=[1.0]),
                      dict(bias=cuda(30, dtype=torch.int32)), dict(row_add=2)):
            with pytest.raises(TypeError):
                given(**wrong)
        for wrong in (dict(x=cuda()), dict(x=cuda(3, 97)), dict(x=cuda(3, 64)), dict(scale=cuda(29, 3, dtype=E8M0)),
                      dict(scale=cuda(30, 4, dtype=E8M0)), dict(weight=cuda(30, 47, dtype=torch.uint8)),
                      dict(weight=cuda(2, 30, 48, dtype=torch.uint8)), dict(scale=cuda(3, dtype=E8M0)),
                      dict(bias=cuda(29)), dict(bias=cuda(1, 30)), dict(activation="tanh"), dict(activation=3),
                      dict(weight=cuda(31, 48, dtype=torch.uint8), scale=cuda(31, 3, dtype=E8M0), activation="swiglu")):
            with pytest.raises(ValueError):
                given(**wrong)


def test_tensors_off_the_gpu_are_refused():
    q, s = fp4.quantize_fp4(torch.randn(6, 64))
    x = torch.randn(2, 64).half()
    for where in (fp4, torch.ops.fused_decode):
        with pytest.raises(ValueError, match="CUDA"):
            where.linear_fp4(x, q, s)
    for args in ((None, q, s), (x, None, s), (x, q, 3)):
        with pytest.raises((TypeError, ValueError)):
            fp4.linear_fp4(*args)


def test_the_fake_kernel_and_a_traced_graph():
    with FakeTensorMode():
        x, q, s = cuda(2, 0, 64), cuda(96, 32, dtype=torch.uint8), cuda(96, 2, dtype=E8M0)
        for f in (torch.ops.fused_decode.linear_fp4, lambda *a: fp4.linear_fp4(*a[:4], activation=a[4])):
            assert f(x, q, s, None, "relu").shape == (2, 0, 96) and f(x, q, s, None, "swiglu").shape == (2, 0, 48)
        graph = make_fx(lambda x, q, s: fp4.linear_fp4(x, q, s, activation="gelu"))(cuda(3, 64), q, s).graph
    assert sum(str(n.target).startswith("fused_decode.linear_fp4") for n in graph.nodes) == 1


class Calls(list):
    """Stands in for the native binding: notes each call and returns FD_OK."""

    def __getattr__(self, name):
        def call(*args):
            self.append((name, args))
            return L.FD_OK
        return call


@pytest.fixture
def calls(monkeypatch):
    stand_in = Calls()
    monkeypatch.setattr(fp4, "native", lambda: stand_in)
    monkeypatch.setattr(fp4, "_raw_stream", lambda dev: 0)
    monkeypatch.setattr(fp4, "_current_device", lambda: None)  # the CPU's index
    monkeypatch.setattr(fp4._lib, "scratch_bytes", lambda *a: 0)
    monkeypatch.setattr(torch.cuda, "device", lambda dev: contextlib.nullcontext())
    monkeypatch.setattr(fp4, "check", lambda op, **a: a)
    ops.clear_plans()
    yield stand_in
    ops.clear_plans()


def test_calls_launch_once_and_keep_a_plan(calls):
    q, s = fp4.quantize_fp4(torch.randn(30, 64))
    x = torch.randn(3, 64).half()
    for _ in range(2):
        assert fp4.linear_fp4(x, q, s, activation="swiglu").shape == (3, 15)
    assert len(calls) == 2 and len(ops._PLANS) == 1
    out = torch.empty(3, 30, dtype=torch.float16)
    before = out._version
    assert fp4.linear_fp4(x, q, s, out=out) is out and out._version > before
    with pytest.raises(ValueError):
        fp4.linear_fp4(x, q, s, out=torch.empty(3, 31, dtype=torch.float16))
    # rows of codes off alignment, or spread, go to the kernels as a copy
    held = torch.zeros(30 * 32 + 1, dtype=torch.uint8)
    held[1:] = q.flatten()
    for codes in (held[1:].view(30, 32), q.t().contiguous().t(), torch.cat([q, q[:, :1]], 1)[:, :32]):
        fp4.linear_fp4(x, codes, s)
        name, args = calls[-1]
        assert args[2] % 16 == 0 and args[2] != codes.data_ptr() and args[13] == 32
    fp4.linear_fp4(x, torch.cat([q, q], 1)[:, :32], s)
    assert calls[-1][1][13] == 64


def test_recorded_calls_go_to_the_custom_op(calls, monkeypatch):
    q, s = fp4.quantize_fp4(torch.randn(30, 64))
    x, b = torch.randn(3, 64).half(), torch.randn(30)
    seen = []

    class Stand:
        def __getattr__(self, name):
            return lambda *a: seen.append(name) or torch.zeros(3, 30, dtype=torch.float16)

    monkeypatch.setattr(torch.ops, "fused_decode", Stand(), raising=False)
    leaf, neg = lambda t: t.clone().requires_grad_(), torch._neg_view
    fp4.linear_fp4(leaf(x), q, s), fp4.linear_fp4(x, q, s, leaf(b)), fp4.linear_fp4(x, q, s, row_add=leaf(b))
    fp4.linear_fp4(neg(x), q, s), fp4.linear_fp4(x, q, s, neg(b)), fp4.linear_fp4(x, q, s, row_add=neg(b))
    assert calls == [] and seen == ["linear_fp4"] * 6
    with torch.no_grad():
        fp4.linear_fp4(leaf(x), q, s)
    assert len(calls) == 1
    with pytest.raises(RuntimeError, match="gradient"):
        fp4.linear_fp4(x, q, s, out=leaf(torch.zeros(3, 30, dtype=torch.float16)))

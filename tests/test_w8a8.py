"""Operators with 8-bit activations on the CPU: what their entry points and the argument contract refuse, the scratch
they ask for, the shapes of their fake kernels, and which calls go to the custom ops."""

from __future__ import annotations

import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

from fused_decode import _lib as L
from fused_decode import ops, w8a8
from fused_decode._checks import check

E4M3 = torch.float8_e4m3fn
# The entry points' checks return before any HIP call; no pointer is read.
nogpu = pytest.mark.skipif(torch.cuda.is_available(), reason="host-only argument checks")
X, W, Y, Q, S, R, P = (0x100000 * i for i in range(1, 8))  # far apart


def rows(a=1, b=1, c=4, n=64, col=1, sc=None):
    return L.FdRows(a, b, c, 0, 0, n if sc is None else sc, col, n)


def refused(status, code, words):
    return status == code and words in L.lib().fd_last_error()


# ------------------------------------------------------------------ rows to codes, the C entries


def quantize(codes=Q, scale=S, x=X, lx=None, act=0):
    return L.lib().fd_quantize_rows_fp8(codes, scale, x, lx or rows(), act, None)


def norm(codes=Q, scale=S, x=X, w=W, wd=2, ws=1, lx=None, eps=1e-6, act=0):
    return L.lib().fd_rms_norm_fp8(codes, scale, x, w, wd, ws, lx or rows(), eps, act, None)


def add_norm(codes=Q, scale=S, ro=Y, x=X, r=R, w=W, wd=2, ws=1, lx=None, lr=None, lro=None, eps=1e-6, act=0):
    return L.lib().fd_add_rms_norm_fp8(codes, scale, ro, x, r, w, wd, ws, lx or rows(), lr or rows(), lro or rows(),
                                       eps, act, None)


@nogpu
@pytest.mark.parametrize("call", [quantize, norm, add_norm])
def test_row_entries_refuse(call):
    assert refused(call(act=2), L.FD_EINVAL, b"act_dtype")
    pointers = ["codes", "scale", "x"] + ["w"] * (call is not quantize) + ["ro", "r"] * (call is add_norm)
    for name in pointers:
        assert refused(call(**{name: None}), L.FD_EINVAL, b"null"), name
    assert call(lx=rows(n=-1)) == L.FD_EINVAL and call(lx=rows(c=-4)) == L.FD_EINVAL
    assert call(lx=rows(col=-1)) == L.FD_EINVAL
    if call is not add_norm:
        assert call(lx=rows(c=0)) == L.FD_OK
    if call is not quantize:
        for eps in (-1.0, float("nan"), float("inf")):
            assert refused(call(eps=eps), L.FD_EINVAL, b"eps")
        assert refused(call(ws=-1), L.FD_EINVAL, b"stride")
        assert refused(call(wd=5), L.FD_EINVAL, b"w_dtype")


@nogpu
@pytest.mark.parametrize("call", [quantize, norm, add_norm])
def test_row_entries_refuse_overlaps(call):
    """Four rows of 64: inputs of 512 bytes (the weights 256), codes of 256, scales of 16."""
    inputs = {"x": X} if call is quantize else {"x": X, "w": W} if call is norm else {"x": X, "r": R, "w": W}
    for name, at in inputs.items():
        last = 255 if name == "w" else 511
        for where in (at, at + last, at - 255):
            assert refused(call(codes=where), L.FD_EINVAL, b"overlap"), (name, where - at)
        for where in (at, at + last - 3, at - 12):
            assert refused(call(scale=where), L.FD_EINVAL, b"overlap"), (name, where - at)
    assert refused(call(codes=Q, scale=Q + 252), L.FD_EINVAL, b"overlap")
    assert refused(call(codes=S + 12, scale=S), L.FD_EINVAL, b"overlap")


@nogpu
def test_a_residual_out_only_over_an_input_as_a_whole():
    assert refused(add_norm(ro=Q - 500), L.FD_EINVAL, b"overlap") and refused(add_norm(ro=S), L.FD_EINVAL, b"overlap")
    assert refused(add_norm(ro=W), L.FD_EINVAL, b"overlap")
    assert refused(add_norm(ro=X + 2), L.FD_EINVAL, b"overlap")
    assert refused(add_norm(ro=R - 128), L.FD_EINVAL, b"overlap")
    assert refused(add_norm(ro=X, lro=rows(sc=128)), L.FD_EINVAL, b"overlap")
    assert refused(add_norm(ro=R, lr=rows(sc=128), lro=rows()), L.FD_EINVAL, b"overlap")
    assert add_norm(lr=rows(c=5)) == L.FD_EINVAL and add_norm(lro=rows(n=32)) == L.FD_EINVAL
    assert add_norm(lx=rows(c=0), lr=rows(c=0), lro=rows(c=0), ro=X) == L.FD_OK


@nogpu
def test_too_many_rows():
    assert refused(quantize(codes=Q << 24, scale=S << 24, lx=rows(c=2**31, n=1, sc=0)), L.FD_EUNSUPPORTED, b"rows")


# ------------------------------------------------------------------ products, the C entry


def linear(y=Y, x=X, xs=S, w=W, ws=S + 0x1000, bias=None, bd=0, act=0, row=None, rd=0, m=40, n=64, k=128, sxm=None,
           swn=None, sb=1, srm=64, srn=1, sym=None, syn=1, scratch=None, size=0, dtype=0):
    nout = n // 2 if act == 5 else n
    return L.lib().fd_linear_w8a8(y, x, xs, w, ws, bias, bd, act, row, rd, m, n, k, k if sxm is None else sxm,
                                  k if swn is None else swn, sb, srm, srn, nout if sym is None else sym, syn, scratch,
                                  size, dtype, None)


def scratch(m, n, k, aligned=1):
    out = ctypes.c_int64(-1)
    return L.lib().fd_linear_w8a8_scratch(m, n, k, aligned, ctypes.byref(out)), out.value


@nogpu
def test_linear_refuses():
    assert refused(linear(dtype=2), L.FD_EINVAL, b"act_dtype")
    for name in ("m", "n", "k"):
        assert refused(linear(**{name: -1}), L.FD_EINVAL, b"size"), name
    for name in ("sxm", "swn", "sb", "srm", "srn", "sym", "syn"):
        assert refused(linear(**{name: -1}), L.FD_EINVAL, b"stride"), name
    assert refused(linear(act=6), L.FD_EINVAL, b"activation") and refused(linear(act=-1), L.FD_EINVAL, b"activation")
    assert refused(linear(act=5, n=63), L.FD_EINVAL, b"even")
    assert refused(linear(bias=P, bd=9), L.FD_EINVAL, b"bias_dtype")
    assert refused(linear(row=P, rd=-1), L.FD_EINVAL, b"row_dtype")
    for name in ("y", "x", "xs", "w", "ws"):
        assert refused(linear(**{name: None}), L.FD_EINVAL, b"null"), name
    assert linear(m=0, y=None) == L.FD_OK and linear(n=0, w=None) == L.FD_OK
    for name in ("m", "n", "k"):
        assert refused(linear(**{name: 2**31 - 1}), L.FD_EUNSUPPORTED, b"large"), name


@nogpu
def test_linear_refuses_an_output_over_an_operand():
    """40 x 64 outputs (5120 bytes) of 40 rows and 64 weight rows of 128 bytes."""
    for at, size in ((X, 5120), (W, 8192), (S, 160), (S + 0x1000, 256)):
        for where in (at, at + size - 1, at - 5119):
            assert refused(linear(y=where, ws=S + 0x1000 if at != S else Q), L.FD_EUNSUPPORTED, b"overlap")
    assert refused(linear(y=P, bias=P + 5118), L.FD_EUNSUPPORTED, b"overlap")
    assert refused(linear(y=P, row=P + 2), L.FD_EUNSUPPORTED, b"overlap")           # one element on
    assert refused(linear(y=P, row=P, rd=2), L.FD_EUNSUPPORTED, b"overlap")         # float32 under 16-bit outputs
    assert refused(linear(y=P, row=P, srm=0), L.FD_EUNSUPPORTED, b"overlap")        # one row under all


@nogpu
def test_rows_off_alignment_need_scratch():
    need = lambda status: refused(status, L.FD_EUNSUPPORTED, b"scratch")
    assert need(linear(k=129)) and need(linear(sxm=136)) and need(linear(swn=136))
    assert need(linear(x=X + 8)) and need(linear(w=W + 1))
    assert need(linear(y=1 << 40, swn=1 << 23))                              # offsets of a tile past 32 bits
    size = (40 + 64) * 144
    assert need(linear(k=129, scratch=P, size=size - 1)) and need(linear(k=129, scratch=None, size=size))
    assert refused(linear(k=129, scratch=P + 8, size=size), L.FD_EUNSUPPORTED, b"aligned")


def test_scratch_sizes():
    assert scratch(-1, 2, 3)[0] == L.FD_EINVAL and scratch(1, 2, -3)[0] == L.FD_EINVAL
    assert L.lib().fd_linear_w8a8_scratch(1, 2, 3, 1, None) == L.FD_EINVAL
    for m, n, k in ((0, 64, 128), (40, 0, 128), (40, 64, 15), (40, 64, 0), (2**31, 64, 128)):
        assert scratch(m, n, k, 0) == (L.FD_OK, 0)
    assert scratch(8, 64, 128) == (L.FD_OK, 0) and scratch(8, 64, 128, 0) == (L.FD_OK, 72 * 128)
    # K of no whole pieces is copied, aligned or not, in rows of whole ones
    assert scratch(8, 64, 129) == scratch(8, 64, 129, 0) == (L.FD_OK, 72 * 144)
    # K splits of few tiles: whole [M, N] sums, behind the copied rows
    (_, sums), (_, both) = scratch(64, 64, 16384), scratch(64, 64, 16384, 0)
    assert sums > 64 * 64 * 4 and sums % (64 * 64 * 4) == 0 and both == sums + 128 * 16384


# ------------------------------------------------------------------ the contract


def cuda(*shape, dtype=torch.float16):
    return torch.empty(shape, dtype=dtype, device="cuda")


def test_row_operators_check_their_arguments():
    with FakeTensorMode():
        x, w = cuda(3, 5, 64), cuda(64, dtype=torch.float32)
        codes, scale = cuda(3, 5, 64, dtype=E4M3), cuda(3, 5, dtype=torch.float32)
        for op, args in (("quantize_rows_fp8", dict(x=x)), ("rms_norm_fp8", dict(x=x, weight=w, eps=1e-6)),
                         ("add_rms_norm_fp8", dict(x=x, residual=x, weight=w, eps=1e-6, residual_out=None))):
            def given(out=None, scale_out=None, **other):
                return check(op, **{**args, **other}, out=out, scale_out=scale_out)

            given(), given(codes, scale)
            for wrong in (dict(x=cuda(3, 5, 64, dtype=torch.float32)), dict(out=cuda(3, 5, 64)), dict(x=None),
                          dict(scale_out=cuda(3, 5)), dict(out=3), dict(scale_out=1.0)):
                with pytest.raises(TypeError):
                    given(**wrong)
            for wrong in (dict(out=cuda(15, 64, dtype=E4M3)), dict(out=cuda(3, 64, 5, dtype=E4M3).transpose(1, 2)),
                          dict(scale_out=cuda(15, dtype=torch.float32)), dict(x=cuda()),
                          dict(scale_out=cuda(5, 3, dtype=torch.float32).t())):
                with pytest.raises(ValueError):
                    given(**wrong)
            if op != "quantize_rows_fp8":
                for wrong in (dict(weight=cuda(63)), dict(weight=cuda(1, 64)), dict(eps=-1.0), dict(eps=float("nan"))):
                    with pytest.raises(ValueError):
                        given(**wrong)
            if op == "add_rms_norm_fp8":
                for wrong in (dict(residual=cuda(3, 5, 32)), dict(residual_out=cuda(5, 3, 64))):
                    with pytest.raises(ValueError):
                        given(**wrong)
                with pytest.raises((TypeError, ValueError)):
                    given(residual=cuda(3, 5, 64, dtype=torch.bfloat16))


def test_linear_checks_its_arguments():
    with FakeTensorMode():
        good = dict(x=cuda(3, 5, 64, dtype=E4M3), x_scale=cuda(3, 5, dtype=torch.float32),
                    weight=cuda(30, 64, dtype=E4M3), scale=cuda(30, dtype=torch.float32), bias=None, activation=None,
                    row_add=None, out=None, dtype=None)
        given = lambda **other: check("linear_w8a8", **{**good, **other})
        assert given()["dtype"] is torch.bfloat16
        assert given(out=cuda(3, 5, 30))["dtype"] is torch.float16
        given(bias=cuda(30, dtype=torch.float32), activation="swiglu", row_add=cuda(15), dtype=torch.float16)
        for wrong in (dict(x=cuda(3, 5, 64)), dict(x=None), dict(x_scale=cuda(3, 5)), dict(x_scale=1.0),
                      dict(weight=cuda(30, 64)), dict(bias=[1.0]), dict(bias=cuda(30, dtype=torch.int32)),
                      dict(row_add=2), dict(dtype=torch.float32), dict(out=cuda(3, 5, 30, dtype=torch.float32)),
                      dict(out=3), dict(out=cuda(3, 5, 30), dtype=torch.bfloat16)):
            with pytest.raises(TypeError):
                given(**wrong)
        for wrong in (dict(x=cuda(dtype=E4M3)), dict(x_scale=cuda(15, dtype=torch.float32)),
                      dict(x_scale=cuda(3, 5, 1, dtype=torch.float32)), dict(weight=cuda(30, 65, dtype=E4M3)),
                      dict(weight=cuda(2, 30, 64, dtype=E4M3)), dict(scale=cuda(29, dtype=torch.float32)),
                      dict(scale=cuda(30)),
                      dict(bias=cuda(29)), dict(bias=cuda(1, 30)), dict(activation="tanh"), dict(activation=3),
                      dict(weight=cuda(31, 64, dtype=E4M3), scale=cuda(31, dtype=torch.float32), activation="swiglu")):
            with pytest.raises(ValueError):
                given(**wrong)


def test_tensors_off_the_gpu_are_refused():
    x, w = torch.randn(2, 64).half(), torch.ones(64)
    q, s = torch.zeros(2, 64, dtype=E4M3), torch.ones(2)
    for call in (lambda f: f.quantize_rows_fp8(x), lambda f: f.rms_norm_fp8(x, w, 1e-6),
                 lambda f: f.add_rms_norm_fp8(x, x, w, 1e-6), lambda f: f.linear_w8a8(q, s, q, s)):
        for where in (w8a8, torch.ops.fused_decode):
            with pytest.raises(ValueError, match="CUDA"):
                call(where)
    for call in (lambda: w8a8.quantize_rows_fp8(None), lambda: w8a8.rms_norm_fp8(x, None),
                 lambda: w8a8.rms_norm_fp8(3, w), lambda: w8a8.add_rms_norm_fp8(x, [1], w),
                 lambda: w8a8.linear_w8a8(q, s, None, s)):
        with pytest.raises((TypeError, ValueError)):
            call()


# ------------------------------------------------------------------ where a call goes


def test_fake_kernels_give_result_shapes():
    from fused_decode.library import OPS_W8A8

    f = torch.ops.fused_decode
    assert all(hasattr(f, name) for name in OPS_W8A8)
    with FakeTensorMode():
        x, w = cuda(2, 0, 3, 64, dtype=torch.bfloat16).transpose(1, 2), cuda(64)
        for got in (f.quantize_rows_fp8(x), f.rms_norm_fp8(x, w), f.add_rms_norm_fp8(x, x, w)):
            codes, scale = got[:2]
            assert codes.shape == (2, 3, 0, 64) and codes.dtype == E4M3 and codes.is_contiguous()
            assert scale.shape == (2, 3, 0) and scale.dtype == torch.float32
        assert got[2].dtype == torch.bfloat16 and got[2].is_contiguous()
        q, s = cuda(96, 64, dtype=E4M3), cuda(96, dtype=torch.float32)
        y = f.linear_w8a8(codes, scale, q, s)
        assert y.shape == (2, 3, 0, 96) and y.dtype == torch.bfloat16
        y = f.linear_w8a8(codes, scale, q, s, None, "swiglu", None, torch.float16)
        assert y.shape == (2, 3, 0, 48) and y.dtype == torch.float16
        # the public functions on tensors without memory
        assert w8a8.linear_w8a8(*w8a8.rms_norm_fp8(x, w), q, s, activation="relu").shape == (2, 3, 0, 96)


class Calls(list):
    """Stands in for the native binding: notes each call and returns FD_OK."""

    def __getattr__(self, name):
        def call(*args):
            self.append(name)
            return L.FD_OK
        return call


@pytest.fixture
def calls(monkeypatch):
    stand_in = Calls()
    monkeypatch.setattr(w8a8, "native", lambda: stand_in)
    monkeypatch.setattr(w8a8, "_raw_stream", lambda dev: 0)
    monkeypatch.setattr(w8a8, "_current_device", lambda: None)  # the CPU's index
    monkeypatch.setattr(w8a8._lib, "scratch_bytes", lambda *a: 0)
    monkeypatch.setattr(torch.cuda, "device", lambda dev: __import__("contextlib").nullcontext())

    def unchecked(op, **a):
        return {**a, "dtype": a.get("dtype") or torch.bfloat16}

    monkeypatch.setattr(w8a8, "check", unchecked)
    ops.clear_plans()
    yield stand_in
    ops.clear_plans()


def arguments():
    x, w = torch.randn(3, 64).half(), torch.ones(64)
    q, s = torch.zeros(30, 64, dtype=E4M3), torch.ones(30)
    return x, w, q, s


def test_plain_calls_launch_once(calls):
    x, w, q, s = arguments()
    codes, scale = w8a8.quantize_rows_fp8(x)
    assert codes.dtype == E4M3 and codes.shape == x.shape and codes.is_contiguous() and scale.shape == (3,)
    w8a8.rms_norm_fp8(x, w)
    w8a8.add_rms_norm_fp8(x, x, w)
    y = w8a8.linear_w8a8(codes, scale, q, s, activation="swiglu", dtype=torch.float16)
    assert y.shape == (3, 15) and y.dtype == torch.float16
    assert calls == ["quantize_rows_fp8", "rms_norm_fp8", "add_rms_norm_fp8", "linear_w8a8"]


def test_a_traced_graph_keeps_the_custom_ops():
    with FakeTensorMode():
        x, w, q, s = cuda(3, 64), cuda(64), cuda(30, 64, dtype=E4M3), cuda(30, dtype=torch.float32)

        def f(x, w, q, s):
            c, t, h = w8a8.add_rms_norm_fp8(x, x, w)
            return w8a8.linear_w8a8(c, t, q, s, row_add=s), w8a8.quantize_rows_fp8(h)

        graph = make_fx(f)(x, w, q, s).graph
    targets = [str(n.target) for n in graph.nodes if n.op == "call_function"]
    for name in ("add_rms_norm_fp8", "linear_w8a8", "quantize_rows_fp8"):
        assert sum(t.startswith(f"fused_decode.{name}") for t in targets) == 1


def test_a_gradient_or_a_negation_does_not_reach_the_plain_launch(calls, monkeypatch):
    x, w, q, s = arguments()
    seen = []

    class Stand:
        def __getattr__(self, name):
            return lambda *a: seen.append(name) or (torch.zeros(3, 64, dtype=E4M3), torch.ones(3), x) \
                if name != "linear_w8a8" else seen.append(name) or torch.zeros(3, 30)

    monkeypatch.setattr(torch.ops, "fused_decode", Stand(), raising=False)
    leaf = lambda t: t.clone().requires_grad_()
    neg = torch._neg_view
    c = torch.zeros(3, 64, dtype=E4M3)
    w8a8.quantize_rows_fp8(leaf(x)), w8a8.quantize_rows_fp8(neg(x))
    w8a8.rms_norm_fp8(x, leaf(w)), w8a8.rms_norm_fp8(x, neg(w)), w8a8.rms_norm_fp8(neg(x), w)
    w8a8.add_rms_norm_fp8(x, leaf(x), w), w8a8.add_rms_norm_fp8(x, neg(x), w)
    w8a8.linear_w8a8(c, torch.ones(3), q, leaf(s)), w8a8.linear_w8a8(c, torch.ones(3), q, s, neg(s))
    w8a8.linear_w8a8(c, torch.ones(3), q, s, row_add=neg(s)), w8a8.linear_w8a8(c, neg(torch.ones(3)), q, s)
    assert calls == [] and len(seen) == 11
    with torch.no_grad():
        w8a8.quantize_rows_fp8(leaf(x))
    assert calls == ["quantize_rows_fp8"]


def test_outputs_that_torch_would_not_write_are_refused(calls):
    x, w, q, s = arguments()
    c, t = torch.zeros(3, 64, dtype=E4M3), torch.ones(3)
    with pytest.raises(RuntimeError, match="gradient"):
        w8a8.add_rms_norm_fp8(x, x, w, residual_out=x.clone().requires_grad_())
    with pytest.raises(RuntimeError, match="gradient"):
        w8a8.rms_norm_fp8(x, w, scale_out=t.clone().requires_grad_())
    with torch.inference_mode():
        out = torch.empty(3, 30, dtype=torch.bfloat16)
        assert w8a8.linear_w8a8(c, t, q, s, out=out) is out
    with pytest.raises(RuntimeError, match="inference"):
        w8a8.linear_w8a8(c, t, q, s, out=out)
    out = torch.empty(3, 30, dtype=torch.bfloat16)
    before = out._version
    w8a8.linear_w8a8(c, t, q, s, out=out)
    assert out._version > before
    with pytest.raises(ValueError):
        w8a8.linear_w8a8(c, t, q, s, out=torch.empty(3, 31, dtype=torch.bfloat16))

"""norm_add_norm on the CPU: what its entry point and the argument contract refuse, its fake kernel, and which calls go to
the custom op."""

from __future__ import annotations

import contextlib

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

from fused_decode import _lib as L
from fused_decode import block_norms, ops
from fused_decode._checks import check

# The entry point's checks return before any HIP call; no pointer is read.
nogpu = pytest.mark.skipif(torch.cuda.is_available(), reason="host-only argument checks")
X, R, Y, RO, G, PW, W = (0x100000 * i for i in range(1, 8))  # far apart


def rows(a=1, b=1, c=4, n=64, col=1, sc=None):
    return L.FdRows(a, b, c, 0, 0, n if sc is None else sc, col, n)


def refused(status, code, words):
    return status == code and words in L.lib().fd_last_error()


def norms(y=Y, ro=RO, x=X, r=R, g=None, gd=2, pw=PW, pd=2, ps=1, w=W, wd=2, ws=1, lx=None, lr=None, lg=None, ly=None,
          lro=None, scale=1.0, eps=1e-6, act=0):
    full = lambda l: l or rows()
    return L.lib().fd_norm_add_norm(y, ro, x, r, g, gd, pw, pd, ps, w, wd, ws, full(lx), full(lr), full(lg), full(ly),
                                    full(lro), scale, eps, act, None)


@nogpu
def test_the_entry_refuses():
    assert refused(norms(act=2), L.FD_EINVAL, b"act_dtype")
    for name in ("y", "ro", "x", "r", "pw", "w"):
        assert refused(norms(**{name: None}), L.FD_EINVAL, b"null"), name
    for name in ("lx", "lr", "ly", "lro"):
        assert norms(**{name: rows(n=-1)}) == L.FD_EINVAL and norms(**{name: rows(c=5)}) == L.FD_EINVAL, name
        assert norms(**{name: rows(col=-1)}) == L.FD_EINVAL, name
    assert norms(g=G, lg=rows(c=5)) == L.FD_EINVAL and norms(g=G, gd=7) == L.FD_EINVAL
    assert refused(norms(pd=4), L.FD_EINVAL, b"post_w_dtype") and refused(norms(wd=-1), L.FD_EINVAL, b"w_dtype")
    assert refused(norms(ps=-1), L.FD_EINVAL, b"stride") and refused(norms(ws=-1), L.FD_EINVAL, b"stride")
    for eps in (-1.0, float("nan"), float("inf")):
        assert refused(norms(eps=eps), L.FD_EINVAL, b"eps")
    for scale in (float("nan"), float("inf"), -float("inf")):
        assert refused(norms(scale=scale), L.FD_EINVAL, b"residual_scale")
    none = dict.fromkeys(("lx", "lr", "ly", "lro"), rows(c=0))
    assert norms(**none) == L.FD_OK
    many = dict.fromkeys(("lx", "lr"), rows(c=2**31, n=1, sc=0))
    assert refused(norms(**many, ly=rows(c=2**31, n=1), lro=rows(c=2**31, n=1)), L.FD_EUNSUPPORTED, b"rows")


@nogpu
def test_the_entry_refuses_overlaps():
    """Four rows of 64: 512 bytes each, the weights 256."""
    for out in ("y", "ro"):
        for at, size in ((PW, 256), (W, 256)):
            for where in (at, at + size - 1, at - 511):
                assert refused(norms(**{out: where}), L.FD_EINVAL, b"weight"), (out, where)
        assert refused(norms(g=G, lg=rows(sc=0), **{out: G + 255}), L.FD_EINVAL, b"gate")
        for at in (X, R):
            for where in (at + 2, at - 510):
                assert refused(norms(**{out: where}), L.FD_EINVAL, b"overlap"), (out, where)
        other = {"y": "ly", "ro": "lro"}[out]
        assert refused(norms(**{out: X, other: rows(sc=128)}), L.FD_EINVAL, b"overlap")
        assert refused(norms(**{other: rows(sc=0)}), L.FD_EINVAL, b"share")
        assert refused(norms(**{other: rows(sc=32)}), L.FD_EINVAL, b"share")
    assert refused(norms(y=RO + 510), L.FD_EINVAL, b"each other")
    assert refused(norms(y=X, ro=X), L.FD_EINVAL, b"each other")


def cuda(*shape, dtype=torch.float16):
    return torch.empty(shape, dtype=dtype, device="cuda")


def test_the_contract():
    with FakeTensorMode():
        x, w = cuda(3, 5, 64), cuda(64, dtype=torch.float32)
        good = dict(x=x, residual=x, post_weight=w, weight=w, eps=1e-6, gate=None, residual_scale=1, out=None,
                    residual_out=None)
        given = lambda **other: check("norm_add_norm", **{**good, **other})
        assert given()["residual_scale"] == 1.0
        for gate in (cuda(64), cuda(5, 1), cuda(3, 1, 64, dtype=torch.float32), cuda(3, 5, 64), cuda()):
            given(gate=gate)
        given(out=cuda(3, 5, 128)[..., ::2], residual_out=x)
        for wrong in (dict(x=cuda(3, 5, 64, dtype=torch.float32)), dict(x=None), dict(gate=2.0), dict(out=3),
                      dict(gate=cuda(64, dtype=torch.int32)), dict(out=cuda(3, 5, 64, dtype=torch.bfloat16)),
                      dict(residual=None), dict(weight=cuda(64, dtype=torch.float64))):
            with pytest.raises(TypeError):
                given(**wrong)
        for wrong in (dict(residual=cuda(3, 5, 32)), dict(post_weight=cuda(63)), dict(weight=cuda(1, 64)),
                      dict(gate=cuda(4, 64)), dict(gate=cuda(1, 3, 5, 64)), dict(eps=-1.0), dict(residual_scale="a"),
                      dict(residual_scale=float("nan")), dict(residual_scale=1e39), dict(out=cuda(5, 3, 64)),
                      dict(residual_out=cuda(1, 5, 64).expand(3, 5, 64)), dict(x=cuda())):
            with pytest.raises(ValueError):
                given(**wrong)


def test_tensors_off_the_gpu_are_refused():
    x, w = torch.randn(2, 64).half(), torch.ones(64)
    for where in (block_norms, torch.ops.fused_decode):
        with pytest.raises(ValueError, match="CUDA"):
            where.norm_add_norm(x, x, w, w)
    for args in ((None, x, w, w), (x, 3, w, w), (x, x, None, w), (x, x, w, [1])):
        with pytest.raises((TypeError, ValueError)):
            block_norms.norm_add_norm(*args)


def test_the_fake_kernel_and_a_traced_graph():
    with FakeTensorMode():
        x, w = cuda(2, 0, 3, 64, dtype=torch.bfloat16).transpose(1, 2), cuda(64)
        for got in (torch.ops.fused_decode.norm_add_norm(x, x, w, w), block_norms.norm_add_norm(x, x, w, w, gate=w)):
            assert [(t.shape, t.dtype, t.is_contiguous()) for t in got] == [((2, 3, 0, 64), torch.bfloat16, True)] * 2
        x = cuda(3, 64)
        graph = make_fx(lambda x, w: block_norms.norm_add_norm(x, x, w, w, residual_scale=0.5))(x, w).graph
    assert sum(str(n.target).startswith("fused_decode.norm_add_norm") for n in graph.nodes) == 1


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
    monkeypatch.setattr(block_norms, "native", lambda: stand_in)
    monkeypatch.setattr(block_norms, "_raw_stream", lambda dev: 0)
    monkeypatch.setattr(block_norms, "_current_device", lambda: None)  # the CPU's index
    monkeypatch.setattr(torch.cuda, "device", lambda dev: contextlib.nullcontext())
    monkeypatch.setattr(block_norms, "check", lambda op, **a: a)
    ops.clear_plans()
    yield stand_in
    ops.clear_plans()


def test_calls_launch_once_and_keep_a_plan(calls):
    x, w = torch.randn(3, 64).half(), torch.ones(64)
    for _ in range(2):
        y, t = block_norms.norm_add_norm(x, x, w, w)
    assert y.shape == t.shape == x.shape and len(calls) == 2 and len(ops._PLANS) == 1
    block_norms.norm_add_norm(x, x, w, w, residual_scale=0.5)
    block_norms.norm_add_norm(x, x, w, w, gate=w)
    assert len(ops._PLANS) == 3 and calls[2][1][17] == 0.5 and calls[3][1][4] == w.data_ptr()
    stream = x.clone()
    before = stream._version
    assert block_norms.norm_add_norm(x, stream, w, w, residual_out=stream)[1] is stream and stream._version > before
    four = torch.zeros(5, 4, 3, 2, 8, dtype=torch.float16).permute(3, 2, 1, 0, 4)  # no two leading dims merge
    y, t = block_norms.norm_add_norm(four, four, w[:8], w[:8], residual_out=four)
    assert t is four and y.is_contiguous()
    wide = torch.zeros(5, 4, 3, 2, 16, dtype=torch.float16).permute(3, 2, 1, 0, 4)
    with pytest.raises(L.FusedDecodeError, match="overlap"):
        block_norms.norm_add_norm(four, four, w[:8], w[:8], out=wide[..., :8], residual_out=wide[..., 8:])


def test_recorded_calls_go_to_the_custom_op(calls, monkeypatch):
    x, w = torch.randn(3, 64).half(), torch.ones(64)
    seen = []

    class Stand:
        def __getattr__(self, name):
            return lambda *a: seen.append(name) or (x.clone(), x.clone())

    monkeypatch.setattr(torch.ops, "fused_decode", Stand(), raising=False)
    leaf, neg = lambda t: t.clone().requires_grad_(), torch._neg_view
    for args, gate in (((leaf(x), x, w, w), None), ((x, leaf(x), w, w), None), ((x, x, leaf(w), w), None),
                       ((x, x, w, leaf(w)), None), ((x, x, w, w), leaf(w)), ((neg(x), x, w, w), None),
                       ((x, x, w, w), neg(w))):
        block_norms.norm_add_norm(*args, gate=gate)
    assert calls == [] and seen == ["norm_add_norm"] * 7
    out = torch.empty_like(x)
    assert block_norms.norm_add_norm(leaf(x), x, w, w, out=out)[0] is out
    with torch.no_grad():
        block_norms.norm_add_norm(leaf(x), x, w, w)
    assert len(calls) == 1
    with pytest.raises(RuntimeError, match="gradient"):
        block_norms.norm_add_norm(x, x, w, w, out=leaf(x))

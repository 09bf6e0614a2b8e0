"""Outputs whose own elements share memory, on the CPU: what finds them, and the operators and entry points that refuse
them. Nothing here is launched: the entry points' checks return before any HIP call, and a layout that passes is given
an output over the weights, which is refused next."""

from __future__ import annotations

import itertools
import random

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from fused_decode import _lib as L
from fused_decode import w8a8
from fused_decode._checks import check
from fused_decode._layout import shares_memory

nogpu = pytest.mark.skipif(torch.cuda.is_available(), reason="host-only argument checks")
X, W, Y, Q, S, R = (0x1000000 * i for i in range(1, 7))  # far apart


def rows(a=1, b=1, c=4, n=64, sa=0, sb=0, sc=64, col=1):
    return L.FdRows(a, b, c, sa, sb, sc, col, n)


def add_norm_fp8(ro, lx, lro):
    return L.lib().fd_add_rms_norm_fp8(Q, S, ro, X, R, W, 2, 1, lx, lx, lro, 1e-6, 0, None)


def add_norm(ro, lx, lro):
    return L.lib().fd_add_rms_norm(Y, ro, X, R, W, 2, 1, lx, lx, lx, lro, 1e-6, 0, None)


def share(status):
    return status == L.FD_EINVAL and b"share memory" in L.lib().fd_last_error()


SHARED = [dict(sc=0), dict(sc=63), dict(sc=32), dict(sc=1), dict(col=0), dict(col=2, sc=64), dict(a=3, sa=0),
          dict(a=3, sa=64), dict(b=2, sb=192), dict(col=4, sc=2, n=8, c=3)]


@nogpu
@pytest.mark.parametrize("call", [add_norm_fp8, add_norm])
@pytest.mark.parametrize("strides", SHARED)
def test_entries_refuse_a_residual_out_whose_rows_share_memory(call, strides):
    """In place (over x, over the residual) and beside."""
    sizes = {k: v for k, v in strides.items() if k in "abcn"}
    lx, lro = rows(**sizes), rows(**strides)
    assert share(call(X + 0x100000, lx, lro)) and share(call(Y + 0x100000, lx, lro))
    lib, e = L.lib(), (1e-6, 0, None)
    if call is add_norm_fp8:
        assert share(lib.fd_add_rms_norm_fp8(Q, S, R, X, R, W, 2, 1, lx, lro, lro, *e))
        assert share(lib.fd_add_rms_norm_fp8(Q, S, X, X, R, W, 2, 1, lro, lx, lro, *e))
    else:
        assert share(lib.fd_add_rms_norm(Y, R, X, R, W, 2, 1, lx, lro, lx, lro, *e))


@nogpu
def test_the_entry_finds_what_an_enumeration_finds():
    r = random.Random(3)
    found = [0, 0]
    for _ in range(3000):
        size = [r.randint(1, 5) for _ in range(4)]
        step = [r.randint(0, 9) if r.random() < 0.6 else r.randint(0, 60) for _ in range(4)]
        at = [sum(i * s for i, s in zip(index, step)) for index in itertools.product(*map(range, size))]
        same = len(set(at)) < len(at)
        a, b, c, n = size
        lx = rows(a, b, c, n, b * c * n, c * n, n)
        lro = rows(a, b, c, n, *step)
        assert add_norm_fp8(W, lx, lro) == L.FD_EINVAL  # over the weights: refused in any case
        assert (b"share memory" in L.lib().fd_last_error()) == same == shares_memory(size, step)
        found[same] += 1
    assert min(found) > 300
    for call in (add_norm_fp8, add_norm):
        assert call(Y + 0x100000, rows(c=0), rows(c=0, sc=0, col=0)) == L.FD_OK  # of no row


def test_views_that_share_nothing():
    t = torch.empty(6, 7, 8, 9)
    for v in (t, t.transpose(0, 2), t[::2, 1:, ::3], t[..., 2:5], t.permute(3, 1, 0, 2), t[:1].transpose(0, 1), t[0, 0, 0],
              torch.empty(9, 9).diagonal(), torch.empty(4, 9, 9).diagonal(dim1=1, dim2=2), torch.empty(3, 0, 5).expand(3, 0, 5),
              torch.empty(1, 4).expand(1, 4), torch.empty(()), torch.empty(8).as_strided((2, 3), (3, 2))):
        assert not shares_memory(v.shape, v.stride())
    for v in (torch.empty(4).expand(3, 4), torch.empty(3, 1).expand(3, 4), torch.empty(20).unfold(0, 8, 4),
              torch.empty(50).as_strided((3, 4, 5), (8, 3, 2)), torch.empty(4, 1, 5).expand(4, 2, 5).transpose(0, 1)):
        assert shares_memory(v.shape, v.stride())


@pytest.mark.parametrize("op", ["add_rms_norm_fp8", "add_rms_norm"])
def test_operators_refuse_them(op):
    with FakeTensorMode():
        x, w = torch.empty(6, 64, dtype=torch.float16, device="cuda"), torch.empty(64, device="cuda")
        args = dict(x=x, weight=w, eps=1e-6, out=None)
        if op == "add_rms_norm_fp8":
            args["scale_out"] = None
        wide = torch.empty(6, 128, dtype=torch.float16, device="cuda")
        for good in (None, x, wide[:, ::2], wide[:, 64:], torch.empty(64, 6, dtype=torch.float16, device="cuda").t()):
            check(op, **args, residual=x, residual_out=good)
        row = torch.empty(64, dtype=torch.float16, device="cuda")
        column = torch.empty(6, 1, dtype=torch.float16, device="cuda")
        long = torch.empty(64 + 5 * 32, dtype=torch.float16, device="cuda")
        for bad in (row.expand(6, 64), column.expand(6, 64), long.unfold(0, 64, 32)):
            for residual in (x, bad):
                with pytest.raises(ValueError, match="residual_out.*share memory"):
                    check(op, **args, residual=residual, residual_out=bad)


def test_a_recorded_call_refuses_them():
    """The way through the custom op, whose result is copied into the output."""
    got = (torch.zeros(6, 64), torch.zeros(6))
    with pytest.raises(ValueError, match="share memory"):
        w8a8._copied(got, torch.zeros(224).unfold(0, 64, 32), None)
    out = torch.ones(6, 64)
    assert w8a8._copied(got, out, None)[0] is out and bool((out == 0).all())


@nogpu
def test_the_product_refuses_an_output_whose_elements_share_memory():
    """40 x 64 outputs, 40 x 32 with SwiGLU; a layout that passes is then refused for its overlap with the weights."""
    def linear(y, sym, syn, act=0, m=40):
        return L.lib().fd_linear_w8a8(y, X, S, W, S + 0x1000, None, 0, act, None, 0, m, 64, 128, 128, 128, 1, 0, 0, sym, syn,
                                      None, 0, 0, None)

    for sym, syn in ((0, 1), (63, 1), (64, 0), (1, 39), (128, 4)):
        assert share(linear(Y, sym, syn)), (sym, syn)
    assert share(linear(Y, 31, 1, act=5)) and share(linear(Y, 0, 0, m=1))
    for sym, syn, m in ((64, 1, 40), (70, 1, 40), (1, 40, 40), (128, 2, 40), (0, 1, 1)):
        assert linear(W, sym, syn, m=m) == L.FD_EUNSUPPORTED and b"overlap" in L.lib().fd_last_error()
    assert linear(W, 32, 1, act=5) == L.FD_EUNSUPPORTED

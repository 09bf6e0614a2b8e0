"""Calls of the operators with 8-bit activations that reach a launch by another way than the plain one, on the CPU with
the library's calls replaced by ones that only note their names."""

from __future__ import annotations

import pytest
import torch
from test_w8a8 import E4M3, arguments, calls, cuda  # noqa: F401 (a fixture)
from torch._subclasses.fake_tensor import FakeTensorMode

from fused_decode import _lib as L
from fused_decode import ops, w8a8


def unmergeable(dtype):
    """Rows of 8 in four leading dims of which no two merge."""
    return torch.zeros(5, 4, 3, 2, 8, dtype=dtype).permute(3, 2, 1, 0, 4)


def test_gathered_rows_refuse_outputs_over_each_other(calls):  # noqa: F811
    """The sums come back by a copy, behind the codes: it must not land on them."""
    x, r, w = unmergeable(torch.float16), unmergeable(torch.float16), torch.ones(8)
    memory = torch.zeros(4 * 960, dtype=torch.uint8)
    residual_out = memory[:1920].view(torch.float16).view(5, 4, 3, 2, 8).permute(3, 2, 1, 0, 4)
    codes = lambda at: memory[at : at + 960].view(E4M3).view(x.shape)
    scale = lambda at: memory[at : at + 480].view(torch.float32).view(x.shape[:-1])
    for out, scale_out in ((codes(0), None), (codes(1919), None), (None, scale(0)), (codes(1920), scale(1916))):
        with pytest.raises(L.FusedDecodeError, match="overlap"):
            w8a8.add_rms_norm_fp8(x, r, w, out=out, scale_out=scale_out, residual_out=residual_out)
    assert calls == []
    got = w8a8.add_rms_norm_fp8(x, r, w, out=codes(1920), scale_out=scale(2880), residual_out=residual_out)
    assert got[2] is residual_out and calls == ["add_rms_norm_fp8"]
    w8a8.add_rms_norm_fp8(x, residual_out, w, residual_out=residual_out)


def test_an_eps_that_changes_is_read_again(calls, monkeypatch):  # noqa: F811
    """A tensor, or a number of numpy's, given as eps: plans are not kept by the tensor's identity."""
    import numpy as np

    x, w, q, s = arguments()
    seen = []
    monkeypatch.setattr(w8a8, "check", lambda op, **a: {"eps": float(a["eps"])})
    monkeypatch.setattr(type(calls), "rms_norm_fp8", lambda self, *a: seen.append(a[7]) or L.FD_OK, raising=False)
    eps = torch.tensor(0.5)
    w8a8.rms_norm_fp8(x, w, eps)
    eps.fill_(0.25)
    w8a8.rms_norm_fp8(x, w, eps)
    w8a8.rms_norm_fp8(x, w, np.float32(0.125))
    w8a8.rms_norm_fp8(x, w, 0.125)
    assert seen == [0.5, 0.25, 0.125, 0.125]
    assert len(ops._PLANS) == 1
    ops._remember(("op", x.shape, x.stride(), (torch.float16, None, b"env"), 1e-6, True), lambda: None)
    assert len(ops._PLANS) == 2


@pytest.mark.parametrize("error", [AttributeError, TypeError, RuntimeError])
def test_an_error_of_the_custom_op_is_the_calls(calls, monkeypatch, error):  # noqa: F811
    """What a trace or a transform raises is not taken for a wrong argument, behind which the launch would follow."""
    x, w, q, s = arguments()

    class Raises:
        def __getattr__(self, name):
            def op(*args):
                raise error(name)
            return op

    monkeypatch.setattr(torch.ops, "fused_decode", Raises(), raising=False)
    leaf, c, t = x.clone().requires_grad_(), torch.zeros(3, 64, dtype=E4M3), torch.ones(3)
    for call in (lambda: w8a8.quantize_rows_fp8(leaf), lambda: w8a8.rms_norm_fp8(leaf, w),
                 lambda: w8a8.add_rms_norm_fp8(x, leaf, w), lambda: w8a8.linear_w8a8(c, t, q, torch._neg_view(s))):
        with pytest.raises(error, match="fp8|w8a8"):
            call()
    assert calls == []


def test_recorded_calls_name_an_output_that_is_no_tensor():
    x = torch.zeros(3, 64)
    with pytest.raises(TypeError, match="output"):
        w8a8._copied((x,), 3)


class Watching(torch.Tensor):
    """A subclass that notes the functions it meets."""

    seen: list = []

    @classmethod
    def __torch_function__(cls, func, types, args=(), kwargs=None):
        cls.seen.append(str(func))
        return super().__torch_function__(func, types, args, kwargs or {})


class Holder(torch.Tensor):
    """A wrapper without memory of its own: a launch on its pointer would read none of the held tensor's."""

    met: list = []

    @staticmethod
    def __new__(cls, held):
        return torch.Tensor._make_wrapper_subclass(cls, held.shape, strides=held.stride(), dtype=held.dtype,
                                                   device=held.device)

    def __init__(self, held):
        self.held = held

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        cls.met.append(str(func))
        return func(*[a.held if isinstance(a, Holder) else a for a in args], **(kwargs or {}))


def each_operator():
    """(name, argument count, call of those tensors) for every operator."""
    x, w, q, s = arguments()
    c, t, r = torch.zeros(3, 64, dtype=E4M3), torch.ones(3), torch.zeros(3, 30)
    return (("quantize_rows_fp8", [x], w8a8.quantize_rows_fp8), ("rms_norm_fp8", [x, w], w8a8.rms_norm_fp8),
            ("add_rms_norm_fp8", [x, x.clone(), w], w8a8.add_rms_norm_fp8),
            ("linear_w8a8", [c, t, q, s, s.clone(), r], lambda *a: w8a8.linear_w8a8(*a[:5], row_add=a[5])))


def test_subclasses_see_the_call(calls):  # noqa: F811
    """Each argument in turn; a Parameter is no such subclass."""
    for name, args, call in each_operator():
        for i in range(len(args)):
            given = list(args)
            Watching.seen.clear()
            given[i] = args[i].as_subclass(Watching)
            call(*given)
            assert any(f"fused_decode.{name}" in f for f in Watching.seen), (name, i)
            Holder.met.clear()
            given[i] = Holder(args[i])
            call(*given)
            assert any(f.startswith(f"fused_decode.{name}") for f in Holder.met), (name, i)
            given[i] = torch.nn.Parameter(args[i], requires_grad=False)
            Watching.seen.clear(), Holder.met.clear()
            call(*given)
            assert not Watching.seen and not Holder.met


def test_a_subclass_as_output_is_written_by_torch(calls):  # noqa: F811
    x, w, q, s = arguments()
    out, t = Holder(torch.empty(3, 30, dtype=torch.bfloat16)), torch.ones(3)
    Holder.met.clear()
    assert w8a8.linear_w8a8(torch.zeros(3, 64, dtype=E4M3), t, q, s, out=out) is out
    assert any("copy_" in f for f in Holder.met)
    residual_out = Holder(x.clone())
    Holder.met.clear()
    assert w8a8.add_rms_norm_fp8(x, x, w, residual_out=residual_out)[2] is residual_out
    assert any("copy_" in f for f in Holder.met)


def test_custom_ops_keep_their_plans(calls, monkeypatch):  # noqa: F811
    """One plan a signature, whatever values the tensors hold; another one for other strides, eps and activations."""
    plans, check = [], w8a8.check
    monkeypatch.setattr(w8a8, "check", lambda op, **a: plans.append(op) or check(op, **a))
    f, (x, w, q, s) = torch.ops.fused_decode, arguments()
    c, t = torch.zeros(3, 64, dtype=E4M3), torch.ones(3)
    for _ in range(3):
        f.quantize_rows_fp8(x.clone()), f.rms_norm_fp8(x, w.clone(), 1e-5), f.add_rms_norm_fp8(x, x.clone(), w, 1e-5)
        f.linear_w8a8(c, t.clone(), q, s, None, "relu"), f.linear_w8a8(c, t, q, s, None, "silu")
        f.linear_w8a8(c, t, q, s, s.clone(), None, torch.zeros(30), torch.float16)
    assert len(calls) == 18 and len(plans) == 6
    f.rms_norm_fp8(x, w, 1e-6), f.quantize_rows_fp8(x.t().contiguous().t()), f.quantize_rows_fp8(x)
    assert len(calls) == 21 and len(plans) == 8


@pytest.mark.parametrize("shape", [(), (0,), (1,), (3, 4), (5, 1, 7), (2, 0, 3)])
def test_plans_hold_no_memory(shape):
    """What a plan makes its results of has their shape, and none of the memory that it was made in."""
    for dtype in (E4M3, torch.float32, torch.bfloat16):
        like = w8a8._like(shape, dtype, torch.device("cpu"))
        assert like.untyped_storage().nbytes() == 0
        made = torch.empty_like(like)
        assert made.shape == shape and made.dtype == dtype and made.is_contiguous()
        assert made.zero_().float().sum() == 0


def test_results_of_no_element_lie_as_the_fake_kernels_say(calls):  # noqa: F811
    """Contiguous, whatever the strides of a batch of no rows: a compiled graph checks what it was told."""
    x, w = torch.empty(2, 0, 3, 64, dtype=torch.bfloat16).transpose(1, 2), torch.ones(64)
    got = w8a8.add_rms_norm_fp8(x, x, w)
    with FakeTensorMode():
        fx, fw = cuda(2, 0, 3, 64, dtype=torch.bfloat16).transpose(1, 2), cuda(64)
        fake = torch.ops.fused_decode.add_rms_norm_fp8(fx, fx, fw)
    assert [(t.shape, t.stride(), t.dtype) for t in got] == [(t.shape, t.stride(), t.dtype) for t in fake]
    assert calls == []


@pytest.mark.parametrize("dynamic", [False, True])
def test_a_compiled_call_with_outputs_stays_whole(dynamic):
    """Sizes that are symbols, outputs given, the residual in place: one graph with the custom op and its copies. (It is run
    only as far as the op, which refuses the CPU.)"""
    graphs = []

    def backend(module, inputs):
        graphs.append([str(n.target) for n in module.graph.nodes if n.op == "call_function"])
        return module.forward

    x, w, q, s = arguments()
    torch._dynamo.reset()
    f = torch.compile(lambda x, r, w, c, t: w8a8.add_rms_norm_fp8(x, r, w, out=c, scale_out=t, residual_out=r),
                      backend=backend, fullgraph=True, dynamic=dynamic)
    wide = torch.zeros(3, 128, dtype=torch.float16)
    for residual in (x.clone(), wide[:, :64]):
        with pytest.raises(ValueError, match="CUDA"):
            f(x, residual, w, torch.zeros(3, 64, dtype=E4M3), torch.ones(3))
    assert graphs and all(sum(t.startswith("fused_decode.add_rms_norm_fp8") for t in g) == 1 for g in graphs)
    torch._dynamo.reset()

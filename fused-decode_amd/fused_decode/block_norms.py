"""The norms around a block: after its output and before the next one, with the block's residual between them.

    y, stream = norm_add_norm(x, residual, post_weight, weight, eps, gate=g, residual_scale=s)

        t = residual + s * g * rms_norm(x, post_weight, eps)        float32
        y = rms_norm(t, weight, eps),  stream = round(t)

in one launch: what ``rms_norm`` of the block's output, the gated addition and ``add_rms_norm``'s norm of the
unrounded sum compute, with one rounding each for ``y`` and the stream. A layer whose blocks are normed on both sides:

    y, h = norm_add_norm(attention(...), x, post_attn_norm, mlp_norm)
    y, x = norm_add_norm(mlp(y), h, post_mlp_norm, next_attn_norm)

Inference only. Where a gradient, a trace or a transform is asked for, the call goes to the custom op of the same name
(``torch.ops.fused_decode.norm_add_norm``), which a graph keeps whole and which says that it has no gradient. There is no
reference counterpart (the reference norms before a block only).
"""

from __future__ import annotations

import math

import torch
from torch.autograd.graph import increment_version

from ._checks import check
from ._layout import contiguous_strides, plan_rows
from ._lib import DTYPE_CODE, FD_EINVAL, FdRows, FusedDecodeError, fail, native
from .ops import _PLANS, _raw_stream, _remember, _sig
from .w8a8 import _PLAIN, _copied, _current_device, _grad, _like, _meet, _out_sig, _subclasses, _watched

__all__ = ["norm_add_norm"]


def norm_add_norm(
    x: torch.Tensor,
    residual: torch.Tensor,
    post_weight: torch.Tensor,
    weight: torch.Tensor,
    eps: float = 1e-6,
    *,
    gate: torch.Tensor | None = None,
    residual_scale: float = 1.0,
    out: torch.Tensor | None = None,
    residual_out: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """``(rms_norm(t, weight), t)`` for ``t = residual + residual_scale * gate * rms_norm(x, post_weight)`` in float32,
    over the last dimension. ``post_weight`` and ``weight`` are ``(N,)``; ``gate`` (None for 1) has any float dtype and
    broadcasts to ``x``: one a channel ``(N,)``, one a row ``(..., 1)``, one an element. ``residual_out=residual`` updates
    the residual stream in place; ``out`` and ``residual_out`` may each be ``x`` or ``residual``, not one another."""
    try:
        recorded = (_watched()
                    or (_grad() and (x.requires_grad or residual.requires_grad or post_weight.requires_grad
                                     or weight.requires_grad or (gate is not None and gate.requires_grad)))
                    or x.is_neg() or residual.is_neg() or post_weight.is_neg() or weight.is_neg()
                    or (gate is not None and gate.is_neg())
                    or (not (x.__class__ in _PLAIN and residual.__class__ in _PLAIN and post_weight.__class__ in _PLAIN
                             and weight.__class__ in _PLAIN and gate.__class__ in _PLAIN and out.__class__ in _PLAIN
                             and residual_out.__class__ in _PLAIN)
                        and _subclasses(x, residual, post_weight, weight, gate, out, residual_out)))
        if not recorded:
            key = ("norm_add_norm", x.shape, x.stride(), x.dtype, x.get_device(), residual.shape, residual.stride(),
                   residual.dtype, residual.get_device(), post_weight.shape, post_weight.stride(), post_weight.dtype,
                   post_weight.get_device(), weight.shape, weight.stride(), weight.dtype, weight.get_device(), eps,
                   None if gate is None else _sig(gate), residual_scale, None if out is None else _out_sig(out),
                   None if residual_out is None else _out_sig(residual_out))
            plan = _PLANS.get(key)
    except (AttributeError, TypeError):  # a non-tensor or unhashable argument: checked below
        recorded, key, plan = False, None, None
    if recorded:
        got = torch.ops.fused_decode.norm_add_norm(x, residual, post_weight, weight, eps, gate, residual_scale)
        return _copied(got, out, residual_out)
    if plan is None:
        plan = _remember(key, _plan_norm_add_norm(x, residual, post_weight, weight, eps, gate, residual_scale, out,
                                                  residual_out))
    return plan(x, residual, post_weight, weight, gate, out, residual_out)


def _plan_norm_add_norm(x, residual, post_weight, weight, eps, gate, residual_scale, out, residual_out):
    """Launch plan of ``norm_add_norm`` for one argument signature."""
    a = check("norm_add_norm", x=x, residual=residual, post_weight=post_weight, weight=weight, eps=eps, gate=gate,
              residual_scale=residual_scale, out=out, residual_out=residual_out)
    eps, scale = a["eps"], a["residual_scale"]
    shape, device, dev = tuple(x.shape), x.device, x.device.index
    like = _like(shape, x.dtype, device)
    if x.numel() == 0:
        return lambda x, r, pw, w, g, o, ro: (torch.empty_like(like) if o is None else o,
                                              torch.empty_like(like) if ro is None else ro)
    dense = contiguous_strides(shape)
    strides = [tuple(x.stride()), tuple(residual.stride()), dense if out is None else tuple(out.stride()),
               dense if residual_out is None else tuple(residual_out.stride())]
    gcode = DTYPE_CODE[x.dtype]
    if gate is not None:
        gcode = DTYPE_CODE[gate.dtype]
        strides.append(tuple(gate.expand(shape).stride()))
    layouts = plan_rows(shape, strides)
    staged = layouts is None  # more than three unmergeable leading dims: the rows are gathered, and written back
    n = shape[-1]
    if staged:
        layouts = [bytes(FdRows(1, 1, math.prod(shape[:-1]), 0, 0, n, 1, n))] * len(strides)
    lx, lr, ly, lro = layouts[:4]
    lg = layouts[4] if gate is not None else lx
    call, act = native().norm_add_norm, DTYPE_CODE[x.dtype]
    pcode, pstride = DTYPE_CODE[post_weight.dtype], int(post_weight.stride(0)) if n > 1 else 1
    wcode, wstride = DTYPE_CODE[weight.dtype], int(weight.stride(0)) if n > 1 else 1

    def run(x, r, pw, w, g, o, ro):
        if _current_device() != dev:  # a launch on the default stream goes to the current device
            with torch.cuda.device(dev):
                return run(x, r, pw, w, g, o, ro)
        y = torch.empty_like(like) if o is None or staged else o
        t = torch.empty_like(like) if ro is None or staged else ro
        if staged:
            if o is not None and ro is not None and _meet(o, ro):
                raise FusedDecodeError("fd_norm_add_norm", FD_EINVAL, "the outputs must not overlap each other")
            x, r, g = x.contiguous(), r.contiguous(), None if g is None else g.expand(shape).contiguous()
        status = call(y.data_ptr(), t.data_ptr(), x.data_ptr(), r.data_ptr(), None if g is None else g.data_ptr(), gcode,
                      pw.data_ptr(), pcode, pstride, w.data_ptr(), wcode, wstride, lx, lr, lg, ly, lro, scale, eps, act,
                      _raw_stream(dev))
        if status:
            fail("fd_norm_add_norm", status)
        if staged:
            y, t = y if o is None else o.copy_(y), t if ro is None else ro.copy_(t)
        elif o is not None or ro is not None:
            increment_version([v for v in (o, ro) if v is not None])
        return y, t
    return run

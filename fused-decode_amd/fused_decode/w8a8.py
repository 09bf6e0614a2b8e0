"""Operators with 8-bit (OCP E4M3) activations: rows to codes, and products of codes.

    codes, scale = quantize_rows_fp8(x)                              # [..., K] -> codes, float32 [...]
    codes, scale = rms_norm_fp8(x, norm_w, eps)
    codes, scale, stream = add_rms_norm_fp8(x, residual, norm_w, eps)
    y = linear_w8a8(codes, scale, q, q_scale, bias, activation="gelu", row_add=r)

A row has one float32 scale, ``max|y| / 448`` for the float32 row ``y`` (never below 2^-126, and 1 for
a row of zeros), and its codes are ``y / scale`` rounded to the nearest E4M3 value: in
``quantize_rows_fp8`` as a division rounds, in the norms by the scale's reciprocal, which takes one
code in about 10^6 to its neighbour. The norms quantise their float32 result, which is never rounded
to 16 bits in between. A row whose largest magnitude is not finite gets a NaN scale and NaN codes.
Weights are those of ``quantize_fp8`` (codes ``[N, K]`` and one scale a row), so that

    y[m, n] = round(act(scale[m] * q_scale[n] * sum_k codes[m, k] q[n, k] + bias[n]) + row_add[m, n])

is computed on the 8-bit matrix cores, with float32 sums and one rounding. A layer's four products
with everything between them but the attention:

    c, s = rms_norm_fp8(x, attn_norm)
    qkv  = linear_w8a8(c, s, *w_qkv, bias)
    c, s = quantize_rows_fp8(attention(qkv))
    h    = linear_w8a8(c, s, *w_o, row_add=x)
    c, s = rms_norm_fp8(h, mlp_norm)
    mid  = linear_w8a8(c, s, *w_gate_up, activation="swiglu")
    c, s = quantize_rows_fp8(mid)
    x    = linear_w8a8(c, s, *w_down, row_add=h)

Inference only. Where a gradient, a trace or a transform is asked for, the call goes to the custom op
of the same name (``torch.ops.fused_decode.*``), which a graph keeps whole and which says that it has
no gradient. There is no reference counterpart (the reference's activations are fp16/bf16 only).
"""

from __future__ import annotations

import math

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from . import _lib
from ._checks import check
from ._lib import ACT_CODE, DTYPE_CODE, FD_EINVAL, FD_EUNSUPPORTED, FdRows, FusedDecodeError, fail, native
from ._layout import contiguous_strides, plan_rows, shares_memory
from .fp8 import FP8_DTYPE
from .ops import (_PLANS, _as_rows, _check_out, _dispatch_modes, _function_modes, _function_modes_watch, _is_tracing,
                  _raw_stream, _remember, _row_add_rows, _sig, _transform, _written)

__all__ = ["add_rms_norm_fp8", "linear_w8a8", "quantize_rows_fp8", "rms_norm_fp8"]

_current_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else (lambda: -1)
_grad, _is_compiling = torch.is_grad_enabled, torch.compiler.is_compiling
_MOST_STRIDE = 1 << 23  # bytes between rows that the product's kernels take as they are; others are copied
_PLAIN = frozenset((torch.Tensor, torch.nn.Parameter, type(None)))


def _watched() -> bool:
    """Whether something would record or transform a call, which a launch on bare pointers would be missing from
    (a tensor whose negation is still to be made takes the same way: the dispatcher makes it)."""
    return (_is_compiling() or forward_ad._current_level >= 0 or _transform() is not None or _is_tracing()
            or _dispatch_modes() > 0 or (_function_modes() > 0 and _function_modes_watch()))


def _subclasses(*tensors) -> bool:
    """Whether one of these is of a tensor subclass, whose memory may be another tensor's and which torch's calls let
    act for themselves: the custom op does. (Asked where a class is not in ``_PLAIN``; a list or a number is left to
    the contract.)"""
    return any(type(t) not in _PLAIN and isinstance(t, torch.Tensor) for t in tensors)


def _out_sig(t: torch.Tensor) -> tuple:
    """Signature of an output that torch would write in place as well."""
    if t.requires_grad and _grad():
        raise RuntimeError("an output that requires a gradient cannot be written in place")
    if t.is_inference() and not torch.is_inference_mode_enabled():
        raise RuntimeError("an inference tensor cannot be written outside inference mode")
    return _sig(t)


def _like(shape: tuple, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    """What ``torch.empty_like`` makes a contiguous ``shape`` of, in the least host time: one element, expanded, and its
    memory given back (a plan made during a capture would keep the graph's pool with it)."""
    one = torch.empty((), dtype=dtype, device=device)
    like = one.expand(shape)
    one.untyped_storage().resize_(0)
    return like


# ------------------------------------------------------------------ rows to codes


def quantize_rows_fp8(
    x: torch.Tensor,
    *,
    out: torch.Tensor | None = None,
    scale_out: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """E4M3 codes of ``x``'s rows (its last dimension) and their float32 scales ``x.shape[:-1]``, in one
    launch. For finite rows the codes and scales that ``quantize_fp8`` gives the same rows."""
    try:
        recorded = (_watched() or (_grad() and x.requires_grad) or x.is_neg()
                    or (not (x.__class__ in _PLAIN and out.__class__ in _PLAIN and scale_out.__class__ in _PLAIN)
                        and _subclasses(x, out, scale_out)))
        if not recorded:
            key = ("quantize_rows_fp8", x.shape, x.stride(), x.dtype, x.get_device(),
                   None if out is None else _out_sig(out), None if scale_out is None else _out_sig(scale_out))
            plan = _PLANS.get(key)
    except AttributeError:  # not a tensor: let the contract say so
        recorded, key, plan = False, None, None
    if recorded:
        return _copied(torch.ops.fused_decode.quantize_rows_fp8(x), out, scale_out)
    if plan is None:
        plan = _remember(key, _plan_rows_fp8("quantize_rows_fp8", x, None, None, 0.0, out, scale_out, None))
    return plan(x, None, None, out, scale_out, None)


def rms_norm_fp8(
    x: torch.Tensor,
    weight: torch.Tensor,
    eps: float = 1e-6,
    *,
    out: torch.Tensor | None = None,
    scale_out: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """``rms_norm`` with E4M3 codes and float32 row scales for its result. ``weight`` is ``(N,)``
    (float16, bfloat16 or float32)."""
    try:
        recorded = (_watched() or (_grad() and (x.requires_grad or weight.requires_grad)) or x.is_neg() or weight.is_neg()
                    or (not (x.__class__ in _PLAIN and weight.__class__ in _PLAIN and out.__class__ in _PLAIN
                             and scale_out.__class__ in _PLAIN) and _subclasses(x, weight, out, scale_out)))
        if not recorded:
            key = ("rms_norm_fp8", x.shape, x.stride(), x.dtype, x.get_device(), weight.shape, weight.stride(),
                   weight.dtype, weight.get_device(), eps, None if out is None else _out_sig(out),
                   None if scale_out is None else _out_sig(scale_out))
            plan = _PLANS.get(key)
    except (AttributeError, TypeError):  # a non-tensor or unhashable argument: checked below
        recorded, key, plan = False, None, None
    if recorded:
        return _copied(torch.ops.fused_decode.rms_norm_fp8(x, weight, eps), out, scale_out)
    if plan is None:
        plan = _remember(key, _plan_rows_fp8("rms_norm_fp8", x, weight, None, eps, out, scale_out, None))
    return plan(x, weight, None, out, scale_out, None)


def add_rms_norm_fp8(
    x: torch.Tensor,
    residual: torch.Tensor,
    weight: torch.Tensor,
    eps: float = 1e-6,
    *,
    out: torch.Tensor | None = None,
    scale_out: torch.Tensor | None = None,
    residual_out: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``add_rms_norm`` with E4M3 codes and float32 row scales for the norm of the float32 sum:
    ``(codes, scale, residual_out)``. ``residual_out=residual`` updates the residual stream in place."""
    try:
        recorded = (_watched()
                    or (_grad() and (x.requires_grad or residual.requires_grad or weight.requires_grad))
                    or x.is_neg() or residual.is_neg() or weight.is_neg()
                    or (not (x.__class__ in _PLAIN and residual.__class__ in _PLAIN and weight.__class__ in _PLAIN
                             and out.__class__ in _PLAIN and scale_out.__class__ in _PLAIN
                             and residual_out.__class__ in _PLAIN)
                        and _subclasses(x, residual, weight, out, scale_out, residual_out)))
        if not recorded:
            key = ("add_rms_norm_fp8", x.shape, x.stride(), x.dtype, x.get_device(), residual.shape, residual.stride(),
                   residual.dtype, residual.get_device(), weight.shape, weight.stride(), weight.dtype,
                   weight.get_device(), eps, None if out is None else _out_sig(out),
                   None if scale_out is None else _out_sig(scale_out),
                   None if residual_out is None else _out_sig(residual_out))
            plan = _PLANS.get(key)
    except (AttributeError, TypeError):
        recorded, key, plan = False, None, None
    if recorded:
        return _copied(torch.ops.fused_decode.add_rms_norm_fp8(x, residual, weight, eps), out, scale_out, residual_out)
    if plan is None:
        plan = _remember(key, _plan_rows_fp8("add_rms_norm_fp8", x, weight, residual, eps, out, scale_out, residual_out))
    return plan(x, weight, residual, out, scale_out, residual_out)


def _planned(make, *args):
    """``make(*args)``, a launch plan, kept by the arguments' signature: for the custom ops, whose calls are no longer
    recorded."""
    key = (make.__name__, *(_sig(a) if isinstance(a, torch.Tensor) else a for a in args))
    return _PLANS.get(key) or _remember(key, make(*args))


def _copied(got: tuple, *outs) -> tuple:
    """A custom op's results, copied where outputs are given."""
    for v, o in zip(got, outs):
        if o is not None and not isinstance(o, torch.Tensor):
            raise TypeError(f"an output must be a tensor or None, got {type(o).__name__}")
        if o is not None and (o.shape != v.shape or o.dtype != v.dtype or o.device != v.device):
            raise ValueError(f"an output must have shape {tuple(v.shape)} and dtype {v.dtype} on {v.device}")
        if o is not None and not _is_compiling() and shares_memory(o.shape, o.stride()):  # (compiled sizes are symbols)
            raise ValueError(f"an output has elements that share memory: shape {tuple(o.shape)} strides {o.stride()}")
    return tuple(v if o is None else o.copy_(v) for v, o in zip(got, outs))


def _meet(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the bytes from first to last element of two tensors overlap, as the library asks it."""
    end = lambda t: t.data_ptr() + (sum((n - 1) * st for n, st in zip(t.shape, t.stride())) + 1) * t.element_size()
    return a.data_ptr() < end(b) and b.data_ptr() < end(a)


def _plan_rows_fp8(op, x, weight, residual, eps, out, scale_out, residual_out):
    """Launch plan of a row operator for one argument signature."""
    add, norm = op == "add_rms_norm_fp8", op != "quantize_rows_fp8"
    args = dict(x=x, out=out, scale_out=scale_out)
    if norm:
        args.update(weight=weight, eps=eps)
    if add:
        args.update(residual=residual, residual_out=residual_out)
    eps = check(op, **args).get("eps", 0.0)
    shape, lead, device = tuple(x.shape), tuple(x.shape[:-1]), x.device
    n, act, dev, rows = shape[-1], DTYPE_CODE[x.dtype], x.device.index, math.prod(lead)
    if rows == 0 or n == 0:  # no value to compute: a row of none has scale 1
        def empty(x, w, r, out, scale_out, residual_out):
            c = torch.empty(shape, dtype=FP8_DTYPE, device=device) if out is None else out
            s = torch.ones(lead, dtype=torch.float32, device=device) if scale_out is None else scale_out.fill_(1.0)
            if not add:
                return c, s
            return c, s, torch.empty(shape, dtype=x.dtype, device=device) if residual_out is None else residual_out
        return empty

    codes_like, scale_like = _like(shape, FP8_DTYPE, device), _like(lead, torch.float32, device)
    dense = contiguous_strides(shape)
    strides = [tuple(x.stride())]
    if add:
        strides += [tuple(residual.stride()), dense if residual_out is None else tuple(residual_out.stride())]
    layouts = plan_rows(shape, strides)
    staged = layouts is None  # more than three unmergeable leading dims: the rows are gathered, and written back
    if staged:
        layouts = [bytes(FdRows(1, 1, rows, 0, 0, n, 1, n))] * len(strides)
    call = getattr(native(), op)
    wcode, wstride = (DTYPE_CODE[weight.dtype], int(weight.stride(0)) if n > 1 else 1) if norm else (act, 1)
    lx = layouts[0]

    if add:
        lr, lro = layouts[1:]
        sum_like = _like(shape, x.dtype, device)

        def run_add(x, w, r, out, scale_out, residual_out):
            if _current_device() != dev:  # a launch on the default stream goes to the current device
                with torch.cuda.device(dev):
                    return run_add(x, w, r, out, scale_out, residual_out)
            c = torch.empty_like(codes_like) if out is None else out
            s = torch.empty_like(scale_like) if scale_out is None else scale_out
            ro = torch.empty_like(sum_like) if residual_out is None or staged else residual_out
            if staged:
                if residual_out is not None and any(o is not None and _meet(o, residual_out) for o in (out, scale_out)):
                    raise FusedDecodeError("fd_add_rms_norm_fp8", FD_EINVAL, "the outputs must not overlap each other")
                x, r = x.contiguous(), r.contiguous()
            status = call(c.data_ptr(), s.data_ptr(), ro.data_ptr(), x.data_ptr(), r.data_ptr(), w.data_ptr(), wcode,
                          wstride, lx, lr, lro, eps, act, _raw_stream(dev))
            if status:
                fail("fd_add_rms_norm_fp8", status)
            if staged and residual_out is not None:
                ro = residual_out.copy_(ro)
            if out is not None or scale_out is not None or residual_out is not None:
                increment_version([t for t in (out, scale_out, residual_out) if t is not None])
            return c, s, ro
        return run_add

    def run(x, w, r, out, scale_out, residual_out):
        if _current_device() != dev:
            with torch.cuda.device(dev):
                return run(x, w, r, out, scale_out, residual_out)
        c = torch.empty_like(codes_like) if out is None else out
        s = torch.empty_like(scale_like) if scale_out is None else scale_out
        if staged:
            x = x.contiguous()
        if norm:
            status = call(c.data_ptr(), s.data_ptr(), x.data_ptr(), w.data_ptr(), wcode, wstride, lx, eps, act,
                          _raw_stream(dev))
        else:
            status = call(c.data_ptr(), s.data_ptr(), x.data_ptr(), lx, act, _raw_stream(dev))
        if status:
            fail("fd_" + op, status)
        if out is not None or scale_out is not None:
            increment_version([t for t in (out, scale_out) if t is not None])
        return c, s
    return run


# ------------------------------------------------------------------ products of codes


def linear_w8a8(
    x: torch.Tensor,
    x_scale: torch.Tensor,
    weight: torch.Tensor,
    scale: torch.Tensor,
    bias: torch.Tensor | None = None,
    *,
    activation: str | None = None,
    row_add: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
    dtype: torch.dtype | None = None,
) -> torch.Tensor:
    """``act(dequantised x @ dequantised weight.T (+ bias)) (+ row_add)`` for E4M3 ``x [..., K]`` with float32
    ``x_scale [...]`` and E4M3 ``weight [N, K]`` with float32 ``scale [N]``, rounded once to ``dtype`` (float16
    or bfloat16; ``out``'s where that is given, else bfloat16).

    ``activation`` is None, "relu", "silu", "gelu" (with erf), "gelu_tanh" or "swiglu", which takes gate rows
    above up rows (``weight [2I, K]``, ``bias [2I]``) and returns ``silu(gate) * up`` ``[..., I]``. ``bias`` and
    ``row_add`` have any float dtype; ``row_add`` broadcasts to the output and is added after the activation.
    Any number of rows and any K (below 2^23 for more than one row); codes whose rows are not 16-byte aligned, whose K
    is no multiple of 16 or whose stride along K is not 1 are copied first."""
    try:
        recorded = (_watched()
                    or (_grad() and (x_scale.requires_grad or scale.requires_grad or x.requires_grad
                                     or weight.requires_grad or (bias is not None and bias.requires_grad)
                                     or (row_add is not None and row_add.requires_grad)))
                    or x_scale.is_neg() or scale.is_neg() or (bias is not None and bias.is_neg())
                    or (row_add is not None and row_add.is_neg())
                    or (not (x.__class__ in _PLAIN and x_scale.__class__ in _PLAIN and weight.__class__ in _PLAIN
                             and scale.__class__ in _PLAIN and bias.__class__ in _PLAIN and row_add.__class__ in _PLAIN
                             and out.__class__ in _PLAIN)
                        and _subclasses(x, x_scale, weight, scale, bias, row_add, out)))
        if not recorded:
            key = ("linear_w8a8", x.shape, x.stride(), x.dtype, x.get_device(), x_scale.shape, x_scale.stride(),
                   x_scale.dtype, x_scale.get_device(), weight.shape, weight.stride(), weight.dtype, weight.get_device(),
                   scale.shape, scale.stride(), scale.dtype, scale.get_device(), None if bias is None else _sig(bias),
                   activation, None if row_add is None else _sig(row_add), None if out is None else _out_sig(out), dtype)
            plan = _PLANS.get(key)
    except (AttributeError, TypeError):  # a non-tensor or unhashable argument: checked below
        recorded, key, plan = False, None, None
    if recorded:
        y = torch.ops.fused_decode.linear_w8a8(x, x_scale, weight, scale, bias, activation, row_add,
                                               dtype or getattr(out, "dtype", torch.bfloat16))
        return _copied((y,), out)[0]
    if plan is None:
        plan = _remember(key, _plan_linear_w8a8(x, x_scale, weight, scale, bias, activation, row_add, out, dtype))
    return plan(x, x_scale, weight, scale, bias, row_add, out)


def _plan_linear_w8a8(x, x_scale, weight, scale, bias, activation, row_add, out, dtype):
    """Launch plan of ``linear_w8a8`` for one argument signature."""
    a = check("linear_w8a8", x=x, x_scale=x_scale, weight=weight, scale=scale, bias=bias, activation=activation,
              row_add=row_add, out=out, dtype=dtype)
    dtype, device, dev = a["dtype"], x.device, x.device.index
    n, k = (int(d) for d in weight.shape)
    nout = n // 2 if activation == "swiglu" else n
    m = math.prod(x.shape[:-1])
    expected = (*x.shape[:-1], nout)
    ra = None if row_add is None else _row_add_rows(row_add, m, nout, expected)
    if out is not None:
        _check_out(out, expected, torch.empty((), dtype=dtype, device=device))
    if m == 0 or nout == 0:
        return lambda x, xs, w, ws, b, r, o: torch.empty(expected, dtype=dtype, device=device) if o is None else o
    xr = _as_rows(x, m)
    x_copy = xr.flat or (k > 1 and xr.col != 1)
    w_copy = k > 1 and weight.stride(1) != 1
    sxm, swn = k if x_copy else xr.row, k if w_copy else int(weight.stride(0))
    s_copy = not (x_scale.is_contiguous() and scale.is_contiguous())
    act, code = ACT_CODE[activation], DTYPE_CODE[dtype]
    bcode, sb = (code, 0) if bias is None else (DTYPE_CODE[bias.dtype], int(bias.stride(0)))
    rcode = code if row_add is None else DTYPE_CODE[row_add.dtype]
    srm, srn, r_flat = ra if ra is not None else (0, 0, False)
    call = native().linear_w8a8
    with torch.cuda.device(dev):
        sizes = [_lib.scratch_bytes("fd_linear_w8a8_scratch", m, n, k, aligned) for aligned in (0, 1)]
    like = _like(expected, dtype, device)
    # by whether the rows are 16-byte aligned, which the pointers say call by call
    scratch = [(_like((size // 4,), torch.float32, device), size) if size else (None, 0) for size in sizes]
    if k % 16 or any(rows > 1 and (step % 16 or step >= _MOST_STRIDE) for rows, step in ((m, sxm), (n, swn))):
        scratch[1] = scratch[0]

    def run(x, xs, w, ws, b, r, o):
        if _current_device() != dev:  # a launch on the default stream goes to the current device
            with torch.cuda.device(dev):
                return run(x, xs, w, ws, b, r, o)
        y = torch.empty_like(like) if o is None else o
        if x_copy:
            x = x.reshape(m, k).contiguous()
        if w_copy:
            w = w.contiguous()
        if s_copy:
            xs, ws = xs.contiguous(), ws.contiguous()
        if r_flat:
            r = r.expand(expected).reshape(m, nout)
        xp, wp = x.data_ptr(), w.data_ptr()
        part_like, part_bytes = scratch[0 if (xp | wp) & 15 else 1]
        part = None if part_like is None else torch.empty_like(part_like)
        args = (xp, xs.data_ptr(), wp, ws.data_ptr(), None if b is None else b.data_ptr(), bcode, act,
                None if r is None else r.data_ptr(), rcode, m, n, k, sxm, swn, sb, srm, srn, nout, 1,
                None if part is None else part.data_ptr(), part_bytes, code, _raw_stream(dev))
        status = call(y.data_ptr(), *args)
        if status == FD_EUNSUPPORTED and o is not None:  # `out` may lie over an operand: write beside it
            beside = torch.empty_like(like)
            status = call(beside.data_ptr(), *args)
            if status == 0:
                return o.copy_(beside)
        if status:
            fail("fd_linear_w8a8", status)
        return y if o is None else _written(o)
    return run

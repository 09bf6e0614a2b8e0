"""4-bit (OCP E2M1) weights with a power-of-two scale for each 32 along K, and their products.

    codes, scale = quantize_fp4(w)                 # [N, K] -> uint8 [N, 16 G], float8_e8m0fnu [N, G], G = ceil(K / 32)
    y = linear_fp4(x, codes, scale, bias, activation="silu", row_add=r)

Two codes a byte, the first in the low half. A group's scale is the smallest power of two that its largest magnitude is
less than 7 of (2^-126 at least; 1 for a group of zeros), and a code is the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their
negatives to w / scale, ties to the even code: a value up to 7 rounds to 6, as far off as halves of E2M1's last step
are. (OCP's own recipe takes the largest magnitude's exponent less 2 for the scale, so that a value of 7 saturates at 6.) A
group that holds an infinity or a NaN gets a NaN scale. Codes and scales are in OCP's MXFP4 format, so weights quantised
elsewhere to it are taken as they are. The kernels decode them exactly and sum in float32:

    y[m, n] = round(act(sum_k x[m, k] * scale[n, k / 32] * e2m1(codes[n, k]) + bias[n]) + row_add[m, n])

The four products of a layer with everything between them but the attention:

    qkv = linear_fp4(rms_norm(x, attn_norm), *w_qkv, bias)
    h   = linear_fp4(attention(qkv), *w_o, row_add=x)
    mid = linear_fp4(rms_norm(h, mlp_norm), *w_gate_up, activation="swiglu")
    x   = linear_fp4(mid, *w_down, row_add=h)

Inference only. Where a gradient, a trace or a transform is asked for, the call goes to the custom op of the same name
(``torch.ops.fused_decode.linear_fp4``), which a graph keeps whole and which says that it has no gradient. There is no
reference counterpart (the reference has fp16/bf16 weights only).
"""

from __future__ import annotations

import math

import torch

from . import _lib
from ._checks import E8M0, FP4_GROUP, check
from ._lib import ACT_CODE, DTYPE_CODE, FD_EUNSUPPORTED, fail, native
from .ops import _PLANS, _as_rows, _check_out, _raw_stream, _remember, _row_add_rows, _sig, _written
from .w8a8 import _PLAIN, _copied, _current_device, _grad, _like, _out_sig, _subclasses, _watched

__all__ = ["dequantize_fp4", "linear_fp4", "quantize_fp4"]

_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def _to_float32(w: torch.Tensor) -> torch.Tensor:
    """Float32 values on the same side of every border between codes or scales as ``w``: float64 is rounded to the odd
    neighbour (the borders are even), so that a second rounding is as if it were the first."""
    v = w.float()
    if w.dtype != torch.float64:
        return v
    back = v.double()
    inexact = (back != w) & torch.isfinite(v)
    bits = v.view(torch.int32)
    return torch.where(inexact, (bits - (back.abs() > w.abs()).int()) | 1, bits).view(torch.float32)


def quantize_fp4(weight: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``[N, K]`` float weight -> (E2M1 codes ``[N, 16 G]`` as uint8, two a byte, E8M0 scales ``[N, G]``) with
    ``G = ceil(K / 32)``; codes past K are 0. (Magnitudes beyond float32's are infinities.)"""
    if not isinstance(weight, torch.Tensor) or weight.ndim != 2:
        raise ValueError("weight must be a rank-2 tensor [N, K]")
    if not weight.is_floating_point():
        raise TypeError("weight must be a floating-point tensor")
    n, k = weight.shape
    groups = -(-k // FP4_GROUP)
    w = torch.nn.functional.pad(_to_float32(weight.detach()), (0, groups * FP4_GROUP - k)).reshape(n, groups, FP4_GROUP)
    top = w.abs().amax(dim=-1) if groups else w.new_zeros(n, 0)
    # the exponent of top / 4, one more from 1.75 times a power of two on
    byte = (((top.view(torch.int32) + 0x200000) >> 23) - 2).clamp(1, 254)
    byte = torch.where(top > 0, byte, 127)
    bad = ~torch.isfinite(top)
    inverse = ((254 - byte) << 23).view(torch.float32)  # exact: byte is 253 at most
    v = torch.where(bad[..., None], 0.0, w * inverse[..., None])
    a = v.abs()
    code = (a > 0.25).to(torch.uint8)
    for edge, up in ((0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        code += (a >= edge) if up else (a > edge)  # ties to the even code
    code += torch.signbit(v).to(torch.uint8) << 3
    code = code.reshape(n, groups * FP4_GROUP)
    scale = torch.where(bad, 255, byte).to(torch.uint8).view(E8M0)
    return code[:, 0::2] | (code[:, 1::2] << 4), scale


def dequantize_fp4(codes: torch.Tensor, scale: torch.Tensor, k: int | None = None) -> torch.Tensor:
    """float32 ``scale * e2m1(codes)``: ``[..., 16 G]`` codes and ``[..., G]`` scales -> ``[..., 32 G]`` (the first ``k``
    columns where that is given)."""
    table = torch.tensor(_VALUES, dtype=torch.float32, device=codes.device)
    v = torch.stack((table[(codes & 15).int()], table[(codes >> 4).int()]), dim=-1)
    v = v.reshape(*scale.shape, FP4_GROUP) * scale.float()[..., None]
    return v.reshape(*scale.shape[:-1], scale.shape[-1] * FP4_GROUP)[..., :k]


def linear_fp4(
    x: torch.Tensor,
    weight: torch.Tensor,
    scale: torch.Tensor,
    bias: torch.Tensor | None = None,
    *,
    activation: str | None = None,
    row_add: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """``act(x @ dequantised weight.T (+ bias)) (+ row_add)`` for float16 or bfloat16 ``x [..., K]`` and the codes and
    scales of ``quantize_fp4``, rounded once to ``x``'s dtype.

    ``activation`` is None, "relu", "silu", "gelu" (with erf), "gelu_tanh" or "swiglu", which takes gate rows
    above up rows (``weight [2I, 16 G]``, ``bias [2I]``) and returns ``silu(gate) * up`` ``[..., I]``. ``bias`` and
    ``row_add`` have any float dtype; ``row_add`` broadcasts to the output and is added after the activation. Any number
    of rows and any K; ``x`` whose stride along K is not 1, and codes whose rows are not 16-byte aligned, are copied
    first."""
    try:
        recorded = (_watched()
                    or (_grad() and (x.requires_grad or scale.requires_grad
                                     or (bias is not None and bias.requires_grad)
                                     or (row_add is not None and row_add.requires_grad)))
                    or x.is_neg() or (bias is not None and bias.is_neg()) or (row_add is not None and row_add.is_neg())
                    or (not (x.__class__ in _PLAIN and weight.__class__ in _PLAIN and scale.__class__ in _PLAIN
                             and bias.__class__ in _PLAIN and row_add.__class__ in _PLAIN and out.__class__ in _PLAIN)
                        and _subclasses(x, weight, scale, bias, row_add, out)))
        if not recorded:
            key = ("linear_fp4", x.shape, x.stride(), x.dtype, x.get_device(), weight.shape, weight.stride(), weight.dtype,
                   weight.get_device(), scale.shape, scale.stride(), scale.dtype, scale.get_device(),
                   None if bias is None else _sig(bias), activation, None if row_add is None else _sig(row_add),
                   None if out is None else _out_sig(out))
            plan = _PLANS.get(key)
    except (AttributeError, TypeError):  # a non-tensor or unhashable argument: checked below
        recorded, key, plan = False, None, None
    if recorded:
        return _copied((torch.ops.fused_decode.linear_fp4(x, weight, scale, bias, activation, row_add),), out)[0]
    if plan is None:
        plan = _remember(key, _plan_linear_fp4(x, weight, scale, bias, activation, row_add, out))
    return plan(x, weight, scale, bias, row_add, out)


def _plan_linear_fp4(x, weight, scale, bias, activation, row_add, out):
    """Launch plan of ``linear_fp4`` for one argument signature."""
    check("linear_fp4", x=x, weight=weight, scale=scale, bias=bias, activation=activation, row_add=row_add)
    dtype, device, dev = x.dtype, x.device, x.device.index
    n, k = int(weight.shape[0]), int(x.shape[-1])
    nout = n // 2 if activation == "swiglu" else n
    m = math.prod(x.shape[:-1])
    expected = (*x.shape[:-1], nout)
    ra = None if row_add is None else _row_add_rows(row_add, m, nout, expected)
    if out is not None:
        _check_out(out, expected, x)
    like = _like(expected, dtype, device)
    if m == 0 or nout == 0:
        return lambda x, w, ws, b, r, o: torch.empty_like(like) if o is None else o
    xr = _as_rows(x, m)
    x_copy = xr.flat or (k > 1 and xr.col != 1)
    sxm = k if x_copy else xr.row
    w_copy = weight.stride(1) != 1 or (n > 1 and weight.stride(0) % 16 != 0)
    s_copy = scale.shape[1] > 1 and scale.stride(1) != 1
    width = int(weight.shape[1])
    swn = int(weight.stride(0))
    ssn = int(scale.shape[1]) if s_copy else int(scale.stride(0))
    act, code = ACT_CODE[activation], DTYPE_CODE[dtype]
    bcode, sb = (code, 0) if bias is None else (DTYPE_CODE[bias.dtype], int(bias.stride(0)))
    rcode = code if row_add is None else DTYPE_CODE[row_add.dtype]
    srm, srn, r_flat = ra if ra is not None else (0, 0, False)
    call = native().linear_fp4
    with torch.cuda.device(dev):
        size = _lib.scratch_bytes("fd_linear_fp4_scratch", m, n, k, code)
    part_like = _like((-(-size // 4),), torch.float32, device) if size else None

    def run(x, w, ws, b, r, o):
        if _current_device() != dev:  # a launch on the default stream goes to the current device
            with torch.cuda.device(dev):
                return run(x, w, ws, b, r, o)
        y = torch.empty_like(like) if o is None else o
        if x_copy:
            x = x.reshape(m, k).contiguous()
        step = swn
        if w_copy or w.data_ptr() & 15:  # (contiguous memory of its own, whatever its strides were)
            w, step = w.clone(memory_format=torch.contiguous_format), width
        if s_copy:
            ws = ws.contiguous()
        if r_flat:
            r = r.expand(expected).reshape(m, nout)
        part = None if part_like is None else torch.empty_like(part_like)
        args = (x.data_ptr(), w.data_ptr(), ws.data_ptr(), None if b is None else b.data_ptr(), bcode, act,
                None if r is None else r.data_ptr(), rcode, m, n, k, sxm, step, ssn, sb, srm, srn, nout, 1,
                None if part is None else part.data_ptr(), size, code, _raw_stream(dev))
        status = call(y.data_ptr(), *args)
        if status == FD_EUNSUPPORTED and o is not None:  # `out` may lie over an operand: write beside it
            beside = torch.empty_like(like)
            status = call(beside.data_ptr(), *args)
            if status == 0:
                return o.copy_(beside)
        if status:
            fail("fd_linear_fp4", status)
        return y if o is None else _written(o)
    return run

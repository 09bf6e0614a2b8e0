"""Argument contract of the public operators, written as data.

Every operator names its checks in ``CONTRACT``: an ordered tuple of rules over
the call's named arguments. ``check(op, **args)`` applies them in order and the
first failure raises ``TypeError`` (wrong kind of object or dtype) or
``ValueError`` (device, shape, value). The operators run this once per distinct
argument signature (``ops`` caches the resulting launch plan), so the rules
can afford clear messages.

What a rule accepts is the drop-in contract of the reference's operators
(src/fused_decode/ops.py:34-69 for the shared checks, :72-315 for each
operator): activations are CUDA float16/bfloat16 tensors, norm weights and
RoPE angles may also be float32, bias is the activation dtype or float32,
row_add is any float dtype broadcastable to the output, eps is finite and
non-negative, and the messages carry the words the reference's tests match
("CUDA", "weight", "even"). fp8 weights (``float8_e4m3fn`` codes with float32
row scales) have rules of their own.
"""

from __future__ import annotations

import math
from typing import Callable

import torch

from ._layout import shares_memory

ACTIVATION = (torch.float16, torch.bfloat16)
FLOAT = (torch.float16, torch.bfloat16, torch.float32)
FP8 = torch.float8_e4m3fn

Rule = Callable[[dict], None]


def _names(dtypes) -> str:
    return " or ".join(str(d).replace("torch.", "") for d in dtypes)


# ------------------------------------------------------------------ rules


def tensor_on_gpu(name: str, dtypes=ACTIVATION) -> Rule:
    """A CUDA (HIP) tensor of one of ``dtypes``."""

    def rule(a: dict) -> None:
        t = a[name]
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
        if not t.is_cuda:
            raise ValueError(f"{name} must be a CUDA tensor (a HIP device), got device {t.device}")
        if t.dtype not in dtypes:
            raise TypeError(f"{name} must be {_names(dtypes)}, got {t.dtype}")

    return rule


def like(name: str, ref: str, *, optional: bool = False) -> Rule:
    """Same shape, dtype and device as ``ref``."""

    def rule(a: dict) -> None:
        t, r = a[name], a[ref]
        if t is None and optional:
            return
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
        if t.device != r.device:
            raise ValueError(f"{name} is on {t.device} but {ref} is on {r.device}")
        if t.shape != r.shape:
            raise ValueError(f"{name} has shape {tuple(t.shape)}, {ref} has {tuple(r.shape)}")
        if t.dtype != r.dtype:
            raise TypeError(f"{name} is {t.dtype}, {ref} is {r.dtype}")

    return rule


def vector_for(name: str, ref: str, *, label: str | None = None, dtypes=FLOAT) -> Rule:
    """A 1-D tensor with one element per column of ``ref`` (its last dim), on
    ``ref``'s device, of one of ``dtypes``. ``label`` names it in messages
    (the norm weight is "weight" whatever the argument is called)."""
    label = label or name

    def rule(a: dict) -> None:
        t, r = a[name], a[ref]
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{label} must be a tensor, got {type(t).__name__}")
        if t.device != r.device:
            raise ValueError(f"{label} is on {t.device} but {ref} is on {r.device}")
        if t.dtype not in dtypes:
            raise TypeError(f"{label} must be {_names(dtypes)}, got {t.dtype}")
        if t.ndim != 1 or t.shape[0] != r.shape[-1]:
            raise ValueError(f"{label} must have shape ({r.shape[-1]},), got {tuple(t.shape)}")

    return rule


def finite_eps(name: str = "eps") -> Rule:
    def rule(a: dict) -> None:
        try:
            v = float(a[name])
        except (TypeError, ValueError) as exc:
            raise ValueError(f"{name} must be a finite value >= 0, got {a[name]!r}") from exc
        if not (math.isfinite(v) and v >= 0):
            raise ValueError(f"{name} must be a finite value >= 0, got {v}")
        a[name] = v

    return rule


def even_last(name: str, what: str = "rope last dimension") -> Rule:
    def rule(a: dict) -> None:
        n = a[name].shape[-1] if a[name].ndim else 0
        if n % 2:
            raise ValueError(f"{what} must be even, got {n}")

    return rule


def broadcast_angles(name: str, ref: str) -> Rule:
    """cos/sin of RoPE: a float tensor on ``ref``'s device whose last dim equals
    ``ref``'s and that broadcasts to ``ref``'s shape (shapes align on the right)."""

    def rule(a: dict) -> None:
        t, r = a[name], a[ref]
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
        if t.device != r.device:
            raise ValueError(f"{name} is on {t.device} but {ref} is on {r.device}")
        if t.dtype not in FLOAT:
            raise TypeError(f"{name} must be {_names(FLOAT)}, got {t.dtype}")
        if t.ndim == 0 or t.shape[-1] != r.shape[-1]:
            raise ValueError(f"{name} last dim {tuple(t.shape)[-1:]} must equal {ref}'s {r.shape[-1]}")
        if not _broadcasts(t.shape, r.shape):
            raise ValueError(f"cannot broadcast {name} shape {tuple(t.shape)} to {tuple(r.shape)}")

    return rule


def _broadcasts(src, dst) -> bool:
    """``src`` expands to ``dst``: no more dims, and each (right-aligned) is 1 or equal."""
    if len(src) > len(dst):
        return False
    return all(s in (1, d) for s, d in zip(reversed(src), reversed(dst)))


def weight_matrix(name: str, ref: str, *, label: str | None = None, fp8: bool = False,
                  dtype_error: type = ValueError) -> Rule:
    """A rank-2 ``[N, K]`` weight on ``ref``'s device: the activation dtype, or
    float8_e4m3fn codes with ``fp8``. A dtype mismatch of a plain weight raises
    ``dtype_error``: ValueError in linear_decode's contract ("weight device and
    dtype must match x"), TypeError for the fused QKV."""
    label = label or name

    def rule(a: dict) -> None:
        w, r = a[name], a[ref]
        if not isinstance(w, torch.Tensor):
            raise TypeError(f"{label} must be a tensor, got {type(w).__name__}")
        if fp8:
            if w.dtype != FP8:
                raise TypeError(f"{label} must hold torch.float8_e4m3fn codes (see quantize_fp8), got {w.dtype}")
            if w.device != r.device:
                raise ValueError(f"{label} is on {w.device} but {ref} is on {r.device}")
        elif w.device != r.device or w.dtype != r.dtype:
            err = dtype_error if w.device == r.device else ValueError
            raise err(f"{label} device and dtype must match {ref}: got {w.device}/{w.dtype}, "
                      f"{ref} is {r.device}/{r.dtype}")
        if w.ndim != 2:
            raise ValueError(f"{label} must have shape [N, K], got {tuple(w.shape)}")

    return rule


def row_scales(name: str, weight: str) -> Rule:
    """float32 per-row scales ``[N]`` of an fp8 weight, on its device."""

    def rule(a: dict) -> None:
        s, w = a[name], a[weight]
        if not isinstance(s, torch.Tensor) or s.dtype != torch.float32 or s.ndim != 1 \
                or s.shape[0] != w.shape[0]:
            got = tuple(s.shape) if isinstance(s, torch.Tensor) else type(s).__name__
            raise ValueError(f"{weight} scale must be float32 of shape ({w.shape[0]},), got {got}")
        if s.device != w.device:
            raise ValueError(f"{weight} scale is on {s.device}, {weight} on {w.device}")

    return rule


def inner_dim(ref: str, weight: str) -> Rule:
    """``ref``'s last dim is the weight's K."""

    def rule(a: dict) -> None:
        k = a[weight].shape[1]
        if a[ref].shape[-1] != k:
            raise ValueError(f"{ref} last dim {a[ref].shape[-1]} != {weight} K {k}")

    return rule


def bias_for(name: str, ref: str, weight: str) -> Rule:
    """Optional ``[N]`` bias in the activation dtype or float32."""

    def rule(a: dict) -> None:
        b = a.get(name)
        if b is None:
            return
        n, r = a[weight].shape[0], a[ref]
        if not isinstance(b, torch.Tensor):
            raise TypeError(f"{name} must be a tensor or None, got {type(b).__name__}")
        if b.ndim != 1 or b.shape[0] != n:
            raise ValueError(f"{name} must have shape ({n},), got {tuple(b.shape)}")
        if b.device != r.device:
            raise ValueError(f"{name} must be on {ref}'s device {r.device}, got {b.device}")
        if b.dtype not in (r.dtype, torch.float32):
            raise TypeError(f"{name} must match {ref} ({r.dtype}) or be float32, got {b.dtype}")

    return rule


def row_add_for(name: str, ref: str, weight: str) -> Rule:
    """Optional epilogue addend: any float dtype, on ``ref``'s device, shaped so
    it indexes the ``[M, N]`` output (``ops`` resolves the broadcast)."""

    def rule(a: dict) -> None:
        t = a.get(name)
        if t is None:
            return
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a tensor or None, got {type(t).__name__}")
        if t.device != a[ref].device:
            raise ValueError(f"{name} must be on {ref}'s device {a[ref].device}, got {t.device}")
        if t.dtype not in FLOAT:
            raise TypeError(f"{name} must be {_names(FLOAT)}, got {t.dtype}")

    return rule


def mlp_weights(gate_up: str, down: str, ref: str, *, fp8: bool = False) -> Rule:
    """``gate_up [2I, H]`` and ``down [H, I]`` for ``ref [..., H]``: rank 2,
    consistent widths, on ``ref``'s device, in its dtype (or fp8 codes)."""

    def rule(a: dict) -> None:
        wgu, wd, r = a[gate_up], a[down], a[ref]
        for nm, w in ((gate_up, wgu), (down, wd)):
            if not isinstance(w, torch.Tensor):
                raise TypeError(f"{nm} must be a tensor, got {type(w).__name__}")
        if fp8:
            for nm, w in ((gate_up, wgu), (down, wd)):
                if w.dtype != FP8:
                    raise TypeError(f"{nm} must hold torch.float8_e4m3fn codes (see quantize_fp8), got {w.dtype}")
        if wgu.ndim != 2 or wd.ndim != 2:
            raise ValueError(f"{gate_up} and {down} must be rank-2, got {wgu.ndim} and {wd.ndim} dims")
        (two_i, h), (h_d, i) = wgu.shape, wd.shape
        if two_i != 2 * i or h != h_d or r.shape[-1] != h:
            raise ValueError(
                f"expected {gate_up} [2I, H] and {down} [H, I] with {ref} [..., H], got "
                f"{tuple(wgu.shape)}, {tuple(wd.shape)}, {tuple(r.shape)}")
        if not fp8 and (wgu.dtype != r.dtype or wd.dtype != r.dtype):
            raise TypeError(f"MLP weights must be {ref}'s dtype {r.dtype}, got {wgu.dtype} and {wd.dtype}")
        if wgu.device != r.device or wd.device != r.device:
            raise ValueError(f"MLP weights must be on {ref}'s device {r.device}")

    return rule


def kind_name(name: str = "kind") -> Rule:
    def rule(a: dict) -> None:
        k = a[name]
        if k is not None and k not in ("dot", "simt"):
            raise ValueError(f"kind must be 'dot' or 'simt' (or None for FUSED_DECODE_LINEAR_KIND), got {k!r}")

    return rule


def output_like(name: str, ref: str) -> Rule:
    """``out`` of a row-wise operator: same shape, dtype and device as the input
    (any strides)."""
    return like(name, ref, optional=True)


def no_shared_elements(name: str) -> Rule:
    """An optional output whose elements all lie at addresses of their own: rows are
    stored while others are still read, and torch would not write it in place either."""

    def rule(a: dict) -> None:
        t = a[name]
        if t is not None and shares_memory(t.shape, t.stride()):
            raise ValueError(f"{name} has elements that share memory: shape {tuple(t.shape)} strides {t.stride()}")

    return rule


# ------------------------------------------------- row-sum (sumsq) entry points
#
# The row-sum forms call C entry points that take bare pointers with no extents
# and, for the MLP and QKV weights, no strides: every operand's layout is fixed
# here, before any launch, so a mis-shaped tensor raises instead of becoming an
# out-of-bounds read or write on the GPU.

SUMSQ_MIN_ROWS = 5  # the MFMA kernels that write and read the sums run from this many rows


def decode_rows(name: str, lo: int = SUMSQ_MIN_ROWS, hi: int = 16) -> Rule:
    """A contiguous rank-2 ``[M, K]`` activation with ``lo <= M <= hi``."""

    def rule(a: dict) -> None:
        t = a[name]
        if t.ndim != 2 or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous [M, K] tensor, got shape {tuple(t.shape)} "
                             f"strides {t.stride()}")
        if not lo <= t.shape[0] <= hi:
            raise ValueError(f"row sums of squares run on the MFMA kernels: {name} needs {lo} to {hi} rows, "
                             f"got {t.shape[0]}")

    return rule


def unit_k_stride(name: str) -> Rule:
    """A weight whose K (last) dim is dense: element stride 1."""

    def rule(a: dict) -> None:
        w = a[name]
        if w.shape[-1] > 1 and w.stride(-1) != 1:
            raise ValueError(f"{name} must have unit stride along K, got strides {w.stride()}")

    return rule


def dense(*names: str) -> Rule:
    """Contiguous tensors (kernels that take no strides for them)."""

    def rule(a: dict) -> None:
        for name in names:
            t = a.get(name)
            if isinstance(t, torch.Tensor) and not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous, got shape {tuple(t.shape)} strides {t.stride()}")

    return rule


def matrix_for(name: str, ref: str, rows: Callable[[dict], int], cols: Callable[[dict], int], *,
               optional: bool = False, dtypes=None) -> Rule:
    """A contiguous ``[rows, cols]`` tensor on ``ref``'s device, in ``ref``'s dtype
    (or one of ``dtypes``): an output, scratch or addend the kernel indexes as
    dense rows."""

    def rule(a: dict) -> None:
        t, r = a.get(name), a[ref]
        if t is None:
            if optional:
                return
            raise ValueError(f"{name} is required")
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
        if t.device != r.device:
            raise ValueError(f"{name} is on {t.device} but {ref} is on {r.device}")
        ok = (r.dtype,) if dtypes is None else dtypes
        if t.dtype not in ok:
            raise TypeError(f"{name} must be {_names(ok)}, got {t.dtype}")
        shape = (rows(a), cols(a))
        if tuple(t.shape) != shape or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous {list(shape)} tensor, got shape {tuple(t.shape)} "
                             f"strides {t.stride()}")

    return rule


def sums_buffer(name: str, ref: str, width: Callable[[dict], int], *, optional: bool = False) -> Rule:
    """Float32 tile sums of squares for a ``width``-column activation: a
    contiguous buffer of ``ceil(width / 16) * 16`` values on ``ref``'s device
    (``sumsq_buffer``)."""

    def rule(a: dict) -> None:
        t = a.get(name)
        if t is None:
            if optional:
                return
            raise ValueError(f"{name} is required")
        w = width(a)
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
        if t.device != a[ref].device:
            raise ValueError(f"{name} is on {t.device} but {ref} is on {a[ref].device}")
        if t.dtype != torch.float32 or not t.is_contiguous() or t.numel() != (w + 15) // 16 * 16:
            raise ValueError(f"{name} must be a contiguous float32 tensor of ceil({w}/16)*16 values "
                             f"(sumsq_buffer), got {t.dtype} shape {tuple(t.shape)}")

    return rule


def _m(ref: str) -> Callable[[dict], int]:
    return lambda a: a[ref].shape[0]


def _rows_of(weight: str) -> Callable[[dict], int]:
    return lambda a: a[weight].shape[0]


def _cols_of(weight: str) -> Callable[[dict], int]:
    return lambda a: a[weight].shape[1]


# ------------------------------------------------------ 8-bit activations (w8a8.py)


def has_rows(name: str) -> Rule:
    """At least one dimension: the last one is the row."""

    def rule(a: dict) -> None:
        if a[name].ndim == 0:
            raise ValueError(f"{name} needs at least one dimension")

    return rule


def codes_out(name: str, ref: str) -> Rule:
    """Optional contiguous E4M3 output of ``ref``'s shape."""

    def rule(a: dict) -> None:
        t, r = a[name], a[ref]
        if t is None:
            return
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
        if t.dtype != FP8:
            raise TypeError(f"{name} must be torch.float8_e4m3fn, got {t.dtype}")
        if t.device != r.device or t.shape != r.shape or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous {tuple(r.shape)} tensor on {r.device}, got shape "
                             f"{tuple(t.shape)} strides {t.stride()} on {t.device}")

    return rule


def scale_of_rows(name: str, ref: str, *, optional: bool = False) -> Rule:
    """float32 scales, one a row of ``ref`` (its shape without the last dimension); as an output
    (``optional``) contiguous."""

    def rule(a: dict) -> None:
        t, r = a[name], a[ref]
        if t is None and optional:
            return
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
        if t.dtype != torch.float32:
            raise TypeError(f"{name} must be float32, got {t.dtype}")
        if t.device != r.device or t.shape != r.shape[:-1] or (optional and not t.is_contiguous()):
            raise ValueError(f"{name} must hold one scale a row of {ref}, shape {tuple(r.shape[:-1])} on {r.device}, "
                             f"got shape {tuple(t.shape)} strides {t.stride()} on {t.device}")

    return rule


ACTIVATIONS = (None, "relu", "silu", "gelu", "gelu_tanh", "swiglu")


def activation_name(name: str, weight: str) -> Rule:
    """An epilogue activation; "swiglu" takes gate rows above up rows of ``weight``."""

    def rule(a: dict) -> None:
        v = a[name]
        if not (v is None or isinstance(v, str)) or v not in ACTIVATIONS:
            raise ValueError(f"{name} must be None or one of {', '.join(map(repr, ACTIVATIONS[1:]))}, got {v!r}")
        if v == "swiglu" and a[weight].shape[0] % 2:
            raise ValueError(f"{name} 'swiglu' needs gate and up rows: {weight} has {a[weight].shape[0]}, must be even")

    return rule


def bias_of(name: str, ref: str, weight: str) -> Rule:
    """Optional ``[N]`` bias of any float dtype."""

    def rule(a: dict) -> None:
        b = a[name]
        if b is None:
            return
        if not isinstance(b, torch.Tensor):
            raise TypeError(f"{name} must be a tensor or None, got {type(b).__name__}")
        if b.ndim != 1 or b.shape[0] != a[weight].shape[0]:
            raise ValueError(f"{name} must have shape ({a[weight].shape[0]},), got {tuple(b.shape)}")
        if b.device != a[ref].device:
            raise ValueError(f"{name} must be on {ref}'s device {a[ref].device}, got {b.device}")
        if b.dtype not in FLOAT:
            raise TypeError(f"{name} must be {_names(FLOAT)}, got {b.dtype}")

    return rule


def output_dtype(name: str, out: str) -> Rule:
    """The output's dtype: ``out``'s where that is given, else bfloat16 by default."""

    def rule(a: dict) -> None:
        d, o = a[name], a[out]
        if o is not None and not isinstance(o, torch.Tensor):
            raise TypeError(f"{out} must be a tensor or None, got {type(o).__name__}")
        if d is None:
            d = torch.bfloat16 if o is None else o.dtype
        if d not in ACTIVATION:
            raise TypeError(f"{name} must be {_names(ACTIVATION)}, got {d}")
        if o is not None and o.dtype != d:
            raise TypeError(f"{out} is {o.dtype}, {name} is {d}")
        a[name] = d

    return rule


# ------------------------------------------------------------------ 4-bit weights (fp4.py)

FP4_GROUP = 32  # values that share a scale
E8M0 = torch.float8_e8m0fnu


def fp4_matrix(name: str, scale: str, ref: str) -> Rule:
    """E2M1 codes ``[N, 16 G]``, two a byte, and their E8M0 scales ``[N, G]``, on ``ref``'s device, for ``ref [..., K]`` with
    ``G = ceil(K / 32)``."""

    def rule(a: dict) -> None:
        w, s, r = a[name], a[scale], a[ref]
        for what, t, dtype in ((name, w, torch.uint8), (scale, s, E8M0)):
            if not isinstance(t, torch.Tensor):
                raise TypeError(f"{what} must be a tensor, got {type(t).__name__}")
            if t.dtype != dtype:
                raise TypeError(f"{what} must be {dtype} (see quantize_fp4), got {t.dtype}")
            if t.device != r.device:
                raise ValueError(f"{what} is on {t.device} but {ref} is on {r.device}")
            if t.ndim != 2:
                raise ValueError(f"{what} must be a rank-2 tensor, got {tuple(t.shape)}")
        groups = -(-r.shape[-1] // FP4_GROUP)
        if w.shape[1] != groups * FP4_GROUP // 2 or s.shape != (w.shape[0], groups):
            raise ValueError(f"{name} and {scale} must have shapes [N, {groups * FP4_GROUP // 2}] and [N, {groups}] for "
                             f"{ref}'s last dimension {r.shape[-1]}, got {tuple(w.shape)} and {tuple(s.shape)}")

    return rule


# ------------------------------------------------------------------ 4-bit key/value cache (kv_fp4.py)

KV_DIMS = (64, 96, 128, 192, 256)


def kv_cache(*names: str) -> Rule:
    """Codes and scales of keys and values: ``[pages, heads, page, dim / 2]`` and ``[pages, heads, page, dim / 32]`` on one
    GPU, slots together, strides alike (those of the scales a sixteenth)."""

    def rule(a: dict) -> None:
        tensors = [a[n] for n in names]
        for i, (n, t) in enumerate(zip(names, tensors)):
            dtype = E8M0 if i % 2 else torch.uint8
            if not isinstance(t, torch.Tensor):
                raise TypeError(f"{n} must be a tensor, got {type(t).__name__}")
            if not t.is_cuda:
                raise ValueError(f"{n} must be a CUDA tensor (a HIP device), got device {t.device}")
            if t.dtype != dtype:
                raise TypeError(f"{n} must be {dtype}, got {t.dtype}")
            if t.ndim != 4:
                raise ValueError(f"{n} must have four dimensions, got shape {tuple(t.shape)}")
        k = tensors[0]
        pages, heads, page, half = k.shape
        if 2 * half not in KV_DIMS:
            raise ValueError(f"a head must have {', '.join(map(str, KV_DIMS))} channels, got {2 * half}")
        if heads == 0 or page == 0:
            raise ValueError(f"a cache has heads and slots, got shape {tuple(k.shape)}")
        for i, (n, t) in enumerate(zip(names, tensors)):
            part = 16 if i % 2 else 1  # a scale for 32 codes, two a byte
            if t.device != k.device:
                raise ValueError(f"{n} is on {t.device} but {names[0]} is on {k.device}")
            if t.shape != (pages, heads, page, half // part):
                raise ValueError(f"{n} must have shape {(pages, heads, page, half // part)}, got {tuple(t.shape)}")
            row = half // part
            want = [s // part for s in k.stride()[:2]] + [row, 1]
            bad = any(size > 1 and st != w for size, st, w in zip(t.shape, t.stride(), want))
            if bad or (i == 0 and any(size > 1 and st % 16 for size, st in zip(t.shape[:2], t.stride()[:2]))):
                raise ValueError(f"a cache's slots must lie together and its tensors' strides be alike, multiples of 16 "
                                 f"and a sixteenth for scales: {n} has strides {t.stride()}, {names[0]} {k.stride()}")

    return rule


def kv_rows(name: str, cache: str, *, multiple: bool = False) -> Rule:
    """``[B, L, heads, dim]`` for a cache's heads (``multiple``: a multiple of them) and head width."""

    def rule(a: dict) -> None:
        t, c = a[name], a[cache]
        if t.device != c.device:
            raise ValueError(f"{name} is on {t.device} but the cache is on {c.device}")
        heads, dim = c.shape[1], 2 * c.shape[3]
        if t.ndim != 4 or t.shape[3] != dim or (t.shape[2] % heads if multiple else t.shape[2] != heads):
            what = f"a multiple of {heads}" if multiple else heads
            raise ValueError(f"{name} must have shape [B, L, {what}, {dim}], got {tuple(t.shape)}")

    return rule


def kv_tokens(lengths: str, pages: str, cache: str, batch: str | None = None) -> Rule:
    """int32 lengths ``[B]`` and, optionally, int32 pages ``[B, n]`` on the cache's device; without pages the cache has one
    for each sequence."""

    def rule(a: dict) -> None:
        n, p, c = a[lengths], a[pages], a[cache]
        for name, t in ((lengths, n), (pages, p)):
            if t is None and name == pages:
                continue
            if not isinstance(t, torch.Tensor):
                raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
            if t.dtype != torch.int32:
                raise TypeError(f"{name} must be int32, got {t.dtype}")
            if t.device != c.device:
                raise ValueError(f"{name} is on {t.device} but the cache is on {c.device}")
        if n.ndim != 1 or (batch is not None and n.shape[0] != a[batch].shape[0]):
            raise ValueError(f"{lengths} must hold one length a sequence, got shape {tuple(n.shape)}")
        if p is not None and (p.ndim != 2 or p.shape[0] != n.shape[0]):
            raise ValueError(f"{pages} must have shape [{n.shape[0]}, n], got {tuple(p.shape)}")
        if p is None and n.shape[0] > c.shape[0]:
            raise ValueError(f"without {pages} each of the {n.shape[0]} sequences has a page: the cache has {c.shape[0]}")

    return rule


def kv_count(name: str) -> Rule:
    def rule(a: dict) -> None:
        v = a[name]
        if isinstance(v, bool) or not hasattr(v, "__index__") or isinstance(v, torch.Tensor):
            raise TypeError(f"{name} must be an integer, got {type(v).__name__}")
        a[name] = v.__index__()
        if a[name] < 0:
            raise ValueError(f"{name} must not be negative, got {v}")

    return rule


def one_of(name: str, values) -> Rule:
    def rule(a: dict) -> None:
        if a[name] not in values:
            raise TypeError(f"{name} must be {_names(values)}, got {a[name]}")

    return rule


def softmax_scale(name: str, ref: str) -> Rule:
    """The scale of the scores, 1 / sqrt(dim) by default."""
    finite = finite_scale(name)

    def rule(a: dict) -> None:
        if a[name] is None:
            a[name] = a[ref].shape[-1] ** -0.5
        finite(a)
        if abs(a[name]) > 1e38:
            raise ValueError(f"{name} must be 1e38 at most, got {a[name]}")

    return rule


def dense_output(name: str, ref: str) -> Rule:
    """Optional contiguous output of ``ref``'s shape, dtype and device."""

    def rule(a: dict) -> None:
        t, r = a[name], a[ref]
        if t is None:
            return
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a tensor or None, got {type(t).__name__}")
        if t.dtype != r.dtype:
            raise TypeError(f"{name} must be {r.dtype}, got {t.dtype}")
        if t.shape != r.shape or t.device != r.device or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous {tuple(r.shape)} tensor on {r.device}, got shape "
                             f"{tuple(t.shape)} strides {t.stride()} on {t.device}")

    return rule


# ------------------------------------------------------ norms around a block (block_norms.py)


def finite_scale(name: str) -> Rule:
    def rule(a: dict) -> None:
        try:
            v = float(a[name])
        except (TypeError, ValueError) as exc:
            raise ValueError(f"{name} must be a finite value, got {a[name]!r}") from exc
        if not abs(v) <= torch.finfo(torch.float32).max:
            raise ValueError(f"{name} must be a finite float32 value, got {v}")
        a[name] = v

    return rule


def gate_for(name: str, ref: str) -> Rule:
    """Optional gate: any float dtype, on ``ref``'s device, broadcastable to its shape."""

    def rule(a: dict) -> None:
        t, r = a[name], a[ref]
        if t is None:
            return
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a tensor or None, got {type(t).__name__}")
        if t.device != r.device:
            raise ValueError(f"{name} is on {t.device} but {ref} is on {r.device}")
        if t.dtype not in FLOAT:
            raise TypeError(f"{name} must be {_names(FLOAT)}, got {t.dtype}")
        if not _broadcasts(t.shape, r.shape):
            raise ValueError(f"cannot broadcast {name} shape {tuple(t.shape)} to {tuple(r.shape)}")

    return rule


# ------------------------------------------------------------------ contract

CONTRACT: dict[str, tuple[Rule, ...]] = {
    "rms_norm": (tensor_on_gpu("x"), vector_for("weight", "x"), finite_eps(), output_like("out", "x")),
    "add_rms_norm": (tensor_on_gpu("x"), tensor_on_gpu("residual"), like("residual", "x"),
                     vector_for("weight", "x"), finite_eps(), output_like("out", "x"),
                     output_like("residual_out", "x"), no_shared_elements("residual_out")),
    "rope": (tensor_on_gpu("x"), even_last("x"), broadcast_angles("cos", "x"),
             broadcast_angles("sin", "x"), output_like("out", "x")),
    "swiglu": (tensor_on_gpu("gate"), tensor_on_gpu("up"), like("up", "gate"), output_like("out", "gate")),
    "linear_decode": (tensor_on_gpu("x"), weight_matrix("weight", "x"), inner_dim("x", "weight"),
                      kind_name(), bias_for("bias", "x", "weight"), row_add_for("row_add", "x", "weight")),
    "post_attn_mlp": (tensor_on_gpu("hidden"), mlp_weights("w_gate_up", "w_down", "hidden"),
                      vector_for("norm_weight", "hidden", label="weight"), finite_eps(), kind_name()),
    "pre_attn_qkv": (tensor_on_gpu("hidden"), weight_matrix("w_qkv", "hidden", dtype_error=TypeError),
                     inner_dim("hidden", "w_qkv"),
                     vector_for("norm_weight", "hidden", label="weight"), finite_eps(), kind_name(),
                     bias_for("bias", "hidden", "w_qkv")),
    "linear_decode_fp8": (tensor_on_gpu("x"), weight_matrix("weight", "x", fp8=True),
                          row_scales("scale", "weight"), inner_dim("x", "weight"),
                          bias_for("bias", "x", "weight"), row_add_for("row_add", "x", "weight")),
    "post_attn_mlp_fp8": (tensor_on_gpu("hidden"), mlp_weights("w_gate_up", "w_down", "hidden", fp8=True),
                          row_scales("gate_up_scale", "w_gate_up"), row_scales("down_scale", "w_down"),
                          vector_for("norm_weight", "hidden", label="weight"), finite_eps()),
    "pre_attn_qkv_fp8": (tensor_on_gpu("hidden"), weight_matrix("w_qkv", "hidden", fp8=True),
                         row_scales("scale", "w_qkv"), inner_dim("hidden", "w_qkv"),
                         vector_for("norm_weight", "hidden", label="weight"), finite_eps(),
                         bias_for("bias", "hidden", "w_qkv")),
}


CONTRACT.update({
    "quantize_rows_fp8": (tensor_on_gpu("x"), has_rows("x"), codes_out("out", "x"),
                          scale_of_rows("scale_out", "x", optional=True)),
    "rms_norm_fp8": (tensor_on_gpu("x"), has_rows("x"), vector_for("weight", "x"), finite_eps(), codes_out("out", "x"),
                     scale_of_rows("scale_out", "x", optional=True)),
    "add_rms_norm_fp8": (tensor_on_gpu("x"), has_rows("x"), tensor_on_gpu("residual"), like("residual", "x"),
                         vector_for("weight", "x"), finite_eps(), codes_out("out", "x"),
                         scale_of_rows("scale_out", "x", optional=True), output_like("residual_out", "x"),
                         no_shared_elements("residual_out")),
    "linear_w8a8": (tensor_on_gpu("x", (FP8,)), has_rows("x"), scale_of_rows("x_scale", "x"),
                    weight_matrix("weight", "x", fp8=True), inner_dim("x", "weight"), row_scales("scale", "weight"),
                    activation_name("activation", "weight"), bias_of("bias", "x", "weight"),
                    row_add_for("row_add", "x", "weight"), output_dtype("dtype", "out")),
})


CONTRACT.update({
    "linear_fp4": (tensor_on_gpu("x"), has_rows("x"), fp4_matrix("weight", "scale", "x"),
                   activation_name("activation", "weight"), bias_of("bias", "x", "weight"),
                   row_add_for("row_add", "x", "weight")),
    "append_kv_fp4": (kv_cache("k", "k_scale", "v", "v_scale"), tensor_on_gpu("new_k"), kv_rows("new_k", "k"),
                      tensor_on_gpu("new_v"), like("new_v", "new_k"), kv_tokens("lengths", "pages", "k", "new_k")),
    "read_kv_fp4": (kv_cache("k", "k_scale", "v", "v_scale"), kv_tokens("lengths", "pages", "k"), kv_count("count"),
                    one_of("dtype", ACTIVATION)),
    "attend_kv_fp4": (kv_cache("k", "k_scale", "v", "v_scale"), tensor_on_gpu("q"), kv_rows("q", "k", multiple=True),
                      kv_tokens("lengths", "pages", "k", "q"), softmax_scale("scale", "q"), dense_output("out", "q")),
    "norm_add_norm": (tensor_on_gpu("x"), has_rows("x"), tensor_on_gpu("residual"), like("residual", "x"),
                      vector_for("post_weight", "x"), vector_for("weight", "x"), finite_eps(), gate_for("gate", "x"),
                      finite_scale("residual_scale"), output_like("out", "x"), no_shared_elements("out"),
                      output_like("residual_out", "x"), no_shared_elements("residual_out")),
})


def dot_kind_if(*sums: str, name: str = "kind") -> Rule:
    """The row sums come from the MFMA kernel, which kind "dot" selects: required
    when any of the ``sums`` buffers is passed."""

    def rule(a: dict) -> None:
        if any(a.get(s) is not None for s in sums) and a[name] != "dot":
            raise ValueError(f"row sums of squares come from the MFMA GEMV: kind must be 'dot', got {a[name]!r}")

    return rule


def _h(a: dict) -> int:
    return a["hidden"].shape[1]


_SUMSQ_LINEAR = (decode_rows("x"), unit_k_stride("weight"),
                 matrix_for("out", "x", _m("x"), _rows_of("weight")),
                 matrix_for("row_add", "x", _m("x"), _rows_of("weight"), optional=True, dtypes=FLOAT),
                 sums_buffer("ss_out", "x", _rows_of("weight")))
_SUMSQ_MLP = (decode_rows("hidden"), dense("norm_weight", "w_gate_up", "w_down"),
              matrix_for("out", "hidden", _m("hidden"), _h),
              matrix_for("mid", "hidden", _m("hidden"), _cols_of("w_down"), optional=True),
              sums_buffer("ss_in", "hidden", _h, optional=True), sums_buffer("ss_out", "hidden", _h, optional=True))
_SUMSQ_QKV = (decode_rows("hidden"), dense("norm_weight", "w_qkv"), sums_buffer("ss_in", "hidden", _h),
              matrix_for("out", "hidden", _m("hidden"), _rows_of("w_qkv")))

# The row-sum forms (rowsq.py): their plain operator's rules, then the layout the
# bare-pointer entry points assume.
CONTRACT.update({
    "linear_sumsq": (*CONTRACT["linear_decode"], dot_kind_if("ss_out"), *_SUMSQ_LINEAR),
    "post_attn_mlp_sumsq": (*CONTRACT["post_attn_mlp"], dot_kind_if("ss_in", "ss_out"), *_SUMSQ_MLP),
    "pre_attn_qkv_sumsq": (*CONTRACT["pre_attn_qkv"], dot_kind_if("ss_in"), *_SUMSQ_QKV),
    "linear_fp8_sumsq": (*CONTRACT["linear_decode_fp8"], *_SUMSQ_LINEAR),
    "post_attn_mlp_fp8_sumsq": (*CONTRACT["post_attn_mlp_fp8"], dense("gate_up_scale", "down_scale"),
                                *_SUMSQ_MLP),
    "pre_attn_qkv_fp8_sumsq": (*CONTRACT["pre_attn_qkv_fp8"], dense("scale"), *_SUMSQ_QKV),
})


def check(op: str, **args) -> dict:
    """Apply ``op``'s rules to its named arguments; returns them with values
    normalised (eps as a float). Raises on the first broken rule."""
    for rule in CONTRACT[op]:
        rule(args)
    return args

"""A key/value cache held in 4 bits (E2M1 codes, a power-of-two scale for each 32 along the head), and attention over it.

    cache = KvCacheFp4.empty(pages, heads, page, dim)
    append_kv_fp4(cache, k, v, lengths, pages)            # k, v [B, L, heads, dim]: the last L of each sequence's tokens
    y = attend_kv_fp4(q, cache, lengths, pages)           # q, y [B, L, query heads, dim]
    k, v = read_kv_fp4(cache, lengths, count, pages)      # tokens 0 .. count - 1 as values

``lengths`` (int32, on the device) are the sequences' tokens, the new ones among them: the same tensor serves the store and
the attention. ``pages`` (int32 ``[B, n]``) are each sequence's pages in order; without it page ``b`` is sequence ``b``'s.
Query ``l`` of ``L`` sees tokens ``0 .. lengths - L + l``; one that sees none gets zeros, and one that sees a key or value
that is no number gets NaN where it counts. Scores, the softmax and its sums are float32; its weights meet the values as
two bfloat16 numbers, within 2^-17 of them (a step of a bfloat16 output is 2^-7). The format is ``quantize_fp4``'s, along the
head. Heads of 64, 96, 128, 192 or 256. A layer of a decode step around it:

    qkv = pre_attn_qkv(x, attn_norm, w_qkv, cos, sin, eps, rope_cols=...)        # q and k rotated
    q, k, v = qkv.view(B, 1, heads + 2 * kv_heads, dim).split([heads, kv_heads, kv_heads], dim=2)
    append_kv_fp4(cache, k, v, lengths, pages)
    h = linear_decode(attend_kv_fp4(q, cache, lengths, pages).view(B, -1), w_o, row_add=x)

Nothing here reads ``lengths`` or ``pages`` on the host: they may change between replays of a captured graph. A page number
outside the cache is not followed (its tokens are neither stored nor seen), nor is a token past what a sequence's pages
hold.

Inference only. Where a trace or a transform is on or a gradient is asked for, a call goes to the custom op of the same
name (``torch.ops.fused_decode.*``). There is no reference counterpart (the reference has no cache and no attention).
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch
from torch.autograd.graph import increment_version

from . import _lib
from ._checks import E8M0, FP4_GROUP, check
from ._lib import DTYPE_CODE, FD_EUNSUPPORTED, FdKvShape, fail, native
from .ops import _PLANS, _raw_stream, _remember, _sig, _written
from .w8a8 import _PLAIN, _copied, _current_device, _grad, _like, _out_sig, _subclasses, _watched

__all__ = ["KvCacheFp4", "append_kv_fp4", "attend_kv_fp4", "read_kv_fp4"]


class KvCacheFp4(NamedTuple):
    """Keys and values as codes ``[pages, heads, page, dim / 2]`` (uint8) and scales ``[pages, heads, page, dim / 32]``
    (float8_e8m0fnu). The four share their strides (scales a sixteenth of the codes'), and slots lie together: one layer
    of a tensor that holds several, or a run of its pages, is a cache too."""

    k: torch.Tensor
    k_scale: torch.Tensor
    v: torch.Tensor
    v_scale: torch.Tensor

    @classmethod
    def empty(cls, pages: int, heads: int, page: int, dim: int, device="cuda") -> KvCacheFp4:
        """A cache of zeros."""
        def pair():
            codes = torch.zeros(pages, heads, page, dim // 2, dtype=torch.uint8, device=device)
            scale = torch.full((pages, heads, page, dim // FP4_GROUP), 127, dtype=torch.uint8, device=device)
            return codes, scale.view(E8M0)
        return cls(*pair(), *pair())


def _plain(cache, lengths, pages, *floats) -> bool:
    """Whether a launch on the pointers of these says all that torch's calls would. (Only floats have gradients, a cache's
    scales among them.)"""
    if _watched():
        return False
    grad = _grad()
    for t in floats:
        if t.__class__ not in _PLAIN or (grad and t.requires_grad) or t.is_neg():
            return not isinstance(t, torch.Tensor)  # anything else is the contract's to name
    k, ks, v, vs = cache
    if grad and (ks.requires_grad or vs.requires_grad):
        return False
    return (k.__class__ is ks.__class__ is v.__class__ is vs.__class__ is lengths.__class__ is torch.Tensor
            and (pages is None or pages.__class__ is torch.Tensor)) or not _subclasses(k, ks, v, vs, lengths, pages)


def _cache_sig(c: KvCacheFp4) -> tuple:
    k, ks, v, vs = c
    return (k.shape, k.stride(), k.dtype, k.get_device(), ks.shape, ks.stride(), ks.dtype, ks.get_device(),
            v.shape, v.stride(), v.dtype, v.get_device(), vs.shape, vs.stride(), vs.dtype, vs.get_device())


def _shape_of(cache: KvCacheFp4) -> tuple[FdKvShape, int]:
    """The ``fd_kv_shape`` of a checked cache, and its slots of a page. (A plan keeps the struct: calls get its address.)"""
    pages, heads, page, half = (int(n) for n in cache.k.shape)
    head = int(cache.k.stride(1)) if heads > 1 else page * half
    step = int(cache.k.stride(0)) if pages > 1 else heads * head
    return FdKvShape(pages, heads, page, 2 * half, step, head), page


class _Where:
    """How a call finds its tokens: the lengths and the table, and copies of them where they are not dense."""

    def __init__(self, lengths, pages, page: int):
        self.lengths_copy = lengths.numel() > 1 and not lengths.is_contiguous()
        self.pages_copy = pages is not None and pages.shape[1] > 1 and pages.stride(1) != 1
        self.step = 0 if pages is None else int(pages.shape[1]) if self.pages_copy else int(pages.stride(0))
        self.count = 0 if pages is None else int(pages.shape[1])
        self.capacity = page if pages is None else self.count * page

    def dense(self, lengths, pages):
        return (lengths.contiguous() if self.lengths_copy else lengths), (pages.contiguous() if self.pages_copy else pages)


def append_kv_fp4(
    cache: KvCacheFp4,
    k: torch.Tensor,
    v: torch.Tensor,
    lengths: torch.Tensor,
    pages: torch.Tensor | None = None,
) -> None:
    """Store ``k`` and ``v`` ``[B, L, heads, dim]`` (float16 or bfloat16) in the cache, in place, as tokens
    ``lengths - L .. lengths - 1`` of each sequence, in one launch. Positions below 0 are skipped, so a batch whose
    sequences have fewer than ``L`` new tokens is padded on the left. Two tokens of one call must
    not share a slot: it may then hold parts of both."""
    try:
        plain = _plain(cache, lengths, pages, k, v)
        key = ("append_kv_fp4", _cache_sig(cache), _sig(k), _sig(v), _sig(lengths), _sig(pages))
        plan = _PLANS.get(key) if plain else None
    except (AttributeError, TypeError, ValueError):  # a non-tensor argument: checked below
        plain, key, plan = True, None, None
    if not plain:
        torch.ops.fused_decode.append_kv_fp4(*cache, k, v, lengths, pages)
        return
    if plan is None:
        plan = _remember(key, _plan_append(*_four(cache), k, v, lengths, pages))
    plan(*cache, k, v, lengths, pages)


def _four(cache) -> tuple:
    if not isinstance(cache, tuple) or len(cache) != 4:
        raise TypeError(f"cache must be a KvCacheFp4, got {type(cache).__name__}")
    return tuple(cache)


def _plan_append(ck, cks, cv, cvs, k, v, lengths, pages):
    cache = KvCacheFp4(ck, cks, cv, cvs)
    check("append_kv_fp4", **cache._asdict(), new_k=k, new_v=v, lengths=lengths, pages=pages)
    kept, page = _shape_of(cache)
    shape = ctypes.addressof(kept)
    dev, act, call = k.device.index, DTYPE_CODE[k.dtype], native().append_kv_fp4
    b, n, heads, dim = (int(s) for s in k.shape)
    where = _Where(lengths, pages, page)
    if where.capacity == 0 or k.numel() == 0:  # no slot, or nothing (an empty tensor has no pointer to pass on)
        return lambda ck, cks, cv, cvs, k, v, lengths, pages: None
    k_copy, v_copy = (dim > 1 and t.stride(3) != 1 for t in (k, v))
    dense = (n * heads * dim, heads * dim, dim)
    sk = dense if k_copy else tuple(int(s) for s in k.stride()[:3])
    sv = dense if v_copy else tuple(int(s) for s in v.stride()[:3])

    def run(ck, cks, cv, cvs, k, v, lengths, pages):
        if _current_device() != dev:  # a launch on the default stream goes to the current device
            with torch.cuda.device(dev):
                return run(ck, cks, cv, cvs, k, v, lengths, pages)
        k, v = k.contiguous() if k_copy else k, v.contiguous() if v_copy else v
        lengths, pages = where.dense(lengths, pages)
        status = call(ck.data_ptr(), cks.data_ptr(), cv.data_ptr(), cvs.data_ptr(), shape, k.data_ptr(), v.data_ptr(),
                      *sk, *sv, lengths.data_ptr(), None if pages is None else pages.data_ptr(), where.step, where.count,
                      b, n, act, _raw_stream(dev))
        if status:
            fail("fd_append_kv_fp4", status)
        increment_version([ck, cks, cv, cvs])
    run.kept = kept
    return run


def read_kv_fp4(
    cache: KvCacheFp4,
    lengths: torch.Tensor,
    count: int,
    pages: torch.Tensor | None = None,
    *,
    dtype: torch.dtype = torch.bfloat16,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values of tokens ``0 .. count - 1`` of each sequence, ``[B, count, heads, dim]`` in ``dtype`` (float16 or
    bfloat16), zeros where a sequence has no such token: what an attention of the caller's own takes, say over a
    prompt's cached prefix."""
    try:
        plain = _plain(cache, lengths, pages)
        key = ("read_kv_fp4", _cache_sig(cache), _sig(lengths), count, _sig(pages), dtype)
        plan = _PLANS.get(key) if plain else None
    except (AttributeError, TypeError, ValueError):
        plain, key, plan = True, None, None
    if not plain:
        return torch.ops.fused_decode.read_kv_fp4(*cache, lengths, count, pages, dtype)
    if plan is None:
        plan = _remember(key, _plan_read(*_four(cache), lengths, count, pages, dtype))
    return plan(*cache, lengths, pages)


def _plan_read(ck, cks, cv, cvs, lengths, count, pages, dtype):
    cache = KvCacheFp4(ck, cks, cv, cvs)
    count = check("read_kv_fp4", **cache._asdict(), lengths=lengths, count=count, pages=pages, dtype=dtype)["count"]
    kept, page = _shape_of(cache)
    shape = ctypes.addressof(kept)
    device, dev, act, call = ck.device, ck.device.index, DTYPE_CODE[dtype], native().read_kv_fp4
    b, heads, dim = int(lengths.shape[0]), int(ck.shape[1]), 2 * int(ck.shape[3])
    where = _Where(lengths, pages, page)
    like = _like((b, count, heads, dim), dtype, device)
    if where.capacity == 0 or ck.shape[0] == 0:
        return lambda ck, cks, cv, cvs, lengths, pages: (torch.zeros_like(like), torch.zeros_like(like))

    def run(ck, cks, cv, cvs, lengths, pages):
        if _current_device() != dev:
            with torch.cuda.device(dev):
                return run(ck, cks, cv, cvs, lengths, pages)
        k, v = torch.empty_like(like), torch.empty_like(like)
        lengths, pages = where.dense(lengths, pages)
        status = call(k.data_ptr(), v.data_ptr(), ck.data_ptr(), cks.data_ptr(), cv.data_ptr(), cvs.data_ptr(), shape,
                      lengths.data_ptr(), None if pages is None else pages.data_ptr(), where.step, where.count, b, count,
                      act, _raw_stream(dev))
        if status:
            fail("fd_read_kv_fp4", status)
        return k, v
    run.kept = kept
    return run


def attend_kv_fp4(
    q: torch.Tensor,
    cache: KvCacheFp4,
    lengths: torch.Tensor,
    pages: torch.Tensor | None = None,
    *,
    scale: float | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Attention of ``q [B, L, query heads, dim]`` (float16 or bfloat16), each sequence's last ``L`` tokens, over the cache:
    ``softmax(scale * q k^T) v`` with ``scale`` 1 / sqrt(dim) by default. Query heads are a multiple of the cache's, each run
    of them reading one. One launch, and another one that joins where a sequence's tokens are cut into shares."""
    try:
        plain = _plain(cache, lengths, pages, q) and (out is None or out.__class__ in _PLAIN)
        key = ("attend_kv_fp4", _sig(q), _cache_sig(cache), _sig(lengths), _sig(pages), scale,
               None if out is None else _out_sig(out))
        plan = _PLANS.get(key) if plain else None
    except (AttributeError, TypeError, ValueError):
        plain, key, plan = True, None, None
    if not plain:
        got = torch.ops.fused_decode.attend_kv_fp4(q, *cache, lengths, pages,
                                                   q.shape[-1] ** -0.5 if scale is None else scale)
        return _copied((got,), out)[0]
    if plan is None:
        plan = _remember(key, _plan_attend(q, *_four(cache), lengths, pages, scale, out))
    return plan(q, *cache, lengths, pages, out)


def _plan_attend(q, ck, cks, cv, cvs, lengths, pages, scale, out):
    cache = KvCacheFp4(ck, cks, cv, cvs)
    scale = check("attend_kv_fp4", q=q, **cache._asdict(), lengths=lengths, pages=pages, scale=scale, out=out)["scale"]
    kept, page = _shape_of(cache)
    shape = ctypes.addressof(kept)
    device, dev, act, call = q.device, q.device.index, DTYPE_CODE[q.dtype], native().attend_kv_fp4
    b, n, heads, dim = (int(s) for s in q.shape)
    where = _Where(lengths, pages, page)
    like = _like((b, n, heads, dim), q.dtype, device)
    if q.numel() == 0:
        return lambda q, ck, cks, cv, cvs, lengths, pages, o: torch.empty_like(like) if o is None else o
    if where.capacity == 0 or cache.k.shape[0] == 0:  # nothing to see
        return lambda q, ck, cks, cv, cvs, lengths, pages, o: torch.zeros_like(like) if o is None else o.zero_()
    q_copy = q.stride(3) != 1
    sq = (n * heads * dim, heads * dim, dim) if q_copy else tuple(int(s) for s in q.stride()[:3])
    with torch.cuda.device(dev):
        size = _lib.scratch_bytes("fd_attend_kv_fp4_scratch", b, n, heads, int(ck.shape[1]), dim, where.capacity)
    part_like = _like((size // 4,), torch.float32, device) if size else None

    def run(q, ck, cks, cv, cvs, lengths, pages, o):
        if _current_device() != dev:
            with torch.cuda.device(dev):
                return run(q, ck, cks, cv, cvs, lengths, pages, o)
        y = torch.empty_like(like) if o is None else o
        if q_copy:
            q = q.contiguous()
        lengths, pages = where.dense(lengths, pages)
        part = None if part_like is None else torch.empty_like(part_like)
        args = (q.data_ptr(), ck.data_ptr(), cks.data_ptr(), cv.data_ptr(), cvs.data_ptr(), shape, *sq,
                lengths.data_ptr(), None if pages is None else pages.data_ptr(), where.step, where.count, b, n, heads,
                scale, None if part is None else part.data_ptr(), size, act, _raw_stream(dev))
        status = call(y.data_ptr(), *args)
        if status == FD_EUNSUPPORTED and o is not None:  # `out` lies over an operand, or off alignment: write beside it
            beside = torch.empty_like(like)
            status = call(beside.data_ptr(), *args)
            if status == 0:
                return o.copy_(beside)
        if status:
            fail("fd_attend_kv_fp4", status)
        return y if o is None else _written(o)
    run.kept = kept
    return run

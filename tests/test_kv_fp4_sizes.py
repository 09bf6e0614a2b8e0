"""Sizes and strides of the 4-bit cache's entry points whose products leave 64 bits are refused like other ones that are too
large, not taken for what is left of them."""

from __future__ import annotations

import ctypes

from test_kv_fp4 import append, attend, nogpu, read, refused, shape

from fused_decode import _lib as L


@nogpu
def test_strides():
    for call in (append, read, attend):
        assert refused(call(s=shape(pages=17, step=1 << 60)), L.FD_EUNSUPPORTED, b"GiB")  # 16 steps are 2^64
        assert refused(call(s=shape(heads=17, head=1 << 60, step=1 << 20)), L.FD_EUNSUPPORTED, b"GiB")
        assert refused(call(s=shape(pages=2**31 - 1, step=(1 << 62) + (1 << 40))), L.FD_EUNSUPPORTED, b"GiB")


@nogpu
def test_tokens_and_queries():
    wide = shape(heads=2**15, dim=128)
    assert refused(append(s=wide, st=[0] * 6, seqs=2**15, new=2**30), L.FD_EUNSUPPORTED, b"large")  # 2^64 lanes
    assert refused(append(s=wide, st=[0] * 6, seqs=2**15, new=2**31), L.FD_EUNSUPPORTED, b"large")
    assert refused(attend(new=1 << 62, hq=8), L.FD_EUNSUPPORTED, b"rows")  # 2^64 query rows of a head
    assert refused(attend(new=1, hq=1 << 62), L.FD_EUNSUPPORTED, b"rows")


def test_scratch_of_what_is_refused():
    for b, new, hq, heads in ((1, 1 << 62, 8, 2), (1, 1, 1 << 62, 2), (1 << 40, 1 << 20, 64, 64), (1, 1 << 20, 64, 1)):
        out = ctypes.c_int64(-1)
        assert L.lib().fd_attend_kv_fp4_scratch(b, new, hq, heads, 64, 100000, ctypes.byref(out)) == L.FD_OK
        assert out.value == 0

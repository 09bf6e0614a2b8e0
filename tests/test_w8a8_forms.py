"""Which kernel fd_linear_w8a8 takes, as its host-only query says (the library's figures are of 256 CUs without a GPU):
the products of test_w8a8_forms_gpu reach every form of tiles, with and without K splits, and every form for few rows."""

from __future__ import annotations

import ctypes

import pytest
import torch
from test_w8a8_forms_gpu import FEW, TILES, form

from fused_decode import _lib as L


def test_the_query():
    out = (ctypes.c_int * 4)()
    lib = L.lib()
    assert lib.fd_linear_w8a8_form(-1, 2, 3, out) == L.FD_EINVAL and lib.fd_linear_w8a8_form(1, 2, 3, None) == L.FD_EINVAL
    for m, n, k in ((0, 64, 64), (8, 0, 64), (2**31, 64, 64)):
        assert form(m, n, k) == (0, 0, 0, 0)
    assert form(9, 64, 15) == form(1, 64, 0) == (1, 0, 0, 0) and form(1, 64, 16) == (2, 0, 0, 0)
    assert form(2, 64, 16) == form(2, 64, 17) == (3, 1, 4, 0) and form(32, 64, 8192) == (3, 2, 8, 0)
    assert form(33, 64, 64)[0] == form(17, 64, 8193)[0] == form(2, 64, 16385)[0] == 4


@pytest.mark.skipif(torch.cuda.is_available(), reason="of 256 CUs")
def test_the_scratch_is_that_of_the_form():
    for m, n, k in [case[:3] for case in TILES] + [(40, 1000, 8209), (9, 70, 33)]:
        f, size = form(m, n, k), ctypes.c_int64()
        assert L.lib().fd_linear_w8a8_scratch(m, n, k, 1, ctypes.byref(size)) == L.FD_OK
        copies = 0 if k % 16 == 0 else (m + n) * (k + 15 & ~15)
        assert size.value == copies + (f[3] * m * n * 4 if f[3] > 1 else 0)


def test_every_form_is_among_the_products():
    tiles = {(form(*case[:3])[1:3], form(*case[:3])[3] > 1) for case in TILES}
    sizes = [(256, 256), (256, 128), (128, 128), (64, 128), (64, 64), (128, 32)]
    assert tiles == {(size, split) for size in sizes for split in (False, True)}
    few = {form(*case)[1:3] for case in FEW}
    assert few == {(1, 4), (1, 8), (1, 16), (2, 4), (2, 8)}

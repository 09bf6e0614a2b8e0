"""The sizes that fd_linear_w8a8 refuses, on the CPU: its checks return before any HIP call."""

from __future__ import annotations

import pytest
import torch

from fused_decode import _lib as L

nogpu = pytest.mark.skipif(torch.cuda.is_available(), reason="host-only argument checks")
X, W, Y, S, T, B = ((1 << 44) * i for i in range(1, 7))  # far apart


def linear(m, n, k, act=0, size=0):
    return L.lib().fd_linear_w8a8(Y, X, S, W, S + (1 << 40), None, 0, act, None, 0, m, n, k, k, k, 1, 0, 0,
                                  n // 2 if act == 5 else n, 1, T if size else None, size, 0, None)


@nogpu
def test_sizes_past_the_kernels():
    said = lambda status, words: status == L.FD_EUNSUPPORTED and words in L.lib().fd_last_error()
    for k in (2**23 - 8, 2**23, 2**23 + 1, 2**28):
        assert said(linear(2, 64, k, size=1 << 42), b"too large to align"), k
        assert said(linear(40, 64, k, size=1 << 42), b"too large to align"), k
    assert said(linear(2, 64, 2**23 - 24, size=64), b"need scratch")  # taken, as far as this goes
    assert said(linear(1, 2**27, 64), b"outputs") and said(linear(1, 2**27, 64, act=5), b"outputs")
    for m, n, k in ((2**31 - 512, 64, 64), (2, 2**31 - 512, 64), (1, 64, 2**31 - 512)):
        assert said(linear(m, n, k), b"too large")

"""norm_add_norm on operands that lie beside each other in one buffer's rows: ranges that cross but share no byte are taken,
others refused."""

from __future__ import annotations

from test_block_norms import G, PW, R, RO, W, X, Y, nogpu, norms, refused, rows

from fused_decode import _lib as L

P = 0x10000000  # a buffer of rows of 128 elements, 256 bytes


def passes(**a):
    """Whether the checks let a call through: what then fails here is the launch."""
    return norms(**a) == L.FD_ELAUNCH


@nogpu
def test_halves_of_a_row():
    half = rows(sc=128)
    assert passes(y=P, ly=half, ro=P + 128, lro=half)
    assert passes(y=P + 128, ly=half, x=P, lx=half) and passes(ro=P, lro=half, r=P + 128, lr=half)
    assert passes(y=P, ly=half, g=P + 128, lg=half, gd=0)
    assert passes(y=P, ly=half, g=P + 128, lg=rows(sc=0), gd=0)  # between the first two rows
    three = rows(b=2, c=2, sc=128)  # planes of two rows
    three.sb = 256
    other = lambda: rows(b=2, c=2)
    planes = dict(lx=other(), lr=other(), ly=three, lro=three)
    planes["lx"].sb = planes["lr"].sb = 128
    assert passes(y=P, ro=P + 128, **planes)


@nogpu
def test_rows_that_share_bytes():
    half = rows(sc=128)
    for d in (2, 126, 254, 130, 126 + 256):  # an element on, and over the next row's first
        assert refused(norms(y=P, ly=half, ro=P + d, lro=half), L.FD_EINVAL, b"each other"), d
        assert refused(norms(y=P + d, ly=half, x=P, lx=half), L.FD_EINVAL, b"overlap"), d
    # rows of other strides, columns of a stride, weights: by their ranges
    assert refused(norms(y=P, ly=half, ro=P + 128, lro=rows(sc=64)), L.FD_EINVAL, b"each other")
    assert refused(norms(y=P, ly=rows(sc=256, col=2), ro=P + 2, lro=rows(sc=256, col=2)), L.FD_EINVAL, b"each other")
    assert refused(norms(y=P, ly=half, pw=P + 128), L.FD_EINVAL, b"weight")
    for d in (2, 130):
        assert refused(norms(y=P, ly=half, g=P + d, lg=rows(sc=0)), L.FD_EINVAL, b"gate"), d

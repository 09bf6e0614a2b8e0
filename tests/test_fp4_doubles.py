"""quantize_fp4 of float64 weights: codes nearest to the weights themselves, not to their float32 roundings."""

from __future__ import annotations

import torch

from fused_decode import fp4

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def nearest(v, unit):
    near = (v.abs() / unit)[..., None].sub(GRID).abs()
    tied = near == near.amin(-1, keepdim=True)
    pick = torch.where(tied & (torch.arange(8) % 2 == 0), 2, tied.int()).argmax(-1)
    return torch.copysign(GRID[pick] * unit, v)


def test_values_beside_the_borders():
    """A hair above, at and below every border between codes and between scales, at several scales."""
    edges = (GRID[1:] + GRID[:-1]) / 2
    hair = 2.0**-45
    v = torch.cat([edges, edges * (1 + hair), edges * (1 - hair)])
    v = torch.cat([v, -v, torch.full((32 * 2 - 2 * len(v),), 6.0, dtype=torch.float64)]).view(2, 32)
    v[:, -1] = 6.0
    for e in (-126, -100, -1, 0, 7, 100, 124):
        codes, scale = fp4.quantize_fp4(v * 2.0**e)
        assert bool((scale.double() == 2.0**e).all())
        got = fp4.dequantize_fp4(codes, scale).double()
        want = nearest(v * 2.0**e, torch.tensor(2.0**e, dtype=torch.float64))
        assert torch.equal(got, want) and torch.equal(torch.signbit(got), torch.signbit(want))


def test_scales_beside_their_border():
    for top, want in ((7.0, 2.0), (7.0 * (1 - 2.0**-45), 1.0), (7.0 * (1 + 2.0**-45), 2.0), (1e-300, 2.0**-126), (0.0, 1.0)):
        w = torch.zeros(1, 32, dtype=torch.float64)
        w[0, 5] = -top
        assert fp4.quantize_fp4(w)[1].double().item() == want
    w = torch.zeros(3, 32, dtype=torch.float64)  # beyond float32: as infinities are
    w[0, 1], w[1, 1], w[2, 1] = 1e39, float("inf"), float("nan")
    assert fp4.quantize_fp4(w)[1].view(torch.uint8).tolist() == [[255]] * 3


def test_float32_weights_keep_their_codes():
    w = torch.randn(50, 96, generator=torch.Generator().manual_seed(1))
    for a, b in zip(fp4.quantize_fp4(w), fp4.quantize_fp4(w.double())):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))

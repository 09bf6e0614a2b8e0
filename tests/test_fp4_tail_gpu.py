"""Codes past K are not used, whatever they and their group's scale are: of small integers every result is exact."""

from __future__ import annotations

import pytest
import torch
from test_fp4_gpu import BOTH, ints, random_codes, weights64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("activation", [None, "swiglu"])
@pytest.mark.parametrize("m", [1, 2, 5, 16, 20, 32, 40, 130])
@pytest.mark.parametrize("k", [1, 31, 33, 100, 257, 2051, 4100])
def test_codes_past_k_under_scales_that_leave_bfloat16(m, k, activation, dtype):
    """The last group's scale 2^126 or 2^127, its codes 0 up to K and 2, 4 or 6 behind it."""
    import fused_decode as fd

    n = 70
    codes, scale = random_codes(n, k, 1)
    x = ints(m, k, seed=2, dtype=dtype)
    first = (k - 1) // 32 * 32  # the last group's
    flat = torch.stack([codes & 15, codes >> 4], -1).flatten(1)
    flat[:, first:k] = 0
    behind = torch.tensor([4, 6, 7, 12, 14, 15], dtype=torch.uint8, device=codes.device)
    dirty = flat.clone()
    dirty[:, k:] = behind[torch.arange(n * (flat.shape[1] - k), device=codes.device) % 6].view(n, -1)
    scale.view(torch.uint8)[::2, -1], scale.view(torch.uint8)[1::2, -1] = 253, 254
    pack = lambda f: f[:, 0::2] | f[:, 1::2] << 4
    flat[:, k:] = 0
    v = x.double() @ weights64(pack(flat), scale, k).t()
    got = fd.linear_fp4(x, pack(dirty), scale, activation=activation)
    assert torch.equal(got, fd.linear_fp4(x, pack(flat), scale, activation=activation))
    if activation is None:
        assert torch.equal(got, v.to(dtype))
    else:
        assert not bool(torch.isnan(got).any())

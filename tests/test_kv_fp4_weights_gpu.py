"""What the softmax weights keep of their bits on their way through the matrix cores.

Two tokens, keys 1 and 0 in one channel and values -6 and 6, so that a query's output is -6 tanh(q / 2), and 4096 queries
from 1e-4 to 2e-3. The score is exact, so the weights are 1 and p = exp(-q) just below 1, held as two bfloat16 numbers: the
first within 2^-9 (half a step below 1), so what it leaves out is at most 2^-9 and is held within half a step of that,
2^-18. The output is off by that over the weights' sum, 2^-19 of 6; p's exponential, the sums and the division add at most
2^-20 of 6 (p's own error of 2^-21 cancels by half in p / (1 + p), and a handful of float32 roundings of 2^-24). Then the
output's rounding to float16."""

from __future__ import annotations

import pytest
import torch
from test_kv_fp4_gpu import DEV, E8M0, i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page", [32, 2])
@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
def test_weights_are_held_in_two_rounded_parts(dim, page):
    import fused_decode as fd

    codes = lambda: torch.zeros(1, 1, page, dim // 2, dtype=torch.uint8, device=DEV)
    scale = torch.full((1, 1, page, dim // 32), 127, dtype=torch.uint8, device=DEV).view(E8M0)
    k, v = codes(), codes()
    k[0, 0, 0, 0] = 0x02  # 1.0 in channel 0
    v[0, 0, 0], v[0, 0, 1] = 0xFF, 0x77  # -6 and 6
    q = torch.zeros(1, 1, 4096, dim, dtype=torch.float16, device=DEV)
    s = (torch.rand(4096, generator=torch.Generator().manual_seed(9)) * 1.9e-3 + 1e-4).half()
    q[0, 0, :, 0] = s.to(DEV)
    y = fd.attend_kv_fp4(q, fd.KvCacheFp4(k, scale, v, scale.clone()), i32([2]), scale=1.0)[0, 0].cpu().double()
    want = -6 * torch.tanh(s.double() / 2)[:, None]
    before = 6 * (2.0**-19 + 2.0**-20)
    assert bool(((y - want).abs() <= before + 2.0**-11 * (want.abs() + before) + 2.0**-25).all())

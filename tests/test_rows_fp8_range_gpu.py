"""Norms to E4M3 codes of rows whose squares leave float32's range: their sum overflows (bfloat16 values above about
1e19) or underflows beside an eps as small (below about 1e-14). The bounds are test_w8a8_gpu.check_codes': the power of two
on such a row rounds nothing, so a row's codes and scale carry the errors of any other."""

from __future__ import annotations

import pytest
import torch
from test_w8a8_gpu import DEV, check_codes, norm64, rnd

pytestmark = pytest.mark.gpu


def rows_at(powers, n, seed, dtype):
    """A row of values up to 1.5 for each power of two, and one of them that is 1 but for its last value."""
    x = rnd(2 * len(powers), n, seed=seed).double().clamp(-1.5, 1.5)
    x[len(powers):, :-1] = 1.0
    p = torch.tensor(powers, device=DEV).double().exp2()[:, None]
    x[: len(powers)] *= p
    x[len(powers):, -1:] *= p
    return x.to(dtype)


# lanes of a row, vectors of a lane, a workgroup a row, and the kernel for any strides
@pytest.mark.parametrize("n", [8, 21, 100, 256, 600, 1025, 2056, 4096, 8193, 20000, 40000])
@pytest.mark.parametrize("eps", [0.0, 1e-30, 1e-12, 1e-5, 1e30])
def test_sums_of_squares_out_of_range(n, eps):
    import fused_decode as fd

    # with eps no smaller than a row's squares its values are t w / sqrt(eps): the rows that keep float32's precision there
    low = [-133, -120, -100, -70, -50, -46, -40] if eps == 0 else [-100, -70, -46, -40] if eps < 1 else [-20]
    for dtype, powers in ((torch.bfloat16, low + [0, 40, 62, 63, 64, 80, 100, 125]), (torch.float16, [-14, 0, 15])):
        x = rows_at(powers, n, n, dtype)
        for w in (rnd(n, seed=1), rnd(n, seed=2, dtype=dtype), rnd(2 * n, seed=3)[::2]):
            codes, scale = fd.rms_norm_fp8(x, w, eps)
            assert bool(scale.isfinite().all())
            check_codes(codes, scale, norm64(x.double(), w, eps), n)
            r = (x.double() / 4).to(dtype)
            codes, scale, ro = fd.add_rms_norm_fp8(x, r, w, eps)
            total = x.float() + r.float()
            check_codes(codes, scale, norm64(total.double(), w, eps), n)
            assert torch.equal(ro, total.to(dtype))


@pytest.mark.parametrize("n", [64, 4096, 40000])
def test_rows_that_stay_what_they_are(n):
    """Zeros, infinities and NaN beside rows out of range, and rows in range, whose codes do not change with them."""
    import fused_decode as fd

    w = torch.ones(n, device=DEV)
    x = rnd(8, n, seed=n, dtype=torch.bfloat16)
    alone = fd.rms_norm_fp8(x[6:].clone(), w, 0.0)
    x[0], x[1], x[2] = 0, 1e30, -1e-30
    x[3, n - 1], x[4, 0], x[5, n // 2] = float("inf"), float("-inf"), float("nan")
    codes, scale = fd.rms_norm_fp8(x, w, 1e-5)
    assert bool((codes[0].float() == 0).all()) and float(scale[0]) == 1
    assert bool((codes[1].float() == 448).all()) and bool(codes[3:6].float().isnan().all())
    assert bool(scale[3:6].isnan().all()) and bool(scale[:3].isfinite().all())
    codes, scale = fd.rms_norm_fp8(x, w, 0.0)  # 0 / 0: no norm to have
    assert bool(codes[0].float().isnan().all()) and bool((codes[2].float() == -448).all())
    assert torch.equal(codes[6:].view(torch.uint8), alone[0].view(torch.uint8)) and torch.equal(scale[6:], alone[1])

"""Products of few rows on either side of the border between the kernels, and those of a caller that has no scratch: of
small integers every result is exact."""

from __future__ import annotations

import pytest
import torch
from test_fp4_gpu import BOTH, ints, random_codes, weights64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("m,n,k", [(2, 70, 8192), (2, 70, 8224), (16, 33, 8192), (16, 33, 16384), (4, 40, 16384),
                                   (17, 48, 4096), (17, 48, 4128), (32, 64, 1535), (32, 64, 1537), (12, 100, 4095),
                                   (13, 20, 4095), (3, 90, 4097), (29, 500, 2051)])
def test_both_sides_of_the_border(m, n, k, dtype):
    import fused_decode as fd

    x, (codes, scale) = ints(m, k, seed=m, dtype=dtype, most=1), random_codes(n, k, n)
    v = x.double() @ weights64(codes, scale, k).t()
    assert torch.equal(fd.linear_fp4(x, codes, scale), v.to(dtype))


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("m,n,k", [(29, 203, 2051), (2, 64, 14336), (13, 64, 14336), (20, 33, 8192), (32, 64, 128)])
def test_few_rows_need_no_scratch(m, n, k, dtype):
    from fused_decode import _lib as L

    x, (codes, scale) = ints(m, k, seed=m, dtype=dtype, most=1), random_codes(n, k, n)
    y = torch.empty(m, n, dtype=dtype, device=x.device)
    g = scale.shape[1]
    code = L.DTYPE_CODE[dtype]
    status = L.lib().fd_linear_fp4(y.data_ptr(), x.data_ptr(), codes.data_ptr(), scale.data_ptr(), None, 0, 0, None, 0, m, n,
                                   k, k, 16 * g, g, 1, n, 1, n, 1, None, 0, code, torch.cuda.current_stream().cuda_stream)
    assert status == L.FD_OK
    assert torch.equal(y, (x.double() @ weights64(codes, scale, k).t()).to(dtype))

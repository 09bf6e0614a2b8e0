"""Which kernel a product of few rows takes, as the scratch it asks for shows (none where its activations stay in
registers)."""

from __future__ import annotations

import pytest

from test_fp4 import scratch

FP16, BF16 = 0, 1


@pytest.mark.parametrize("m,n,k,dtype", [
    (2, 6144, 4096, FP16), (32, 28672, 4096, FP16), (32, 4096, 4096, BF16), (16, 2048, 8192, FP16), (16, 2048, 8192, BF16),
    (4, 4096, 14336, BF16), (12, 16384, 3001, FP16), (16, 28672, 2051, BF16), (32, 4096, 1001, FP16), (2, 5, 1, BF16)])
def test_activations_in_registers(m, n, k, dtype):
    assert scratch(m, n, k, dtype) == (0, 0)


@pytest.mark.parametrize("m,n,k,dtype", [
    (29, 5003, 2051, FP16), (17, 5003, 2051, BF16), (2, 4096, 14336, FP16), (13, 4096, 14336, BF16), (17, 2048, 8192, FP16),
    (32, 4096, 5120, BF16), (2, 4096, 28672, BF16), (8, 5003, 4099, FP16), (33, 64, 128, BF16)])
def test_tiles(m, n, k, dtype):
    status, size = scratch(m, n, k, dtype)
    assert status == 0 and size >= m * -(-k // 128) * 128 * (4 if dtype == FP16 else 2)

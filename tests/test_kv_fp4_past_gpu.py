"""Attention over the 4-bit cache where lengths pass what a sequence's pages hold, and where page numbers lie outside the
cache, on the path whose steps are runs of slots."""

from __future__ import annotations

import pytest
import torch
from test_kv_fp4_gpu import BOTH, check_attention, i32, random_cache, rnd

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [32, 33, 63, 64, 100, 1000, 4111])
def test_lengths_past_the_only_page(page, dim, dtype):
    """Without a table a sequence has its page's tokens, each once, however far its length goes past them."""
    import fused_decode as fd

    cache = random_cache(1, 2, page, dim, seed=page)
    whole = -(-page // 32) * 32
    for new in (1, 2, 5):
        q = rnd(1, new, 4, dim, seed=6, dtype=dtype)
        for length in (page - 1, page, page + 1, whole - 1, whole, whole + new - 1, whole + new, 2 * page + 7, 2**31 - 1):
            n = i32([length])
            check_attention(fd.attend_kv_fp4(q, cache, n), q, cache, n)


@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("page", [32, 64])
def test_lengths_and_pages_outside_the_cache_in_whole_steps(page, dim):
    """Pages of whole steps: lengths past them and below zero, page numbers that no page has."""
    import fused_decode as fd

    cache = random_cache(9, 2, page, dim, seed=7)
    table = i32([[0, 3, 8], [9, 1, -1], [-5, 1 << 30, 2], [4, 4, 4], [-1, -1, 9], [5, 6, 7]])
    q = rnd(6, 3, 4, dim, seed=8, dtype=torch.bfloat16)
    for lengths in ([3 * page, 70, 75, 3 * page - 1, 60, 33], [3 * page + 1, 1000, 2**31 - 1, 2, -3, -(2**31)],
                    [3 * page + 2, page + 1, page, page - 1, 0, 3 * page + 34]):
        n = i32(lengths)
        check_attention(fd.attend_kv_fp4(q, cache, n, table), q, cache, n, table)

"""Attention over the 4-bit cache where scores are infinite."""

from __future__ import annotations

import math

import pytest
import torch
from test_kv_fp4_gpu import BOTH, DEV, check_attention, i32, random_cache, rnd

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page", [0, 32, 64, 24])
@pytest.mark.parametrize("dim", [64, 128, 192])
def test_scores_of_minus_infinity(page, dim):
    """Scores that fall below float32 (bfloat16's largest queries times a negative key) weigh nothing beside finite ones,
    and a query of which all scores do has no softmax: NaN, not the zeros of one that sees no token."""
    import fused_decode as fd

    size, count = page or 192, 192
    per = count // size
    q = rnd(1, 2, 2, dim, seed=1, dtype=torch.bfloat16)
    q[..., 0] = 3e38
    for first, last in ((0, 32), (0, 96), (96, 192), (31, 33), (0, 191)):  # the tokens whose scores are below float32
        cache = random_cache(per, 1, size, dim, seed=3)
        k = cache.k.view(1, count, dim // 2) if per == 1 else cache.k.view(count, dim // 2)[None]
        k[0, :, 0] &= 0xF0  # channel 0: 0 for the others
        k[0, first:last, 0] |= 0x0E  # -4
        cache.k_scale.view(torch.uint8).view(count, -1)[first:last, 0] = 127
        table = torch.arange(per, dtype=torch.int32, device=DEV)[None] if page else None
        y = fd.attend_kv_fp4(q, cache, i32([count]), table)
        held = cache.k_scale.view(torch.uint8).view(count, -1)
        rest = [t for t in range(count) if not first <= t < last]
        # the same with the other tokens alone, in one page, each query's own
        for l in range(2):
            seen = [t for t in rest if t <= count - 2 + l]
            if not seen:
                assert bool(torch.isnan(y[0, l]).all())
                continue
            part = fd.KvCacheFp4(*(t.view(torch.uint8).view(count, -1)[seen].view(1, 1, len(seen), -1).contiguous().view(t.dtype)
                                   for t in cache))
            few = q[:, l : l + 1].clone()
            few[..., 0] = 0.0
            check_attention(y[:, l : l + 1].contiguous(), few, part, i32([len(seen)]))
        assert held.shape[0] == count
    assert not fd.attend_kv_fp4(q, cache, i32([0]), table).any()


def test_a_row_of_minus_infinity_beside_one_that_finds_more():
    """Tokens 0 to 31 have scores of minus infinity, 32 to 127 are in no page, 128 is the second query's only: its wave
    raises a maximum while the first query's stays."""
    import fused_decode as fd

    cache = random_cache(17, 1, 8, 128, seed=6)
    cache.k[:4, ..., 0] = cache.k[:4, ..., 0] & 0xF0 | 0x0E  # -4
    cache.k[16, ..., 0] &= 0xF0
    cache.k_scale.view(torch.uint8)[:4, ..., 0] = 127
    q = rnd(1, 2, 1, 128, seed=7, dtype=torch.bfloat16)
    q[..., 0] = 3e38
    table = i32([[0, 1, 2, 3, *[-1] * 12, 16]])
    y = fd.attend_kv_fp4(q, cache, i32([129]), table)
    assert bool(torch.isnan(y[0, 0]).all())
    want = fd.read_kv_fp4(cache, i32([129]), 129, table)[1][0, 128]
    assert torch.equal(y[0, 1], want)  # all of the weight is on token 128


@pytest.mark.parametrize("dtype", BOTH)
def test_infinite_queries(dtype):
    """Minus infinity times keys above zero: every score is minus infinity, and the softmax of nothing else is NaN; plus
    infinity among the scores is NaN as well."""
    import fused_decode as fd

    for length in (1, 20, 200, 5000):
        cache = random_cache(1, 1, length, 128, seed=4)
        cache.k[..., 0] = cache.k[..., 0] & 0xF0 | 0x04  # channel 0: 2
        q = rnd(1, 1, 3, 128, seed=5, dtype=dtype)
        clean = fd.attend_kv_fp4(q, cache, i32([length]))
        for bad in (-math.inf, math.inf):
            one = q.clone()
            one[0, 0, 1, 0] = bad
            y = fd.attend_kv_fp4(one, cache, i32([length]))
            assert bool(torch.isnan(y[0, 0, 1]).all()) and torch.equal(y[0, 0, ::2], clean[0, 0, ::2])

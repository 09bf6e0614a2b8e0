"""Attention over the 4-bit cache where scores are no numbers: NaN stands where it has to, and the rest of such a call is
the call without it, bit for bit (no other row's sums have another operand or another order)."""

from __future__ import annotations

import pytest
import torch
from test_kv_fp4_gpu import BOTH, DEV, gen, i32, random_cache, rnd

pytestmark = pytest.mark.gpu

# page (0: no table) and tokens: a wave's only step, several waves', a last step that ends inside, shares
PLACES = [(0, 1), (0, 40), (0, 128), (0, 5000), (64, 20), (64, 300), (64, 6000), (24, 20), (24, 128), (24, 5000)]


def cache_of(page, length, heads, dim, seqs=2):
    per = -(-length // page) if page else 1
    cache = random_cache(seqs * per, heads, page or length, dim, seed=length)
    table = torch.randperm(seqs * per, generator=gen(length)).view(seqs, per).to(torch.int32).to(DEV) if page else None
    return cache, table


def slot_of(table, page, b, t):
    return (b, t) if table is None else (int(table[b, t // page]), t % page)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("dim", [64, 128, 192])
@pytest.mark.parametrize("page,length", PLACES)
def test_a_query_of_no_numbers_gets_none(page, length, dim, dtype):
    """All of a sequence's queries NaN (a tile of nothing else), or one head's among others."""
    import fused_decode as fd

    cache, table = cache_of(page, length, 2, dim)
    n = i32([length, length])
    for group, new in ((1, 1), (4, 1), (5, 4)):
        q = rnd(2, new, 2 * group, dim, seed=1, dtype=dtype)
        clean = fd.attend_kv_fp4(q, cache, n, table)
        sees = length - new + torch.arange(new, device=DEV) >= 0  # a query that sees no token has zeros
        all_nan, one_nan = q.clone(), q.clone()
        all_nan[0] = float("nan")
        y = fd.attend_kv_fp4(all_nan, cache, n, table)
        assert bool(torch.isnan(y[0, sees]).all()) and not y[0, ~sees].any() and torch.equal(y[1], clean[1])
        one_nan[1, :, group, 3] = float("nan")
        y = fd.attend_kv_fp4(one_nan, cache, n, table)
        assert bool(torch.isnan(y[1, sees, group]).all()) and not y[1, ~sees].any()
        rest = [h for h in range(2 * group) if h != group]
        assert torch.equal(y[0], clean[0]) and torch.equal(y[1][:, rest], clean[1][:, rest])


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("dim", [64, 128, 192])
@pytest.mark.parametrize("page,length", PLACES)
def test_a_key_of_no_numbers_is_every_later_querys(page, length, dim, dtype):
    """A NaN scale of one token's key, the first, a middle or the last one: NaN for each query that sees it, whatever else
    its wave, its share or its sequence holds; other heads' and sequences' results as they were."""
    import fused_decode as fd

    cache, table = cache_of(page, length, 2, dim)
    n = i32([length, length])
    raw = cache.k_scale.view(torch.uint8)
    for new, group in ((1, 1), (1, 4), (3, 2)):
        q = rnd(2, new, 2 * group, dim, seed=2, dtype=dtype)
        clean = fd.attend_kv_fp4(q, cache, n, table)
        for t in sorted({0, length // 2, length - 1}):
            page_id, slot = slot_of(table, page, 0, t)
            held = int(raw[page_id, 1, slot, 1])
            raw[page_id, 1, slot, 1] = 255
            y = fd.attend_kv_fp4(q, cache, n, table)
            raw[page_id, 1, slot, 1] = held
            bad = torch.zeros_like(y, dtype=torch.bool)
            bad[0, max(0, t - length + new) :, group:] = True  # query l sees tokens up to length - new + l
            assert bool(torch.isnan(y[bad]).all()) and torch.equal(y[~bad], clean[~bad]), (new, group, t)

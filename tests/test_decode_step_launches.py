"""How many launches the decode step in 4 bits says it issues: what its operators' scratch says they need."""

from __future__ import annotations

import pytest
import torch

from fused_decode.decode_step import DecodeStep


def step(m, context, dtype=torch.float16, h=4096, i=14336):
    ds = DecodeStep.__new__(DecodeStep)
    ds.m, ds.h, ds.i, ds.dtype, ds.context = m, h, i, dtype, context
    ds.fp4, ds.fp8, ds.fused, ds.rowsq, ds.kind = True, False, True, False, None
    ds.qkv_n, ds.qk_heads = h // 128 * 3 // 2 * 128, h // 128 * 5 // 4
    return ds


@pytest.mark.parametrize("m,context,dtype,want", [
    (1, 256, torch.float16, 9),     # one share of tokens, four products of one launch
    (1, 1024, torch.float16, 10),   # the shares are joined
    (4, 1024, torch.bfloat16, 10),
    (4, 256, torch.bfloat16, 9),
    (8, 1024, torch.float16, 12),   # the down projection in tiles: copied activations and K splits
    (16, 1024, torch.bfloat16, 11),  # K splits alone
])
def test_launches_of_a_layer(m, context, dtype, want):
    assert step(m, context, dtype).launches_per_layer == want

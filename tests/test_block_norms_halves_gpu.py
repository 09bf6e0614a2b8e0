"""norm_add_norm on halves of one buffer's rows: the values and nothing else."""

from __future__ import annotations

import pytest
import torch
from test_block_norms_gpu import DEV, check, rnd

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [8, 100, 1000, 4096, 33000, 3])
def test_halves_of_a_buffer(n, dtype):
    import fused_decode as fd

    w, pw = rnd(n, seed=3), rnd(n, seed=4)
    x, r, gate = (rnd(5, n, seed=s, dtype=dtype) for s in (1, 2, 5))
    wide = torch.full((5, 2 * n + 1), 7.0, dtype=dtype, device=DEV)
    left, right = wide[:, :n], wide[:, n : 2 * n]
    got = fd.norm_add_norm(x, r, pw, w, gate=gate, out=left, residual_out=right)
    assert got[0] is left and got[1] is right and bool((wide[:, -1] == 7.0).all())
    check(got, x, r, pw, w, 1e-6, gate)
    for a, b in ((x, r), (r, x)):  # each input beside the output that is not over it
        left.copy_(a), right.copy_(b)
        other = torch.empty_like(x)
        args = (left, r) if a is x else (x, left)
        fd.norm_add_norm(*args, pw, w, gate=gate, out=right, residual_out=other)
        check((right, other), x, r, pw, w, 1e-6, gate)
        assert torch.equal(left, a)

"""What stays of a capture that made the launch plans of the 8-bit operators: results, and no memory of its pool."""

from __future__ import annotations

import gc

import pytest
import torch
from test_w8a8_gpu import DEV, rnd

pytestmark = pytest.mark.gpu


def test_a_captured_plan_leaves_the_graphs_pool():
    import fused_decode as fd
    from fused_decode import ops

    x, w = rnd(90, 2048, seed=1, dtype=torch.bfloat16), rnd(2048, seed=2)
    q, qs = fd.quantize_fp8(rnd(600, 2048, seed=3))
    odd, odds = fd.quantize_fp8(rnd(70, 2047, seed=4))

    def run():
        c, s, h = fd.add_rms_norm_fp8(x, x, w)
        d, t = fd.quantize_rows_fp8(h[:, 1:])
        return fd.linear_w8a8(c, s, q, qs, activation="silu"), fd.linear_w8a8(d, t, odd, odds), fd.rms_norm_fp8(h, w)[1]

    pools = lambda: {tuple(s["segment_pool_id"]) for s in torch.cuda.memory_snapshot()}
    run()
    torch.cuda.synchronize()
    before = pools()
    ops.clear_plans()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    assert pools() > before
    for _ in range(3):
        graph.replay()
        want = run()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    del got, graph
    gc.collect()
    torch.cuda.empty_cache()
    assert pools() <= before
    assert all(torch.equal(a, b) for a, b in zip(run(), want))

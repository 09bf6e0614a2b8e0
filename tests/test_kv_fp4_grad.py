"""A cache whose scales ask for a gradient: its calls go to the custom ops, which say that they have none."""

from __future__ import annotations

import torch
from test_kv_fp4 import calls, cpu_cache  # noqa: F401 (a fixture)

from fused_decode import kv_fp4


def test_scales_that_ask_for_a_gradient(calls, monkeypatch):  # noqa: F811
    c, n = cpu_cache(), torch.tensor([3, 4], dtype=torch.int32)
    new, q = torch.zeros(2, 1, 2, 64).half(), torch.zeros(2, 1, 4, 64).half()
    seen = []

    class Stand:
        def __getattr__(self, name):
            return lambda *a: seen.append(name) or torch.zeros(2, 1, 4, 64).half()

    monkeypatch.setattr(torch.ops, "fused_decode", Stand(), raising=False)
    for name in ("k_scale", "v_scale"):
        leaf = c._replace(**{name: getattr(c, name).clone().requires_grad_()})
        seen.clear()
        kv_fp4.append_kv_fp4(leaf, new, new, n)
        kv_fp4.read_kv_fp4(leaf, n, 3)
        kv_fp4.attend_kv_fp4(q, leaf, n, scale=1.0)
        assert calls == [] and seen == ["append_kv_fp4", "read_kv_fp4", "attend_kv_fp4"]
    with torch.no_grad():
        kv_fp4.attend_kv_fp4(q, leaf, n, scale=1.0)
    assert len(calls) == 1

"""Plans of the attention over a cache in 8 bits, what of them no GPU is needed for."""
from __future__ import annotations

import torch

from test_cache8_host import metas

from pulse_infer_amd.ops import cache8


def test_a_plan_is_one_devices(monkeypatch):
    """A plan for "cuda" is for the device that is the current one when it is made, and says so (its lists lie there)."""
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 3)
    plan = cache8.AttentionPlan(metas([(0, 3)]), 1, 1, 32, page_size=16, dtype=torch.float32)      # (one that has no lists)
    assert plan.device == torch.device("cuda", 3)
    assert cache8.AttentionPlan(metas([(0, 3)]), 1, 1, 32, page_size=16, dtype=torch.float32, device="cuda:1").device.index == 1

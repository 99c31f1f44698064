"""Plans of the attention over a cache in 8 bits, what of them no GPU is needed for."""
from __future__ import annotations

import pytest
import torch

from test_cache8_host import metas

from pulse_infer_amd.cache import CacheManager, Paged8KVSpec, PagedKVSpec
from pulse_infer_amd.ops import KernelError, cache8


def test_a_plan_is_one_devices(monkeypatch):
    """A plan for "cuda" is for the device that is the current one when it is made, and says so (its lists lie there)."""
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 3)
    plan = cache8.AttentionPlan(metas([(0, 3)]), 1, 1, 32, page_size=16, dtype=torch.float32)      # (one that has no lists)
    assert plan.device == torch.device("cuda", 3)
    assert cache8.AttentionPlan(metas([(0, 3)]), 1, 1, 32, page_size=16, dtype=torch.float32, device="cuda:1").device.index == 1


@pytest.mark.parametrize("seed", range(300))
def test_rows_that_lie_apart(seed):
    """Against the bytes themselves, marked one by one."""
    import random

    r = random.Random(seed)
    buffer = torch.zeros(4000, dtype=torch.bfloat16)
    rows, a_columns, b_columns = r.randint(1, 6), r.randint(1, 40), r.randint(1, 40)
    a_step = a_columns + r.randint(0, 60)
    b_step = a_step if r.random() < 0.6 and a_step >= b_columns else b_columns + r.randint(0, 60)
    a = buffer.as_strided((rows, a_columns), (a_step, 1), r.randint(0, 300))
    b = buffer.as_strided((rows, b_columns), (b_step, 1), r.randint(0, 300))
    a.fill_(1.0)
    share = bool((b == 1.0).any())
    got = cache8._apart(rows, 2, a.data_ptr(), a_step, a_columns, b.data_ptr(), b_step, b_columns)
    if rows == 1 or a_step == b_step:
        assert got == (not share)
    else:                        # (rows of two steps that interleave are taken to overlap)
        assert not (got and share)


@pytest.mark.parametrize("n", [21844, 21846, 30000, 65533, 65534])
def test_many_requests_and_one_long(n):
    """Items that are too many for each to have two pieces more are cut into fewer, or not at all."""
    plan = cache8.AttentionPlan(metas([(100_000, 1)] + [(5, 1)] * n), 4, 2, 32, page_size=16, dtype=torch.bfloat16, device="cpu")
    (_, _, _, items, room, columns, _), (_, _, slots, *_) = plan.calls[0], plan.works[0]
    assert items == n + 1 <= room <= 65535 and (columns == 0) == (room == items)
    assert slots >= 1 and (room == items or room >= items + slots)


def test_windows_and_chunks_beyond_32_bits_hide_nothing():
    for given in (dict(window=2 ** 31), dict(chunk=2 ** 31), dict(window=2 ** 40), dict(chunk=10 ** 12)):
        plan = cache8.AttentionPlan(metas([(70, 1), (2 ** 31 - 3, 2)]), 2, 1, 32, page_size=16, dtype=torch.bfloat16, device="cpu", **given)
        assert (plan.window, plan.chunk) == (0, 0) and plan._tiles(70, 1) == 2
    plan = cache8.AttentionPlan(metas([(70, 1)]), 2, 1, 32, page_size=16, dtype=torch.bfloat16, device="cpu", window=2 ** 31 - 1)
    assert plan.window == 2 ** 31 - 1


@pytest.mark.parametrize("page", [1, 4, 8, 16, 24, 48, 64])
@pytest.mark.parametrize("heads", [1, 3, 8])
def test_bytes_of_the_storage(page, heads):
    """What the manager says of its pools is what their tensors take: of 8 bits with scales for every block, whatever the page."""
    manager = CacheManager([Paged8KVSpec(heads, 32), PagedKVSpec(2, 16), Paged8KVSpec(heads, 32)], page_size=page, num_pages=5, max_requests=2)
    manager.allocate_storage("cpu", torch.bfloat16)
    assert manager.storage_bytes(2) == sum(t.numel() * t.element_size() for g in manager.groups for t in g.spec.tensors(g.storage))


def test_portions_of_uneven_walks_are_cut_where_they_fill_the_gpu(monkeypatch):
    """A slot each by themselves: two pieces an item where one walk is far longer than a slot's share of all, else whole; of 256 channels, of which a
    compute unit holds one workgroup, no more pieces than items."""
    monkeypatch.setattr(cache8, "compute_units", lambda: 256)

    def room(entries, d=128):
        plan = cache8.AttentionPlan(metas(entries), 32, 8, d, page_size=16, dtype=torch.bfloat16, device="cpu")
        (name, _, _, items, pieces, _, _), = plan.calls
        assert name == "pulse_attn8_many" and items * 8 >= 512
        return pieces / items

    assert room([(8000, 300), (0, 2000)]) == room([(6000, 600), (0, 2000)]) == 3      # (the items and twice as many)
    assert room([(0, 2048)]) == room([(0, 2600)]) == room([(0, 1044), (0, 1668)]) == room([(8000, 2048)]) == 1
    assert room([(8000, 300), (0, 2000)], d=256) == 2


@pytest.mark.parametrize("send", [lambda v: torch.tensor(v), lambda v: torch.tensor(v, dtype=torch.int32)[:-1], lambda v: torch.tensor(v + v, dtype=torch.int32)[::2],
                                  lambda v: torch.tensor(v, dtype=torch.int32, device="meta")])
def test_lists_that_are_not_what_the_kernels_read_are_refused(send):
    with pytest.raises(KernelError, match="to_device"):
        cache8.AttentionPlan(metas([(40, 1), (0, 3)]), 4, 2, 32, page_size=16, dtype=torch.bfloat16, device="cpu", to_device=send)

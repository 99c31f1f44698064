"""What a step's kernels are told about its rows and pages: the same integers whether host or device puts them together."""
from __future__ import annotations

import random
from types import SimpleNamespace

import pytest
import torch

from conftest import require_gpu

pytestmark = pytest.mark.gpu


def runner_over(specs, page_size, num_pages, max_requests=64):
    """The step function's host side over a cache without storage."""
    from pulse_infer_amd.cache import CacheManager
    from pulse_infer_amd.engine.runner import ModelRunner, _Staging

    runner = ModelRunner.__new__(ModelRunner)
    runner.device = torch.device("cuda:0")
    runner.cache = CacheManager(specs, page_size, num_pages, max_requests)
    runner._staging = _Staging(runner.device)
    runner.model = SimpleNamespace(workspace=None, vocab_size=1000)
    runner.max_positions = 10 ** 9
    return runner


def contexts(runner, entries, feed=None):
    """The step's context made on the host and on the device."""
    from pulse_infer_amd.parts.base import contexts_uneven

    metas = runner._check(entries)
    want = [m.first_row + int(w) for e, m in zip(entries, metas) for w in e.want]
    out = []
    for runner.MAPS_FROM in (10 ** 9, 1):
        out.append(runner._context_of_step(entries, metas, want, max(m.start + m.count for m in metas), contexts_uneven(metas), feed))
    del runner.MAPS_FROM
    return metas, out


def same(runner, entries, feed=None):
    metas, (host, dev) = contexts(runner, entries, feed)
    for name in ("token_ids", "positions", "token_entry", "entry_start", "entry_count", "entry_first_row", "entry_slot", "want_rows", "live_context"):
        a, b = getattr(host, name), getattr(dev, name)
        assert a.dtype == b.dtype == torch.int32 and a.tolist() == b.tolist(), name
    for name in ("num_tokens", "num_wanted", "max_count", "max_context", "uneven", "entries"):
        assert getattr(host, name) == getattr(dev, name), name
    assert set(host.block_tables) == set(dev.block_tables) == set(range(len(runner.cache.groups)))
    for gi, g in enumerate(runner.cache.groups):
        a, b = host.block_tables[gi].tolist(), dev.block_tables[gi].tolist()
        assert [len(r) for r in a] == [len(r) for r in b]
        for m, x, y in zip(metas, a, b):      # (behind the tokens that it has the host lists pages that are reserved already)
            n = g.pages_for(m.start + m.count)
            assert x[:n] == y[:n] and set(y[n:]) <= {-1}, (gi, m)
    for m in metas:
        runner.cache.advance(m.request, m.start + m.count)


def test_pools_of_more_slots_than_32_bits_number():
    require_gpu()
    from pulse_infer_amd.cache import PagedKVSpec
    from pulse_infer_amd.engine.runner import StepEntry

    runner = runner_over([PagedKVSpec(2, 32)], 1 << 20, 1 << 11)
    for r in range(9):
        runner.add_request(r)
        runner.reserve(r, 40)
    same(runner, [StepEntry(r, [r + 1] * (r + 1), [0]) for r in range(9)])

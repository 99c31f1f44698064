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


@pytest.mark.parametrize("seed", range(6))
def test_host_and_device_agree(seed):
    """Groups with and without windows and chunks, pages that were given back, portions of uneven lengths, pages reserved ahead, ids that
    come from the device."""
    require_gpu()
    from pulse_infer_amd.cache import Paged8KVSpec, PagedKVSpec
    from pulse_infer_amd.engine.runner import StepEntry

    r = random.Random(seed)
    page = r.choice([1, 4, 16, 24])
    specs = [PagedKVSpec(2, 32), PagedKVSpec(2, 32, window=r.randint(1, 40)), PagedKVSpec(1, 64, chunk=r.randint(2, 50)), PagedKVSpec(2, 32),
             Paged8KVSpec(2, 32, window=r.randint(1, 40))]
    runner = runner_over(specs, page, 12_000)
    live, gone = [], False
    for step in range(12):
        for _ in range(r.randint(0, 6) if step else 9):
            live.append((seed, step, len(live)))
            runner.add_request(live[-1])
        if step > 4 and len(live) > 9:
            runner.free_request(live.pop(r.randrange(len(live))))
        entries = []
        for name in r.sample(live, r.randint(1, len(live))):
            n = r.choice([1, 1, 1, r.randint(1, 100)])
            runner.reserve(name, runner.cache.computed(name) + n + r.choice([0, 0, 70]))
            entries.append(StepEntry(name, [r.randrange(1000) for _ in range(n)], sorted(r.sample(range(n), r.randint(0, min(n, 3))))))
        total = sum(len(e.tokens) for e in entries)
        feed = None
        if step % 3 == 1:
            places = r.sample(range(total), r.randint(1, total))
            source = torch.tensor([r.randrange(1000) for _ in range(total + 2)], dtype=torch.int32, device="cuda:0")
            feed = (source, places, [r.randrange(total + 2) for _ in places])
        same(runner, entries, feed)
        gone = gone or any(-1 in t for g in runner.cache.groups for t in g.tables.values())
    assert gone and len(runner.cache.groups) == 4


def test_a_model_that_pages_nothing():
    require_gpu()
    from pulse_infer_amd.cache import StateSpec
    from pulse_infer_amd.engine.runner import StepEntry

    runner = runner_over([StateSpec((4, 4), "float32"), None], 16, 8)
    for r in range(10):
        runner.add_request(r)
        runner.reserve(r, 50)
    same(runner, [StepEntry(r, list(range(1, 2 + 3 * r)), [0] if r % 2 else []) for r in (9, 0, 3, 4, 5, 6, 7, 8, 1)])
    same(runner, [StepEntry(r, [5], [0]) for r in range(10)])

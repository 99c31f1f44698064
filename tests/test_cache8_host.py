"""A cache of keys and values in 8 bits, what of it is host code: the spec, the plan's items, and the refusals that no GPU is needed for."""
from __future__ import annotations

import pytest
import torch

from plain import cache8_plain as plain

from pulse_infer_amd.cache.manager import CacheManager
from pulse_infer_amd.cache.specs import Paged8CacheView, Paged8KVSpec, PagedKVSpec, block_tokens
from pulse_infer_amd.ops import KernelError, cache8
from pulse_infer_amd.parts.base import EntryMeta


def metas(entries):
    out, row = [], 0
    for i, (s, c) in enumerate(entries):
        out.append(EntryMeta(i, i, s, c, row))
        row += c
    return out


def test_spec_and_manager():
    """Shapes, bytes, pages given back below a window; runs of equal specs share a pool, others have their own."""
    spec = Paged8KVSpec(2, 32, window=20)
    manager = CacheManager([spec, PagedKVSpec(2, 32, window=20), spec, Paged8KVSpec(2, 32)], page_size=16, num_pages=8, max_requests=2)
    assert [len(g.runs) for g in manager.groups] == [2, 1, 1]
    manager.allocate_storage("cpu", torch.bfloat16)
    view = manager.view(2, writable=False)
    assert type(view) is Paged8CacheView and not view.writable and view.group == 0
    assert view.keys.shape == (8, 2, 16, 32) and view.values.shape == (8, 2, 1, 32, 16) and view.scales.shape == (8, 2, 1, 2)
    assert view.keys.dtype == view.values.dtype == torch.float8_e4m3fn and view.scales.dtype == torch.float32
    assert spec.bytes_per_token(2) == spec.bytes_per_token(4) == 2 * 2 * 32 + 1
    manager.add_request("r")
    manager.reserve("r", 100)
    manager.advance("r", 90)
    assert manager.table(0, "r")[:4] == [-1] * 4 and manager.table(0, "r")[4] >= 0 and -1 not in manager.table(2, "r")
    manager.free_request("r")
    manager.check()


@pytest.mark.parametrize("page,block", [(1, 1), (8, 8), (16, 16), (24, 24), (32, 16), (48, 16), (256, 16)])
def test_blocks(page, block):
    assert block_tokens(page) == block
    entries = [(0, 1), (page - 1, 2), (3 * page + 1, 5 * page), (7, 0)]
    want = plain.maps([e for e in entries if e[1]], list(range(40)), page, 100, 12)
    assert cache8.blocks_touched(metas(entries), page) == len(want["blocks"])


@pytest.mark.parametrize("nq,nkv", [(1, 1), (8, 2), (6, 2), (7, 1), (32, 1), (40, 2), (130, 1)])
def test_items_cover_every_row_once(nq, nkv):
    entries = metas([(0, 1), (50, 1), (3, 5), (0, 700), (9, 33), (4, 0)])
    sent = []
    plan = cache8.AttentionPlan(entries, nq, nkv, 64, page_size=16, dtype=torch.bfloat16, device="cpu",
                                to_device=lambda flat: sent.append(flat) or torch.tensor(flat, dtype=torch.int32))
    rows = sorted((row + i, entry) for flat in sent for row, n, entry in zip(flat[0::4], flat[1::4], flat[2::4]) for i in range(n))
    assert rows == [(e.first_row + i, e.request) for e in entries for i in range(e.count)]
    group = nq // nkv
    for (name, *_), flat in zip(plan.calls, sent):
        most = 16 if name == "pulse_attn8_few" else 128
        assert all(n * min(group, most) <= max(most, group if name == "pulse_attn8_few" else 0) for n in flat[1::4])
    assert plan.rows == sum(e.count for e in entries)


def test_the_nearest_byte():
    """The plain form's rounding against torch's conversion, and its exponents against their definition."""
    x = torch.linspace(-448, 448, 20001, dtype=torch.float64)
    x = torch.cat([x, x * 2.0 ** -12, torch.tensor([0.0, 2.0 ** -10, 3 * 2.0 ** -10, 17.0, 19.0, 232.0], dtype=torch.float64)])
    assert torch.equal(plain.nearest(x), x.float().to(torch.float8_e4m3fn).double())
    for a in (448.0, 448.0000001, 1.0, 1.75, 1.7500001, 3e38, 1e-44, 0.0, 0.875):
        e = float(plain.exponent(torch.tensor(a, dtype=torch.float64)))
        assert e == plain.LEAST or (a <= 448 * 2.0 ** e and a > 448 * 2.0 ** (e - 1))
    b = torch.arange(256, dtype=torch.uint8)
    assert torch.equal(torch.nan_to_num(plain.decode(b), nan=1e9), torch.nan_to_num(b.view(torch.float8_e4m3fn).double(), nan=1e9))


def test_refusals_without_a_gpu():
    spec = Paged8KVSpec(1, 32)
    view = spec.view(spec.allocate(1, 2, 16, "cpu", torch.bfloat16), 0, 0, 16, True)
    ints = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    qkv, pos = torch.zeros((3, 96)), ints([0, 1, 2])
    with pytest.raises(KernelError, match="GPU"):
        cache8.store(qkv, qkv, 1, 1, 32, view, pos, ints([[0, 3, 0, 0]]))
    with pytest.raises(KernelError, match="GPU"):
        cache8.step_maps(ints([0]), ints([3]), page_size=16, num_pages=2, pages=ints([0]), slots=pos.clone())
    plan = cache8.AttentionPlan(metas([(0, 3)]), 1, 1, 32, page_size=16, dtype=torch.bfloat16, device="cpu")
    with pytest.raises(KernelError, match="GPU"):
        plan.cut(pos)
    with pytest.raises(KernelError, match="GPU"):
        cache8.attention(qkv, qkv, plan, view, pos, pos, ints([[0]]), 1.0)
    for bad in (dict(nq=4, nkv=3), dict(d=0), dict(d=513), dict(window=-1), dict(window=2, chunk=2), dict(dtype=torch.float16)):
        args = dict(nq=4, nkv=2, d=32, window=0, chunk=0, dtype=torch.bfloat16, **{}) | bad
        with pytest.raises(KernelError):
            cache8.AttentionPlan(metas([(0, 3)]), args.pop("nq"), args.pop("nkv"), args.pop("d"), page_size=16, device="cpu", **args)
    with pytest.raises(KernelError, match="too many"):
        cache8.AttentionPlan(metas([(0, 1)] * 70000), 4, 2, 32, page_size=16, dtype=torch.bfloat16, device="cpu")


@pytest.mark.parametrize("entries", [[(0, 3, 1)], [(0, 3, 0), (5, 2, 2)], [(0, 3, 0), (5, 2, 4)], [(-1, 2, 0)], [(0, 2, 0), (0, -1, 2)]])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_that_do_not_follow_each_other_are_refused(entries, dtype):
    step = [EntryMeta(i, i, start, count, row) for i, (start, count, row) in enumerate(entries)]
    with pytest.raises(KernelError, match="expected the next"):
        cache8.AttentionPlan(step, 4, 2, 32, page_size=16, dtype=dtype, device="cpu")


def test_options():
    from pulse_infer_amd.cli import build_parser
    from pulse_infer_amd.models.causal_lm import CausalLM

    assert build_parser().parse_args(["m", "--cache-dtype", "float8_e4m3"]).cache_dtype == "float8_e4m3"
    assert build_parser().parse_args(["m"]).cache_dtype == "auto"

    class Spec:
        def validate(self):
            pass

    with pytest.raises(ValueError, match="unknown cache dtype"):
        CausalLM(Spec(), None, device="cpu", options={"cache_dtype": "int4"})

"""A cache of keys and values in 8 bits: maps, store and attention against plain float64, at the sizes and masks where they can go wrong.

Tolerances, fixed before the first run: integers, bytes of rows that are stored as they come, and scales are equal; what goes through
norm or rotation first is the e4m3 number nearest to a value that float32 arithmetic has to 1e-5 of the row's largest.  Attention in
bfloat16: the weights are rounded once (2^-8 of sum w|v|), the result once (2^-8 of itself), the rest is float32 (1e-5 of sum w|v|, and
2^-22 of the row's sum |q||k| for its scores).  In float32: 2^-24 times (channels + 2) times sum |q||k| for a score, twice that
relative to sum w|v|, and 1e-6 of it for exponentials and sums."""
from __future__ import annotations

import math

import pytest
import torch

from conftest import require_gpu
from plain import cache8_plain as plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F64 = torch.float64


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def view_of(cache):
    from pulse_infer_amd.cache.specs import Paged8CacheView

    keys, values, scales = (t.to(DEV) for t in cache.tensors())
    return Paged8CacheView(0, keys, values, scales, cache.page)


def metas(entries):
    from pulse_infer_amd.parts.base import EntryMeta

    out, row = [], 0
    for i, (s, c) in enumerate(entries):
        out.append(EntryMeta(i, i, s, c, row))
        row += c
    return out


def layout(entries, page, seed, spare=3):
    """(list of all requests' pages, pages of the pool, table rows)"""
    held = [-(-(s + c) // page) for s, c in entries]
    pool = sum(held) + spare
    order = torch.randperm(pool, generator=torch.Generator().manual_seed(seed)).tolist()
    pages, rows = order[:sum(held)], []
    for h in held:
        at = sum(len(r) for r in rows)
        rows.append(pages[at:at + h])
    return pages, pool, rows


# ---------------------------------------------------------------------------------------------------------------- maps
MAPS = [
    ([(0, 1)], 16, 0), ([(4095, 1)], 16, 0), ([(0, 17), (15, 1), (16, 1), (31, 40)], 16, 2), ([(5, 0), (0, 3), (7, 0), (9, 2)], 4, 0),
    ([(i * 13, 1 + i % 5) for i in range(300)], 32, 1), ([(0, 1)] * 700, 16, 0), ([(1000, 777), (3, 5)], 24, 0), ([(100, 30)], 64, -1),
]


@pytest.mark.parametrize("entries,page,extra", MAPS)
def test_maps(entries, page, extra):
    require_gpu()
    from pulse_infer_amd.ops import cache8

    pages, pool, rows = layout(entries, page, 3)
    width = max(1, max(len(r) for r in rows) + extra)
    want = plain.maps(entries, pages, page, pool, width)
    total, n = sum(c for _, c in entries), len(want["blocks"])
    assert n == cache8.blocks_touched(metas(entries), page)
    got = dict(first_row=ints([-9] * (len(entries) + 1)), positions=ints([-9] * (total + 5)), token_entry=ints([-9] * (total + 5)),
               slots=ints([-9] * (total + 5)), table=torch.full((len(entries), width), -9, dtype=torch.int32, device=DEV),
               blocks=torch.full((n + 2, 4), -9, dtype=torch.int32, device=DEV))
    start, count = ints([s for s, _ in entries]), ints([c for _, c in entries])
    cache8.step_maps(start, count, page_size=page, num_pages=pool, pages=ints(pages), **got)
    for name in ("positions", "token_entry", "slots"):
        assert got[name].tolist() == want[name] + [-9] * 5, name       # (rows behind the last request's stay as they were)
    assert got["first_row"].tolist() == want["first_row"] and got["table"].tolist() == want["table"]
    assert got["blocks"].tolist() == want["blocks"] + [[0, 0, -1, 0]] * 2
    if extra >= 0:      # the same from the table
        slots, blocks = ints([-9] * total), torch.zeros((n, 4), dtype=torch.int32, device=DEV)
        cache8.step_maps(start, count, page_size=page, num_pages=pool, table=got["table"], slots=slots, blocks=blocks)
        assert slots.tolist() == want["slots"] and blocks.tolist() == want["blocks"]


def test_maps_of_pages_that_are_none():
    """Pages outside the pool and pages that the list does not have give no slot and no block."""
    require_gpu()
    from pulse_infer_amd.ops import cache8

    entries, pages = [(30, 10), (0, 20)], [5, -1, 99, 2]      # the second request's second page is missing
    want = plain.maps(entries, pages, 16, 8, 3)
    slots, blocks, table = ints([0] * 30), torch.zeros((len(want["blocks"]), 4), dtype=torch.int32, device=DEV), ints([[0] * 3] * 2)
    cache8.step_maps(ints([30, 0]), ints([10, 20]), page_size=16, num_pages=8, pages=ints(pages), table=table, slots=slots, blocks=blocks)
    assert slots.tolist() == want["slots"] and blocks.tolist() == want["blocks"] and table.tolist() == want["table"]
    assert -1 in want["slots"]


def test_maps_of_lengths_whose_pages_leave_32_bits():
    """Four requests of 2^30 + 1 pages of one token each, and a list of three pages: all but the first two of the first's are none."""
    require_gpu()
    from pulse_infer_amd.ops import cache8

    slots, blocks, table = ints([5] * 4), torch.zeros((4, 4), dtype=torch.int32, device=DEV), ints([[7, 7]] * 4)
    cache8.step_maps(ints([1 << 30] * 4), ints([1] * 4), page_size=1, num_pages=4, pages=ints([3, 1, 2]), table=table, slots=slots, blocks=blocks)
    assert slots.tolist() == [-1] * 4 and blocks.tolist() == [[i, 1, -1, 0] for i in range(4)]
    assert table.tolist() == [[3, 1], [-1, -1], [-1, -1], [-1, -1]]


# --------------------------------------------------------------------------------------------------------------- store
STORE = [   # nq, nkv, d, page, dtype, norm, rotary, pairing, entries
    (4, 2, 128, 16, torch.bfloat16, True, 128, 1, [(0, 40), (15, 1), (16, 1), (33, 20)]),
    (4, 2, 128, 16, torch.bfloat16, False, 0, 0, [(0, 16), (7, 9), (5, 3), (0, 1)]),
    (6, 1, 32, 16, torch.float32, True, 32, 0, [(0, 70), (9, 1), (3, 33)]),
    (3, 3, 48, 8, torch.bfloat16, True, 16, 1, [(0, 21), (6, 1), (7, 1)]),
    (2, 1, 10, 4, torch.float32, False, 6, 0, [(0, 9), (2, 1)]),
    (2, 2, 256, 32, torch.bfloat16, "plain", 64, 1, [(0, 50), (31, 2)]),
    (1, 1, 512, 16, torch.float32, True, 512, 1, [(3, 20)]),
    (4, 4, 64, 24, torch.bfloat16, False, 64, 0, [(0, 30), (23, 1)]),
    (4, 2, 20, 16, torch.bfloat16, True, 12, 1, [(0, 18), (4, 1)]),
]


@pytest.mark.parametrize("nq,nkv,d,page,dtype,norm,rotary,pairing,entries", STORE)
@pytest.mark.parametrize("in_place", [False, True])
def test_store(nq, nkv, d, page, dtype, norm, rotary, pairing, entries, in_place):
    require_gpu()
    from pulse_infer_amd.ops import cache8

    g = torch.Generator().manual_seed(nq * d + page)
    pages, pool, _ = layout(entries, page, 5)
    want = plain.maps(entries, pages, page, pool, 1)
    total = sum(c for _, c in entries)
    cache = plain.Cache(pool, nkv, page, d)
    old = torch.randn((pool * page, nkv, d), generator=g, dtype=F64) * 0.3       # what earlier steps left, at smaller scales
    cache.store(old, old * 5, [[i * cache.block, cache.block, i, 0] for i in range(pool * cache.nb)])
    view = view_of(cache)
    qkv = (torch.randn((total, (nq + 2 * nkv) * d + 8), generator=g) * 2).to(dtype).to(DEV)[:, :(nq + 2 * nkv) * d]
    w = [(1 + 0.2 * torch.rand(d, generator=g)).to(dtype).to(DEV) for _ in range(2)] if norm is True else [None, None]
    angles = torch.tensor(want["positions"], dtype=F64)[:, None] * 10.0 ** -(torch.arange(rotary // 2, dtype=F64) / 9) if rotary else None
    cos, sin = (torch.cos(angles).float().to(DEV), torch.sin(angles).float().to(DEV)) if rotary else (None, None)
    temperature = (0.1, 7) if norm == "plain" else None
    q, k, v = plain.prepared(qkv, nq, nkv, d, None, w[0], w[1], 1e-6, norm == "plain", angles, rotary, pairing, temperature,
                             torch.tensor(want["positions"]))
    cache.store(k, v, want["blocks"])
    q_out = qkv if in_place else torch.zeros((total, nq * d), dtype=dtype, device=DEV)
    cache8.store(qkv, q_out, nq, nkv, d, view, ints(want["positions"]), ints(want["blocks"]), q_weight=w[0], k_weight=w[1], eps=1e-6, cos=cos,
                 sin=sin, rotary_dim=rotary, pairing=pairing, plain_norm=norm == "plain", q_temperature=temperature)
    got_q = q_out[:, :nq * d].cpu().to(F64).view(total, nq, d)
    size = q.abs().amax(-1, keepdim=True)
    assert ((got_q - q).abs() <= torch.finfo(dtype).eps / 2 * q.abs() + 1e-5 * size).all()
    keys, values, scales = cache.tensors()
    assert torch.equal(view.scales.cpu(), scales)
    assert torch.equal(view.values.cpu().view(torch.uint8), values.view(torch.uint8))
    if not norm and not rotary:
        assert torch.equal(view.keys.cpu().view(torch.uint8), keys.view(torch.uint8))
    else:
        a, b = plain.decode(view.keys), plain.decode(keys)
        # (a value within 1e-5 of a border may fall to the neighbour: a step of 2^-3 of it, of 2^-9 below 2^-6)
        assert ((a - b).abs() <= torch.maximum(b.abs() * 2.0 ** -3, torch.tensor(2.0 ** -9, dtype=F64))).all()
        assert (a != b).double().mean() < 1e-3


@pytest.mark.parametrize("nq,nkv,d,page,norm,rotary,pairing,shares,entries", [
    (4, 2, 128, 16, True, 128, 1, 4, [(0, 40), (15, 1), (16, 1), (33, 20)]), (4, 1, 64, 32, False, 0, 0, 1, [(0, 16), (7, 9)]),
    (2, 2, 256, 48, "plain", 64, 1, 7, [(0, 50), (31, 2)]), (1, 1, 512, 16, True, 512, 0, 2, [(3, 20)]), (3, 3, 40, 16, False, 16, 1, 9, [(0, 33)])])
def test_store_of_rows_in_shares(nq, nkv, d, page, norm, rotary, pairing, shares, entries):
    """Shares that are multiples of 2^-10 below 8: their sums are exact, and what is stored is what the plain form stores of the sums."""
    require_gpu()
    from pulse_infer_amd.ops import cache8

    g = torch.Generator().manual_seed(shares)
    pages, pool, _ = layout(entries, page, 6)
    want = plain.maps(entries, pages, page, pool, 1)
    total, columns = sum(c for _, c in entries), (nq + 2 * nkv) * d
    cache = plain.Cache(pool, nkv, page, d)
    old = torch.randn((pool * page, nkv, d), generator=g, dtype=F64) * 0.3
    cache.store(old, old * 5, [[i * cache.block, cache.block, i, 0] for i in range(pool * cache.nb)])
    view = view_of(cache)
    parts = torch.round(torch.randn((shares, total, columns + 4), generator=g).clamp(-7, 7) * 1024) / 1024
    w = [(1 + 0.2 * torch.rand(d, generator=g)).to(torch.bfloat16).to(DEV) for _ in range(2)] if norm is True else [None, None]
    angles = torch.tensor(want["positions"], dtype=F64)[:, None] * 10.0 ** -(torch.arange(rotary // 2, dtype=F64) / 9) if rotary else None
    cos, sin = (torch.cos(angles).float().to(DEV), torch.sin(angles).float().to(DEV)) if rotary else (None, None)
    q, k, v = plain.prepared(parts.to(F64).sum(0)[:, :columns], nq, nkv, d, None, w[0], w[1], 1e-6, norm == "plain", angles, rotary, pairing, None,
                             torch.tensor(want["positions"]))
    cache.store(k, v, want["blocks"])
    qkv = torch.full((total, columns), math.nan, dtype=torch.bfloat16, device=DEV)
    cache8.store(qkv, qkv, nq, nkv, d, view, ints(want["positions"]), ints(want["blocks"]), q_weight=w[0], k_weight=w[1], eps=1e-6, cos=cos, sin=sin,
                 rotary_dim=rotary, pairing=pairing, plain_norm=norm == "plain", parts=parts.to(DEV))
    got_q = qkv[:, :nq * d].cpu().to(F64).view(total, nq, d)
    assert ((got_q - q).abs() <= 2.0 ** -8 * q.abs() + 1e-5 * q.abs().amax(-1, keepdim=True)).all() and torch.isnan(qkv[:, nq * d:]).all()
    keys, values, scales = cache.tensors()
    assert torch.equal(view.scales.cpu(), scales) and torch.equal(view.values.cpu().view(torch.uint8), values.view(torch.uint8))
    a, b = plain.decode(view.keys), plain.decode(keys)
    assert ((a - b).abs() <= torch.maximum(b.abs() * 2.0 ** -3, torch.tensor(2.0 ** -9, dtype=F64))).all()
    assert (a != b).double().mean() < 1e-3 and (norm or rotary or torch.equal(a, b))


def test_store_token_by_token_grows_its_scale():
    """One token after the other, each larger than those before: what the block holds is what the plain form's appends give, byte by
    byte, and within one rounding of the token at the final scale."""
    require_gpu()
    from pulse_infer_amd.ops import cache8

    nkv, d = 2, 64
    cache = plain.Cache(3, nkv, 16, d)
    view = view_of(cache)
    g = torch.Generator().manual_seed(1)
    rows = torch.randn((16, 3 * nkv * d), generator=g).to(torch.bfloat16) * (2.0 ** torch.arange(-6, 10))[:, None].to(torch.bfloat16)
    dev = rows.to(DEV)
    for t in range(16):
        block = [[0, 1, 1, t]]
        _, k, v = plain.prepared(rows[t:t + 1], nkv, nkv, d)
        cache.store(k, v, block)
        cache8.store(dev[t:t + 1], torch.empty((1, nkv * d), dtype=torch.bfloat16, device=DEV), nkv, nkv, d, view, ints([t]), ints(block))
    keys, values, scales = cache.tensors()
    assert torch.equal(view.keys.cpu().view(torch.uint8), keys.view(torch.uint8))
    assert torch.equal(view.values.cpu().view(torch.uint8), values.view(torch.uint8)) and torch.equal(view.scales.cpu(), scales)
    _, k, _ = plain.prepared(rows, nkv, nkv, d)
    got = plain.decode(view.keys[1]) * view.scales[1, :, 0, 0].cpu().to(F64)[:, None, None]
    exact, s = k.transpose(0, 1), view.scales[1, :, 0, 0].cpu().to(F64)[:, None, None]
    # an append rounds again only what falls below the smallest normal number: at most half a step of 2^-9 s for each of fifteen
    assert ((got - exact).abs() <= 2.0 ** -4 * exact.abs() + 15 * 2.0 ** -10 * s).all()


def test_store_of_what_is_not_finite():
    require_gpu()
    from pulse_infer_amd.ops import cache8

    nkv, d = 1, 32
    cache = plain.Cache(2, nkv, 16, d)
    view = view_of(cache)
    x = torch.randn((20, 3 * d), generator=torch.Generator().manual_seed(2))
    x[3, d + 4], x[5, d + 1], x[7, 2 * d + 9], x[8, 2 * d] = math.inf, math.nan, -math.inf, math.nan
    x[9, 2 * d + 1] = 3e38
    blocks = [[0, 16, 1, 0], [16, 4, 0, 0]]
    _, k, v = plain.prepared(x, 1, nkv, d)
    cache.store(k, v, blocks)
    cache8.store(x.to(DEV), torch.empty((20, d), device=DEV), 1, nkv, d, view, ints(list(range(20))), ints(blocks))
    got_k, got_v = plain.decode(view.keys), plain.decode(view.values).transpose(3, 4)
    assert torch.equal(torch.isnan(got_k).view(-1), torch.isnan(cache.x[0]).view(-1)) and torch.isnan(got_k).sum() == 2
    assert torch.equal(torch.nan_to_num(got_v), torch.nan_to_num(cache.x[1])) and torch.isnan(got_v).sum() == 2
    assert torch.equal(view.scales.cpu(), cache.tensors()[2]) and view.scales[1, 0, 0, 1] < 0 < view.scales[0, 0, 0, 1]
    # a block that is begun anew holds nothing of what was there
    cache8.store(x[10:12].to(DEV), torch.empty((2, d), device=DEV), 1, nkv, d, view, ints([0, 1]), ints([[0, 2, 1, 0]]))
    assert view.scales[1, 0, 0, 1] > 0 and not torch.isnan(plain.decode(view.values)).any()
    assert (view.keys[1, 0, 2:].view(torch.uint8) == 0).all()


def test_store_leaves_other_blocks_alone():
    """Places of the list without rows, blocks of no page, blocks that the pool does not have."""
    require_gpu()
    from pulse_infer_amd.ops import cache8

    cache = plain.Cache(2, 1, 16, 32)
    old = torch.randn((32, 1, 32), generator=torch.Generator().manual_seed(3), dtype=F64)
    cache.store(old, old, [[0, 16, 0, 0], [16, 16, 1, 0]])
    view = view_of(cache)
    before = [t.clone() for t in (view.keys.view(torch.uint8), view.values.view(torch.uint8), view.scales)]
    x = torch.randn((4, 96), device=DEV)
    cache8.store(x, torch.empty((4, 32), device=DEV), 1, 1, 32, view, ints([0] * 4), ints([[0, 4, -1, 0], [0, 0, 1, 0], [0, 4, 2, 0], [0, 4, 1, 13], [2, 3, 1, 0],
                                                                                             [2 ** 31 - 2, 4, 1, 0], [0, 4, 1, 2 ** 31 - 2], [0, 2 ** 31 - 1, 1, 1]]))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(before, (view.keys.view(torch.uint8), view.values.view(torch.uint8), view.scales)))


# ----------------------------------------------------------------------------------------------------------- attention
def bound_of(dtype, d, want, mass, size):
    if dtype == torch.float32:
        return (2 * 2.0 ** -24 * (d + 2) * size + 1e-6) * mass + 2.0 ** -24 * want.abs()
    return 2.0 ** -8 * (mass + want.abs()) + (1e-5 + 2.0 ** -22 * size) * mass


def attend(entries, nq, nkv, d, page, dtype=torch.bfloat16, seed=0, window=0, chunk=0, softcap=0.0, sink=False, gate=None, none=(), pad=0,
           spoil=None, extra_rows=0, unwritten=None):
    """Kernel and plain on one random cache; asserts the bound and returns (got, want)."""
    require_gpu()
    from pulse_infer_amd.ops import cache8
    from pulse_infer_amd.parts.base import Workspace

    g = torch.Generator().manual_seed(seed + d + nq)
    pages, pool, rows = layout(entries, page, seed)
    if unwritten is not None:      # nobody has the first page, nor the last ones
        pool, rows = pool + 1, [[p + 1 for p in r] for r in rows]
    total = sum(c for _, c in entries)
    cache = plain.Cache(pool, nkv, page, d)
    k, v = (torch.randn((pool * page, nkv, d), generator=g, dtype=F64) * torch.exp(torch.randn((1, nkv, d), generator=g, dtype=F64) * 0.4) for _ in range(2))
    if spoil is not None:
        spoil(k, v, rows, page)
    cache.store(k, v, [[i * cache.block, cache.block, i, 0] for i in range(pool * cache.nb)])
    view = view_of(cache)
    if unwritten is not None:
        free = sorted(set(range(pool)) - {p for r in rows for p in r})
        view.scales[free] = unwritten
        view.keys.view(torch.uint8)[free] = view.values.view(torch.uint8)[free] = 0x7f
    width = max(len(r) for r in rows) + 1
    table = [r + [-1] * (width - len(r)) for r in rows]
    for b, j in none:
        table[b][j] = -1 if j % 2 else pool
    q = torch.randn((total + extra_rows, nq * d + pad), generator=g).to(dtype).to(DEV)[:, :nq * d]
    out = torch.full((total + extra_rows, nq * d + pad), 7.0, dtype=dtype, device=DEV)[:, :nq * d]
    sinks = torch.randn(nq, generator=g).to(DEV) if sink else None
    width_g = 0 if gate is None else gate
    gates = torch.randn((total + extra_rows, nq * max(1, width_g) + 3), generator=g).to(dtype).to(DEV) if gate is not None else None
    m = metas(entries)
    positions = ints([p for s, c in entries for p in range(s, s + c)] + [0] * extra_rows)
    token_entry = ints([b for b, (_, c) in enumerate(entries) for _ in range(c)] + [-1] * extra_rows)
    scale = 1.3 * d ** -0.5
    ws = Workspace(torch.device(DEV))
    # as the plan has it, and every portion that can be in items of 128 columns, joined by a launch and by their last pieces
    was, outs = (cache8.AttentionPlan.FEW_WALKS, cache8.AttentionPlan.MANY_HERE), []
    try:
        for cache8.AttentionPlan.FEW_WALKS, cache8.AttentionPlan.MANY_HERE in (was, (0, 0), (0, 10 ** 6)):
            out.fill_(7.0)
            made = cache8.plan(m, nq, nkv, d, positions, page_size=page, dtype=dtype, window=window, chunk=chunk, workspace=ws)
            cache8.attention(q, out, made, view, positions, token_entry, ints(table), scale, gate=gates, gate_width=width_g, sink=sinks,
                             softcap=softcap)
            outs.append(out[:total].cpu().to(F64).reshape(total, nq, d))
            assert not extra_rows or (out[total:] == 7.0).all()
    finally:
        cache8.AttentionPlan.FEW_WALKS, cache8.AttentionPlan.MANY_HERE = was
    want, mass, size = plain.attention(q[:total].cpu().to(F64).reshape(total, nq, d), cache, entries, table, scale, window, chunk, softcap,
                                       sinks, gates[:total] if gates is not None else None, width_g, pool)
    bound = bound_of(dtype, d, want, mass, size)
    fine = torch.isfinite(want)
    for got in outs:
        assert torch.equal(fine, torch.isfinite(got)), (fine != torch.isfinite(got)).nonzero()[:5]
        off = ((got - want).abs() - bound)[fine]
        assert (off <= 1e-12).all(), (float(off.max()), ((got - want).abs() / (bound + 1e-30))[fine].max())
    return outs[0], want


ONE = [(0, 1), (1, 1), (15, 1), (16, 1), (62, 1), (63, 1), (64, 1), (200, 1)]
MIX = [(0, 1), (0, 5), (40, 3), (0, 33), (130, 70), (17, 1)]


@pytest.mark.parametrize("d", [16, 32, 48, 64, 80, 96, 112, 128, 144, 160, 192, 224, 256])
def test_attention_head_sizes(d):
    attend(ONE, 4, 2, d, 16)
    attend(MIX, 4, 2, d, 16, seed=1)


@pytest.mark.parametrize("d", [48, 80, 112])
def test_attention_of_heads_that_end_inside_an_operand(d):
    """Heads whose channels do not fill the last operand: keys and values that are not finite reach their own heads and channels only."""
    def spoil(k, v, rows, page):
        k[rows[3][130 // page] * page + 130 % page, 0, :] = math.nan      # a key of one head that rows of request 3 see from position 130 on
        v[rows[5][9 // page] * page + 9 % page, 1, d - 1] = math.nan      # the last channel of the other head

    entries = [(700, 1), (0, 150), (63, 1), (100, 64), (5, 1), (9, 1)]
    got, _ = attend(entries, 6, 2, d, 32, seed=21, spoil=spoil, gate=16, sink=True)
    bad = torch.isnan(got)
    assert bad[182:216, :3].all() and not bad[182:216, 3:].any() and not bad[:182].any() and not bad[216].any()
    assert bad[217, 3:, d - 1].all() and not bad[217, :, :d - 1].any() and not bad[217, :3].any()
    attend([(900, 1), (1300, 300)], 8, 1, d, 16, seed=22, window=500, pad=8)


@pytest.mark.parametrize("nq,nkv", [(1, 1), (3, 3), (6, 2), (7, 1), (16, 1), (20, 1), (32, 2), (33, 1), (130, 1)])
def test_attention_shared_heads(nq, nkv):
    attend([(0, 1), (77, 1), (3, 9)] if nq > 16 else MIX, nq, nkv, 32, 16, seed=2)


@pytest.mark.parametrize("page", [1, 8, 16, 24, 32, 48, 64, 256])
def test_attention_pages(page):
    attend(MIX, 4, 2, 64, page, seed=3)


@pytest.mark.parametrize("d", [20, 32, 130, 300, 512])
@pytest.mark.parametrize("page", [4, 16])
def test_attention_float32(d, page):
    attend([(0, 1), (9, 4), (100, 1), (0, 17)], 3, 1, d, page, torch.float32, seed=4)


@pytest.mark.parametrize("window,chunk", [(1, 0), (5, 0), (64, 0), (100, 0), (0, 1), (0, 48), (0, 64), (0, 100)])
@pytest.mark.parametrize("dtype,page", [(torch.bfloat16, 16), (torch.bfloat16, 32), (torch.float32, 16), (torch.bfloat16, 12)])
def test_attention_windows_and_chunks(window, chunk, dtype, page):
    attend(MIX + [(300, 1)], 4, 2, 32, page, dtype, seed=5, window=window, chunk=chunk)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("softcap,sink,gate", [(5.0, False, None), (0.0, True, None), (0.0, False, 0), (20.0, True, 24), (0.0, True, 64)])
def test_attention_caps_sinks_gates(dtype, softcap, sink, gate):
    attend(MIX, 4, 2, 64, 16, dtype, seed=6, softcap=softcap, sink=sink, gate=gate, pad=16, extra_rows=3)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_long_axis_is_joined(dtype):
    """Contexts that are cut into many pieces beside ones of a few tokens."""
    attend([(3000, 1), (2, 1), (1025, 1)], 2, 1, 64, 16, dtype, seed=7)
    attend([(2500, 40), (0, 90), (700, 1)], 2, 1, 32, 16, dtype, seed=8, window=900)


@pytest.mark.parametrize("entries,nq,nkv", [([(i * 7 % 300, 1) for i in range(70)], 16, 8), ([(0, 512)], 128, 32), ([(5, 600), (0, 40)], 64, 16)])
def test_attention_of_items_that_fill_the_gpu(entries, nq, nkv):
    """Many items: nothing is cut; with a window most of a long walk falls away."""
    attend(entries, nq, nkv, 32, 16, seed=20)
    attend(entries, nq, nkv, 32, 16, seed=21, window=70, sink=True)


@pytest.mark.parametrize("seed", range(24))
def test_attention_drawn(seed):
    """Sizes, layouts and masks drawn over the range, odd ones among them."""
    import random

    r = random.Random(seed)
    nq, nkv = r.choice([(4, 4), (6, 2), (7, 1), (12, 4), (20, 4), (18, 1), (5, 5)])
    long = lambda most: int(math.exp(r.uniform(0, math.log(most))))  # noqa: E731
    entries = [(long(1500) - 1, 1 if r.random() < 0.6 else long(200)) for _ in range(r.randint(1, 9))]
    window, chunk = r.choice([(0, 0), (0, 0), (long(700), 0), (0, long(300))])
    attend(entries, nq, nkv, r.choice([32, 40, 64, 96, 128, 192]), r.choice([4, 16, 16, 32, 48]), r.choice([torch.bfloat16] * 3 + [torch.float32]),
           seed=100 + seed, window=window, chunk=chunk, softcap=r.choice([0.0, 0.0, 8.0]), sink=r.random() < 0.4,
           gate=r.choice([None, None, 0, 16]), pad=r.choice([0, 8]), extra_rows=r.choice([0, 2]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("sink", [False, True])
def test_attention_rows_that_see_nothing(dtype, sink):
    """Pages that are not there hide their keys; a row left with none is zeros."""
    got, _ = attend([(20, 1), (5, 1), (0, 40), (100, 1)], 2, 1, 32, 16, dtype, seed=9, sink=sink, none=[(1, 0), (2, 0), (3, 3), (3, 2)])
    assert (got[1] == 0).all() and (got[2:18] == 0).all() and (got[18:] != 0).any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("page", [16, 20])
def test_attention_what_is_not_finite_stays_with_those_who_see_it(dtype, page):
    def spoil(k, v, rows, page):
        at = lambda b, pos: rows[b][pos // page] * page + pos % page  # noqa: E731
        v[at(0, 50), 0, 3] = math.nan      # rows of request 0 from position 50 on
        k[at(1, 30), 0, 5] = math.inf      # rows of request 1 from position 30 on
        v[at(2, 41), 0, 0] = math.inf      # beyond request 2's last row
        v[at(3, 10), 0, 7] = math.nan      # below request 3's window

    entries = [(20, 60), (10, 60), (35, 6), (95, 2), (20, 1)]
    got, want = attend(entries, 2, 1, 32, page, dtype, seed=10, window=40, spoil=spoil)
    bad = torch.isnan(got)
    assert not bad[:30].any() and bad[30:60, :, 3].all() and not bad[30:60, :, 4].any()
    assert not bad[60:80].any() and bad[80:110].all() and not bad[120:].any()


@pytest.mark.parametrize("d,page,dtype", [(32, 16, torch.bfloat16), (96, 48, torch.bfloat16), (128, 32, torch.bfloat16), (40, 12, torch.float32)])
@pytest.mark.parametrize("scale", [math.nan, -math.inf, -3.0e38])
def test_attention_of_a_pool_with_pages_that_nobody_wrote(d, page, dtype, scale):
    attend([(70, 1), (0, 140), (0, 1), (333, 40), (15, 1)], 4, 2, d, page, dtype, seed=12, none=((0, 1), (3, 2)), unwritten=scale)


@pytest.mark.parametrize("d,page,dtype", [(32, 16, torch.bfloat16), (32, 20, torch.bfloat16), (64, 32, torch.float32)])
@pytest.mark.parametrize("rows", [1, 40])
def test_attention_of_positions_far_behind_the_table(d, page, dtype, rows):
    """Rows at the last positions that 32 bits have see what the table has, as rows right behind it do.  (The two are cut differently, and portions among them take
    kernels that round their weights at different maxima: each is held to the bound that a kernel's result has.)"""
    require_gpu()
    from pulse_infer_amd.ops import cache8

    pages = 9
    cache = plain.Cache(pages, 2, page, d)
    x = torch.randn((pages * page, 2, d), generator=torch.Generator().manual_seed(5), dtype=F64)
    cache.store(x, x.flip(0), [[i * cache.block, cache.block, i, 0] for i in range(pages * cache.nb)])
    view, table = view_of(cache), ints([list(range(pages))])
    q = torch.randn((rows, 4 * d), generator=torch.Generator().manual_seed(6)).to(dtype).to(DEV)
    want, mass, size = plain.attention(q.cpu().to(F64).reshape(rows, 4, d), cache, [(pages * page, rows)], [list(range(pages)) + [-1] * rows], d ** -0.5)
    for start in (pages * page, 2 ** 31 - 1 - rows):
        positions = torch.arange(start, start + rows, dtype=torch.int64).to(torch.int32).to(DEV)
        made = cache8.plan(metas([(start, rows)]), 4, 2, d, positions, page_size=page, dtype=dtype)
        out = torch.full_like(q, 7.0)
        cache8.attention(q, out, made, view, positions, ints([0] * rows), table, d ** -0.5)
        assert ((out.cpu().to(F64).reshape(rows, 4, d) - want).abs() <= bound_of(dtype, d, want, mass, size) + 1e-12).all()


def test_attention_of_pages_beyond_32_bits():
    """Pages whose bytes lie beyond 2^32 of the cache's first."""
    require_gpu()
    from pulse_infer_amd.cache.specs import Paged8KVSpec
    from pulse_infer_amd.ops import cache8

    nkv, d, pages = 8, 128, 280_000                     # 4.6 GB of keys, as much of values
    spec = Paged8KVSpec(nkv, d)
    storage = spec.allocate(1, pages, 16, torch.device(DEV), torch.bfloat16)
    view = spec.view(storage, 0, 0, 16, True)
    small = plain.Cache(3, nkv, 16, d)
    used = [pages - 1, 270_001, 1]
    entries = [(0, 33), (32, 1)]
    g = torch.Generator().manual_seed(11)
    qkv = torch.randn((33, 3 * nkv * d), generator=g).to(torch.bfloat16).to(DEV)
    want = plain.maps([(0, 33)], used, 16, pages, 3)
    q = torch.empty((33, nkv * d), dtype=torch.bfloat16, device=DEV)
    cache8.store(qkv, q, nkv, nkv, d, view, ints(want["positions"]), ints(want["blocks"]))
    _, k, v = plain.prepared(qkv, nkv, nkv, d)
    small.store(k, v, [[0, 16, 0, 0], [16, 16, 1, 0], [32, 1, 2, 0]])
    for i, p in enumerate(used):
        assert torch.equal(view.keys[p].cpu().view(torch.uint8), small.tensors()[0][i].view(torch.uint8))
    positions, token_entry = ints(list(range(33)) + [32]), ints([0] * 33 + [1])
    qs = torch.cat([q, q[32:33]])
    out = torch.empty_like(qs)
    made = cache8.plan(metas(entries), nkv, nkv, d, positions, page_size=16, dtype=torch.bfloat16)
    cache8.attention(qs, out, made, view, positions, token_entry, ints([used, used]), d ** -0.5)
    ref, mass, size = plain.attention(qs.cpu().to(F64).view(34, nkv, d), small, entries, [[0, 1, 2]] * 2, d ** -0.5)
    off = (out.cpu().to(F64).view(34, nkv, d) - ref).abs() - (2.0 ** -8 * (mass + ref.abs()) + (1e-5 + 2.0 ** -22 * size) * mass)
    assert (off <= 0).all()


# ------------------------------------------------------------------------------------------------------------ together
def test_a_step_recorded_and_replayed():
    """Maps, store and attention of decoding steps, recorded once and replayed with other lengths: every replay is the eager step."""
    require_gpu()
    from pulse_infer_amd.ops import cache8
    from pulse_infer_amd.parts.base import Workspace

    nq, nkv, d, page, b = 8, 2, 64, 16, 3
    lengths = [(600, 3, 40), (601, 4, 41), (1100, 15, 47), (100, 16, 48)]
    width, pool = 80, 300
    table = torch.randperm(pool, generator=torch.Generator().manual_seed(1)).to(torch.int32)[:b * width].view(b, width).contiguous().to(DEV)

    def fresh():
        cache = plain.Cache(pool, nkv, page, d)
        g = torch.Generator().manual_seed(2)
        k, v = (torch.randn((pool * page, nkv, d), generator=g, dtype=F64) for _ in range(2))
        cache.store(k, v, [[i * 16, 16, i, 0] for i in range(pool)])
        return view_of(cache)

    start, count = ints([0] * b), ints([1] * b)
    qkv = torch.zeros((b, (nq + 2 * nkv) * d), dtype=torch.bfloat16, device=DEV)
    rows = [torch.randn(qkv.shape, generator=torch.Generator().manual_seed(i)).to(torch.bfloat16).to(DEV) for i in range(len(lengths))]

    def program(view):
        m = dict(positions=ints([0] * b), token_entry=ints([0] * b), blocks=torch.zeros((b, 4), dtype=torch.int32, device=DEV))
        q, out = (torch.zeros((b, nq * d), dtype=torch.bfloat16, device=DEV) for _ in range(2))
        ws = Workspace(torch.device(DEV))
        made = cache8.plan(metas([(0, 1)] * b), nq, nkv, d, m["positions"], page_size=page, dtype=torch.bfloat16, workspace=ws)

        def step():
            cache8.step_maps(start, count, page_size=page, num_pages=pool, table=table, **m)
            made.cut(m["positions"])
            cache8.store(qkv, q, nq, nkv, d, view, m["positions"], m["blocks"])
            cache8.attention(q, out, made, view, m["positions"], m["token_entry"], table, d ** -0.5)

        return step, out

    def run(step, i):
        start.copy_(ints(list(lengths[i])))
        qkv.copy_(rows[i])
        step()

    eager_view, view = fresh(), fresh()
    eager, want = program(eager_view)
    step, out = program(view)
    run(step, 0)
    run(eager, 0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in [0, 1, 2, 3, 1, 2]:
        run(eager, i)
        run(graph.replay, i)
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
        assert torch.equal(view.keys.view(torch.uint8), eager_view.keys.view(torch.uint8))
        assert torch.equal(view.scales, eager_view.scales)


@pytest.mark.parametrize("d,page", [(128, 16), (64, 48)])
def test_two_steps_on_two_streams_at_once(d, page):
    """Plans, workspaces and outputs of their own over one cache: whatever runs beside them, the results are those of each alone, bit for bit."""
    require_gpu()
    from pulse_infer_amd.ops import cache8
    from pulse_infer_amd.parts.base import Workspace

    nq, nkv = 8, 2
    steps = [[(3000, 1), (17, 1), (2500, 1), (700, 1)], [(1200, 200), (64, 1), (900, 33)]]
    pages, pool, _ = layout([(max(s[i][0] + s[i][1] if i < len(s) else 1 for s in steps), 0) for i in range(4)], page, 8)
    cache = plain.Cache(pool, nkv, page, d)
    g = torch.Generator().manual_seed(4)
    k, v = (torch.randn((pool * page, nkv, d), generator=g, dtype=F64) for _ in range(2))
    cache.store(k, v, [[i * cache.block, cache.block, i, 0] for i in range(pool * cache.nb)])
    view, runs = view_of(cache), []
    for entries in steps:
        total, held = sum(c for _, c in entries), [-(-(s + c) // page) for s, c in entries]
        at = [sum(held[:i]) for i in range(len(held))]
        table = ints([(pages[a:a + h] + [-1] * max(held))[:max(held)] for a, h in zip(at, held)])
        q = torch.randn((total, nq * d), generator=g).to(torch.bfloat16).to(DEV)
        positions = ints([p for s, c in entries for p in range(s, s + c)])
        token_entry = ints([b for b, (_, c) in enumerate(entries) for _ in range(c)])
        made = cache8.plan(metas(entries), nq, nkv, d, positions, page_size=page, dtype=torch.bfloat16, workspace=Workspace(torch.device(DEV)))
        runs.append((q, made, positions, token_entry, table, torch.cuda.Stream()))

    def go(run):
        q, made, positions, token_entry, table, _ = run
        out = torch.empty_like(q)
        cache8.attention(q, out, made.cut(positions), view, positions, token_entry, table, d ** -0.5)
        return out

    alone = [go(run) for run in runs]
    torch.cuda.synchronize()
    outs = []
    for _ in range(10):
        for n, run in enumerate(runs):
            with torch.cuda.stream(run[-1]):
                outs.append((n, go(run)))
    torch.cuda.synchronize()
    assert all(torch.equal(out, alone[n]) for n, out in outs) and all(torch.isfinite(out).all() for out in alone)


def test_prompts_and_decoding_on_another_stream():
    """A prompt whole, then tokens one by one, on a stream of the program's own, against the plain forms of the same steps."""
    require_gpu()
    from pulse_infer_amd.ops import cache8

    nq, nkv, d, page = 6, 2, 64, 16
    steps = [[(0, 45), (0, 3)], [(45, 1), (3, 1)], [(46, 1), (4, 20)], [(47, 1), (24, 1)]]
    rows = [[4, 0, 6, 2], [1, 5, 3, 7]]
    cache = plain.Cache(8, nkv, page, d)
    view = view_of(cache)
    stream = torch.cuda.Stream()
    for n, entries in enumerate(steps):
        total = sum(c for _, c in entries)
        qkv = torch.randn((total, (nq + 2 * nkv) * d), generator=torch.Generator().manual_seed(n)).to(torch.bfloat16)
        pages = [p for r, (s, c) in zip(rows, entries) for p in r[:-(-(s + c) // page)]]
        want = plain.maps(entries, pages, page, 8, 4)
        q, k, v = plain.prepared(qkv, nq, nkv, d)
        cache.store(k, v, want["blocks"])
        ref, mass, size = plain.attention(q, cache, entries, want["table"], d ** -0.5)
        with torch.cuda.stream(stream):
            m = dict(positions=ints([0] * total), token_entry=ints([0] * total), table=ints([[0] * 4] * 2),
                     blocks=torch.zeros((len(want["blocks"]), 4), dtype=torch.int32, device=DEV))
            cache8.step_maps(ints([s for s, _ in entries]), ints([c for _, c in entries]), page_size=page, num_pages=8, pages=ints(pages), **m)
            dev = qkv.to(DEV)
            out = torch.empty((total, nq * d), dtype=torch.bfloat16, device=DEV)
            cache8.store(dev, dev, nq, nkv, d, view, m["positions"], m["blocks"])
            made = cache8.plan(metas(entries), nq, nkv, d, m["positions"], page_size=page, dtype=torch.bfloat16)
            cache8.attention(dev[:, :nq * d], out, made, view, m["positions"], m["token_entry"], m["table"], d ** -0.5)
        stream.synchronize()
        off = (out.cpu().to(F64).view(total, nq, d) - ref).abs() - (2.0 ** -8 * (mass + ref.abs()) + (1e-5 + 2.0 ** -22 * size) * mass)
        assert (off <= 0).all(), n
        assert torch.equal(view.values.cpu().view(torch.uint8), cache.tensors()[1].view(torch.uint8))


# ------------------------------------------------------------------------------------------------------------ refusals
def test_refusals():
    require_gpu()
    from pulse_infer_amd.cache.specs import Paged8CacheView
    from pulse_infer_amd.ops import KernelError, cache8

    cache = plain.Cache(4, 2, 16, 32)
    view = view_of(cache)
    e = metas([(0, 3)])
    pos, ent, table = ints([0, 1, 2]), ints([0] * 3), ints([[0, 1]])
    q = torch.zeros((3, 128), dtype=torch.bfloat16, device=DEV)
    qkv = torch.zeros((3, 256), dtype=torch.bfloat16, device=DEV)
    blocks = ints([[0, 3, 0, 0]])
    made = cache8.plan(e, 4, 2, 32, pos, page_size=16, dtype=torch.bfloat16)

    def bad(fn, *a, **k):
        with pytest.raises(KernelError):
            fn(*a, **k)

    go = lambda **k: cache8.attention(k.pop("q", q), k.pop("out", q.clone()), made, k.pop("view", view), k.pop("pos", pos), ent, k.pop("table", table), k.pop("scale", 1.0), **k)  # noqa: E731
    go()
    bad(go, q=q.float())
    bad(go, out=q.float())
    bad(go, q=q[:, :96])
    bad(go, q=q[:2], out=q[:2].clone())
    bad(go, q=q.t().contiguous().t())
    bad(go, pos=pos.long())
    bad(go, pos=pos[:2])
    bad(go, pos=pos.cpu())
    bad(go, table=table.long())
    bad(go, scale=0.0)
    bad(go, scale=-1.0)
    bad(go, softcap=-1.0)
    bad(go, sink=torch.zeros(3, device=DEV))
    bad(go, gate=torch.zeros((3, 4), device=DEV))
    bad(go, gate=torch.zeros((3, 4), dtype=torch.bfloat16, device=DEV), gate_width=2)
    bad(go, view=Paged8CacheView(0, view.keys, view.values, view.scales.double(), 16))
    bad(go, view=Paged8CacheView(0, view.keys[:, :1], view.values, view.scales, 16))
    bad(go, view=Paged8CacheView(0, view.keys.view(torch.uint8), view.values, view.scales, 16))
    bad(go, view=Paged8CacheView(0, view.keys, view.values[:3], view.scales, 16))
    uncut = cache8.AttentionPlan(e, 4, 2, 32, page_size=16, dtype=torch.bfloat16)
    bad(cache8.attention, q, q.clone(), uncut, view, pos, ent, table, 1.0)
    bad(cache8.plan, e, 4, 3, 32, pos, page_size=16, dtype=torch.bfloat16)
    bad(cache8.plan, e, 4, 2, 600, pos, page_size=16, dtype=torch.bfloat16)
    bad(cache8.plan, e, 4, 2, 32, pos, page_size=16, dtype=torch.bfloat16, window=3, chunk=4)
    bad(cache8.plan, e, 4, 2, 32, pos[:2], page_size=16, dtype=torch.bfloat16)
    put = lambda **k: cache8.store(k.pop("qkv", qkv), k.pop("q", q), 4, 2, 32, k.pop("view", view), k.pop("pos", pos), k.pop("blocks", blocks), **k)  # noqa: E731
    put()
    bad(put, qkv=qkv[:, :200])
    bad(put, q=q[:2])
    bad(put, q=q.float())
    bad(put, pos=pos[:2])
    bad(put, blocks=blocks[:, :3])
    bad(put, blocks=blocks.long())
    bad(put, q_weight=torch.ones(32, device=DEV))
    bad(put, q_weight=torch.ones(16, device=DEV), k_weight=torch.ones(16, device=DEV))
    bad(put, cos=torch.zeros((3, 16), device=DEV))
    bad(put, cos=torch.zeros((3, 16), device=DEV), sin=torch.zeros((3, 16), device=DEV), rotary_dim=30)
    bad(put, cos=torch.zeros((3, 16), device=DEV), sin=torch.zeros((3, 16), device=DEV), rotary_dim=32, pairing=2)
    bad(put, q_temperature=(0.1, 0))
    put(parts=torch.zeros((2, 3, 256), device=DEV))
    bad(put, parts=torch.zeros((2, 3, 252), device=DEV))
    bad(put, parts=torch.zeros((2, 3, 258), device=DEV))
    bad(put, parts=torch.zeros((3, 256), device=DEV))
    bad(put, parts=torch.zeros((2, 3, 256), dtype=torch.bfloat16, device=DEV))
    bad(put, parts=torch.zeros((2, 3, 256), device=DEV), qkv=qkv.float(), q=q.float())
    bad(put, view=Paged8CacheView(0, view.keys, view.values, view.scales, 16, writable=False))
    maps = lambda **k: cache8.step_maps(k.pop("start", ints([0])), k.pop("count", ints([3])), page_size=k.pop("page_size", 16), num_pages=k.pop("num_pages", 4), **k)  # noqa: E731
    maps(pages=ints([1]), slots=ints([0] * 3))
    bad(maps, slots=ints([0] * 3))
    bad(maps, pages=ints([1]), slots=ints([0] * 3), positions=ints([0] * 4))
    bad(maps, pages=ints([1]), block=5, blocks=blocks)
    bad(maps, pages=ints([1]).long(), slots=ints([0] * 3))
    bad(maps, start=ints([0, 1]))
    bad(maps, start=ints([0] * 5000), count=ints([0] * 5000))
    bad(maps, num_pages=1 << 28, pages=ints([1]), slots=ints([0] * 3))
    bad(maps, pages=ints([1]), table=ints([[0], [0]]))

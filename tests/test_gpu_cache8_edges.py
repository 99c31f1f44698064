"""A cache of keys and values in 8 bits at its edges: the largest numbers, the last positions, calls without rows, rows that overlap, other
streams.  Tolerances are those of test_gpu_cache8.py, from whose plain forms the expected values come."""
from __future__ import annotations

import pytest
import torch

from conftest import require_gpu
from plain import cache8_plain as plain
from test_gpu_cache8 import DEV, F64, MIX, attend, bound_of, ints, metas, view_of

pytestmark = pytest.mark.gpu


def held(view, page):
    """The plain cache that holds what the kernels' cache holds."""
    pages, nkv, _, d = view.keys.shape
    cache = plain.Cache(pages, nkv, page, d)
    cache.x[0].copy_(plain.decode(view.keys).view(cache.x[0].shape))
    cache.x[1].copy_(plain.decode(view.values).transpose(3, 4))
    cache.e.copy_(torch.log2(view.scales.cpu().to(F64).abs()))
    return cache


# --------------------------------------------------------------------------------------------------- the largest numbers
LARGE = [torch.finfo(torch.bfloat16).max, 248.0 * 2.0 ** 120, 247.0 * 2.0 ** 120, -255.0 * 2.0 ** 120, 225.0 * 2.0 ** 120]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("page", [16, 20])
def test_store_of_the_largest_numbers(dtype, page):
    """At the greatest exponent the largest byte is 240's, in a block that is begun and in one whose earlier bytes move: nothing stands for more
    than a float32 number, and everything is within 2^-4 of what came."""
    require_gpu()
    from pulse_infer_amd.ops import cache8

    d = 32
    view = view_of(plain.Cache(2, 1, page, d))
    x = torch.randn((page + 3, 3 * d), generator=torch.Generator().manual_seed(0)).to(dtype)
    for i, v in enumerate(LARGE):
        x[i, d + i], x[i + 4, 2 * d + 7 + i], x[page + 2, d + 3 * i], x[page + 2, 2 * d + 5 * i] = v, v, -v, v
    if dtype == torch.float32:
        x[page + 1, d + 20] = torch.finfo(torch.float32).max
    dev = x.to(DEV)
    for first, rows, block, at in ((0, page, 1, 0), (page, 2, 0, 0), (page + 2, 1, 0, 2)):
        cache8.store(dev[first:first + rows], torch.empty((rows, d), dtype=dtype, device=DEV), 1, 1, d, view, ints([0] * rows), ints([[0, rows, block, at]]))
    cache = held(view, page)
    assert (view.scales == 2.0 ** 120).all()      # (every block holds one of them, and none that is not finite)
    keys, values = (c[:, 0, :].to(F64) for c in (cache.x[0][:, :, 0] * 2.0 ** 120, cache.x[1][:, :, 0] * 2.0 ** 120))
    for got, first in ((keys, d), (values, 2 * d)):
        want = x[:, first:first + d].to(F64)
        got = torch.cat([got[1], got[0, :3]])
        assert (got.abs() <= 240 * 2.0 ** 120).all() and (got.abs() == 240 * 2.0 ** 120).any()
        assert ((got - want).abs() <= 2.0 ** -4 * want.abs())[want.abs() > 1.0e38].all()


@pytest.mark.parametrize("d,page", [(32, 16), (64, 32), (128, 16), (192, 16)])
@pytest.mark.parametrize("few", [True, False])
def test_the_largest_numbers_stay_with_those_who_see_them(d, page, few, monkeypatch):
    """bfloat16's largest number as a value and as a key: rows before it are what they are without it."""
    require_gpu()
    from pulse_infer_amd.ops import cache8

    nq, nkv, rows, at = 4, 2, 45, 30
    if not few:
        monkeypatch.setattr(cache8.AttentionPlan, "FEW_WALKS", 0)
    view = view_of(plain.Cache(4, nkv, page, d))
    g = torch.Generator().manual_seed(d)
    qkv = torch.randn((rows, (nq + 2 * nkv) * d), generator=g)
    qkv[at, (nq + nkv) * d + 3] = qkv[at + 2, nq * d + d + 5] = torch.finfo(torch.bfloat16).max
    qkv[at, nq * d + 1] = -torch.finfo(torch.bfloat16).max
    qkv = qkv.to(torch.bfloat16).to(DEV)
    positions = ints(list(range(rows)))
    pages = [3, 1, 0][:-(-rows // page)]
    want = plain.maps([(0, rows)], pages, page, 4, 3)
    q, out = (torch.zeros((rows, nq * d), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    cache8.store(qkv, q, nq, nkv, d, view, positions, ints(want["blocks"]))
    made = cache8.plan(metas([(0, rows)]), nq, nkv, d, positions, page_size=page, dtype=torch.bfloat16)
    cache8.attention(q, out, made, view, positions, ints([0] * rows), ints(want["table"]), d ** -0.5)
    ref, mass, size = plain.attention(q[:at].cpu().to(F64).view(at, nq, d), held(view, page), [(0, at)], want["table"], d ** -0.5)
    got = out[:at].cpu().to(F64).view(at, nq, d)
    assert torch.isfinite(got).all()
    assert ((got - ref).abs() <= bound_of(torch.bfloat16, d, ref, mass, size) + 1e-12).all()


# ------------------------------------------------------------------------------------------------------ the last positions
@pytest.mark.parametrize("d,page,dtype", [(32, 20, torch.bfloat16), (64, 16, torch.float32), (300, 16, torch.bfloat16), (32, 16, torch.bfloat16), (128, 32, torch.bfloat16)])
@pytest.mark.parametrize("window,chunk", [(5, 0), (700, 0), (0, 48), (2 ** 31 - 1, 0), (2 ** 31 - 100, 0), (0, 2 ** 30)])
@pytest.mark.parametrize("rows,back", [(1, 0), (40, 0), (600, 300), (1, 3000)])
def test_attention_of_the_last_positions_behind_a_mask(d, page, dtype, window, chunk, rows, back):
    """Rows at the last positions that 32 bits have, whose window or chunk begins behind the table (rows of zeros) or reaches into it."""
    require_gpu()
    from pulse_infer_amd.ops import cache8

    pages, start = 9, 2 ** 31 - rows - back
    cache = plain.Cache(pages, 2, page, d)
    x = torch.randn((pages * page, 2, d), generator=torch.Generator().manual_seed(5), dtype=F64)
    cache.store(x, x.flip(0), [[i * cache.block, cache.block, i, 0] for i in range(pages * cache.nb)])
    q = torch.randn((rows, 4 * d), generator=torch.Generator().manual_seed(6)).to(dtype).to(DEV)
    positions = torch.arange(start, start + rows, dtype=torch.int64)
    low = positions // chunk * chunk if chunk else (positions - window + 1).clamp_min(0)
    made = cache8.plan(metas([(start, rows)]), 4, 2, d, positions.to(torch.int32).to(DEV), page_size=page, dtype=dtype, window=window, chunk=chunk)
    out = torch.full_like(q, 7.0)
    cache8.attention(q, out, made, view_of(cache), positions.to(torch.int32).to(DEV), ints([0] * rows), ints([list(range(pages))]), d ** -0.5)
    got = out.cpu().to(F64).reshape(rows, 4, d)
    keys, values = cache.rows(list(range(pages)))
    seen = torch.arange(pages * page) >= low[:, None]
    for h in range(4):
        qh = q[:, h * d:(h + 1) * d].cpu().to(F64)
        s = torch.where(seen, qh @ keys[h // 2].T * d ** -0.5, torch.full((), -float("inf"), dtype=F64))
        p = torch.where(seen.any(-1, keepdim=True), torch.softmax(s, -1), torch.zeros((), dtype=F64))
        want, mass, size = p @ values[h // 2], p @ values[h // 2].abs(), (qh.abs() @ keys[h // 2].abs().T).amax(-1, keepdim=True) * d ** -0.5
        assert ((got[:, h] - want).abs() <= bound_of(dtype, d, want, mass, size) + 1e-12).all()
        assert (got[:, h][~seen.any(-1)] == 0).all()


# -------------------------------------------------------------------------------------------------------- no rows at all
@pytest.mark.parametrize("dtype,page", [(torch.bfloat16, 16), (torch.float32, 20)])
def test_steps_without_rows(dtype, page):
    """Requests that bring no tokens: nothing is stored, attended or listed, and nothing is refused."""
    require_gpu()
    from pulse_infer_amd.ops import cache8

    nkv, d, entries = 2, 32, [(3, 0), (0, 0)]
    view = view_of(plain.Cache(2, nkv, page, d))
    before = [t.clone().view(torch.uint8) for t in (view.keys, view.values, view.scales)]
    empty, none = torch.zeros((0, 3 * nkv * d), dtype=dtype, device=DEV), ints([])
    blocks = torch.full((2, 4), 9, dtype=torch.int32, device=DEV)
    cache8.step_maps(ints([s for s, _ in entries]), ints([c for _, c in entries]), page_size=page, num_pages=2, table=ints([[1], [-1]]), blocks=blocks,
                     positions=none, token_entry=none, slots=none)
    assert blocks.tolist() == [[0, 0, -1, 0]] * 2
    for listed in (blocks, blocks[:0]):
        cache8.store(empty, empty[:, :nkv * d], nkv, nkv, d, view, none, listed)
    cache8.store(empty, empty[:, :nkv * d], nkv, nkv, d, view, none, blocks, cos=torch.zeros((0, 16), device=DEV), sin=torch.zeros((0, 16), device=DEV),
                 rotary_dim=32, plain_norm=True, q_temperature=(0.1, 3))
    made = cache8.plan(metas(entries), nkv, nkv, d, none, page_size=page, dtype=dtype)
    cache8.attention(empty, empty.clone(), made, view, none, none, ints([[1], [-1]]), 1.0)
    out = torch.full((3, nkv * d), 7.0, dtype=dtype, device=DEV)      # (rows that no entry has)
    cache8.attention(torch.zeros_like(out), out, made, view, ints([0] * 3), ints([-1] * 3), ints([[1], [-1]]), 1.0)
    assert (out == 7.0).all()
    assert all(torch.equal(a, b.view(torch.uint8)) for a, b in zip(before, (view.keys, view.values, view.scales)))


# ------------------------------------------------------------------------------------------------------------- streams
@pytest.mark.parametrize("recut,room", [(False, False), (True, False), (False, True)])
def test_a_plan_that_is_dropped_before_its_stream_has_come_to_it(recut, room):
    """Made on one stream, used on another that is busy, dropped at once (with its workspace): nobody gets its lists' memory, or the workspace's, before
    they have been read."""
    require_gpu()
    from pulse_infer_amd.ops import cache8
    from pulse_infer_amd.parts.base import Workspace

    nq, nkv, d, page, entries = 8, 2, 64, 16, [(700, 1), (0, 150), (300, 40), (1200, 1)]
    view = view_of(plain.Cache(200, nkv, page, d))
    view.keys.copy_(torch.randn(view.keys.shape, device=DEV).to(view.keys.dtype))
    view.values.copy_(torch.randn(view.values.shape, device=DEV).to(view.values.dtype))
    view.scales.fill_(1.0)
    total = sum(c for _, c in entries)
    table = torch.randperm(200, generator=torch.Generator().manual_seed(1))[:4 * 50].to(torch.int32).view(4, 50).contiguous().to(DEV)
    positions = ints([p for s, c in entries for p in range(s, s + c)])
    token_entry = ints([b for b, (_, c) in enumerate(entries) for _ in range(c)])
    table[3, 40:] = -1
    q = torch.randn((total, nq * d), generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(DEV)
    want, out = torch.zeros_like(q), torch.zeros_like(q)
    work, busy = torch.randn((8192, 8192), device=DEV).to(torch.bfloat16), torch.cuda.Stream()

    def plan(ws=None):
        return cache8.plan(metas(entries), nq, nkv, d, positions, page_size=page, dtype=torch.bfloat16, workspace=ws)

    cache8.attention(q, want, plan(), view, positions, token_entry, table, d ** -0.5)
    with torch.cuda.stream(busy):
        product = work @ work      # (the library is loaded and its scratch there)
    torch.cuda.synchronize()
    ws = Workspace(torch.device(DEV)) if room else None
    made = plan(ws)
    lists = [(t.data_ptr(), t.numel()) for w in made.works for t in (w[0], w[-1])]
    if room:      # (the workspace's buffers are the first stream's)
        cache8.attention(q, out, made, view, positions, token_entry, table, d ** -0.5)
        lists += [(t.data_ptr(), t.numel()) for r in made.rooms.values() for t in r]
        assert len(lists) >= 4
        out.zero_()
    done = torch.cuda.Event()
    busy.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(busy):
        for _ in range(100):
            torch.mm(work, work, out=product)
        if recut:
            made.cut(positions)
        cache8.attention(q, out, made, view, positions, token_entry, table, d ** -0.5)
        done.record()
    del made, ws
    others = [torch.empty(n, dtype=torch.int32, device=DEV) for _ in range(8) for _, n in lists]      # (nothing is written to them)
    assert not done.query()
    assert not {t.data_ptr() for t in others} & {at for at, _ in lists}
    torch.cuda.synchronize()
    assert torch.equal(out, want)


# ------------------------------------------------------------------------------------------------------ rows that overlap
def test_rows_that_overlap_what_is_still_read_are_refused():
    """q_out among k and v, out among other rows of q; beside each other in one buffer and in place they are served."""
    require_gpu()
    from pulse_infer_amd.ops import KernelError, cache8

    nq, nkv, d, rows = 4, 2, 32, 5
    view = view_of(plain.Cache(1, nkv, 16, d))
    columns = (nq + 2 * nkv) * d
    positions, blocks = ints(list(range(rows))), ints([[0, rows, 0, 0]])
    buffer = torch.randn((rows, columns + nq * d), generator=torch.Generator().manual_seed(0)).to(torch.bfloat16).to(DEV)

    def store(qkv, q_out, **k):
        cache8.store(qkv, q_out, nq, nkv, d, view, positions[:qkv.shape[0]], ints([[0, qkv.shape[0], 0, 0]]), **k)

    for n in (1, rows):
        with pytest.raises(KernelError, match="overlaps"):
            store(buffer[:n], buffer[:n, d:])
        with pytest.raises(KernelError, match="overlaps"):
            store(buffer[:n], buffer[:n, columns - d:])
        with pytest.raises(KernelError, match="among"):
            store(buffer[:n], buffer[:n], v_head0=nq - 1)
        store(buffer[:n], torch.empty_like(buffer[:n]), v_head0=0)      # (from rows of their own values may be any columns)
    with pytest.raises(KernelError, match="overlaps"):
        store(buffer[1:], buffer[:rows - 1])
    with pytest.raises(KernelError, match="overlaps"):
        store(buffer[:, :columns], buffer.view(-1)[:rows * nq * d].view(rows, nq * d))
    q, out, token_entry, table = buffer[:, :nq * d].clone(), torch.empty((rows, nq * d), dtype=torch.bfloat16, device=DEV), ints([0] * rows), ints([[0]])
    store(buffer[:, :columns], buffer[:, columns:])
    assert torch.equal(buffer[:, columns:], q)      # (no norm, no rotation: q as it came)
    store(buffer, buffer)
    made = cache8.plan(metas([(0, rows)]), nq, nkv, d, positions, page_size=16, dtype=torch.bfloat16)

    def attend(q, out):
        cache8.attention(q, out, made, view, positions, token_entry, table, 0.2)

    for bad in (buffer[:, d:], buffer[:, 8:]):
        with pytest.raises(KernelError, match="overlaps"):
            attend(buffer, bad)
    longer = torch.zeros((rows + 1, nq * d), dtype=torch.bfloat16, device=DEV)
    with pytest.raises(KernelError, match="overlaps"):
        attend(longer[:rows], longer[1:])
    attend(buffer, out)
    attend(buffer, buffer[:, nq * d:])
    assert torch.equal(buffer[:, nq * d:2 * nq * d], out)


@pytest.mark.parametrize("d,page,dtype,entries", [(64, 16, torch.bfloat16, [(2000, 1), (3, 1), (700, 1)]), (64, 16, torch.bfloat16, [(2500, 300), (0, 90), (40, 1)]),
                                                  (64, 8, torch.bfloat16, [(100, 40)]), (128, 16, torch.float32, [(300, 9)])])
def test_attention_in_place(d, page, dtype, entries):
    """out = q, through every kernel and join."""
    require_gpu()
    from pulse_infer_amd.ops import cache8

    nq, nkv = 8, 2
    held = [-(-(s + c) // page) for s, c in entries]
    pool = sum(held)
    view = view_of(plain.Cache(pool, nkv, page, d))
    view.keys.copy_(torch.randn(view.keys.shape, device=DEV).to(view.keys.dtype))
    view.values.copy_(torch.randn(view.values.shape, device=DEV).to(view.values.dtype))
    view.scales.fill_(1.0)
    at = [sum(held[:i]) for i in range(len(held))]
    table = ints([list(range(a, a + n)) + [-1] * (max(held) - n) for a, n in zip(at, held)])
    positions = ints([p for s, c in entries for p in range(s, s + c)])
    token_entry = ints([b for b, (_, c) in enumerate(entries) for _ in range(c)])
    q = torch.randn((positions.numel(), nq * d + 8), device=DEV).to(dtype)
    made = cache8.plan(metas(entries), nq, nkv, d, positions, page_size=page, dtype=dtype)
    out = torch.empty_like(q)
    cache8.attention(q, out, made, view, positions, token_entry, table, d ** -0.5)
    cache8.attention(q, q, made, view, positions, token_entry, table, d ** -0.5)
    assert torch.isfinite(out[:, :nq * d]).all() and torch.equal(q[:, :nq * d], out[:, :nq * d])


# ---------------------------------------------------------------------------------------------------------------- caps
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("cap", [0.01, 30.0, 256.0, 256.1, 1e4, 1e6, 1e30])
def test_attention_of_every_cap(dtype, cap):
    """Scores under a cap far above them are the scores themselves."""
    attend(MIX + [(600, 1)], 4, 2, 64, 16, dtype, seed=31, softcap=cap, sink=True, gate=0)
    attend(MIX, 4, 2, 128, 16, dtype, seed=32, softcap=cap, window=33)


@pytest.mark.parametrize("bad", [dict(softcap=float("inf")), dict(softcap=float("nan")), dict(scale=float("inf")), dict(scale=float("nan"))])
def test_caps_and_scales_that_are_no_numbers_are_refused(bad):
    require_gpu()
    from pulse_infer_amd.ops import KernelError, cache8

    view, pos = view_of(plain.Cache(1, 1, 16, 32)), ints([0])
    q = torch.zeros((1, 32), dtype=torch.bfloat16, device=DEV)
    made = cache8.plan(metas([(0, 1)]), 1, 1, 32, pos, page_size=16, dtype=torch.bfloat16)
    with pytest.raises(KernelError, match="finite"):
        cache8.attention(q, q.clone(), made, view, pos, pos, ints([[0]]), bad.get("scale", 1.0), softcap=bad.get("softcap", 0.0))


# ------------------------------------------------------------------------------------------------------- many requests
def test_attention_of_many_requests_and_one_long():
    """A long context beside 30,000 short ones, or as many as a launch has room for, that are alike: the same rows as of the long one beside three."""
    require_gpu()
    from pulse_infer_amd.ops import cache8

    nq, nkv, d, pages = 4, 2, 32, 1251
    view = view_of(plain.Cache(pages, nkv, 16, d))
    view.keys.copy_(torch.randn(view.keys.shape, device=DEV).to(view.keys.dtype))
    view.values.copy_(torch.randn(view.values.shape, device=DEV).to(view.values.dtype))
    view.scales.fill_(1.0)
    outs = []
    for n in (3, 30_000, 65_534):
        entries = [(20_000, 1)] + [(9, 1)] * n
        table = torch.full((n + 1, pages), -1, dtype=torch.int32, device=DEV)
        table[0], table[1:, 0] = torch.arange(pages, dtype=torch.int32, device=DEV), 7
        q = torch.randn((2, nq * d), generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(DEV)
        q = torch.cat([q[:1], q[1:].expand(n, -1)])
        positions = ints([s for s, _ in entries])
        made = cache8.plan(metas(entries), nq, nkv, d, positions, page_size=16, dtype=torch.bfloat16)
        out = torch.zeros_like(q)
        cache8.attention(q, out, made, view, positions, ints(list(range(n + 1))), table, d ** -0.5)
        assert torch.equal(out[1:], out[1:2].expand(n, -1))
        outs.append(out[:2].double())
    assert torch.equal(outs[0][1], outs[1][1]) and torch.equal(outs[0][1], outs[2][1]) and torch.isfinite(torch.stack(outs)).all()
    # (the long one is cut differently: one rounding of the weights and one of the result on either side, of no more than the largest value)
    assert ((outs[0][0] - torch.stack(outs)[:, 0]).abs() <= 4 * 2.0 ** -8 * view.values.float().abs().max().double()).all()


@pytest.mark.parametrize("n,tokens", [(65_535, 2_500_001), (40_000, 4_000_000)])
def test_attention_of_a_context_of_millions_beside_many(n, tokens):
    """The last keys of a context of millions of tokens count, however many requests are beside it."""
    require_gpu()
    from pulse_infer_amd.ops import cache8

    d, page = 32, 4096
    view = view_of(plain.Cache(2, 1, page, d))
    g = torch.Generator().manual_seed(n)
    view.keys.copy_((torch.randn(view.keys.shape, generator=g) * 0.1).to(DEV).to(view.keys.dtype))
    view.values.copy_(torch.randn(view.values.shape, generator=g).to(DEV).to(view.values.dtype))
    view.scales.fill_(1.0)
    q = torch.randn((1, d), generator=g).to(torch.bfloat16)
    view.keys[1, 0, :9] = (torch.sign(q) * 4).to(DEV).to(view.keys.dtype)      # (a few keys of the last page outweigh all that is before them)
    last = (tokens - 1) // page
    table = torch.full((n, last + 1), -1, dtype=torch.int32, device=DEV)
    table[:, 0], table[0] = 0, 0
    table[0, last] = 1
    positions = ints([tokens - 1] + [20] * (n - 1))
    made = cache8.plan(metas([(tokens - 1, 1)] + [(20, 1)] * (n - 1)), 1, 1, d, positions, page_size=page, dtype=torch.bfloat16)
    rows = q.to(DEV).expand(n, -1).contiguous()
    out = torch.zeros_like(rows)
    cache8.attention(rows, out, made, view, positions, ints(list(range(n))), table, 1.0)
    keys, values = (x[:, 0] for x in (plain.decode(view.keys), plain.decode(view.values).transpose(3, 4).reshape(2, 1, page, d)))
    s = [keys[i] @ q[0].to(F64) for i in (0, 1)]
    s[1] = s[1][:(tokens - 1) % page + 1]
    top = max(float(x.max()) for x in s)
    p = [torch.exp(x - top) * w for x, w in zip(s, (last, 1))]
    total = sum(x.sum() for x in p)
    want, mass = (sum(x @ f(v[:x.numel()]) for x, v in zip(p, values)) / total for f in (lambda v: v, torch.abs))
    size = max(float((keys[i].abs() @ q[0].abs().to(F64)).max()) for i in (0, 1))
    assert ((out[0].cpu().to(F64) - want).abs() <= bound_of(torch.bfloat16, d, want, mass, size)).all()
    assert float(p[1][:9].sum() / total) > 0.5


@pytest.mark.parametrize("window", [0, 900])
def test_attention_of_portions_that_fill_the_gpu_and_are_cut(window):
    """A short portion far behind beside a longer one from the start, whose items have a place each by themselves."""
    require_gpu()
    from pulse_infer_amd.ops import cache8

    entries = [(4000, 40), (0, 500)]
    plan = cache8.AttentionPlan(metas(entries), 128, 32, 96, page_size=16, dtype=torch.bfloat16)
    assert plan.calls[0][3] * 32 >= 512 and plan.calls[0][4] == 3 * plan.calls[0][3]
    attend(entries, 128, 32, 96, 16, seed=40, window=window)


# ---------------------------------------------------------------------------------------------------------- recordings
def test_a_recording_outlives_the_workspace_it_was_recorded_with():
    """A workspace that grows behind a recording, for another recording and for eager calls: each replay is the eager call, in whatever order."""
    require_gpu()
    from pulse_infer_amd.ops import cache8
    from pulse_infer_amd.parts.base import Workspace

    nq, nkv, d, page = 8, 2, 64, 16
    view = view_of(plain.Cache(300, nkv, page, d))
    view.keys.copy_(torch.randn(view.keys.shape, device=DEV).to(view.keys.dtype))
    view.values.copy_(torch.randn(view.values.shape, device=DEV).to(view.values.dtype))
    view.scales.fill_(1.0)
    table = torch.randperm(300, generator=torch.Generator().manual_seed(1))[:4 * 75].to(torch.int32).view(4, 75).contiguous().to(DEV)
    shared, programs = Workspace(torch.device(DEV)), []
    for entries in ([(900, 1), (1100, 1)], [(1000, 1)] * 3, [(700, 300), (0, 90), (1000, 1)], [(900, 200), (800, 100), (900, 200), (1000, 1)]):
        total = sum(c for _, c in entries)
        positions = ints([p for s, c in entries for p in range(s, s + c)])
        token_entry = ints([b for b, (_, c) in enumerate(entries) for _ in range(c)])
        q = torch.randn((total, nq * d), generator=torch.Generator().manual_seed(total)).to(torch.bfloat16).to(DEV)
        out = torch.zeros_like(q)

        def call(plan, out=out, q=q, positions=positions, token_entry=token_entry):
            cache8.attention(q, out, plan, view, positions, token_entry, table, d ** -0.5)

        make = lambda ws: cache8.plan(metas(entries), nq, nkv, d, positions, page_size=page, dtype=torch.bfloat16, workspace=ws)  # noqa: E731
        call(make(None))
        want, plan = out.clone(), make(shared)
        call(plan)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):      # (which gives the pool's free memory back to the device)
            call(plan)
        programs.append((plan, call, graph, out, want))
    current = {shared.buffer("attention8.part_o", 1, 1, torch.float32).data_ptr()}
    rooms = [{at for at, _, _ in plan.rooms} for plan, *_ in programs]
    assert all(rooms) and len(set().union(*rooms)) > 1 and any(not r & current for r in rooms)      # (some were recorded with what has been replaced)
    assert all(o.data_ptr() == at for plan, *_ in programs for (at, _, _), (o, _) in plan.rooms.items())
    torch.cuda.empty_cache()
    for i in (0, 3, 1, 2, 0, 0, 3):
        plan, call, graph, out, want = programs[i]
        for run in (graph.replay, lambda: call(plan), graph.replay):
            out.zero_()
            run()
            torch.cuda.synchronize()
            assert torch.equal(out, want), i


# ---------------------------------------------------------------------------------------------------- the last positions' maps
@pytest.mark.parametrize("start,count", [(2 ** 31 - 40, 39), (2 ** 31 - 16, 15), (2 ** 31 - 2, 1), (2 ** 31 - 17, 1)])
def test_maps_of_the_last_positions(start, count):
    """Rows up to the last position that a length of 32 bits leaves, in pages of 2^20 tokens."""
    require_gpu()
    from pulse_infer_amd.ops import cache8

    page, pool = 1 << 20, 2047
    pages = [(7 * i) % pool for i in range(2048)]
    want = plain.maps([(start, count), (0, 3)], pages + [5], page, pool, 2048)
    n = count + 3
    got = dict(positions=ints([-9] * n), token_entry=ints([-9] * n), slots=ints([-9] * n), first_row=ints([-9] * 3),
               blocks=torch.full((len(want["blocks"]), 4), -9, dtype=torch.int32, device=DEV), table=torch.full((2, 2048), -9, dtype=torch.int32, device=DEV))
    assert cache8.blocks_touched(metas([(start, count), (0, 3)]), page) == len(want["blocks"])
    cache8.step_maps(ints([start, 0]), ints([count, 3]), page_size=page, num_pages=pool, pages=ints(pages + [5]), **got)
    for name, t in got.items():
        assert t.tolist() == want[name], name


def test_a_workspace_of_another_device_is_refused():
    """Room for joined pieces that the GPU's kernels cannot write to."""
    require_gpu()
    from pulse_infer_amd.ops import KernelError, cache8
    from pulse_infer_amd.parts.base import Workspace

    view, positions = view_of(plain.Cache(80, 2, 16, 32)), ints([1200])
    q = torch.zeros((1, 128), dtype=torch.bfloat16, device=DEV)
    table = ints([list(range(76))])
    for ws, call in ((Workspace(torch.device("cpu")), None), (None, Workspace(torch.device("cpu")))):
        made = cache8.plan(metas([(1200, 1)]), 4, 2, 32, positions, page_size=16, dtype=torch.bfloat16, workspace=ws)
        assert made.calls[0][5] > 0
        for _ in range(2):
            with pytest.raises(KernelError, match="workspace"):
                cache8.attention(q, q.clone(), made, view, positions, ints([0]), table, 1.0, workspace=call)


def test_the_first_cut_is_no_recorded_one():
    """Behind a recording that has not been replayed nothing is shared out: a call outside it would follow a list that nobody has written."""
    require_gpu()
    from pulse_infer_amd.ops import KernelError, cache8

    view, positions, table = view_of(plain.Cache(80, 2, 16, 32)), ints([1200]), ints([list(range(76))])
    q = torch.zeros((1, 128), dtype=torch.bfloat16, device=DEV)
    out, other = q.clone(), q.clone()
    made = cache8.AttentionPlan(metas([(1200, 1)]), 4, 2, 32, page_size=16, dtype=torch.bfloat16)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        other.add_(1.0)
        with pytest.raises(KernelError, match="first cut"):
            made.cut(positions)
    with pytest.raises(KernelError, match="not been cut"):
        cache8.attention(q, out, made, view, positions, ints([0]), table, 1.0)
    made.cut(positions)
    cache8.attention(q, out, made, view, positions, ints([0]), table, 1.0)
    again = torch.cuda.CUDAGraph()
    zero = ints([0])
    torch.cuda.synchronize()
    with torch.cuda.graph(again):
        made.cut(positions)
        cache8.attention(q, out, made, view, positions, zero, table, 1.0)
    for _ in range(3):
        graph.replay()
        again.replay()
        torch.cuda.synchronize()
    assert (other == 3.0).all() and torch.isfinite(out).all()

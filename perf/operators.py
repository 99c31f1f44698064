"""Keys and values held in 8 bits: what a step has to know about its pages, what it puts into them, what it reads from them.

Three operators, and a step that runs them together, as cases that can be timed and checked:

``maps``    from the requests' lengths and the list of their pages: rows, positions, block tables, slots and the blocks written.
``store``   the norm and the rotation of a step's queries and keys, and its keys and values into the cache in 8 bits.
``attend``  attention over that cache: single tokens, portions of prompts, both in one step.
``step``    the maps once, then store and attention of several layers.

The cache.  Pages of ``page`` tokens; a block is 16 tokens of a page (the whole page where 16 does not divide its size).  A block of a
head has one scale for its keys and one for its values, a power of two: the least 2^e (e >= -118) with max |x| <= 448 * 2^e over the
finite values that the block holds; a value x is kept as the e4m3 number nearest to x / 2^e.  Keys lie as [page, head, token, channel],
values as [page, head, block, channel, token], scales as [page, head, block, (key, value)].
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda:0"
F8 = torch.float8_e4m3fn
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
LEAST = -118         # the smallest exponent of a scale
THETA = 1e6
EPS = 1e-6


# ---------------------------------------------------------------------------------------------------- the cases
def _case(kind, **more):
    return {**dict(kind=kind, heads=32, kv_heads=8, dim=128, page=16, dtype="bf16", singles=0, shortest=1, longest=1, portions=0,
                   portion=1, behind=0, window=0, cap=0.0, sink=False, gate=False, norm=False, layers=1), **more}


def listed():
    return [
        # A full batch decodes: 64 requests at about 4,096 tokens, a token each.
        _case("maps", name="maps-decode-64", singles=64, shortest=3900, longest=4300),
        # A busy step: prompts in portions behind contexts of all lengths, one of them long, beside decoding requests.
        _case("maps", name="maps-mixed-8192", singles=48, shortest=17, longest=32000, portions=16, portion=600, behind=8000),
        # One user's next token: the latency of a launch.
        _case("store", name="store-decode-1", singles=1, shortest=4095, longest=4095, norm=True),
        # The benchmark's prompt: 2,048 tokens at once.
        _case("store", name="store-prompt-2048", portions=1, portion=2048, norm=True),
        # One user, a context of 4,096: few rows and a long axis.
        _case("attend", name="attend-decode-1", singles=1, shortest=4096, longest=4096),
        # A server's usual step: 24 requests of all lengths, a window and capped scores.
        _case("attend", name="attend-decode-24-uneven", singles=24, shortest=150, longest=12000, window=4096, cap=30.0, sink=True),
        # The benchmark's full batch.
        _case("attend", name="attend-decode-64", singles=64, shortest=3968, longest=4223),
        # Long contexts at a full batch, 64 query heads: the 32B shape.
        _case("attend", name="attend-decode-64-long", heads=64, singles=64, shortest=8192, longest=8192),
        # The benchmark's prompt.
        _case("attend", name="attend-prompt-2048", portions=1, portion=2048),
        # A portion of a long prompt beside short ones, odd lengths, narrow heads on pages of 32.
        _case("attend", name="attend-portions-odd", heads=40, dim=64, page=32, portions=3, portion=509, behind=7001),
        # The true 32-bit run of a small model: 6 heads on one, 32 channels.
        _case("attend", name="attend-float32", heads=6, kv_heads=1, dim=32, dtype="f32", singles=2, shortest=9, longest=90, portions=4,
              portion=70),
        # What a decoding step does with it, four layers deep.
        _case("step", name="step-decode-32", singles=32, shortest=1000, longest=5000, layers=4, norm=True),
    ]


HEADS = [(32, 8), (64, 8), (40, 8), (16, 16), (12, 4), (6, 2), (6, 1), (7, 1), (32, 1)]


def draw(rng):
    spread = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))  # noqa: E731
    kind = rng.choice(["maps", "store", "attend", "attend", "attend", "step"])
    heads, kv_heads = rng.choice(HEADS)
    c = _case(kind, heads=heads, kv_heads=kv_heads, dim=rng.choice([32, 64, 80, 96, 128, 128, 128, 192, 256]),
              page=rng.choice([8, 16, 16, 16, 32, 64]), norm=rng.random() < 0.5, layers=rng.randint(1, 4) if kind == "step" else 1)
    if rng.random() < 0.15:
        c["dtype"] = "f32"
    small = c["dtype"] == "f32" or c["page"] % 16 or c["dim"] % 32
    if rng.random() < 0.7 or kind == "step":
        c["singles"] = spread(1, 24 if small else 64)
        c["longest"] = spread(1, 2000 if small else 8000)
        c["shortest"] = rng.randint(1, c["longest"])
    if not c["singles"] or rng.random() < 0.3:
        c["portions"] = rng.randint(1, 3)
        c["portion"] = spread(2, 300 if small else 1500)
        c["behind"] = rng.choice([0, spread(1, 600 if small else 5000)])
    if rng.random() < 0.3:
        c["window"] = spread(1, 4000)
    if rng.random() < 0.3:
        c["cap"] = rng.choice([15.0, 30.0, 50.0])
    c["sink"], c["gate"] = rng.random() < 0.3, rng.random() < 0.2
    while work(c)["flops"] > 9e10 or work(c)["bytes"] > 1e9:      # (the largest listed ones: 1.1e11 and 1.1e9)
        c["longest"], c["portion"], c["behind"] = c["longest"] // 2 + 1, c["portion"] // 2 + 1, c["behind"] // 2
        c["shortest"] = min(c["shortest"], c["longest"])
    return c


def entries_of(case):
    """(tokens in the cache, tokens of this step) of every request: lengths spread evenly, portions of odd lengths."""
    n, lo, hi = case["singles"], case["shortest"], case["longest"]
    out = [(lo - 1 + (hi - lo) * i // max(1, n - 1), 1) for i in range(n)]
    for i in range(case["portions"]):
        out.append((case["behind"] - i * 97 % (case["behind"] // 2 + 1), max(1, case["portion"] - i * 37 % (case["portion"] // 2 + 1))))
    return out


def block_of(page):
    return 16 if page % 16 == 0 else page


def work(case):
    e, t = entries_of(case), sum(c for _, c in entries_of(case))
    nq, nkv, d, size = case["heads"], case["kv_heads"], case["dim"], 4 if case["dtype"] == "f32" else 2
    block, w = block_of(case["page"]), case["window"]
    pages = [(s + c + case["page"] - 1) // case["page"] for s, c in e]
    touched = sum((s + c - 1) // block - s // block + 1 for s, c in e)
    maps = 4 * (2 * len(e) + sum(pages) + len(e) + 1 + len(e) * max(pages) + 3 * t + 4 * touched)
    store = t * (nq + 2 * nkv) * d * size + t * nq * d * size + 2 * t * nkv * d + 8 * touched * nkv + 4 * t * d
    kept = sum(min(s + c, w + c - 1) if w else s + c for s, c in e)
    seen = sum(min(p + 1, w) if w else p + 1 for s, c in e for p in range(s, s + c))
    attend = 2 * t * nq * d * size + kept * nkv * (2 * d + 8 / block)
    products = 4 * nq * d * seen
    rotation = t * (nq + nkv) * d * 4
    if case["kind"] == "maps":
        return {"bytes": maps, "flops": 0}
    if case["kind"] == "store":
        return {"bytes": store, "flops": rotation}
    if case["kind"] == "attend":
        return {"bytes": attend, "flops": products}
    return {"bytes": maps + case["layers"] * (store + attend), "flops": case["layers"] * (rotation + products)}


# --------------------------------------------------------------------------------------------------- the inputs
def _to8(x, exponent):
    """float32 values at 2^exponent as e4m3 (every finite value fits by the choice of the exponent)."""
    return torch.ldexp(x, -exponent).to(F8)


def _exponent(amax):
    m, e = torch.frexp(amax)                 # amax = m 2^e, m in [1/2, 1); 448 = 7/8 2^9
    e = e - 9 + (m > 0.875).to(e.dtype)
    return torch.where(amax > 0, e, torch.full_like(e, LEAST)).clamp_min(LEAST)


def _filled_cache(g, owner_len, page, nkv, d):
    """Pages with keys and values of ``owner_len`` [pages] tokens each (what earlier steps left)."""
    block = block_of(page)
    pages, nb = owner_len.numel(), page // block
    here = (torch.arange(page, device=DEVICE) < owner_len[:, None]).view(pages, 1, page, 1)
    out = []
    for spread in (0.5, 0.2):                # keys have channels that stand out, values fewer
        x = torch.randn((pages, nkv, page, d), generator=g, device=DEVICE)
        x *= torch.exp(spread * torch.randn((1, nkv, 1, d), generator=g, device=DEVICE))
        x = torch.where(here, x, torch.zeros((), device=DEVICE)).view(pages, nkv, nb, block, d)
        e = _exponent(x.abs().amax(dim=(3, 4)))
        out.append((_to8(x, e[..., None, None]), torch.ldexp(torch.ones_like(e, dtype=torch.float32), e)))
    (k, ks), (v, vs) = out
    return {"keys": k.view(pages, nkv, page, d).contiguous(),
            "values": v.view(torch.uint8).transpose(3, 4).contiguous().view(F8),
            "scales": torch.stack([ks, vs], dim=-1).contiguous()}


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    e, page = entries_of(case), case["page"]
    nq, nkv, d, dtype, kind = case["heads"], case["kv_heads"], case["dim"], TYPES[case["dtype"]], case["kind"]
    block = block_of(page)
    starts, counts = [s for s, _ in e], [c for _, c in e]
    total, nums = sum(counts), [(s + c + page - 1) // page for s, c in e]
    first = [sum(counts[:i]) for i in range(len(e) + 1)]
    num_pages = sum(nums) + 3
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEVICE)  # noqa: E731
    shuffled = torch.randperm(num_pages, generator=g, device=DEVICE).to(torch.int32)[:sum(nums)].contiguous()
    width = max(nums)
    touched = sum((s + c - 1) // block - s // block + 1 for s, c in e)
    state = {"case": case, "entries": e, "page": page, "block": block, "num_pages": num_pages, "start": ints(starts), "count": ints(counts),
             "pages": shuffled, "pages_at": ints([sum(nums[:i]) for i in range(len(e))])}
    # what the maps operator fills (a step's integers); the other operators' programs have them filled
    state["maps"] = {"first_row": ints([0] * (len(e) + 1)), "positions": ints([0] * total), "token_entry": ints([0] * total),
                     "table": torch.zeros((len(e), width), dtype=torch.int32, device=DEVICE), "slots": ints([0] * total),
                     "blocks": torch.zeros((touched, 4), dtype=torch.int32, device=DEVICE)}
    _plain_maps(state)
    if kind == "maps":
        for t in state["maps"].values():
            t.fill_(-7)
        return state
    # tokens that the pages hold: before this step for a store, after it for attention alone
    at = torch.zeros(num_pages, dtype=torch.int64, device=DEVICE)
    have = [(s if kind != "attend" else s + c) for s, c in e]
    fill = [min(page, max(0, h - j * page)) for h, n in zip(have, nums) for j in range(n)]
    at[shuffled.long()] = torch.tensor(fill, device=DEVICE)
    rand = lambda *shape: torch.randn(shape, generator=g, device=DEVICE)  # noqa: E731
    layers = []
    for _ in range(case["layers"]):
        layer = dict(_filled_cache(g, at, page, nkv, d))
        layer["q"] = torch.zeros((total, nq * d), dtype=dtype, device=DEVICE)
        if kind == "attend":
            layer["q"].copy_(1.5 * rand(total, nq * d))
        else:
            layer["qkv"] = rand(total, (nq + 2 * nkv) * d).to(dtype)
        if case["norm"]:
            layer["q_weight"] = (0.9 + 0.2 * torch.rand(d, generator=g, device=DEVICE)).to(dtype)
            layer["k_weight"] = (0.9 + 0.2 * torch.rand(d, generator=g, device=DEVICE)).to(dtype)
        if kind != "store":
            layer["out"] = torch.zeros((total, nq * d), dtype=dtype, device=DEVICE)
            layer["sink"] = rand(nq) if case["sink"] else None
            layer["gate"] = rand(total, nq).to(dtype) if case["gate"] else None
        layers.append(layer)
    state["layers"] = layers
    angle = state["maps"]["positions"].double()[:, None] * torch.pow(torch.tensor(THETA, dtype=torch.float64, device=DEVICE),
                                                                     -torch.arange(d // 2, device=DEVICE).double() * (2.0 / d))
    state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
    # the rows of the single tokens' and of the portions' queries, side by side (a place without a row: the last, of zeros)
    groups = []
    for which in ([i for i, x in enumerate(counts) if x == 1], [i for i, x in enumerate(counts) if x > 1]):
        if which:
            most = max(counts[i] for i in which)
            rows = [[first[i] + j if j < counts[i] else total for j in range(most)] for i in which]
            wide = max(nums[i] for i in which)
            groups.append((torch.tensor(which, device=DEVICE), torch.tensor(rows, device=DEVICE), wide))
    state["groups"] = groups
    if own:
        from pulse_infer_amd.cache.specs import Paged8CacheView
        from pulse_infer_amd.ops import cache8
        from pulse_infer_amd.parts.base import EntryMeta, Workspace

        for layer in layers:
            layer["view"] = Paged8CacheView(0, layer["keys"], layer["values"], layer["scales"], page)
        state["metas"] = [EntryMeta(i, i, s, c, first[i]) for i, (s, c) in enumerate(e)]
        state["workspace"] = Workspace(torch.device(DEVICE))
        # (made once a step, for all its layers; a step of the same shape cuts it anew)
        state["plan"] = cache8.plan(state["metas"], nq, nkv, d, state["maps"]["positions"], page_size=page, dtype=dtype,
                                    window=case["window"], workspace=state["workspace"])
    return state


# ------------------------------------------------------------------------------------------------ the plain forms
def _plain_maps(st):
    start, count, page, block, m = st["start"].long(), st["count"].long(), st["page"], st["block"], st["maps"]
    end = start + count
    first = torch.cat([torch.zeros(1, dtype=torch.int64, device=DEVICE), count.cumsum(0)])
    m["first_row"].copy_(first)
    row = torch.arange(m["positions"].numel(), device=DEVICE)
    entry = torch.searchsorted(first[1:], row, right=True)
    pos = start[entry] + row - first[entry]
    m["positions"].copy_(pos)
    m["token_entry"].copy_(entry)
    held = (end + page - 1) // page
    j = torch.arange(m["table"].shape[1], device=DEVICE)
    at = (held.cumsum(0) - held)[:, None] + j
    table = torch.where(j < held[:, None], st["pages"].long()[at.clamp_max(st["pages"].numel() - 1)], -1)
    m["table"].copy_(table)
    of = table[entry, pos // page]
    m["slots"].copy_(torch.where((of >= 0) & (of < st["num_pages"]), of * page + pos % page, -1))
    n_blocks = (end - 1) // block - start // block + 1
    upto = n_blocks.cumsum(0)
    i = torch.arange(m["blocks"].shape[0], device=DEVICE)
    b = torch.searchsorted(upto, i, right=True)
    number = start[b] // block + i - (upto - n_blocks)[b]
    lo = torch.maximum(number * block, start[b])
    rows = torch.minimum((number + 1) * block, end[b]) - lo
    of = table[b, number * block // page]
    here = torch.where((of >= 0) & (of < st["num_pages"]), of * (page // block) + number % (page // block), -1)
    m["blocks"].copy_(torch.stack([first[b] + lo - start[b], rows, here, lo % block], dim=1))
    return m


def _plain_store(st, layer):
    case, m = st["case"], st["maps"]
    nq, nkv, d, block = case["heads"], case["kv_heads"], case["dim"], st["block"]
    x = layer["qkv"].float()
    total = x.shape[0]
    q, k, v = (t.reshape(total, -1, d) for t in x.split([nq * d, nkv * d, nkv * d], dim=1))
    if case["norm"]:
        q = q / torch.sqrt((q * q).mean(-1, keepdim=True) + EPS) * layer["q_weight"].float()
        k = k / torch.sqrt((k * k).mean(-1, keepdim=True) + EPS) * layer["k_weight"].float()
    cos, sin = st["cos"][:, None], st["sin"][:, None]

    def turn(t):
        a, b = t[..., :d // 2], t[..., d // 2:]
        return torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)

    layer["q"].copy_(turn(q).reshape(total, nq * d))
    # the blocks that the step writes to: earlier bytes at their scale, the new tokens, one new scale over both
    first, rows, number, at = m["blocks"].long().unbind(1)
    place = torch.arange(block, device=DEVICE)
    new = (place >= at[:, None]) & (place < (at + rows)[:, None])
    row = (first[:, None] + place - at[:, None]).clamp(0, total - 1)
    earlier = (at > 0)[:, None, None]
    nb = case["page"] // block
    keys = layer["keys"].view(torch.uint8).view(st["num_pages"], nkv, nb, block, d)
    values, scales = layer["values"].view(torch.uint8), layer["scales"]
    page, inner = number // nb, number % nb
    for which, held, fresh in ((0, keys, turn(k)), (1, values, v)):
        old = held[page, :, inner].view(F8).float()
        old = old if which == 0 else old.transpose(2, 3)                                    # [blocks, heads, token, channel]
        was = torch.frexp(scales[page, :, inner, which])[1] - 1
        was = torch.where(earlier[:, :, 0], was, torch.full_like(was, LEAST))
        old = torch.where(earlier[..., None], old, torch.zeros((), device=DEVICE))
        token = fresh[row].transpose(1, 2)                                                  # [blocks, heads, token, channel]
        mask = new[:, None, :, None]
        amax = torch.where(mask, token.abs(), torch.zeros((), device=DEVICE)).amax(dim=(2, 3))
        e = torch.maximum(was, _exponent(amax))
        both = torch.where(mask, _to8(token, e[..., None, None]).float(), _to8(old, (e - was)[..., None, None]).float()).to(F8)
        both = both.view(torch.uint8)
        held[page, :, inner] = both if which == 0 else both.transpose(2, 3)
        scales[page, :, inner, which] = torch.ldexp(torch.ones_like(e, dtype=torch.float32), e)
    return {"q": layer["q"], "keys": layer["keys"], "values": layer["values"], "scales": layer["scales"]}


def _plain_attend(st, layer):
    case, m = st["case"], st["maps"]
    nq, nkv, d, page, block = case["heads"], case["kv_heads"], case["dim"], case["page"], st["block"]
    group = nq // nkv
    q = torch.cat([layer["q"].float(), torch.zeros((1, nq * d), device=DEVICE)]).view(-1, nkv, group, d)
    positions = torch.cat([m["positions"].long(), torch.full((1,), -1, device=DEVICE)])
    out = torch.zeros((q.shape[0], nkv, group, d), device=DEVICE)
    nb = page // block
    for which, rows, width in st["groups"]:      # (at most two: the single tokens, the portions)
        n, most = rows.shape
        at = m["table"][which, :width].long()
        at = at.clamp_min(0)                     # (pages that a shorter request has not: their keys are masked)
        scale = layer["scales"][at]
        keys = layer["keys"].view(torch.uint8)[at].view(F8).float().view(n, width, nkv, nb, block, d)
        keys = (keys * scale[..., 0, None, None]).permute(0, 2, 1, 3, 4, 5).reshape(n, nkv, width * page, d)
        values = layer["values"].view(torch.uint8)[at].view(F8).float().view(n, width, nkv, nb, d, block)
        values = (values * scale[..., 1, None, None]).permute(0, 2, 1, 3, 5, 4).reshape(n, nkv, width * page, d)
        qs = q[rows].permute(0, 2, 3, 1, 4).reshape(n, nkv, group * most, d)
        s = torch.matmul(qs, keys.transpose(2, 3).contiguous()).view(n, nkv, group, most, width * page) * d ** -0.5
        if case["cap"]:
            s = case["cap"] * torch.tanh(s / case["cap"])
        pos = positions[rows][:, None, None, :, None]
        j = torch.arange(width * page, device=DEVICE)
        seen = j <= pos
        if case["window"]:
            seen = seen & (j > pos - case["window"])
        s = torch.where(seen, s, torch.full((), -math.inf, device=DEVICE))
        top = s.amax(-1, keepdim=True)
        if layer["sink"] is not None:
            top = torch.maximum(top, layer["sink"].view(1, nkv, group, 1, 1))
        top = torch.where(torch.isinf(top), torch.zeros((), device=DEVICE), top)
        p = torch.exp(s - top)
        total = p.sum(-1, keepdim=True)
        if layer["sink"] is not None:
            total = total + torch.exp(layer["sink"].view(1, nkv, group, 1, 1) - top)
        o = torch.matmul(p.view(n, nkv, group * most, -1), values).view(n, nkv, group, most, d)
        out[rows] = (o / torch.where(total > 0, total, torch.ones((), device=DEVICE))).permute(0, 3, 1, 2, 4)
    out = out[:-1].reshape(-1, nq, d)
    if layer["gate"] is not None:
        out = out * torch.sigmoid(layer["gate"].float())[..., None]
    layer["out"].copy_(out.reshape(-1, nq * d))
    return layer["out"]


# ------------------------------------------------------------------------------------------------------- a pass
def _maps(st):
    if not own:
        return _plain_maps(st)
    from pulse_infer_amd.ops import cache8

    cache8.step_maps(st["start"], st["count"], page_size=st["page"], num_pages=st["num_pages"], pages=st["pages"], block=st["block"],
                     **st["maps"])
    return st["maps"]


def _store(st, layer):
    if not own:
        return _plain_store(st, layer)
    from pulse_infer_amd.ops import cache8

    case, m = st["case"], st["maps"]
    cache8.store(layer["qkv"], layer["q"], case["heads"], case["kv_heads"], case["dim"], layer["view"], m["positions"], m["blocks"],
                 q_weight=layer.get("q_weight"), k_weight=layer.get("k_weight"), eps=EPS, cos=st["cos"], sin=st["sin"],
                 rotary_dim=case["dim"], pairing=1)
    return {"q": layer["q"], "keys": layer["keys"], "values": layer["values"], "scales": layer["scales"]}


def _attend(st, layer):
    if not own:
        return _plain_attend(st, layer)
    from pulse_infer_amd.ops import cache8

    case, m = st["case"], st["maps"]
    cache8.attention(layer["q"], layer["out"], st["plan"], layer["view"], m["positions"], m["token_entry"], m["table"],
                     case["dim"] ** -0.5, gate=layer["gate"], sink=layer["sink"], softcap=case["cap"])
    return layer["out"]


def run(st):
    kind = st["case"]["kind"]
    if kind == "maps":
        return dict(_maps(st))
    if kind == "store":
        return _store(st, st["layers"][0])
    if kind == "attend":
        return _attend(st, st["layers"][0])
    _maps(st)
    if own:
        st["plan"].cut(st["maps"]["positions"])
    out = {}
    for i, layer in enumerate(st["layers"]):
        out[f"stored{i}"] = _store(st, layer)
        out[f"out{i}"] = _attend(st, layer)
    return out


# ------------------------------------------------------------------------------------------- the same in 64 bits
def _round8(x):
    """The e4m3 number nearest to x (float64, |x| <= 448), ties to the even one: steps of 2^-3 of the value's power of two, of 2^-9
    below 2^-6."""
    e = torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -20))).clamp_min(-6)
    step = torch.pow(torch.tensor(2.0, dtype=torch.float64, device=x.device), e - 3)
    return torch.round(x / step) * step


def _decode8(b):
    """What bytes stand for, in float64: sign, four bits of exponent (bias 7), three of fraction."""
    b = b.view(torch.uint8).to(torch.int64)
    e, f = (b >> 3) & 15, (b & 7).double()
    size = torch.where(e > 0, (1 + f / 8) * torch.pow(torch.tensor(2.0, dtype=torch.float64, device=b.device), (e - 7).double()), f * 2.0 ** -9)
    return torch.where(b >= 128, -size, size)


def _exact_maps(case, st):
    page, block, pages = case["page"], st["block"], st["pages"].tolist()
    out = {k: [] for k in ("first_row", "positions", "token_entry", "table", "slots", "blocks")}
    row = at = 0
    for b, (s, c) in enumerate(st["entries"]):
        mine = pages[at:at + -(-(s + c) // page)]
        at += len(mine)
        out["first_row"].append(row)
        out["table"].append(mine + [-1] * (st["maps"]["table"].shape[1] - len(mine)))
        for p in range(s, s + c):
            out["positions"].append(p)
            out["token_entry"].append(b)
            out["slots"].append(mine[p // page] * page + p % page)
        p = s
        while p < s + c:
            n = min(block - p % block, s + c - p)
            out["blocks"].append([row + p - s, n, mine[p // page] * (page // block) + p % page // block, p % block])
            p += n
        row += c
    out["first_row"].append(row)
    return {k: torch.tensor(v, dtype=torch.int32) for k, v in out.items()}


def _exact_store(case, st, layer):
    nq, nkv, d, block, page = case["heads"], case["kv_heads"], case["dim"], st["block"], case["page"]
    x = layer["qkv"].double().view(-1, nq + 2 * nkv, d)
    angle = st["maps"]["positions"].double()[:, None] / THETA ** (torch.arange(d // 2, device=DEVICE).double() * 2 / d)
    spin = torch.polar(torch.ones_like(angle), angle)[:, None]

    def made(heads, weight):
        if weight is not None:
            heads = heads * torch.rsqrt(heads.square().mean(-1, keepdim=True) + EPS) * weight.double()
        z = torch.complex(heads[..., :d // 2], heads[..., d // 2:]) * spin
        return torch.cat([z.real, z.imag], -1)

    q, k, v = made(x[:, :nq], layer.get("q_weight")), made(x[:, nq:nq + nkv], layer.get("k_weight")), x[:, nq + nkv:]
    keys, values = _decode8(layer["keys"]), _decode8(layer["values"])
    scales = layer["scales"].double().clone()
    nb = page // block
    for first, rows, number, at in st["maps"]["blocks"].tolist():
        p, inner = divmod(number, nb)
        for which, new, held in ((0, k, keys[p, :, inner * block:(inner + 1) * block]), (1, v, values[p, :, inner].transpose(1, 2))):
            token = new[first:first + rows].transpose(0, 1)
            need = (torch.ceil(torch.log2(token.abs().amax(dim=(1, 2)) / 448).clamp_min(LEAST)))
            was = torch.log2(scales[p, :, inner, which]) if at else torch.full_like(need, LEAST)
            if not at:
                held.zero_()
            e = torch.maximum(was, need)
            held.copy_(_round8(held * torch.pow(2.0, was - e)[:, None, None]))
            held[:, at:at + rows] = _round8(token * torch.pow(2.0, -e)[:, None, None])
            scales[p, :, inner, which] = torch.pow(2.0, e)
    return {"q": q.reshape(q.shape[0], -1), "keys": keys, "values": values, "scales": scales}


def _exact_attend(case, st, q, keys, values, scales, layer):
    nq, nkv, d, page, block = case["heads"], case["kv_heads"], case["dim"], case["page"], st["block"]
    out = torch.zeros((q.shape[0], nq, d), dtype=torch.float64, device=DEVICE)
    q = q.double().view(-1, nq, d)
    row = 0
    for b, (s, c) in enumerate(st["entries"]):
        length = s + c
        lo = max(0, s - case["window"] + 1) if case["window"] else 0
        at = st["maps"]["table"][b, lo // page:-(-length // page)].long()
        base = lo // page * page
        w = at.numel() * page
        size = scales[at].double().repeat_interleave(block, dim=2).transpose(0, 1).reshape(nkv, w, 2)
        k = keys(at).transpose(0, 1).reshape(nkv, w, d) * size[..., :1]
        v = values(at).transpose(3, 4).transpose(0, 1).reshape(nkv, w, d) * size[..., 1:]
        j, i = torch.arange(base, base + w, device=DEVICE), torch.arange(s, length, device=DEVICE)[:, None]
        hidden = (j > i) | (j <= i - case["window"]) if case["window"] else j > i
        for h in range(nq):
            x = q[row:row + c, h] @ k[h * nkv // nq].T.contiguous() / math.sqrt(d)
            if case["cap"]:
                x = torch.tanh(x / case["cap"]) * case["cap"]
            x = x.masked_fill(hidden, -math.inf)
            if layer["sink"] is not None:
                x = torch.cat([x, layer["sink"][h].double().expand(c, 1)], 1)
            o = torch.softmax(x, -1)[:, :w] @ v[h * nkv // nq]
            if layer["gate"] is not None:
                o = o * torch.sigmoid(layer["gate"][row:row + c, h].double())[:, None]
            out[row:row + c, h] = o
        row += c
    return out.reshape(-1, nq * d)


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "maps":
        return _exact_maps(case, st)
    if case["kind"] == "store":
        return _exact_store(case, st, st["layers"][0])
    if case["kind"] == "attend":
        layer = st["layers"][0]
        return _exact_attend(case, st, layer["q"], lambda at: _decode8(layer["keys"].view(torch.uint8)[at]),
                             lambda at: _decode8(layer["values"].view(torch.uint8)[at]), layer["scales"], layer)
    if sum((c + 15) // 16 + 1 for _, c in st["entries"]) * case["layers"] > 4000:
        return None
    out = {}
    for n, layer in enumerate(st["layers"]):
        put = _exact_store(case, st, layer)
        # (the attention reads the queries as they are stored)
        q = put["q"].to(TYPES[case["dtype"]])
        out[f"stored{n}"] = put
        out[f"out{n}"] = _exact_attend(case, st, q, lambda at: put["keys"][at], lambda at: put["values"][at], put["scales"], layer)
    return out

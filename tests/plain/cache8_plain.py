"""A cache of keys and values in 8 bits in plain torch, float64, on the CPU: the maps, the store and the attention, each from its formula."""
from __future__ import annotations

import math

import torch

LEAST = -118
F64 = torch.float64


def block_of(page):
    return 16 if page % 16 == 0 else page


def decode(b):
    """What e4m3 bytes stand for."""
    b = b.cpu().view(torch.uint8).long()
    e, f = (b >> 3) & 15, (b & 7).to(F64)
    x = torch.where(e > 0, (1 + f / 8) * 2.0 ** (e - 7).to(F64), f * 2.0 ** -9)
    x = torch.where((b & 127) == 127, torch.full_like(x, math.nan), x)
    return torch.where(b >= 128, -x, x)


def nearest(x):
    """The e4m3 number nearest to x, |x| <= 448, ties to even; NaN for what is not finite."""
    ok = torch.isfinite(x)
    y = torch.where(ok, x, torch.zeros_like(x))
    e = torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -20))).clamp_min(-6)
    step = 2.0 ** (e - 3)
    return torch.where(ok, torch.round(y / step) * step, torch.full_like(x, math.nan))


def exponent(amax):
    """The least e >= LEAST with amax <= 448 2^e."""
    e = torch.ceil(torch.log2(amax.clamp_min(2.0 ** -140) / 448.0))
    e = torch.where(amax > 448.0 * 2.0 ** e, e + 1, e)
    e = torch.where(amax <= 448.0 * 2.0 ** (e - 1), e - 1, e)
    return e.clamp_min(LEAST)


def maps(entries, pages, page, num_pages, width, block=None):
    """entries [(start, count)], pages: the list of all requests' pages."""
    block = block or block_of(page)
    out = {k: [] for k in ("first_row", "positions", "token_entry", "table", "slots", "blocks")}
    row = at = 0
    for b, (s, c) in enumerate(entries):
        held = -(-(s + c) // page)
        mine = [pages[i] if i < len(pages) else -1 for i in range(at, at + held)]
        at += held
        ok = [0 <= p < num_pages for p in mine]
        out["first_row"].append(row)
        out["table"].append((mine + [-1] * width)[:width])
        for p in range(s, s + c):
            out["positions"].append(p)
            out["token_entry"].append(b)
            out["slots"].append(mine[p // page] * page + p % page if ok[p // page] else -1)
        p = s
        while p < s + c:
            n = min(block - p % block, s + c - p)
            out["blocks"].append([row + p - s, n, mine[p // page] * (page // block) + p % page // block if ok[p // page] else -1, p % block])
            p += n
        row += c
    out["first_row"].append(row)
    return out


def prepared(qkv, nq, nkv, d, v_head0=None, q_w=None, k_w=None, eps=0.0, plain_norm=False, angles=None, rotary_dim=0, pairing=0,
             temperature=None, positions=None):
    """(q, k, v) [T, heads, d] after norm, temperature and rotation."""
    x = qkv.cpu().to(F64)
    t = x.shape[0]
    v0 = nq + nkv if v_head0 is None else v_head0
    q, k, v = (x[:, a * d:(a + n) * d].reshape(t, n, d).clone() for a, n in ((0, nq), (nq, nkv), (v0, nkv)))

    def norm(h, w):
        h = h / torch.sqrt(h.square().mean(-1, keepdim=True) + eps)
        return h if w is None else h * w.cpu().to(F64)

    if q_w is not None or plain_norm:
        q, k = norm(q, q_w), norm(k, k_w)
    if temperature is not None:
        coef, every = temperature
        f = 1 + coef * torch.log(torch.div(positions.cpu().to(F64) + 1, every, rounding_mode="floor") + 1)
        q = q * f[:, None, None]
    if angles is not None:
        half = rotary_dim // 2
        a, b = (slice(0, rotary_dim, 2), slice(1, rotary_dim, 2)) if pairing == 0 else (slice(0, half), slice(half, rotary_dim))
        cos, sin = torch.cos(angles.cpu().to(F64))[:, None], torch.sin(angles.cpu().to(F64))[:, None]
        for h in (q, k):
            u, w = h[..., a].clone(), h[..., b].clone()
            h[..., a], h[..., b] = u * cos - w * sin, u * sin + w * cos
    return q, k, v


class Cache:
    """Values at exponents, whole: keys and values [pages, heads, blocks, block, d] (float64 e4m3 numbers), exponents [..., 2]."""

    def __init__(self, pages, nkv, page, d):
        self.page, self.block = page, block_of(page)
        self.nb = page // self.block
        shape = (pages, nkv, self.nb, self.block, d)
        self.x = [torch.zeros(shape, dtype=F64), torch.zeros(shape, dtype=F64)]
        self.e = torch.full((pages, nkv, self.nb, 2), LEAST, dtype=F64)
        self.marked = torch.zeros((pages, nkv, self.nb), dtype=torch.bool)

    def store(self, k, v, blocks):
        for first, rows, number, at in blocks:
            if rows <= 0 or number < 0:
                continue
            p, inner = divmod(number, self.nb)
            for which, new in ((0, k), (1, v)):
                held, tok = self.x[which][p, :, inner], new[first:first + rows].transpose(0, 1)
                if at == 0:
                    held.zero_()
                    self.e[p, :, inner, which] = LEAST
                    if which == 1:
                        self.marked[p, :, inner] = False
                ok = torch.isfinite(tok)
                amax = torch.where(ok, tok.abs(), torch.zeros_like(tok)).amax(dim=(1, 2))
                was = self.e[p, :, inner, which].clone()
                e = torch.maximum(was, exponent(amax))
                held.copy_(nearest(held * 2.0 ** (was - e)[:, None, None]))
                held[:, at:at + rows] = nearest(tok * 2.0 ** -e[:, None, None])
                self.e[p, :, inner, which] = e
                if which == 1:
                    self.marked[p, :, inner] |= ~ok.all(dim=2).all(dim=1)

    def tensors(self):
        """As the kernels hold them."""
        pages, nkv, nb, block, d = self.x[0].shape
        keys = self.x[0].to(torch.float32).to(torch.float8_e4m3fn).view(pages, nkv, self.page, d)
        values = self.x[1].to(torch.float32).to(torch.float8_e4m3fn).view(torch.uint8).transpose(3, 4).contiguous().view(torch.float8_e4m3fn)
        scales = (2.0 ** self.e).to(torch.float32)
        scales[..., 1] = torch.where(self.marked, -scales[..., 1], scales[..., 1])
        return keys, values, scales

    def rows(self, pages):
        """Keys and values [heads, tokens, d] of a request's pages, as float64."""
        out = []
        for which in (0, 1):
            x = self.x[which][pages] * (2.0 ** self.e[pages][..., which])[..., None, None]     # [n, heads, nb, block, d]
            out.append(x.permute(1, 0, 2, 3, 4).reshape(x.shape[1], -1, x.shape[-1]))
        return out


def attention(q, cache, entries, table, scale, window=0, chunk=0, softcap=0.0, sink=None, gate=None, gate_width=0, num_pages=None):
    """(out, sum of weights times |values|, largest sum |q||k| scale of a row) [T, nq, d]: the rows of ``entries`` [(start, count)]."""
    t, nq, d = q.shape
    nkv = cache.x[0].shape[1]
    out, mass, size = torch.zeros_like(q), torch.zeros_like(q), torch.zeros((t, nq, 1), dtype=F64)
    num_pages = num_pages or cache.x[0].shape[0]
    row = 0
    for b, (s, c) in enumerate(entries):
        held = -(-(s + c) // cache.page)
        pages = [int(p) for p in table[b][:held]]
        there = torch.tensor([0 <= p < num_pages for p in pages]).repeat_interleave(cache.page)
        keys, values = cache.rows([p if 0 <= p < num_pages else 0 for p in pages])
        j, pos = torch.arange(held * cache.page), torch.arange(s, s + c)[:, None]
        lo = pos - pos % chunk if chunk else (pos - window + 1).clamp_min(0) if window else torch.zeros_like(pos)
        seen = (j >= lo) & (j <= pos) & there
        hides = seen[:, :, None]
        for h in range(nq if c else 0):
            kk, vv = keys[h * nkv // nq], values[h * nkv // nq]
            # (what is not finite counts where it is seen alone)
            x = torch.where(seen, q[row:row + c, h] @ torch.nan_to_num(kk).T * scale, torch.full((), -math.inf, dtype=F64))
            x = torch.where(seen & torch.isnan(kk).any(-1), torch.full((), math.nan, dtype=F64), x)
            size[row:row + c, h, 0] = torch.where(seen, q[row:row + c, h].abs() @ torch.nan_to_num(kk).abs().T, torch.zeros((), dtype=F64)).amax(-1) * scale
            if softcap:
                x = torch.where(seen, softcap * torch.tanh(x / softcap), x)
            if sink is not None:
                x = torch.cat([x, sink[h].cpu().to(F64).expand(c, 1)], 1)
            p = torch.where(seen.any(-1, keepdim=True), torch.softmax(x, -1)[:, :j.numel()], torch.zeros((), dtype=F64))
            out[row:row + c, h] = p @ torch.nan_to_num(vv)
            mass[row:row + c, h] = p @ torch.nan_to_num(vv).abs()
            spoilt = (hides & torch.isnan(vv)[None]).any(1) if torch.isnan(vv).any() else torch.zeros((c, d), dtype=torch.bool)
            out[row:row + c, h][spoilt] = math.nan
        row += c
    if gate is not None:
        g = torch.sigmoid(gate.cpu().to(F64))
        f = torch.ones_like(out)
        if gate_width:
            f[..., :gate_width] = g[:, :nq * gate_width].reshape(t, nq, gate_width)
        else:
            f = f * g[:, :nq, None]
        out, mass = out * f, mass * f
    return out, mass, size

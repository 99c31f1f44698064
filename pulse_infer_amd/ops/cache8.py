"""A cache of keys and values in 8 bits: the step's maps, the store and the attention over it.

Bytes are e4m3 numbers.  A block is 16 tokens of a page (the whole page where 16 does not divide its size); of a block and kv head the keys
share a scale and the values another, powers of two that grow with what the block holds (``csrc/cache8.h`` has the formulas).  The pages are
a ``Paged8CacheView``'s; ``cache/specs.py`` allocates them.

A step makes its maps once (``step_maps``: rows, positions, block tables, slots and the blocks it writes to, from the requests' lengths),
plans its attention once (``plan``, and ``cut`` for every further step of the same shape), and then calls ``store`` and ``attention`` in
every layer.  As elsewhere in this package, tensors are checked on the host, kernels are queued on torch's current stream, and nothing
falls back to another implementation.
"""
from __future__ import annotations

import struct
from typing import Any, Callable, List, Optional, Sequence, Tuple

import torch

from ..cache.specs import Paged8CacheView, block_tokens
from .device import compute_units
from .kernels import _TAG, _gpu, _i32, _need, _ptr, _stream, _tag
from .library import KernelError, call

MAX_REQUESTS = 4096          # of step_maps
MAX_HEAD_DIM = 512           # of store and of attention
INF = float("inf")
MAX_PIECES = 65535           # of a launch's grid
PIECE_INTS = 12              # of a piece of work (csrc/cache8_attn.h)
TILE = 64                    # keys of a step of the matrix-core kernels
MATRIX_CAP = 256.0           # the largest cap of those kernels, which have a capped score to 2^-22 of the cap: of 256 6e-5, where a weight is rounded by 2^-8
FEW, MANY = 16, 128          # columns (rows times the heads that share a kv head) of an item of the two matrix-core kernels


def _refuse(what: str, why: str) -> None:
    raise KernelError(f"{what}: {why}")


# (The checks are plain conditions whose messages are put together only when they fail: a dozen formatted messages that nobody reads
# took longer than the kernels of a decoding step do.)
def _here(what: str, tensors: Sequence[Optional[torch.Tensor]]) -> None:
    """All of them on the current GPU, whose stream the kernels are queued on."""
    current = -1
    for t in tensors:
        if t is None:
            continue
        index = t.get_device()
        if current < 0:
            _gpu(what, t)
            current = torch.cuda.current_device()
        if index != current:
            _gpu(what, t)
            _refuse(what, f"a tensor lies on {t.device}, the current GPU is cuda:{current}")


def _ints(what: str, name: str, t: torch.Tensor, n: int) -> None:
    if t.dtype != torch.int32 or not t.is_contiguous() or t.numel() < n:
        _refuse(what, f"{name} must be a contiguous int32 tensor of {n} numbers at least")


def _pages(what: str, view: Paged8CacheView, nkv: int, d: int) -> Tuple[int, int]:
    """(pages, tokens a page) of a cache that is what the kernels take it for."""
    keys, values, scales, page = view.keys, view.values, view.scales, view.page_size
    block = 16 if page % 16 == 0 else page      # (block_tokens)
    shape = keys.shape
    pages = shape[0]
    if shape != (pages, nkv, page, d) or values.shape != (pages, nkv, page // block, d, block) or scales.shape != (pages, nkv, page // block, 2):
        _refuse(what, f"the cache is {tuple(keys.shape)}, {tuple(values.shape)}, {tuple(scales.shape)}, expected {(pages, nkv, page, d)}, "
                      f"{(pages, nkv, page // block, d, block)}, {(pages, nkv, page // block, 2)}")
    if keys.dtype != torch.float8_e4m3fn or values.dtype != torch.float8_e4m3fn or scales.dtype != torch.float32:
        _refuse(what, "keys and values must be float8_e4m3fn, their scales float32")
    if not (keys.is_contiguous() and values.is_contiguous() and scales.is_contiguous()) or (keys.data_ptr() | values.data_ptr() | scales.data_ptr()) % 16:
        _refuse(what, "the cache must be contiguous and aligned to 16 bytes")
    return pages, page


def _apart(rows: int, size: int, at_a: int, step_a: int, a: int, at_b: int, step_b: int, b: int) -> bool:
    """Whether ``rows`` rows of ``a`` numbers of ``size`` bytes from address ``at_a`` on, ``step_a`` numbers apart, have no byte in common with as
    many rows of ``b`` from ``at_b`` on."""
    if at_b >= at_a + ((rows - 1) * step_a + a) * size or at_a >= at_b + ((rows - 1) * step_b + b) * size:
        return True
    between = (at_b - at_a) % (step_a * size) if step_a else 0      # (rows of one buffer beside each other)
    return rows > 1 and step_a == step_b and between >= a * size and between + b * size <= step_a * size


# The arguments of the entry points as the structures of csrc/cache8_maps.hip, cache8_store.hip and cache8_attn.h, put together at once.
_MAPS = struct.Struct("@9Q8i")
_STORE = struct.Struct("@QqQq9Q14i2fQ3q")
_ATTN = struct.Struct("@QqQq7Qq5Q16i2f")


def _at(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _block_list(what: str, blocks: torch.Tensor) -> int:
    shape = blocks.shape
    if blocks.dtype != torch.int32 or len(shape) != 2 or shape[1] != 4 or not blocks.is_contiguous() or blocks.data_ptr() % 16:
        _refuse(what, "blocks must be contiguous int32 [n, 4], aligned to 16 bytes")
    return shape[0]


# ------------------------------------------------------------------------------------------------------------- the maps
def step_maps(start: torch.Tensor, count: torch.Tensor, *, page_size: int, num_pages: int, pages: Optional[torch.Tensor] = None,
              table: Optional[torch.Tensor] = None, first_row: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None,
              token_entry: Optional[torch.Tensor] = None, slots: Optional[torch.Tensor] = None, blocks: Optional[torch.Tensor] = None,
              block: int = 0) -> None:
    """What a step's kernels have to know about rows and pages, from its requests' lengths, in one launch.

    ``start``, ``count`` int32 [B]: tokens of each request in the cache, tokens of this step (0: the request brings none).  ``pages``
    int32: the requests' pages one request after the other, ceil((start + count) / page_size) each.  All further tensors are int32
    and filled where given: ``first_row`` [B + 1] (sums of counts), ``positions``, ``token_entry``, ``slots`` [T] (page * page_size +
    place in the page, -1 where the page is none of the pool's ``num_pages``), ``table`` [B, width] (a request's pages, then -1; pages
    beyond the width are left out) and ``blocks`` [n, 4]: the blocks of ``block`` tokens that the step writes to, request by request
    (first row, rows, the block's number page * (page_size / block) + block in the page or -1, place in the block of the first row);
    places that are left over say "no rows".  Without ``pages``, ``table`` is read instead of written.  Rows behind the last request's are
    left as they were; what does not fit is left out.  T < 2^31, start + count < 2^31,
    num_pages * page_size < 2^31, B <= 4096."""
    what = "step_maps"
    _here(what, (start, count, pages, table, first_row, positions, token_entry, slots, blocks))
    n = start.numel()
    _ints(what, "start", start, 1)
    _ints(what, "count", count, 1)
    if n > MAX_REQUESTS or count.numel() != n:
        _refuse(what, f"lengths of {n} and {count.numel()} requests (1 to {MAX_REQUESTS})")
    if page_size <= 0 or num_pages <= 0 or page_size * num_pages >= 2 ** 31:
        _refuse(what, f"{num_pages} pages of {page_size} tokens")
    block = block or block_tokens(page_size)
    if block <= 0 or page_size % block:
        _refuse(what, f"blocks of {block} tokens do not divide pages of {page_size}")
    listed = width = places = 0
    rows = -1
    for name, t in (("positions", positions), ("token_entry", token_entry), ("slots", slots)):
        if t is not None:
            _ints(what, name, t, 0)
            if rows >= 0 and t.numel() != rows:
                _refuse(what, f"{name} of {t.numel()} rows beside {rows}")
            rows = t.numel()
    if first_row is not None:
        _ints(what, "first_row", first_row, n + 1)
    if pages is not None:
        _ints(what, "pages", pages, 1)
        listed = pages.numel()
    if table is not None:
        shape = table.shape
        if table.dtype != torch.int32 or len(shape) != 2 or not table.is_contiguous() or shape[0] != n or shape[1] < 1:
            _refuse(what, f"the table must be contiguous int32 [{n}, width]")
        width = shape[1]
    if pages is None and table is None and not (slots is None and blocks is None):
        _refuse(what, "slots and blocks need the pages or the table")
    if blocks is not None:
        places = _block_list(what, blocks)
    call("pulse_step_maps", _MAPS.pack(start.data_ptr(), count.data_ptr(), _at(pages), _at(first_row), _at(positions), _at(token_entry),
                                       _at(slots), _at(table), _at(blocks), n, listed, page_size, num_pages, block, max(rows, 0), width,
                                       places), _stream())


def blocks_touched(entries: Sequence[Any], page_size: int) -> int:
    """Places of ``step_maps``'s ``blocks`` that a step of these entries takes."""
    block = block_tokens(page_size)
    return sum((e.start + e.count - 1) // block - e.start // block + 1 for e in entries if e.count > 0)


# ------------------------------------------------------------------------------------------------------------- the store
def store(qkv: torch.Tensor, q_out: torch.Tensor, nq: int, nkv: int, d: int, view: Paged8CacheView, positions: torch.Tensor,
          blocks: torch.Tensor, *, q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, eps: float = 0.0,
          cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None, rotary_dim: int = 0, pairing: int = 0,
          plain_norm: bool = False, v_head0: Optional[int] = None, q_temperature: Optional[tuple] = None,
          parts: Optional[torch.Tensor] = None) -> None:
    """A step's rows of the fused projection: norm and rotation of q (to ``q_out`` [T, >= nq * d], which may be the front of ``qkv``) and k,
    k and v into the blocks that ``step_maps`` listed.  The options are those of ``kernels.qk_rope_kv``.

    Of a block that is begun (its first token among the new ones) nothing that it held before stays; behind the new tokens it holds
    zeros.  Of another the earlier bytes stay, moved to the new scale where that has grown.  A block may be listed once: requests do
    not share pages that a step writes to.  ``qkv`` [T, columns] bfloat16 or float32 with contiguous rows; heads of an even number of
    channels up to 512.  ``parts`` float32 [shares, T, columns]: the rows are the sum of these shares, in their order, and of ``qkv``
    nothing is read (``store_takes_parts``)."""
    what = "store"
    _here(what, (qkv, q_out, view.keys, view.values, view.scales, positions, blocks, q_weight, k_weight, cos, sin, parts))
    if not view.writable:
        _refuse(what, "the cache is another run's")
    if nq <= 0 or nkv <= 0 or d <= 0 or d % 2 or d > MAX_HEAD_DIM:
        _refuse(what, f"heads of {d} channels (even, up to {MAX_HEAD_DIM})")
    pages, page = _pages(what, view, nkv, d)
    v_head0 = nq + nkv if v_head0 is None else int(v_head0)
    columns = max(nq + nkv, v_head0 + nkv) * d
    shape, to = qkv.shape, q_out.shape
    if len(shape) != 2 or v_head0 < 0 or shape[1] < columns or qkv.stride(1) != 1:
        _refuse(what, f"qkv must be [T, {columns}] with contiguous rows")
    tokens = shape[0]
    if len(to) != 2 or to[0] != tokens or to[1] < nq * d or q_out.stride(1) != 1 or q_out.dtype != qkv.dtype:
        _refuse(what, f"q_out must be [{tokens}, {nq * d}] of qkv's storage type with contiguous rows")
    stride, q_stride = qkv.stride(0), q_out.stride(0)
    if tokens > 1 and (stride < columns or q_stride < nq * d):
        _refuse(what, "rows that overlap")
    qkv_at, q_at = qkv.data_ptr(), q_out.data_ptr()
    if tokens and parts is None:
        if qkv_at == q_at and (tokens == 1 or stride == q_stride):
            if v_head0 < nq:
                _refuse(what, f"values from head {v_head0} on lie among the {nq} heads of q that q_out takes the place of")
        elif not _apart(tokens, qkv.element_size(), qkv_at, stride, columns, q_at, q_stride, nq * d):
            _refuse(what, "q_out overlaps rows of qkv (it may be their front, or lie apart)")
    _ints(what, "positions", positions, tokens)
    places = _block_list(what, blocks)
    if (q_weight is None) != (k_weight is None) or (plain_norm and q_weight is not None):
        _refuse(what, "bad norm options")
    w_tag = rotated = 0
    if q_weight is not None:
        if (q_weight.numel() != d or k_weight.numel() != d or q_weight.dtype != k_weight.dtype or not q_weight.is_contiguous()
                or not k_weight.is_contiguous()):
            _refuse(what, f"the two norm weights must hold {d} values of one storage type")
        w_tag = _tag(q_weight, what)
    if (cos is None) != (sin is None):
        _refuse(what, "the rotation needs both of its tables")
    if cos is not None:
        rotated = rotary_dim
        if rotary_dim % 2 or not 0 < rotary_dim <= d or pairing not in (0, 1):
            _refuse(what, f"bad rotation of {rotary_dim} channels")
        shape = cos.shape
        if (shape != sin.shape or len(shape) != 2 or shape[0] < tokens or shape[1] != rotary_dim // 2 or cos.dtype != torch.float32
                or sin.dtype != torch.float32 or not cos.is_contiguous() or not sin.is_contiguous()):
            _refuse(what, f"cos/sin must be float32 [T, {rotary_dim // 2}]")
    coef, every = 0.0, 0
    if q_temperature is not None:
        coef, every = float(q_temperature[0]), int(q_temperature[1])
        if every <= 0:
            _refuse(what, "the query temperature's interval must be positive")
    shares = part_stride = part_row = 0
    if parts is not None:
        if parts.dtype != torch.float32 or parts.dim() != 3 or parts.shape[1] != tokens or parts.shape[2] < columns or not parts.is_contiguous():
            _refuse(what, f"the shares must be contiguous float32 [shares, {tokens}, {columns}]")
        shares, part_stride, part_row = parts.shape[0], parts.stride(0), parts.shape[2]
        if not store_takes_parts(qkv, d, rotated, page, parts, q_out, q_weight, k_weight, cos, sin) or part_row % 4 or q_stride % 4 or shares < 1:
            _refuse(what, "shares need bfloat16 rows, aligned, in chunks of eight channels, and pages of a multiple of 16 tokens")
    if tokens == 0:       # (whose tensors have no addresses)
        return
    call("pulse_store8", _STORE.pack(
        qkv_at, stride, q_at, q_stride, _at(q_weight), _at(k_weight), _at(cos), _at(sin), view.keys.data_ptr(),
        view.values.data_ptr(), view.scales.data_ptr(), positions.data_ptr(), blocks.data_ptr(), _tag(qkv, what), w_tag, rotated, pairing,
        pages, page, places, tokens, nq, nkv, d, plain_norm, v_head0, every, eps, coef, _at(parts), part_stride, part_row, shares), _stream())


def store_takes_parts(qkv: torch.Tensor, d: int, rotary_dim: int, page_size: int, *others: Optional[torch.Tensor]) -> bool:
    """Whether ``store`` takes these rows as float32 shares: in pieces that neither heads nor rotation cut (``others``: the norms' weights
    and the rotation's tables)."""
    return (qkv.dtype == torch.bfloat16 and d % 8 == 0 and rotary_dim % 8 == 0 and page_size % 16 == 0 and qkv.stride(0) % 4 == 0
            and all(t is None or t.data_ptr() % 16 == 0 for t in (qkv, *others)))


# --------------------------------------------------------------------------------------------------------- the attention
def matrix_cores(d: int, page_size: int, dtype: torch.dtype) -> bool:
    """Whether attention runs on the matrix cores; anything else goes to the kernel that serves every size."""
    return dtype == torch.bfloat16 and d % 16 == 0 and 32 <= d <= 256 and (d % 32 == 0 or d < 128) and page_size % 16 == 0


PLAIN_CALLS = [("pulse_attn8_plain", 0, 0, 0, 0, 0, 0)]      # (of AttentionPlan.calls)


class AttentionPlan:
    """A step's attention: which rows go together, and how the keys are shared out over the GPU.  The first depends on the step's shape
    alone (how many tokens each request brings); the second is made on the GPU from the positions, by ``cut``, once a step for all
    layers that are alike in heads, window and chunk.  ``plain``: everything goes to the kernel that serves every size."""

    # Workgroups a compute unit that a kernel's keys are shared out over ("slots") and the fewest tiles of 64 keys of a piece.  Of attn8_many's a
    # unit's registers hold three where heads have 32 or 64 channels (two / three, us: 2,048 tokens 42 / 34.5, 2 portions of 509 behind 7,000
    # at 40 heads 133 / 107); pieces for as many in attn8_few read no faster (64 contexts of 4,096 95 / 104).
    FEW_SLOTS, FEW_LEAST = 2, 8
    MANY_SLOTS, MANY_NARROW_SLOTS, MANY_LEAST = 2, 3, 8
    # How many times the items there may be pieces in any case, where the items have not and where they have a slot each by themselves (32 heads on
    # 8 of 128, us).  attn8_few, once / twice / three times: contexts of 3,000 on the average, the longest 15,000, 40 of them 53 / 60 / 59, 64
    # 139 / 89 / 86, 100 of 2,000 106 / 90 / 91; 40 of 6,000 that are alike 110 / 101.  attn8_many: 1,500 tokens 36.6 / 42.8, 3 portions of 500
    # behind 1,000 49.7 / 60 / 63; 300 behind 8,000 beside 2,000 229 / 106 / 117, 600 behind 12,000 beside six of 500 343 / 192 / 196.  (Of 256
    # channels a unit holds one workgroup of attn8_many: five portions up to 2,009 132 / 160.)
    FEW_ROUNDS, MANY_ROUNDS = (2, 2), (1, 2)
    # Up to so many pieces an item on the average the last one joins them (in a launch of its own / by the last, us: 1,024 tokens 39 / 28, 3
    # portions of 300 behind 2,000 59 / 48, 512 behind 8,192 98 / 96; at 10 an item 74 / 109).
    MANY_HERE = 6
    # Nothing is cut (and nothing joined) where the items have a slot each by themselves and the longest is not much more than a slot's share of all:
    # so many times of attn8_few's, at most so many tiles more of attn8_many's.  Whole / cut, us, 32 heads on 8 of 128: 64 contexts of 4,000 on the
    # average 94 / 107 (1.05 times), 96 / 110 (1.15), 101 / 111 (1.3), 106 / 110 (1.5), 114 / 112 (1.8), but 96 of 3,000 118 / 122 (1.0), 124 / 122 (1.2),
    # 129 / 123 (1.5) and 128 of 2,000 113 / 111 (0.9), 117 / 112 (1.15), 121 / 112 (1.3).  Portions: 1,044 and 1,668 tokens 54 / 62 (11 tiles more), 2,600
    # 79 / 84 (14), 2,048 63 / 59 to 71 (16), 600 behind 3,000 beside 2,000 107 / 95 (26), 1,200 behind 4,000 beside 1,500 158 / 136 (30), 600 behind
    # 6,000 beside 2,000 183 / 132 (59).
    FEW_EVEN, MANY_LONGER = 1.15, 24
    # Of attn8_few, where every unit has an item, neither are those cut whose lengths are (on the GPU, in a step's own positions) within so many
    # hundredths of their mean, unless some units had two and most one.  Cut / whole, us, 32 heads on 8 of 128, contexts of 1,000 / 4,000 / 8,000: 32 of
    # them 19.6 / 16.6, 52.9 / 49.2, 98 / 93; 40 24.6 / 26, 71 / 76, 129 / 147; 48, where it changes with the length, 25.7 / 24.7, 77.8 / 79.9, 143 / 152; 56 33 / 25.7,
    # 94 / 84, 175 / 160.  Of 64 channels 40 14.2 / 11.6, 39 / 36, 71 / 68.
    FEW_ALIKE = 110
    # Portions go through attn8_few up to so many columns, and altogether while they walk no more tiles a compute unit for it.  One portion
    # of 128 rows, 32 heads on 8, many / few, us: from the start 14.5 / 11.6, behind 1,000 tokens 22.1 / 12.7, behind 8,000 42.5 / 47; of 200
    # behind 1,000 23.9 / 19.3, of 240 24.4 / 32.2; of 300 from the start 16.0 / 11.6, of 500 19.6 / 16.6; sixteen of 64 behind 1,000 31 / 40.
    FEW_COLUMNS, FEW_WALKS = 32, 36

    def __init__(self, entries: Sequence[Any], nq: int, nkv: int, d: int, *, page_size: int, dtype: torch.dtype, window: int = 0,
                 chunk: int = 0, device: Any = "cuda", workspace: Any = None, to_device: Optional[Callable] = None, plain: bool = False):
        _need(nq > 0 and nkv > 0 and nq % nkv == 0, f"plan: {nq} query heads are not a multiple of {nkv} key/value heads")
        _need(0 < d <= MAX_HEAD_DIM, f"plan: heads of {d} channels (up to {MAX_HEAD_DIM})")
        _need(window >= 0 and chunk >= 0 and not (window and chunk), "plan: a window and chunks at once, or a negative one")
        _need(dtype in (torch.bfloat16, torch.float32), f"plan: storage type {dtype} is not supported (float32 or bfloat16)")
        self.nq, self.nkv, self.d, self.page_size, self.dtype = nq, nkv, d, int(page_size), dtype
        # (one that no position of 32 bits reaches beyond hides nothing)
        self.window, self.chunk = (0 if v >= 2 ** 31 else int(v) for v in (window, chunk))
        self.workspace = workspace
        self.tag, self.size = _TAG[dtype], dtype.itemsize
        self.rows, self.entries = 0, len(entries)
        for e in entries:
            if e.first_row != self.rows or e.count < 0 or e.start < 0:
                _refuse("plan", f"an entry of {e.count} rows from position {e.start} on, at row {e.first_row}: expected the next, row {self.rows}")
            self.rows += e.count
        self.matrix = not plain and matrix_cores(d, page_size, dtype)
        self.device = torch.device(device)
        if self.device.type == "cuda" and self.device.index is None:      # (the one that its lists lie on, whichever is the current one later)
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.ready = not self.matrix      # whether the keys have been shared out
        self.works: List[Tuple] = []      # (items on the GPU, their number, slots, least, room for pieces, counters an item, hundredths of the mean, longer pieces, cut)
        self.calls: List[Tuple] = []      # (entry point, items, cut, number of items, room for pieces, columns of the room for joined pieces, joined by the last)
        self.rooms: dict = {}             # what its calls had of the workspace: a recording goes on writing there when the workspace has grown
        self.streams: set = set()         # whose work the lists' memory waits for when the plan goes
        if not self.matrix:
            self.calls = PLAIN_CALLS
            return
        if self.device.type == "cuda":
            self.streams.add(_stream().value)
        units, group = compute_units(), nq // nkv
        few, many = [], []
        each, wide, groups = max(1, FEW // group), MANY // group, nkv * ((group + FEW - 1) // FEW)
        # every 16 columns of attn8_few walk the keys for themselves
        walks = sum(-(-e.count // each) * (self._tiles(e.start, e.count)) for e in entries if e.count * group > self.FEW_COLUMNS) * groups
        narrow = wide == 0 or walks <= self.FEW_WALKS * units
        for i, e in enumerate(entries):
            to, step = (few, each) if narrow or e.count * group <= self.FEW_COLUMNS else (many, wide)
            to += [(e.start + at, e.first_row + at, min(step, e.count - at), i) for at in range(0, e.count, step)]
        to_device = to_device or (lambda flat: torch.tensor(flat, dtype=torch.int32, device=self.device))

        def add(name: str, columns: int, items: List[Tuple], groups: int, slots: int, least: int, rounds: Tuple[int, int]) -> None:
            n = len(items)
            if not n:
                return
            tiles = [self._tiles(start, rows) for start, _, rows, _ in items]
            _need(n <= MAX_PIECES, f"plan: {n} items are too many")
            filled = n * groups >= slots * units
            share = sum(tiles) * groups / (slots * units)
            whole = n == MAX_PIECES or filled and max(tiles) <= (share + self.MANY_LONGER if columns == MANY else self.FEW_EVEN * share)
            slots = max(1, min(max(slots * units // groups, rounds[filled] * n), MAX_PIECES - n))      # (fewer than the items: nothing is cut)
            room = n if whole else n + slots
            if not whole and columns == MANY:      # the longest pieces first, as far as can be told from the starts
                low = max(least, -(-sum(tiles) // slots))
                high = max(low, max(tiles))
                while low < high:                  # (the length that attn8_cut finds)
                    middle = (low + high) // 2
                    if sum(-(-t // middle) for t in tiles) <= slots:
                        high = middle
                    else:
                        low = middle + 1
                items = [it for _, it in sorted(zip(tiles, items), key=lambda x: -(-x[0] // -(-x[0] // low)), reverse=True)]
            on_gpu = to_device([v for _, row, rows, entry in items for v in (row, rows, entry, 0)])
            _need(on_gpu.dtype == torch.int32 and on_gpu.device == self.device and on_gpu.is_contiguous() and on_gpu.numel() >= 4 * n,
                  f"plan: to_device must give {4 * n} contiguous int32 numbers on {self.device}")
            here = int(columns == FEW or slots <= self.MANY_HERE * n)
            counters = n * groups if here else 0
            cut = torch.empty(PIECE_INTS * room + 2 * n + counters, dtype=torch.int32, device=self.device)
            # (what the units' turns at n * groups workgroups are above what they would be if these could be shared out evenly)
            turns = -(-n * groups // units) * units / (n * groups)
            alike = self.FEW_ALIKE if columns == FEW and n * groups >= units and turns <= (1.7 if d <= 64 else 1.35) else 0
            self.works.append((on_gpu, n, slots, least, room, counters // n, alike, int(columns == FEW), cut))
            self.calls.append((name, on_gpu.data_ptr(), cut.data_ptr(), n, room, 0 if whole else room * groups * columns, here))

        add("pulse_attn8_few", FEW, few, groups, self.FEW_SLOTS, self.FEW_LEAST, self.FEW_ROUNDS)
        # The longest walks first; where two workgroups share a unit, the second ones' from the other end, the shortest beside the longest.
        many.sort(key=lambda it: -it[0])
        first = max(1, units // nkv)
        if first < len(many) <= 2 * first:
            many[first:] = many[:first - 1:-1]
        add("pulse_attn8_many", MANY, many, nkv, self.MANY_NARROW_SLOTS if d in (32, 64) else self.MANY_SLOTS, self.MANY_LEAST,
            self.MANY_ROUNDS if d < 256 else (1, 1))

    def on(self, stream: Any) -> None:
        """``stream``, the current one, reads the lists from now on: they may have been made on another, and the plan be dropped before it
        has come to them."""
        if stream.value not in self.streams:
            self.streams.add(stream.value)
            for work in self.works:
                for t in (work[0], work[-1]):
                    t.record_stream(torch.cuda.current_stream())

    def _tiles(self, start: int, count: int) -> int:
        """Tiles that hold keys of ``count`` tokens from position ``start`` on."""
        low = start - start % self.chunk if self.chunk else max(0, start - self.window + 1) if self.window else 0
        return (start + count - 1) // TILE + 1 - low // TILE

    def cut(self, positions: torch.Tensor) -> "AttentionPlan":
        """Shares the keys out for the rows' ``positions``: for every step, before its first ``attention``; the first time outside a recording."""
        _here("plan", (positions,))
        _ints("plan", "positions", positions, self.rows)
        if self.device.index is not None and positions.device != self.device:
            _refuse("plan", f"it was made for {self.device}, the positions lie on {positions.device}")
        if not self.ready and self.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            _refuse("plan", "its first cut cannot be a recorded one, behind which nothing has been shared out yet")
        self.ready = True
        stream = _stream()
        self.on(stream)
        for items, n, slots, least, room, groups, even, shrink, cut in self.works:
            call("pulse_attn8_cut", _ptr(items), _i32(n), _ptr(positions), _i32(self.window), _i32(self.chunk), _i32(slots), _i32(least),
                 _i32(room), _i32(groups), _i32(even), _i32(shrink), _ptr(cut), stream)
        return self


def plan(entries: Sequence[Any], nq: int, nkv: int, d: int, positions: torch.Tensor, *, page_size: int, dtype: torch.dtype,
         window: int = 0, chunk: int = 0, workspace: Any = None, to_device: Optional[Callable] = None) -> AttentionPlan:
    """The attention of a step of ``entries`` (``EntryMeta``: start, count, first_row; one's rows behind the other's from row 0 on, at positions
    that follow each other) whose rows stand at ``positions``, for layers of these heads.  It is made outside a recording; a step of the same
    shape takes the same plan, cut anew (``AttentionPlan.cut``, which may be recorded).  A plan, its counters among it, serves calls that follow
    each other, on whichever stream.  ``workspace`` (a ``Workspace``): where the room for joined pieces comes from, for calls and replays that
    follow each other; without one every call takes it from torch's pool.  A recording needs its plan (the lists, and the room that it was
    recorded with) for as long as it is replayed."""
    return AttentionPlan(entries, nq, nkv, d, page_size=page_size, dtype=dtype, window=window, chunk=chunk, device=positions.device,
                         workspace=workspace, to_device=to_device).cut(positions)


def attention(q: torch.Tensor, out: torch.Tensor, plan: AttentionPlan, view: Paged8CacheView, positions: torch.Tensor,
              token_entry: torch.Tensor, table: torch.Tensor, scale: float, *, gate: Optional[torch.Tensor] = None, gate_width: int = 0,
              sink: Optional[torch.Tensor] = None, softcap: float = 0.0, workspace: Any = None) -> None:
    """Causal attention of a step's rows over a cache in 8 bits, as ``plan`` has it: ``q``, ``out`` [T, >= nq * d] of one storage type (bfloat16
    or float32; rows may be strided, ``out`` may be ``q``), ``positions`` (those that the plan was cut for) and ``token_entry`` int32 [T], ``table`` int32
    [entries, width].

    A row sees the keys of its request from its window's (chunk's) first to its own position, in pages that are there: a table entry
    outside the pool hides its keys.  A row that sees none is zeros.  ``scale`` > 0; ``softcap``: scores become cap * tanh(score / cap)
    (of caps above ``MATRIX_CAP`` by the kernel that serves every size);
    ``sink`` float32 [nq]: exp(sink) is one more term of the denominator; ``gate`` [T, nq] of q's storage type: head h is multiplied by
    sigmoid(gate[:, h]), or with ``gate_width`` [T, nq * gate_width] its first channels each by one of its own.  What is not finite
    reaches the rows that see it and no others.  Rows that no entry of the plan has are left as they were."""
    what = "attention"
    _here(what, (q, out, view.keys, view.values, view.scales, positions, token_entry, table, gate, sink))
    nq, nkv, d = plan.nq, plan.nkv, plan.d
    pages, page = _pages(what, view, nkv, d)
    if plan.device.index is not None and plan.device.index != q.get_device():
        _refuse(what, f"the plan was made for {plan.device}, q lies on {q.device}")
    if page != plan.page_size or q.dtype != plan.dtype:
        _refuse(what, f"the plan is for pages of {plan.page_size} and {plan.dtype}")
    shape, to = q.shape, out.shape
    if (len(shape) != 2 or len(to) != 2 or q.dtype != out.dtype or shape[0] != to[0] or shape[1] < nq * d or to[1] < nq * d
            or q.stride(1) != 1 or out.stride(1) != 1):
        _refuse(what, f"q and out must be [T, {nq * d}] of one storage type with contiguous rows")
    tokens = shape[0]
    q_stride, o_stride = (q.stride(0), out.stride(0)) if tokens > 1 else (nq * d, nq * d)
    if q_stride < nq * d or o_stride < nq * d:
        _refuse(what, "rows that overlap")
    q_at, out_at = q.data_ptr(), out.data_ptr()
    if tokens and not (q_at == out_at and q_stride == o_stride) and not _apart(tokens, plan.size, q_at, q_stride, nq * d, out_at, o_stride, nq * d):
        _refuse(what, "out overlaps rows of q (it may be the same, or lie apart)")
    if plan.rows > tokens:
        _refuse(what, f"the plan has {plan.rows} rows, q {tokens}")
    if not plan.ready:
        _refuse(what, "the plan has not been cut for any positions")
    if not 0.0 < scale < INF or not 0.0 <= softcap < INF:
        _refuse(what, "the scale must be positive and the cap not negative, and both finite")
    _ints(what, "positions", positions, tokens)
    _ints(what, "token_entry", token_entry, tokens)
    shape = table.shape
    if table.dtype != torch.int32 or len(shape) != 2 or not table.is_contiguous() or shape[0] < max(1, plan.entries) or shape[1] < 1:
        _refuse(what, f"the table must be contiguous int32 [{plan.entries}, width]")
    gate_stride = 0
    if gate is None:
        gate_width = 0
    else:
        if (not 0 <= gate_width <= d or gate.dtype != q.dtype or gate.dim() != 2 or gate.shape[0] != tokens
                or gate.shape[1] < nq * max(1, gate_width) or gate.stride(1) != 1):
            _refuse(what, f"the gate must be [{tokens}, {nq * max(1, gate_width)}] of q's storage type")
        gate_stride = gate.stride(0) if tokens > 1 else 0
    if sink is not None and (sink.dtype != torch.float32 or sink.numel() != nq or not sink.is_contiguous()):
        _refuse(what, f"the sinks must be float32 [{nq}]")
    if tokens == 0:
        return
    workspace = workspace if workspace is not None else plan.workspace
    stream = _stream()
    if stream.value not in plan.streams:
        plan.on(stream)
    calls = plan.calls if softcap <= MATRIX_CAP else PLAIN_CALLS
    if calls is not PLAIN_CALLS and (q_at % 16 or q_stride % 8 or out_at % 8 or o_stride % 4):
        _refuse(what, "rows must be aligned to 16 bytes")
    for name, items, cut, n_items, room, rows, here in calls:
        part_o = part_ml = 0
        if rows:
            if workspace is not None:
                o = workspace.buffer("attention8.part_o", rows, d, torch.float32)
                ml = workspace.buffer("attention8.part_ml", rows, 2, torch.float32)
                part_o, part_ml = o.data_ptr(), ml.data_ptr()
                place = part_o, part_ml, stream.value
                if place not in plan.rooms:
                    if o.get_device() != q.get_device():
                        _refuse(what, f"the workspace is on {o.device}, q on {q.device}")
                    plan.rooms[place] = o, ml
                    for t in (o, ml):          # (made on another stream, perhaps)
                        t.record_stream(torch.cuda.current_stream())
            else:
                o = torch.empty((rows, d), dtype=torch.float32, device=q.device)
                ml = torch.empty((rows, 2), dtype=torch.float32, device=q.device)
                part_o, part_ml = o.data_ptr(), ml.data_ptr()
        call(name, _ATTN.pack(
            q_at, q_stride, out_at, o_stride, view.keys.data_ptr(), view.values.data_ptr(), view.scales.data_ptr(), positions.data_ptr(),
            token_entry.data_ptr(), table.data_ptr(), _at(gate), gate_stride, _at(sink), items, cut, part_o, part_ml, plan.tag, plan.rows,
            shape[0], shape[1], nq, nkv, d, page, pages, plan.window, plan.chunk, gate_width, n_items, room, here, 0, scale, softcap),
            stream)

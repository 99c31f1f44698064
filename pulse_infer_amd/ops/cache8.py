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

import ctypes
from typing import Any, Callable, List, Optional, Sequence, Tuple

import torch

from ..cache.specs import Paged8CacheView, block_tokens
from .device import compute_units
from .kernels import _f32, _gpu, _i32, _i64, _int_vec, _need, _ptr, _stream, _tag
from .library import call, load

MAX_REQUESTS = 4096          # of step_maps
MAX_HEAD_DIM = 512           # of store and of attention
FEW, MANY = 16, 128          # columns (rows times the heads that share a kv head) of an item of the two matrix-core kernels


def _here(what: str, *tensors: Optional[torch.Tensor]) -> None:
    """All of them on the current GPU, whose stream the kernels are queued on."""
    _gpu(what, *tensors)
    current = torch.cuda.current_device()
    for t in tensors:
        if t is not None and t.device.index != current:
            _need(False, f"{what}: a tensor lies on {t.device}, the current GPU is cuda:{current}")


def _pages(what: str, view: Paged8CacheView, nkv: int, d: int) -> Tuple[int, int]:
    """(pages, tokens a page) of a cache that is what the kernels take it for."""
    keys, values, scales = view.keys, view.values, view.scales
    _need(keys.dim() == 4 and keys.shape[1] == nkv and keys.shape[3] == d and keys.shape[2] == view.page_size,
          f"{what}: the keys are {tuple(keys.shape)}, expected [pages, {nkv}, {view.page_size}, {d}]")
    pages, _, page, _ = keys.shape
    block = block_tokens(page)
    _need(tuple(values.shape) == (pages, nkv, page // block, d, block),
          f"{what}: the values are {tuple(values.shape)}, expected {(pages, nkv, page // block, d, block)}")
    _need(tuple(scales.shape) == (pages, nkv, page // block, 2) and scales.dtype == torch.float32,
          f"{what}: the scales must be float32 {(pages, nkv, page // block, 2)}")
    _need(keys.dtype == values.dtype == torch.float8_e4m3fn, f"{what}: keys and values must be float8_e4m3fn")
    _need(all(t.is_contiguous() and t.data_ptr() % 16 == 0 for t in (keys, values, scales)),
          f"{what}: the cache must be contiguous and aligned to 16 bytes")
    return pages, page


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
    left as they were; what does not fit is left out.  T < 2^31, num_pages * page_size < 2^31, B <= 4096."""
    what = "step_maps"
    _here(what, start, count, pages, table, first_row, positions, token_entry, slots, blocks)
    n = start.numel()
    _int_vec(f"{what}: start", start)
    _int_vec(f"{what}: count", count)
    _need(0 < n <= MAX_REQUESTS and count.numel() == n, f"{what}: lengths of {n} and {count.numel()} requests (1 to {MAX_REQUESTS})")
    _need(page_size > 0 and num_pages > 0 and page_size * num_pages < 2 ** 31, f"{what}: {num_pages} pages of {page_size} tokens")
    block = block or block_tokens(page_size)
    _need(block > 0 and page_size % block == 0, f"{what}: blocks of {block} tokens do not divide pages of {page_size}")
    for name, t in (("pages", pages), ("positions", positions), ("token_entry", token_entry), ("slots", slots)):
        if t is not None:
            _int_vec(f"{what}: {name}", t)
    if first_row is not None:
        _int_vec(f"{what}: first_row", first_row, n + 1)
    _need(pages is None or pages.numel() > 0 or (slots is None and blocks is None and table is None), f"{what}: the list of pages is empty")
    rows = [t.numel() for t in (positions, token_entry, slots) if t is not None]
    _need(len(set(rows)) <= 1, f"{what}: positions, token_entry and slots of {rows} rows")
    width = 0
    if table is not None:
        _need(table.dim() == 2 and table.dtype == torch.int32 and table.is_contiguous() and table.shape[0] == n and table.shape[1] > 0,
              f"{what}: the table must be contiguous int32 [{n}, width]")
        width = table.shape[1]
    _need(pages is not None or table is not None or (slots is None and blocks is None), f"{what}: slots and blocks need the pages or the table")
    if blocks is not None:
        _need(blocks.dim() == 2 and blocks.shape[1] == 4 and blocks.dtype == torch.int32 and blocks.is_contiguous()
              and blocks.data_ptr() % 16 == 0, f"{what}: blocks must be contiguous int32 [n, 4], aligned to 16 bytes")
    call("pulse_step_maps", _ptr(start), _ptr(count), _i32(n), _ptr(pages), _i32(pages.numel() if pages is not None else 0),
         _i32(page_size), _i32(num_pages), _i32(block), _ptr(first_row), _ptr(positions), _ptr(token_entry), _ptr(slots),
         _i32(rows[0] if rows else 0), _ptr(table), _i32(width), _ptr(blocks), _i32(blocks.shape[0] if blocks is not None else 0), _stream())


def blocks_touched(entries: Sequence[Any], page_size: int) -> int:
    """Places of ``step_maps``'s ``blocks`` that a step of these entries takes."""
    block = block_tokens(page_size)
    return sum((e.start + e.count - 1) // block - e.start // block + 1 for e in entries if e.count > 0)


# ------------------------------------------------------------------------------------------------------------- the store
def store(qkv: torch.Tensor, q_out: torch.Tensor, nq: int, nkv: int, d: int, view: Paged8CacheView, positions: torch.Tensor,
          blocks: torch.Tensor, *, q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, eps: float = 0.0,
          cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None, rotary_dim: int = 0, pairing: int = 0,
          plain_norm: bool = False, v_head0: Optional[int] = None, q_temperature: Optional[tuple] = None) -> None:
    """A step's rows of the fused projection: norm and rotation of q (to ``q_out`` [T, >= nq * d], which may be the front of ``qkv``) and k,
    k and v into the blocks that ``step_maps`` listed.  The options are those of ``kernels.qk_rope_kv``.

    Of a block that is begun (its first token among the new ones) nothing that it held before stays; behind the new tokens it holds
    zeros.  Of another the earlier bytes stay, moved to the new scale where that has grown.  A block may be listed once: requests do
    not share pages that a step writes to.  ``qkv`` [T, columns] bfloat16 or float32 with contiguous rows; heads of an even number of
    channels up to 512."""
    what = "store"
    _here(what, qkv, q_out, view.keys, view.values, view.scales, positions, blocks, q_weight, k_weight, cos, sin)
    _need(view.writable, f"{what}: the cache is another run's")
    _need(nq > 0 and nkv > 0 and d > 0 and d % 2 == 0 and d <= MAX_HEAD_DIM, f"{what}: heads of {d} channels (even, up to {MAX_HEAD_DIM})")
    pages, page = _pages(what, view, nkv, d)
    tokens = qkv.shape[0]
    v_head0 = nq + nkv if v_head0 is None else int(v_head0)
    _need(qkv.dim() == 2 and qkv.stride(1) == 1 and v_head0 >= 0 and qkv.shape[1] >= max(nq + nkv, v_head0 + nkv) * d,
          f"{what}: qkv must be [T, {max(nq + nkv, v_head0 + nkv) * d}] with contiguous rows")
    _need(q_out.dim() == 2 and q_out.shape[0] == tokens and q_out.shape[1] >= nq * d and q_out.stride(1) == 1 and q_out.dtype == qkv.dtype,
          f"{what}: q_out must be [{tokens}, {nq * d}] of qkv's storage type with contiguous rows")
    _need(tokens <= 1 or (qkv.stride(0) >= qkv.shape[1] and q_out.stride(0) >= q_out.shape[1]), f"{what}: rows that overlap")
    _int_vec(f"{what}: positions", positions, tokens)
    _need(blocks.dim() == 2 and blocks.shape[1] == 4 and blocks.dtype == torch.int32 and blocks.is_contiguous() and blocks.data_ptr() % 16 == 0,
          f"{what}: blocks must be contiguous int32 [n, 4], aligned to 16 bytes")
    _need((q_weight is None) == (k_weight is None) and not (plain_norm and q_weight is not None), f"{what}: bad norm options")
    w_tag = 0
    if q_weight is not None:
        _need(q_weight.numel() == d and k_weight.numel() == d and q_weight.dtype == k_weight.dtype and q_weight.is_contiguous()
              and k_weight.is_contiguous(), f"{what}: the two norm weights must hold {d} values of one storage type")
        w_tag = _tag(q_weight, what)
    _need((cos is None) == (sin is None), f"{what}: the rotation needs both of its tables")
    if cos is not None:
        _need(rotary_dim % 2 == 0 and 0 < rotary_dim <= d and pairing in (0, 1), f"{what}: bad rotation of {rotary_dim} channels")
        for t in (cos, sin):
            _need(t.dtype == torch.float32 and t.is_contiguous() and t.dim() == 2 and t.shape[0] >= tokens and t.shape[1] == rotary_dim // 2,
                  f"{what}: cos/sin must be float32 [T, {rotary_dim // 2}]")
    coef, every = (float(q_temperature[0]), int(q_temperature[1])) if q_temperature is not None else (0.0, 0)
    _need(q_temperature is None or every > 0, f"{what}: the query temperature's interval must be positive")
    call("pulse_store8", _ptr(qkv), _i32(_tag(qkv, what)), _i64(qkv.stride(0)), _ptr(q_out), _i64(q_out.stride(0)), _ptr(q_weight),
         _ptr(k_weight), _i32(w_tag), _f32(eps), _ptr(cos), _ptr(sin), _i32(rotary_dim if cos is not None else 0), _i32(pairing),
         _ptr(view.keys), _ptr(view.values), _ptr(view.scales), _i32(pages), _i32(page), _ptr(positions), _ptr(blocks),
         _i32(blocks.shape[0]), _i32(tokens), _i32(nq), _i32(nkv), _i32(d), _i32(1 if plain_norm else 0), _i32(v_head0), _f32(coef),
         _i32(every), _stream())


# --------------------------------------------------------------------------------------------------------- the attention
class _Attn8(ctypes.Structure):
    # as PulseAttn8 of csrc/cache8_attn.h
    _fields_ = ([("q", ctypes.c_void_p), ("q_stride", ctypes.c_int64), ("out", ctypes.c_void_p), ("o_stride", ctypes.c_int64)]
                + [(n, ctypes.c_void_p) for n in ("keys", "values", "scales", "positions", "token_entry", "table", "gate")]
                + [("gate_stride", ctypes.c_int64)] + [(n, ctypes.c_void_p) for n in ("sink", "items", "cut", "part_o", "part_ml")]
                + [(n, ctypes.c_int) for n in ("dtype", "tokens", "entries", "table_width", "nq", "nkv", "d", "page_size", "num_pages",
                                               "window", "chunk", "gate_width", "n_items", "max_work")]
                + [("scale", ctypes.c_float), ("softcap", ctypes.c_float)])


def matrix_cores(d: int, page_size: int, dtype: torch.dtype) -> bool:
    """Whether attention runs on the matrix cores; anything else goes to the kernel that serves every size."""
    return dtype == torch.bfloat16 and d % 32 == 0 and d <= 256 and page_size % 16 == 0


class _Work:
    """The items of one of the two matrix-core kernels, and how they are cut for the step at hand."""

    def __init__(self, what: str, columns: int, items: List[int], slots: int, least: int, device: torch.device, to_device: Callable):
        self.what, self.columns = what, columns
        self.n = len(items) // 4
        self.items = to_device(items)
        self.slots, self.least = slots, least
        self.max_work = self.n + slots if slots > 0 else self.n
        ints = 4 + 4 * self.max_work + 2 * self.n
        self.cut = torch.empty(ints, dtype=torch.int32, device=device)


class AttentionPlan:
    """A step's attention: which rows go together, and how the keys are shared out over the GPU.  The first depends on the step's shape
    alone (how many tokens each request brings); the second is made on the GPU from the positions, by ``cut``, once a step for all
    layers that are alike in heads, window and chunk."""

    FEW_SLOTS = 2        # workgroups of attn8_few a compute unit that a step is shared out over
    FEW_LEAST = 4        # tiles of 64 keys of a piece: one a wavefront
    MANY_SLOTS = 2
    MANY_LEAST = 8
    FEW_ROWS = 32        # columns up to which a portion goes through attn8_few

    def __init__(self, entries: Sequence[Any], nq: int, nkv: int, d: int, *, page_size: int, dtype: torch.dtype, window: int = 0,
                 chunk: int = 0, device: Any = None, to_device: Optional[Callable] = None):
        _need(nq > 0 and nkv > 0 and nq % nkv == 0, f"plan: {nq} query heads are not a multiple of {nkv} key/value heads")
        _need(0 < d <= MAX_HEAD_DIM, f"plan: heads of {d} channels (up to {MAX_HEAD_DIM})")
        _need(window >= 0 and chunk >= 0 and not (window and chunk), "plan: a window and chunks at once, or a negative one")
        self.nq, self.nkv, self.d, self.page_size, self.dtype = nq, nkv, d, int(page_size), dtype
        self.window, self.chunk = int(window), int(chunk)
        self.rows = max((e.first_row + e.count for e in entries), default=0)
        self.device = torch.device(device if device is not None else "cuda")
        self.works: List[_Work] = []
        if not matrix_cores(d, page_size, dtype):
            return
        group = nq // nkv
        few, many = [], []
        each, wide = max(1, FEW // group), MANY // group
        for i, e in enumerate(entries):
            to, step = (few, each) if e.count * group <= self.FEW_ROWS or wide == 0 else (many, wide)
            to += [(e.first_row + at, min(step, e.count - at), i, 0) for at in range(0, e.count, step)]
        # (a prompt's last rows see the most keys: their walks start first)
        many.sort(key=lambda it: -(entries[it[2]].start + it[0] - entries[it[2]].first_row))
        if to_device is None:
            to_device = lambda flat: torch.tensor(flat, dtype=torch.int32, device=self.device)  # noqa: E731
        units = compute_units()
        groups = nkv * ((group + FEW - 1) // FEW)
        if few:
            self.works.append(_Work("pulse_attn8_few", FEW, [v for it in few for v in it], max(1, self.FEW_SLOTS * units // groups),
                                    self.FEW_LEAST, self.device, to_device))
        if many:
            self.works.append(_Work("pulse_attn8_many", MANY, [v for it in many for v in it], max(1, self.MANY_SLOTS * units // nkv),
                                    self.MANY_LEAST, self.device, to_device))
        for w in self.works:
            _need(w.max_work <= 65535, f"plan: {w.n} items are too many")

    def cut(self, positions: torch.Tensor) -> "AttentionPlan":
        """Shares the keys out for the rows' ``positions``: for every step, before its first ``attention``."""
        _here("plan", positions)
        _int_vec("plan: positions", positions, self.rows)
        for w in self.works:
            call("pulse_attn8_cut", _ptr(w.items), _i32(w.n), _ptr(positions), _i32(self.window), _i32(self.chunk), _i32(max(1, w.slots)),
                 _i32(w.least), _i32(w.max_work), _ptr(w.cut), _stream())
        return self

    def parts(self, w: _Work) -> Tuple[int, int]:
        """Rows of the room for pieces that are joined: (columns of all pieces, channels)."""
        group = self.nq // self.nkv
        groups = self.nkv * ((group + FEW - 1) // FEW) if w.columns == FEW else self.nkv
        return (w.max_work * groups * w.columns, self.d) if w.max_work > w.n else (0, self.d)


def plan(entries: Sequence[Any], nq: int, nkv: int, d: int, positions: torch.Tensor, *, page_size: int, dtype: torch.dtype,
         window: int = 0, chunk: int = 0, workspace: Any = None, to_device: Optional[Callable] = None) -> AttentionPlan:
    """The attention of a step of ``entries`` (``EntryMeta``: start, count, first_row) whose rows stand at ``positions``, for layers of these
    heads.  A step of the same shape takes the same plan, cut anew (``AttentionPlan.cut``); ``workspace`` holds the room for joined pieces
    and serves the steps of one stream one after the other."""
    made = AttentionPlan(entries, nq, nkv, d, page_size=page_size, dtype=dtype, window=window, chunk=chunk, device=positions.device,
                         to_device=to_device)
    made.workspace = workspace
    return made.cut(positions)


def attention(q: torch.Tensor, out: torch.Tensor, plan: AttentionPlan, view: Paged8CacheView, positions: torch.Tensor,
              token_entry: torch.Tensor, table: torch.Tensor, scale: float, *, gate: Optional[torch.Tensor] = None, gate_width: int = 0,
              sink: Optional[torch.Tensor] = None, softcap: float = 0.0, workspace: Any = None) -> None:
    """Causal attention of a step's rows over a cache in 8 bits, as ``plan`` has it: ``q``, ``out`` [T, >= nq * d] of one storage type (bfloat16
    or float32; rows may be strided), ``positions`` and ``token_entry`` int32 [T], ``table`` int32 [entries, width].

    A row sees the keys of its request from its window's (chunk's) first to its own position, in pages that are there: a table entry
    outside the pool hides its keys.  A row that sees none is zeros.  ``scale`` > 0; ``softcap``: scores become cap * tanh(score / cap);
    ``sink`` float32 [nq]: exp(sink) is one more term of the denominator; ``gate`` [T, nq] of q's storage type: head h is multiplied by
    sigmoid(gate[:, h]), or with ``gate_width`` [T, nq * gate_width] its first channels each by one of its own.  What is not finite
    reaches the rows that see it and no others.  Rows that no entry of the plan has are left as they were."""
    what = "attention"
    _here(what, q, out, view.keys, view.values, view.scales, positions, token_entry, table, gate, sink)
    nq, nkv, d = plan.nq, plan.nkv, plan.d
    pages, page = _pages(what, view, nkv, d)
    tokens = q.shape[0]
    _need(page == plan.page_size and q.dtype == plan.dtype, f"{what}: the plan is for pages of {plan.page_size} and {plan.dtype}")
    _need(q.dim() == 2 and out.dim() == 2 and q.stride(1) == 1 and out.stride(1) == 1 and q.dtype == out.dtype and out.shape[0] == tokens
          and q.shape[1] >= nq * d and out.shape[1] >= nq * d,
          f"{what}: q and out must be [T, {nq * d}] of one storage type with contiguous rows")
    _need(tokens <= 1 or (q.stride(0) >= nq * d and out.stride(0) >= nq * d), f"{what}: rows that overlap")
    _need(plan.rows <= tokens, f"{what}: the plan has {plan.rows} rows, q {tokens}")
    _need(scale > 0.0 and softcap >= 0.0, f"{what}: the scale must be positive and the cap not negative")
    _int_vec(f"{what}: positions", positions, tokens)
    _int_vec(f"{what}: token_entry", token_entry, tokens)
    _need(table.dim() == 2 and table.dtype == torch.int32 and table.is_contiguous() and table.numel() > 0,
          f"{what}: the table must be contiguous int32 [entries, width]")
    if gate is not None:
        _need(0 <= gate_width <= d and gate.dtype == q.dtype and gate.dim() == 2 and gate.shape[0] == tokens
              and gate.shape[1] >= nq * max(1, gate_width) and gate.stride(1) == 1,
              f"{what}: the gate must be [{tokens}, {nq * max(1, gate_width)}] of q's storage type")
    if sink is not None:
        _need(sink.dtype == torch.float32 and sink.is_contiguous() and sink.numel() == nq, f"{what}: the sinks must be float32 [{nq}]")
    if tokens == 0:
        return
    tag = _tag(q, what)
    wide = lambda t: t.stride(0) if tokens > 1 else nq * d  # noqa: E731
    args = _Attn8(q=q.data_ptr(), q_stride=wide(q), out=out.data_ptr(), o_stride=wide(out), keys=view.keys.data_ptr(),
                  values=view.values.data_ptr(), scales=view.scales.data_ptr(), positions=positions.data_ptr(),
                  token_entry=token_entry.data_ptr(), table=table.data_ptr(), gate=gate.data_ptr() if gate is not None else 0,
                  gate_stride=gate.stride(0) if gate is not None and tokens > 1 else 0, sink=sink.data_ptr() if sink is not None else 0,
                  dtype=tag, tokens=tokens, entries=table.shape[0], table_width=table.shape[1], nq=nq, nkv=nkv, d=d, page_size=page,
                  num_pages=pages, window=plan.window, chunk=plan.chunk, gate_width=gate_width if gate is not None else 0, scale=scale,
                  softcap=softcap)
    if not matrix_cores(d, page, q.dtype):
        call("pulse_attn8_plain", ctypes.byref(args), _stream())
        return
    _need(q.data_ptr() % 16 == 0 and (tokens <= 1 or q.stride(0) % 8 == 0) and out.data_ptr() % 8 == 0
          and (tokens <= 1 or out.stride(0) % 4 == 0), f"{what}: rows must be aligned to 16 bytes")
    workspace = workspace if workspace is not None else getattr(plan, "workspace", None)
    for w in plan.works:
        rows, _ = plan.parts(w)
        if rows:
            if workspace is not None:
                o = workspace.buffer("attention8.part_o", rows, d, torch.float32)
                ml = workspace.buffer("attention8.part_ml", rows, 2, torch.float32)
            else:
                o = torch.empty((rows, d), dtype=torch.float32, device=q.device)
                ml = torch.empty((rows, 2), dtype=torch.float32, device=q.device)
            args.part_o, args.part_ml = o.data_ptr(), ml.data_ptr()
        args.items, args.cut, args.n_items, args.max_work = w.items.data_ptr(), w.cut.data_ptr(), w.n, w.max_work
        call(w.what, ctypes.byref(_Attn8.from_buffer_copy(args)), _stream())     # (its own: calls may be kept and made again)

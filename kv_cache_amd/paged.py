"""A paged K/V cache for requests of different lengths: its page table, its
writes and the attention over it (MI355X).

K and V lie in pages of ``page`` tokens that requests take from one pool:
``k_pages`` / ``v_pages`` [pages, Hkv, page, D] (bf16 or fp16), and
``table`` int32 [requests, width] holds the page of each request's token t at
t // page.  A serving step does, once,

1. ``plan_step``  -- pages for the step's new tokens from the stack of free
                    ones, and each row's slot and position, decided on the
                    GPU from the request lengths (``PageTable.step``);

then for each layer

2. ``append``     -- the rows' K and V into their slots;
3. ``attention``  -- the rows over the cache: single tokens, drafted tokens,
                    chunks of prompts, whole prompts, mixed as they come;
                    scores may be capped by a tanh and biased by distance,
                    the mask may have a two-sided prefix and documents;

and ``release_pages`` gives back the pages of requests that ended or of
tokens that were rejected.  Pages may hold codes of 8 or 4 bits with scales
(``quantized_pages``); ``read`` gives cached tokens back as rows.  Requests
may continue another one's tokens: ``share_rows`` gathers a step's rows by
parent, and ``attention(..., shared=...)`` reads a parent's keys for all of
them together.  No length is needed on the host, so a step can be
captured into a graph and replayed while the requests grow.

No reference counterpart: the reference keeps HF's dense cache, every
sequence of a batch at one length, and prefills with dense attention
(evaluate_qwen3_top2_head_limit3_ppl.py:7079-7111).  Everything runs on the
GPU on the current stream and raises RuntimeError on bad input.  The pages
hold no graph: there are no gradients.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _lib


def _require(cond: bool, msg: str) -> None:
    if not cond:
        raise RuntimeError(msg)


class StepPlan(NamedTuple):
    """What ``plan_step`` decides of a step: request b's rows are
    ``cu_rows[b] .. cu_rows[b + 1] - 1`` and it holds ``kv_lens[b]`` tokens
    after the step (0 if it was not served); ``slots`` and ``positions`` of
    every row (-1 where it has no token); ``failed`` [1] counts the requests
    whose new tokens found no room."""

    cu_rows: torch.Tensor     # int32 [requests + 1]
    kv_lens: torch.Tensor     # int32 [requests]
    slots: torch.Tensor       # int64 [rows]
    positions: torch.Tensor   # int32 [rows]
    failed: torch.Tensor      # int32 [1]

    @classmethod
    def empty(cls, requests: int, rows: int, device) -> "StepPlan":
        """Buffers for a step of ``rows`` rows."""
        kv = torch.empty(requests, dtype=torch.int32, device=device)
        return cls(kv.new_empty(requests + 1), kv, kv.new_empty(rows, dtype=torch.int64), kv.new_empty(rows),
                   kv.new_empty(1))


# The checks below run several times a call of ten microseconds: they ask tensors the cheapest way there is
# (get_device() for the device, numel() and dim() for a shape of one axis).


def _i32(name: str, t: torch.Tensor, n: int, idx: int) -> None:
    if (t.dtype is not torch.int32 or t.numel() != n or t.dim() != 1 or not t.is_contiguous()
            or t.get_device() != idx):
        raise RuntimeError(f"{name} must be contiguous int32 [{n}] on cuda:{idx}")


def _check_table(table: torch.Tensor) -> tuple[int, int, int, int]:
    """(device index, requests, width, row stride) of a page table."""
    if not table.is_cuda or table.dtype is not torch.int32 or table.dim() != 2:
        raise RuntimeError("table must be CUDA int32 [requests, width] with contiguous rows")
    ld, one = table.stride()
    if one != 1:
        raise RuntimeError("table must be CUDA int32 [requests, width] with contiguous rows")
    return (table.get_device(), *table.shape, ld)


def plan_step(new_lens: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, free: torch.Tensor,
              count: torch.Tensor, page: int, rows: int, *, padded: int = 0, out: StepPlan | None = None) -> StepPlan:
    """Adds ``new_lens[b]`` tokens to every request: takes their pages from
    the stack ``free`` int32 [pages] (``count`` int32 [1] entries, top last)
    into ``table`` int32 [requests, width], raises ``lens`` int32 [requests],
    and gives every one of the step's ``rows`` rows its slot and position.

    Rows are packed, ``new_lens[b]`` for each request, or, with ``padded`` =
    n, n for each with its tokens last (a left-padded batch; ``rows`` is then
    requests * n).  The rows before them have slot and position -1; over the
    cache they are queries of the request's earlier tokens, so ``attention``
    gives zeros only where there are none.  Rows behind the last request's have no token.  A request
    whose tokens do not fit its table row, the pool or ``rows`` is left as it
    is, with kv_lens 0, and counted in ``failed``.  At most 4096 requests,
    2^20 pages, 2^20 rows; ``page`` a power of two in [16, 4096]."""
    lib = _lib.load()
    idx, n, width, ld = _check_table(table)
    pages = free.numel()
    _i32("new_lens", new_lens, n, idx)
    _i32("lens", lens, n, idx)
    _i32("free", free, pages, idx)
    _i32("count", count, 1, idx)
    if out is None:
        out = StepPlan.empty(n, rows, table.device)
    else:
        _i32("out.cu_rows", out.cu_rows, n + 1, idx)
        _i32("out.kv_lens", out.kv_lens, n, idx)
        _i32("out.positions", out.positions, rows, idx)
        _i32("out.failed", out.failed, 1, idx)
        _check_slots(out.slots, rows, idx)
    cu, kv, slots, positions, failed = out
    guard = _lib.enter_device(idx)
    try:
        rc = lib.qkv_paged_plan(new_lens.data_ptr(), table.data_ptr(), ld, lens.data_ptr(), free.data_ptr(),
                                count.data_ptr(), n, width, pages, page, rows, padded, cu.data_ptr(), kv.data_ptr(),
                                slots.data_ptr(), positions.data_ptr(), failed.data_ptr(), _lib.stream_on(idx))
    finally:
        _lib.leave_device(guard)
    _lib.check(rc)
    return out


def release_pages(keep: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, free: torch.Tensor,
                  count: torch.Tensor, page: int) -> None:
    """Cuts every request to its first ``keep[b]`` tokens (0 ends it, its
    length or more leaves it) and gives the pages behind them back to
    ``free``; the last step's tokens released leave the stack as it was."""
    lib = _lib.load()
    idx, n, width, ld = _check_table(table)
    pages = free.numel()
    _i32("keep", keep, n, idx)
    _i32("lens", lens, n, idx)
    _i32("free", free, pages, idx)
    _i32("count", count, 1, idx)
    guard = _lib.enter_device(idx)
    try:
        rc = lib.qkv_paged_release(keep.data_ptr(), table.data_ptr(), ld, lens.data_ptr(), free.data_ptr(),
                                   count.data_ptr(), n, width, pages, page, _lib.stream_on(idx))
    finally:
        _lib.leave_device(guard)
    _lib.check(rc)


class PageTable:
    """The page table of ``requests`` requests of at most ``capacity`` tokens
    over a pool of ``pages`` pages, one for all layers: ``table``, ``lens``,
    ``free`` and ``count`` as ``plan_step`` takes them, all on the GPU."""

    def __init__(self, requests: int, capacity: int, pages: int, page: int, device):
        _require(requests >= 1 and capacity >= 1 and pages >= 1, "requests, capacity and pages must be positive")
        _require(16 <= page <= 4096 and page & (page - 1) == 0, "page must be a power of two in [16, 4096]")
        self.page, self.pages, self.capacity = int(page), int(pages), int(capacity)
        dev = torch.device(device)
        self.table = torch.full((requests, -(-capacity // page)), -1, dtype=torch.int32, device=dev)
        self.lens = torch.zeros(requests, dtype=torch.int32, device=dev)
        self.free = torch.arange(pages - 1, -1, -1, dtype=torch.int32, device=dev)   # page 0 on top
        self.count = torch.full((1,), pages, dtype=torch.int32, device=dev)

    def step(self, new_lens: torch.Tensor, rows: int, *, padded: int = 0, out: StepPlan | None = None) -> StepPlan:
        """``plan_step`` on this table."""
        return plan_step(new_lens, self.table, self.lens, self.free, self.count, self.page, rows, padded=padded,
                         out=out)

    def release(self, keep: torch.Tensor) -> None:
        """``release_pages`` on this table."""
        release_pages(keep, self.table, self.lens, self.free, self.count, self.page)


def _check_slots(slots: torch.Tensor, rows: int, idx: int) -> None:
    if (slots.dtype is not torch.int64 or slots.numel() != rows or slots.dim() != 1 or not slots.is_contiguous()
            or slots.get_device() != idx):
        raise RuntimeError(f"slots must be contiguous int64 [{rows}] on cuda:{idx}")


def _check_pages(k_pages: torch.Tensor, v_pages: torch.Tensor) -> tuple[int, tuple, tuple]:
    """(dtype code, strides of k_pages, of v_pages) of a layer's pages, checked."""
    code = _lib.half_code("k_pages", k_pages)
    if (not k_pages.is_cuda or k_pages.dim() != 4 or k_pages.shape != v_pages.shape
            or v_pages.dtype is not k_pages.dtype or v_pages.get_device() != k_pages.get_device()
            or k_pages.stride(3) != 1 or v_pages.stride(3) != 1):
        raise RuntimeError("k_pages and v_pages must be CUDA [pages, kv_heads, page, dim] of one shape, dtype and "
                           "device with contiguous channels")
    return code, k_pages.stride(), v_pages.stride()


class SharedRows:
    """What ``share_rows`` decides of a step, one int32 ``buffer`` for all of
    it; ``positions`` [rows] is where each row's token is, its parent's
    tokens before its request's own (-1 where a row has no token)."""

    __slots__ = ("buffer", "rows", "requests", "positions")

    def __init__(self, requests: int, rows: int, device):
        if not (1 <= requests <= 4096 and 1 <= rows <= 1 << 20):
            raise RuntimeError(f"share_rows takes 1 to 4096 requests and 1 to 2^20 rows, got {requests} and {rows}")
        # qkv_paged_share_words
        self.buffer = torch.empty(3 * rows + 4 * requests + 1, dtype=torch.int32, device=device)
        self.rows, self.requests, self.positions = rows, requests, self.buffer[:rows]


def share_rows(parents: torch.Tensor, cu_rows: torch.Tensor, kv_lens: torch.Tensor, lens: torch.Tensor, rows: int, *,
               out: SharedRows | None = None) -> SharedRows:
    """Of a step whose requests may continue the tokens of another one: the
    rows gathered by parent, for ``attention(..., shared=...)`` of every
    layer.  ``parents`` int32 [requests] is each request's parent, a request
    of the same page table, or -1; ``lens`` int32 [requests] the tokens that
    requests hold as parents (``PageTable.lens``); ``cu_rows`` and ``kv_lens``
    are the step's (``plan_step``).  A request then stands behind all tokens
    of its parent, wherever their last page ends; its own pages hold only its
    own tokens.  The parent's own parent does not count.  Release a parent
    after its last child."""
    lib = _lib.load()
    n, idx = parents.numel(), parents.get_device()
    if idx < 0:
        raise RuntimeError("parents must be CUDA")
    _i32("parents", parents, n, idx)
    _i32("cu_rows", cu_rows, n + 1, idx)
    _i32("kv_lens", kv_lens, n, idx)
    _i32("lens", lens, n, idx)
    if out is None:
        out = SharedRows(n, rows, parents.device)
    else:
        _require(out.rows == rows and out.requests == n and out.buffer.get_device() == idx,
                 f"out must be SharedRows({n}, {rows}) on cuda:{idx}")
    guard = _lib.enter_device(idx)
    try:
        rc = lib.qkv_paged_share(parents.data_ptr(), cu_rows.data_ptr(), kv_lens.data_ptr(), lens.data_ptr(), n, rows,
                                 out.buffer.data_ptr(), _lib.stream_on(idx))
    finally:
        _lib.leave_device(guard)
    _lib.check(rc)
    return out


# Quantised pages: codes of 8 bits (e4m3) or of 4 (e2m1, two to a byte, the even channel in the low half), and one scale
# byte s for each 32 channels of a token's head, under which a code stands for its value times 2^(s - 127).
_CODES = {torch.float8_e4m3fn: 1, torch.uint8: 2}
_BLOCK = 32
_HALF = (torch.bfloat16, torch.float16)


def quantized_pages(pages: int, kv_heads: int, page: int, head_dim: int, kind: str,
                    device) -> tuple[torch.Tensor, torch.Tensor]:
    """Quantised pages of K or of V for a layer, and their scales: ``kind``
    "fp8" (float8_e4m3fn [pages, Hkv, page, D]) or "fp4" (uint8 [pages, Hkv,
    page, D / 2]), scales uint8 [pages, Hkv, page, D / 32]; contents as the
    allocator gives them."""
    _require(kind in ("fp8", "fp4"), f"kind must be fp8 or fp4, got {kind!r}")
    _require(head_dim % _BLOCK == 0, f"head_dim must be a multiple of {_BLOCK}, got {head_dim}")
    scales = torch.empty((pages, kv_heads, page, head_dim // _BLOCK), dtype=torch.uint8, device=device)
    if kind == "fp8":
        return scales.new_empty((pages, kv_heads, page, head_dim), dtype=torch.float8_e4m3fn), scales
    return scales.new_empty((pages, kv_heads, page, head_dim // 2)), scales


def _check_codes(k_pages: torch.Tensor, v_pages: torch.Tensor, k_scales, v_scales) -> tuple:
    """(code, device index, shape of the values, strides of the pages, strides
    of the scales) of a layer's quantised pages, checked."""
    code, idx, shape, ps = _CODES.get(k_pages.dtype), k_pages.get_device(), k_pages.shape, k_pages.stride()
    if code is None:
        raise RuntimeError(f"quantised pages must be float8_e4m3fn or uint8, got {k_pages.dtype}")
    if (idx < 0 or len(shape) != 4 or v_pages.shape != shape or v_pages.dtype is not k_pages.dtype
            or v_pages.get_device() != idx):
        raise RuntimeError("k_pages and v_pages must be CUDA [pages, kv_heads, page, dim] of one shape, dtype and "
                           "device with contiguous channels")
    if v_pages.stride() != ps or ps[3] != 1:
        raise RuntimeError("k_pages and v_pages must have the same strides, with contiguous channels")
    pages, heads, page, dim = shape
    dim *= code   # two to a byte
    if dim % _BLOCK or k_scales is None or v_scales is None:
        raise RuntimeError(f"quantised pages have k_scales and v_scales and a multiple of {_BLOCK} channels")
    blocks, ss = dim // _BLOCK, k_scales.stride()
    if (k_scales.dtype is not torch.uint8 or v_scales.dtype is not torch.uint8 or k_scales.get_device() != idx
            or v_scales.get_device() != idx or k_scales.shape != (pages, heads, page, blocks)
            or v_scales.shape != k_scales.shape or v_scales.stride() != ss or ss[3] != 1 or ss[2] != blocks):
        raise RuntimeError(f"k_scales and v_scales must be uint8 {[pages, heads, page, blocks]} on {k_pages.device} of "
                           "the same strides, a head's tokens without gaps")
    return code, idx, (pages, heads, page, dim), ps, ss[:2]


def append(key: torch.Tensor, value: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
           slots: torch.Tensor, *, k_scales: torch.Tensor | None = None,
           v_scales: torch.Tensor | None = None) -> None:
    """Writes the rows' K and V, [rows, Hkv, D] at any strides with contiguous
    channels, to their ``slots`` (int64 [rows], as ``plan_step`` gives them;
    a row with -1 is skipped, no slot may come twice).

    Into quantised pages (``quantized_pages``, with their scales), bf16 or
    fp16 rows are rounded to the nearest code, halves to the even one, under
    the smallest power of two (from 2^-100 on) that keeps a block's largest
    magnitude within half a step: an fp8 value is off by at most 2^-4 of
    itself or 2^-10 of the scale, an fp4 one by 2^-2 or 2^-2.  A block with an
    infinity or NaN is stored as NaN; magnitudes that would read back as more
    than the dtype holds (fp16 over 61440, in fp4 over 49152) are stored as
    that."""
    if k_scales is not None or v_scales is not None or k_pages.dtype in _CODES:
        return _append_codes(key, value, k_pages, v_pages, slots, k_scales, v_scales)
    lib = _lib.load()
    _, ks, vs = _check_pages(k_pages, v_pages)
    pages, heads, page, dim = k_pages.shape
    idx = k_pages.get_device()
    rows = slots.numel()
    _check_slots(slots, rows, idx)
    for name, t in (("key", key), ("value", value)):
        if (t.shape != (rows, heads, dim) or t.dtype is not k_pages.dtype or t.get_device() != idx
                or t.stride(2) != 1):
            raise RuntimeError(f"{name} must be {k_pages.dtype} [{rows}, {heads}, {dim}] on {k_pages.device} with "
                               "contiguous channels: key, value and slots have as many rows")
    # row and head strides of the rows, page, head and token strides of the pages, in one array
    st = _lib.strides(*key.stride()[:2], *value.stride()[:2], *ks[:3], *vs[:3])
    at = ctypes.addressof(st)
    guard = _lib.enter_device(idx)
    try:
        rc = lib.qkv_paged_append(key.data_ptr(), at, value.data_ptr(), at + 16, k_pages.data_ptr(), at + 32,
                                  v_pages.data_ptr(), at + 56, pages, page, heads, dim, slots.data_ptr(), rows,
                                  _lib.stream_on(idx))
    finally:
        _lib.leave_device(guard)
    _lib.check(rc)


def _append_codes(key, value, k_pages, v_pages, slots, k_scales, v_scales) -> None:
    lib = _lib.load()
    code, idx, (pages, heads, page, dim), ps, ss = _check_codes(k_pages, v_pages, k_scales, v_scales)
    rows = slots.numel()
    _check_slots(slots, rows, idx)
    dtype = _lib.half_code("key", key)
    for name, t in (("key", key), ("value", value)):
        if t.shape != (rows, heads, dim) or t.dtype is not key.dtype or t.get_device() != idx or t.stride(2) != 1:
            raise RuntimeError(f"{name} must be {key.dtype} [{rows}, {heads}, {dim}] on {k_pages.device} with "
                               "contiguous channels: key, value and slots have as many rows")
    # row and head strides of the rows, page, head and token strides of the pages, page and head strides of the scales
    st = _lib.strides(*key.stride()[:2], *value.stride()[:2], *ps[:3], *ss)
    at = ctypes.addressof(st)
    guard = _lib.enter_device(idx)
    try:
        rc = lib.qkv_paged_append_codes(key.data_ptr(), at, value.data_ptr(), at + 16, k_pages.data_ptr(),
                                        v_pages.data_ptr(), at + 32, k_scales.data_ptr(), v_scales.data_ptr(), at + 56,
                                        code, pages, page, heads, dim, slots.data_ptr(), rows, dtype,
                                        _lib.stream_on(idx))
    finally:
        _lib.leave_device(guard)
    _lib.check(rc)


def read(k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor, cu_rows: torch.Tensor,
         kv_lens: torch.Tensor, rows: int, *, k_scales: torch.Tensor | None = None,
         v_scales: torch.Tensor | None = None, dtype: torch.dtype | None = None,
         out: tuple[torch.Tensor, torch.Tensor] | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """K and V of cached tokens, [rows, Hkv, D] each: row i of request b is
    the token at kv_lens[b] - (cu_rows[b + 1] - cu_rows[b]) + i, so that
    cu_rows = the sums of kv_lens reads whole requests; zeros where a request
    has no token.  Channels are a multiple of 32.  Quantised pages give ``dtype`` (bf16 if not said), which
    holds what they stand for without a rounding (fp16 below 2^-14 with fewer
    bits, and infinities past 65504); others their own.  Rows of ``out`` (two
    tensors, any row and head strides of 16 bytes) behind the last request are
    left as they were."""
    lib = _lib.load()
    if k_scales is not None or v_scales is not None or k_pages.dtype in _CODES:
        code, on, (pages, heads, page, dim), ps, ss = _check_codes(k_pages, v_pages, k_scales, v_scales)
        if dtype is None:
            dtype = torch.bfloat16
        elif dtype not in _HALF:
            raise RuntimeError(f"dtype must be bfloat16 or float16, got {dtype}")
    else:
        _, ps, vs = _check_pages(k_pages, v_pages)
        _require(vs == ps, "k_pages and v_pages must have the same strides")
        _require(dtype is None or dtype is k_pages.dtype, f"pages of {k_pages.dtype} are not read as {dtype}")
        code, on, ss, dtype = 0, k_pages.get_device(), (0, 0), k_pages.dtype   # (no scales)
        pages, heads, page, dim = k_pages.shape
    idx, n, width, ld = _check_table(table)
    if on != idx:
        raise RuntimeError(f"table must be on {k_pages.device}")
    _i32("cu_rows", cu_rows, n + 1, idx)
    _i32("kv_lens", kv_lens, n, idx)
    if rows < 0:
        raise RuntimeError("rows must not be negative")
    if out is None:
        key = torch.empty((rows, heads, dim), dtype=dtype, device=k_pages.device)
        value = torch.empty_like(key)
    else:
        key, value = out
        for t in out:
            _require(t.shape == (rows, heads, dim) and t.dtype is dtype and t.get_device() == idx and t.stride(2) == 1,
                     f"out must be two {dtype} [{rows}, {heads}, {dim}] on {k_pages.device} with contiguous channels")
    st = _lib.strides(*ps[:3], *ss, *key.stride()[:2], *value.stride()[:2])
    at = ctypes.addressof(st)
    guard = _lib.enter_device(idx)
    try:
        rc = lib.qkv_paged_read(k_pages.data_ptr(), v_pages.data_ptr(), at, _lib.ptr(k_scales), _lib.ptr(v_scales),
                                at + 24, code, pages, page, heads, dim, table.data_ptr(), ld, width, n,
                                cu_rows.data_ptr(), kv_lens.data_ptr(), rows, key.data_ptr(), at + 40,
                                value.data_ptr(), at + 56, _lib.DTYPE_CODES[dtype], _lib.stream_on(idx))
    finally:
        _lib.leave_device(guard)
    _lib.check(rc)
    return key, value


def attention_workspace(rows: int, max_rows: int, requests: int, width: int, page: int, q_heads: int, kv_heads: int,
                        head_dim: int, device, *, shared: bool = False) -> torch.Tensor:
    """A workspace for ``attention`` calls of these sizes, with ``shared``
    rows or without (contents irrelevant).  Calls that share one must not
    overlap in time."""
    lib = _lib.load()
    size = lib.qkv_paged_attention_shared_workspace_bytes if shared else lib.qkv_paged_attention_workspace_bytes
    need = size(rows, max_rows, requests, width, page, q_heads, kv_heads, head_dim)
    _require(need >= 0, "attention_workspace: sizes that attention does not take")
    return torch.empty(need // 4, dtype=torch.float32, device=device)


def attention(query: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor,
              cu_rows: torch.Tensor, kv_lens: torch.Tensor, scaling: float, *, max_rows: int | None = None,
              softcap: float = 0.0, slopes: torch.Tensor | None = None, prefix_lens: torch.Tensor | None = None,
              first_keys: torch.Tensor | None = None, out: torch.Tensor | None = None,
              workspace: torch.Tensor | None = None, k_scales: torch.Tensor | None = None,
              v_scales: torch.Tensor | None = None, shared: SharedRows | None = None) -> torch.Tensor:
    """query [rows, Hq, D] over the cached keys of the rows' requests, whose
    own K and V were appended before.  Row i of request b is the token at
    p = kv_lens[b] - (cu_rows[b + 1] - cu_rows[b]) + i and sees the keys j
    with first_keys[row] <= j < max(p + 1, prefix_lens[b]) that the request
    holds; a row that sees none gets zeros.

    ``softcap`` > 0 caps scores to softcap * tanh(scaling * q.k / softcap);
    ``slopes`` f32 [Hq] then takes slopes[h] * |p - j| off; ``prefix_lens``
    int32 [requests] opens the first keys to every row; ``first_keys`` int32
    [rows] hides the keys before a row's document (or window: p + 1 - w), a
    prefix's among them.  ``max_rows``, the most rows a request has where the
    caller knows it (1 in a decode step), spares workgroups and workspace;
    saying less than there is changes the result by its rounding at most.
    ``workspace`` (``attention_workspace``) spares an allocation.  Quantised
    pages come with ``k_scales`` and ``v_scales`` (``quantized_pages``) and
    are attended to as the values of the query's dtype that they stand for.

    ``shared`` (``share_rows`` of the same step) puts requests behind their
    parents: with n = the parent's tokens, row i of request b is the token at
    p = n + kv_lens[b] - (cu_rows[b + 1] - cu_rows[b]) + i of the parent's
    tokens and its own behind them, first_keys and prefix_lens count from the
    parent's first, and rows before a request's own first token get zeros.  A
    parent's keys are read for all rows behind it together, once for every 128
    (row, query head)s of a KV head.  The workspace then holds partial outputs
    of every (row, query head), about 33 KB a row with 32 heads of 128
    channels; rows times query heads stay below 2^26.

    Returns [rows, Hq, D] in the query's dtype; rows of ``out`` behind the
    last request are left as they were."""
    lib = _lib.load()
    if k_scales is not None or v_scales is not None or k_pages.dtype in _CODES:
        code, on, (pages, kv_heads, page, dim), ks, ss = _check_codes(k_pages, v_pages, k_scales, v_scales)
        dtype = _lib.half_code("query", query)
    else:
        dtype, ks, vs = _check_pages(k_pages, v_pages)
        if vs != ks:
            raise RuntimeError("k_pages and v_pages must have the same strides")
        if query.dtype is not k_pages.dtype:
            raise RuntimeError(f"query must be {k_pages.dtype} [rows, q_heads, dim] on {k_pages.device} with contiguous "
                               "channels")
        code, on, ss = 0, k_pages.get_device(), ()
        pages, kv_heads, page, dim = k_pages.shape
    idx, n, width, ld = _check_table(table)
    if on != idx:
        raise RuntimeError(f"table must be on {k_pages.device}")
    if query.dim() != 3 or query.get_device() != idx or query.stride(2) != 1 or query.size(2) != dim:
        raise RuntimeError(f"query must be {query.dtype} [rows, q_heads, {dim}] on {k_pages.device} with contiguous "
                           "channels")
    rows, q_heads, _ = query.shape
    _i32("cu_rows", cu_rows, n + 1, idx)
    _i32("kv_lens", kv_lens, n, idx)
    if prefix_lens is not None:
        _i32("prefix_lens", prefix_lens, n, idx)
    if first_keys is not None:
        _i32("first_keys", first_keys, rows, idx)
    if slopes is not None:
        _require(slopes.dtype is torch.float32 and slopes.get_device() == idx and slopes.shape == (q_heads,)
                 and slopes.is_contiguous(), f"slopes must be contiguous float32 [{q_heads}] on cuda:{idx}")
    if out is None:
        out = torch.empty_like(query, memory_format=torch.contiguous_format)
    else:
        _require(out.shape == query.shape and out.dtype is query.dtype and out.get_device() == idx
                 and out.stride(2) == 1, "out must have the query's shape, dtype and device with contiguous channels")
    most = rows if max_rows is None else max_rows
    ws_ptr, ws_bytes = None, 0
    if shared is not None and (shared.rows != rows or shared.requests != n or shared.buffer.get_device() != idx):
        raise RuntimeError(f"shared must be share_rows of {n} requests and {rows} rows on cuda:{idx}")
    if workspace is None:
        size = lib.qkv_paged_attention_workspace_bytes if shared is None else lib.qkv_paged_attention_shared_workspace_bytes
        ws_bytes = size(rows, most, n, width, page, q_heads, kv_heads, dim)
        if ws_bytes > 0:
            workspace = torch.empty(ws_bytes // 4, dtype=torch.float32, device=query.device)
            ws_ptr = workspace.data_ptr()
    else:
        _require(workspace.get_device() == idx and workspace.is_contiguous(),
                 f"workspace must be contiguous on cuda:{idx}")
        ws_ptr, ws_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    slopes_ptr = None if slopes is None else slopes.data_ptr()
    prefix_ptr = None if prefix_lens is None else prefix_lens.data_ptr()
    first_ptr = None if first_keys is None else first_keys.data_ptr()
    # row and head strides of the query, page, head and token strides of the pages, row and head strides of out, page
    # and head strides of the scales
    st = _lib.strides(*query.stride()[:2], *ks[:3], *out.stride()[:2], *ss)
    at = ctypes.addressof(st)
    guard = _lib.enter_device(idx)
    try:
        if shared is not None:
            rc = lib.qkv_paged_attention_shared(
                query.data_ptr(), at, k_pages.data_ptr(), v_pages.data_ptr(), at + 16, _lib.ptr(k_scales),
                _lib.ptr(v_scales), at + 56, code, shared.buffer.data_ptr(), pages, page, table.data_ptr(), ld, width, n,
                cu_rows.data_ptr(), kv_lens.data_ptr(), rows, most, q_heads, kv_heads, dim, scaling, softcap, slopes_ptr,
                prefix_ptr, first_ptr, ws_ptr, ws_bytes, out.data_ptr(), at + 40, dtype, _lib.stream_on(idx))
        elif code:
            rc = lib.qkv_paged_attention_codes(
                query.data_ptr(), at, k_pages.data_ptr(), v_pages.data_ptr(), at + 16, k_scales.data_ptr(),
                v_scales.data_ptr(), at + 56, code, pages, page, table.data_ptr(), ld, width, n, cu_rows.data_ptr(),
                kv_lens.data_ptr(), rows, most, q_heads, kv_heads, dim, scaling, softcap, slopes_ptr, prefix_ptr,
                first_ptr, ws_ptr, ws_bytes, out.data_ptr(), at + 40, dtype, _lib.stream_on(idx))
        else:
            rc = lib.qkv_paged_attention(
                query.data_ptr(), at, k_pages.data_ptr(), v_pages.data_ptr(), at + 16, pages, page, table.data_ptr(), ld,
                width, n, cu_rows.data_ptr(), kv_lens.data_ptr(), rows, most, q_heads, kv_heads, dim, scaling, softcap,
                slopes_ptr, prefix_ptr, first_ptr, ws_ptr, ws_bytes, out.data_ptr(), at + 40, dtype,
                _lib.stream_on(idx))
    finally:
        _lib.leave_device(guard)
    _lib.check(rc)
    return out

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
tokens that were rejected.  No length is needed on the host, so a step can be
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


def append(key: torch.Tensor, value: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
           slots: torch.Tensor) -> None:
    """Writes the rows' K and V, [rows, Hkv, D] at any strides with contiguous
    channels, to their ``slots`` (int64 [rows], as ``plan_step`` gives them;
    a row with -1 is skipped, no slot may come twice)."""
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


def attention_workspace(rows: int, max_rows: int, requests: int, width: int, page: int, q_heads: int, kv_heads: int,
                        head_dim: int, device) -> torch.Tensor:
    """A workspace for ``attention`` calls of these sizes (contents
    irrelevant).  Calls that share one must not overlap in time."""
    need = _lib.load().qkv_paged_attention_workspace_bytes(rows, max_rows, requests, width, page, q_heads, kv_heads,
                                                           head_dim)
    _require(need >= 0, "attention_workspace: sizes that attention does not take")
    return torch.empty(need // 4, dtype=torch.float32, device=device)


def attention(query: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor,
              cu_rows: torch.Tensor, kv_lens: torch.Tensor, scaling: float, *, max_rows: int | None = None,
              softcap: float = 0.0, slopes: torch.Tensor | None = None, prefix_lens: torch.Tensor | None = None,
              first_keys: torch.Tensor | None = None, out: torch.Tensor | None = None,
              workspace: torch.Tensor | None = None) -> torch.Tensor:
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
    ``workspace`` (``attention_workspace``) spares an allocation.  Returns
    [rows, Hq, D] in the query's dtype; rows of ``out`` behind the last
    request are left as they were."""
    lib = _lib.load()
    code, ks, vs = _check_pages(k_pages, v_pages)
    idx, n, width, ld = _check_table(table)
    pages, kv_heads, page, dim = k_pages.shape
    if k_pages.get_device() != idx:
        raise RuntimeError(f"table must be on {k_pages.device}")
    if vs != ks:
        raise RuntimeError("k_pages and v_pages must have the same strides")
    if (query.dim() != 3 or query.dtype is not k_pages.dtype or query.get_device() != idx or query.stride(2) != 1
            or query.size(2) != dim):
        raise RuntimeError(f"query must be {k_pages.dtype} [rows, q_heads, {dim}] on {k_pages.device} with contiguous "
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
    if workspace is None:
        ws_bytes = lib.qkv_paged_attention_workspace_bytes(rows, most, n, width, page, q_heads, kv_heads, dim)
        if ws_bytes > 0:
            workspace = torch.empty(ws_bytes // 4, dtype=torch.float32, device=query.device)
            ws_ptr = workspace.data_ptr()
    else:
        _require(workspace.get_device() == idx and workspace.is_contiguous(),
                 f"workspace must be contiguous on cuda:{idx}")
        ws_ptr, ws_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    # row and head strides of the query, page, head and token strides of the pages, row and head strides of out
    st = _lib.strides(*query.stride()[:2], *ks[:3], *out.stride()[:2])
    at = ctypes.addressof(st)
    guard = _lib.enter_device(idx)
    try:
        rc = lib.qkv_paged_attention(
            query.data_ptr(), at, k_pages.data_ptr(), v_pages.data_ptr(), at + 16, pages, page, table.data_ptr(), ld,
            width, n, cu_rows.data_ptr(), kv_lens.data_ptr(), rows, most, q_heads, kv_heads, dim, scaling, softcap,
            None if slopes is None else slopes.data_ptr(), None if prefix_lens is None else prefix_lens.data_ptr(),
            None if first_keys is None else first_keys.data_ptr(), ws_ptr, ws_bytes, out.data_ptr(), at + 40, code,
            _lib.stream_on(idx))
    finally:
        _lib.leave_device(guard)
    _lib.check(rc)
    return out

"""HuggingFace transformers integration: decode-time append of the int4 K
structures inside a ``Cache``, and an attention function that runs the int4
sparse decode step on it.

The reference reaches its selection through HF's eager attention, which it
patches (evaluate_qwen3_top2_head_limit3_ppl.py:6934-6944), and keeps an
auxiliary K copy (dim-major bf16) that it grows by one column per decode step
(EV:2018-2042).  Here the auxiliary structure is the int4 cache of
``int4.Int4KCache``: after prefill the packed K, the static channel subset and
the subset slab are built once; every later token is quantized into them in
place (``int4_pack_k`` / ``build_slab`` over ``[t, t+1)``) as HF appends it to
the bf16 (or fp16) cache.  K/V live in preallocated buffers of a fixed capacity, so no
step reallocates or copies the history.

Use:

    from kv_cache_amd import hf
    hf.register()                                         # attn_implementation "int4_sparse"
    model.config._attn_implementation = "int4_sparse"
    cache = hf.Int4SparseCache(capacity=40960, group=32, selected=32, block=16, topk=128)
    out = model(input_ids, past_key_values=cache, use_cache=True)       # prefill: dense SDPA
    out = model(next_ids, past_key_values=cache, use_cache=True)        # decode: int4 sparse

Prefill (more than one query per call) runs dense SDPA on the GPU, as the
reference's prefill runs dense HF attention (EV:7079-7111), with transformers'
SDPA mask (``register`` registers it for the new name, so padding is applied).
Decode steps with one query per sequence run the int4 path with the
reference's decode semantics (EV:4419-4460, 2938-2982): the blocks are chosen
over the history (every cached token but the current one), and the attention
covers them plus the protected tokens -- ``protect_sink`` first tokens,
``protect_recent`` last history tokens and, with ``keep_self`` (the
reference's default), the current token.  The int4 kernels take no per-token
mask, so a decode step on a padded batch (a mask that hides cached positions)
raises instead of attending to the padding.  The channel subset is the one
chosen when the int4 structures are built at the first decode step (the
static per-KV-head subset of the int4 design); later tokens are quantized
into it.

The reference's other decode modes run through ``register_mode(mode,
capacity)``: the candidate-reuse modes (``qabs{S}cand{pct}reuse…``), the
lagged modes (``lagtop2`` / ``lagrefresh{N}`` / ``qdrift…`` / ``pconf{T}`` +
``qabs{S}cand{pct}``), the exact candidate attention (``qabs{S}cand{pct}
[append|r{N}]attn``) and the block selectors (``qbb…`` / ``brep…`` /
``qboracle…``), each through its native decode step (``reuse.ReuseDecodeStep``,
``reuse.LaggedReuseDecodeStep``, ``reuse.QabsCandidateAttentionStep``,
``blocksel.BlockSelectDecodeStep``), one per attention layer, on any HF cache
(K/V [B, Hkv, T, D] with the current token last).  As the reference's hook
dispatches these modes only for one query per sequence (EV:6236, 6308,
6414-6448), prefill stays dense SDPA.

``PagedCache`` with the implementation of ``register_paged`` keeps K/V in pages
(``paged``) and runs prompts, chunks and decode steps densely over them,
left-padded batches included: padding takes no slot, and every sequence has
its own length on the GPU.  Masks are compared with what the pages show: any
other than causal with left padding and the layer's window raises.

    hf.register_paged()                                   # attn_implementation "paged"
    model.config._attn_implementation = "paged"
    cache = hf.PagedCache(capacity=40960, page=64)
    out = model.generate(**tokenizer(prompts, padding=True), past_key_values=cache)
"""

from __future__ import annotations

import functools
import math
import weakref

import torch

from . import int4 as K
from . import paged

# Cache layers by the address of their K buffer: the attention function gets
# K as a view of that buffer and finds the layer's int4 state through it.
# Weak references, so a freed cache's address cannot match a later tensor.
_LAYERS: "weakref.WeakValueDictionary[int, Int4CacheLayer]" = weakref.WeakValueDictionary()


class Int4CacheLayer:
    """One layer's K/V (bf16 or fp16) in preallocated buffers plus its int4 structures."""

    is_sliding = False
    is_compileable = False
    supports_early_init = False

    def __init__(self, capacity: int, group: int, selected: int, block: int, topk: int, protect_sink: int = 0,
                 protect_recent: int = 0, keep_self: bool = True):
        self.capacity = K.round_capacity(capacity)
        self.group, self.selected, self.block, self.topk = int(group), int(selected), int(block), int(topk)
        self.protect = dict(protect_sink=max(0, int(protect_sink)), protect_recent=max(0, int(protect_recent)),
                            keep_self=bool(keep_self))
        self.keys = self.values = None
        self.is_initialized = False
        self.length = 0
        self.int4 = None          # Int4KCache once built
        self.bufs = None          # decode-step buffers

    def __repr__(self):
        return f"Int4CacheLayer(length={self.length}, capacity={self.capacity})"

    # -- CacheLayerMixin protocol ------------------------------------------
    def lazy_initialization(self, key_states: torch.Tensor, value_states: torch.Tensor) -> None:
        b, h, _, d = key_states.shape
        dev = key_states.device
        self.dtype, self.device = key_states.dtype, dev
        self._k = torch.empty((b, h, self.capacity, d), dtype=key_states.dtype, device=dev)
        self._v = torch.empty((b, h, self.capacity, d), dtype=value_states.dtype, device=dev)
        _LAYERS[self._k.data_ptr()] = self
        self.is_initialized = True

    def update(self, key_states: torch.Tensor, value_states: torch.Tensor, *args, **kwargs):
        if not self.is_initialized:
            self.lazy_initialization(key_states, value_states)
        n = key_states.size(-2)
        t0, t1 = self.length, self.length + n
        if t1 > self.capacity:
            raise RuntimeError(f"Int4 cache capacity {self.capacity} exceeded ({t1} tokens)")
        self._k[:, :, t0:t1].copy_(key_states)
        self._v[:, :, t0:t1].copy_(value_states)
        self.length = t1
        self.keys, self.values = self._k[:, :, :t1], self._v[:, :, :t1]
        if self.int4 is not None:
            self.append_int4(t0, t1)
        return self.keys, self.values

    def get_mask_sizes(self, query_length: int):
        return self.length + query_length, 0

    def get_seq_length(self) -> int:
        return self.length

    def get_max_length(self) -> int:
        return self.capacity

    def reset(self) -> None:
        self.length = 0
        self.int4 = None

    def offload(self):
        raise RuntimeError("Int4CacheLayer cannot be offloaded")

    prefetch = offload

    # -- int4 structures ---------------------------------------------------
    def build_int4(self) -> None:
        """Pack the cached tokens, choose the channel subset, build the slab."""
        if self.keys.dtype not in (torch.bfloat16, torch.float16):
            raise RuntimeError(f"the int4 path needs bfloat16 or float16 K/V, got {self.keys.dtype}")
        t = self.length
        packed, scales = K.int4_pack_k(self._k, self.group, capacity=self.capacity, t_end=t)
        chan, _ = K.select_channels(packed, scales, t, self.group, self.selected)
        slab, slab_scales = K.build_slab(self._k, chan, capacity=self.capacity, t_end=t)
        self.int4 = K.Int4KCache(packed, scales, chan, slab, slab_scales, t, self.group)

    def append_int4(self, t0: int, t1: int) -> None:
        """Quantize tokens [t0, t1) into the packed K and the slab (the channel
        subset stays the one chosen at prefill)."""
        c = self.int4
        K.int4_pack_k(self._k, self.group, packed=c.packed, scales=c.scales, t_begin=t0, t_end=t1)
        K.build_slab(self._k, c.chan_idx, slab=c.slab, slab_scales=c.slab_scales, t_begin=t0, t_end=t1)
        c.tokens = t1

    def decode_buffers(self, batch: int, q_heads: int, kv_heads: int, head_dim: int):
        """Block maxima, selection, workspaces and output sized for the full
        capacity, allocated once (flat, so that each step takes a contiguous
        view of its own size)."""
        if self.bufs is None:
            nb = math.ceil(self.capacity / self.block)
            k = min(self.topk, nb)
            dev = self.device
            n_ws = K.protected_workspace_blocks(k, self.block, self.capacity - 1, **self.protect)
            self.bufs = {
                "bmax": torch.empty(batch * kv_heads * nb, dtype=torch.float32, device=dev),
                "sel": torch.empty(batch * kv_heads * k, dtype=torch.int32, device=dev),
                "topk_ws": K.topk_workspace(batch * kv_heads, nb, k, dev),
                "attn_ws": K.attention_workspace(batch, q_heads, kv_heads, head_dim, n_ws, self.block, dev),
            }
        return self.bufs


class Int4SparseCache:
    """A transformers ``Cache`` whose layers keep K/V in preallocated buffers
    and append the int4 structures at every decode step."""

    def __new__(cls, capacity: int, group: int = 32, selected: int = 32, block: int = 16, topk: int = 128, *,
                protect_sink: int = 0, protect_recent: int = 0, keep_self: bool = True):
        from transformers.cache_utils import Cache, CacheLayerMixin

        layer_cls = _layer_class(CacheLayerMixin)
        cache = Cache(layer_class_to_replicate=functools.partial(
            layer_cls, capacity, group, selected, block, topk, protect_sink, protect_recent, keep_self))
        return cache


@functools.lru_cache(maxsize=1)
def _layer_class(mixin):
    # Int4CacheLayer registered as a CacheLayerMixin so transformers' checks accept it.
    return type("Int4CacheLayerHF", (Int4CacheLayer, mixin), {"__init__": Int4CacheLayer.__init__})


def int4_sparse_attention_forward(module, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor,
                                  attention_mask, scaling: float | None = None, dropout: float = 0.0, **kwargs):
    """HF attention interface (query [B,Hq,q,D]; key/value [B,Hkv,T,D]) ->
    (out [B,q,Hq,D], None).  One query per sequence on an Int4SparseCache:
    int4 scoring of the history + top-k blocks + GQA sparse attention over
    them and the protected tokens; otherwise dense SDPA."""
    from transformers.integrations.sdpa_attention import sdpa_attention_forward

    layer = _LAYERS.get(key.data_ptr())
    if query.size(2) != 1 or layer is None or layer.keys is None or key.size(2) != layer.length:
        return sdpa_attention_forward(module, query, key, value, attention_mask, dropout=dropout, scaling=scaling,
                                      **kwargs)
    if layer.int4 is None:
        # once per sequence, when the int4 structures are built: the cached
        # positions' padding does not change later, and new tokens are real
        if attention_mask is not None and not _all_visible(attention_mask, layer.length):
            raise RuntimeError("int4 sparse decode does not support padded batches (the attention mask hides cached "
                               "positions); decode such batches with dense attention")
        layer.build_int4()
    b, hq, _, d = query.shape
    hkv = key.size(1)
    t = layer.length
    history = t - 1                       # the current token is not a candidate (EV:4414-4415)
    if history < 1:
        return sdpa_attention_forward(module, query, key, value, attention_mask, dropout=dropout, scaling=scaling,
                                      **kwargs)
    scaling = d ** -0.5 if scaling is None else float(scaling)
    bufs = layer.decode_buffers(b, hq, hkv, d)
    c = layer.int4
    nb = math.ceil(history / layer.block)
    k = min(layer.topk, nb)
    q = query[:, :, 0, :].contiguous()
    bmax = bufs["bmax"][: b * hkv * nb].view(b, hkv, nb)
    K.decode_scores(q, c.chan_idx, c.slab, c.slab_scales, history, layer.block, bmax=bmax)
    sel = bufs["sel"][: b * hkv * k].view(b, hkv, k)
    if nb <= K.SELECT_MAX_BLOCKS:
        out = K.sparse_attention_select(q, layer.keys, layer.values, bmax, k, layer.block, history, scaling,
                                        workspace=bufs["attn_ws"], sel_out=sel, **layer.protect)
    else:
        K.block_topk(bmax, k, out=sel, workspace=bufs["topk_ws"])
        out = K.sparse_attention(q, layer.keys, layer.values, sel, layer.block, history, scaling,
                                 workspace=bufs["attn_ws"], **layer.protect)
    # a fresh output per call: callers may keep a step's attention output
    # (hooks, captured activations) while later steps run
    return out[:, None].to(query.dtype), None


def _all_visible(mask: torch.Tensor, length: int) -> bool:
    """True when a decode step's attention mask ([B, 1, q, T], bool or
    additive float) hides none of the first ``length`` positions."""
    m = mask[..., -1, :length]
    return bool(m.all()) if m.dtype == torch.bool else bool((m == 0).all())


def register(name: str = "int4_sparse") -> str:
    """Register the attention function with transformers under ``name``."""
    from transformers import AttentionInterface
    from transformers.masking_utils import AttentionMaskInterface, sdpa_mask

    AttentionInterface.register(name, int4_sparse_attention_forward)
    # without a mask function of its own a custom implementation gets no mask
    # at all, padding included; SDPA's mask is the one its prefill path uses
    AttentionMaskInterface.register(name, sdpa_mask)
    return name


def native_step_class(mode: str):
    """The decode step that serves a reference mode string, or ValueError."""
    from . import blocksel, reuse

    if reuse.is_lagged_mode(mode):
        return reuse.LaggedReuseDecodeStep
    for parse, cls in ((reuse.parse_reuse_mode, reuse.ReuseDecodeStep),
                       (reuse.parse_qabs_attn_mode, reuse.QabsCandidateAttentionStep),
                       (blocksel.parse_block_mode, blocksel.BlockSelectDecodeStep)):
        try:
            parse(mode)
        except (RuntimeError, ValueError):
            continue
        return cls
    raise ValueError(f"{mode!r} is not a mode served by a native decode step")


def register_mode(mode: str, capacity: int, *, name: str | None = None, **step_kwargs) -> str:
    """Register an attention implementation (default name ``qkv_<mode>``) that
    runs ``mode``'s native decode step for one query per sequence and dense
    SDPA otherwise.  ``capacity`` bounds the cached tokens per sequence;
    ``step_kwargs`` go to the step (``top_fraction``, ``protect_sink``,
    ``protect_recent``, ``keep_self``, ``candidate_selection``, …, as the
    reference's flags).  The steps, one per attention module, are in the
    returned function's ``steps`` (``ATTENTION_STEPS[name]``); each starts a
    new sequence by itself when the history does not continue its last call's
    (EV:1651's query-token check)."""
    from transformers import AttentionInterface
    from transformers.integrations.sdpa_attention import sdpa_attention_forward
    from transformers.masking_utils import AttentionMaskInterface, sdpa_mask

    cls = native_step_class(mode)
    steps: weakref.WeakKeyDictionary = weakref.WeakKeyDictionary()

    def forward(module, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, attention_mask,
                scaling: float | None = None, dropout: float = 0.0, **kwargs):
        if query.size(2) != 1:
            return sdpa_attention_forward(module, query, key, value, attention_mask, dropout=dropout,
                                          scaling=scaling, **kwargs)
        if attention_mask is not None and not _all_visible(attention_mask, key.size(2)):
            raise RuntimeError(f"{mode} decode does not support padded batches (the attention mask hides cached "
                               "positions); decode such batches with dense attention")
        b, hq, _, d = query.shape
        hkv = key.size(1)
        step = steps.get(module)
        if (step is None or (step.batch, step.q_heads, step.kv_heads, step.head_dim) != (b, hq, hkv, d)
                or step.dtype != query.dtype):
            step = cls(mode, b, hq, hkv, d, capacity, device=query.device, **{**step_kwargs, "dtype": query.dtype})
            steps[module] = step
        scaling = d ** -0.5 if scaling is None else float(scaling)
        out = step(query[:, :, 0, :], key, value, scaling)
        # the step's output buffer is overwritten by its next call
        return out[:, None].clone(), None

    forward.steps = steps
    name = name or f"qkv_{mode}"
    AttentionInterface.register(name, forward)
    AttentionMaskInterface.register(name, sdpa_mask)
    ATTENTION_STEPS[name] = steps
    return name


ATTENTION_STEPS: dict = {}


# An additive mask hides a key with this or less: its weight is zero beside any score.
_HIDDEN = -1.0e4


class _PagedState:
    """What the layers of one PagedCache share: the page table, which columns
    hold tokens, and the plan of the step that the first layer to reach it
    made."""

    def __init__(self, capacity: int, page: int):
        self.capacity, self.page = int(capacity), int(page)
        self.table = self.plan = None
        self.real = None         # bool [batch, columns]: those with a token; None while no step had a mask
        self.masks = []          # (mask, window) of the step's layers, compared with what the pages show
        self.length = self.new = 0   # columns stepped, padding included; of the last step
        self.open = False        # an update's columns have not been attended over yet

    def check_closed(self) -> None:
        """Raises if the attention function did not take an earlier update:
        its columns are in no page."""
        if self.open:
            raise RuntimeError("K and V of an earlier update of this PagedCache were not taken: run the model with the "
                               "attention implementation of register_paged, and reset() the cache")

    def step(self, length: int, n: int, batch: int, device, attention_mask, window) -> paged.StepPlan:
        """The plan of the step that brings the sequences to ``length``
        columns with ``n`` new ones; raises where a layer's mask is not what
        its attention over the pages shows."""
        first = self.length != length
        if length - n != (self.length if first else self.length - self.new):
            raise RuntimeError(f"the layers of a PagedCache step together: a layer steps from {length - n} columns to "
                               f"{length}, the cache holds {self.length}")
        if first:
            self.masks = []
            if self.length == 0:
                self.real = None     # a refused step's, of whatever batch
        # layers share a mask or two: one host read for each in a step
        if attention_mask is not None and not any(m is attention_mask and w == window for m, w in self.masks):
            self._compare(length, n, batch, device, attention_mask, window, first)
            self.masks.append((attention_mask, window))
        elif first and self.real is not None:
            self.real = torch.cat((self.real[:, :self.length], self.real.new_ones((batch, n))), 1)
        if not first:
            return self.plan
        if self.table is None or (self.length == 0 and self.table.lens.numel() != batch):
            pages = batch * -(-self.capacity // self.page)
            self.table = paged.PageTable(batch, self.capacity, pages, self.page, device)
        if attention_mask is None:
            new = torch.full((batch,), n, dtype=torch.int32, device=device)
        else:
            new = self.real[:, length - n:length].sum(-1, dtype=torch.int32)
        self.plan = self.table.step(new, batch * n, padded=n)
        self.length, self.new = length, n
        return self.plan

    def _compare(self, length: int, n: int, batch: int, device, mask, window, first: bool) -> None:
        """Takes the padding of the step's columns from the mask (``first``)
        and compares the rest of it: a token's query has to see its sequence's
        tokens up to its own, within the window.  The rows of padding may see
        anything."""
        if (mask.dim() != 4 or mask.size(0) not in (1, batch) or mask.size(2) not in (1, n) or mask.size(3) < length
                or not (mask.dtype == torch.bool or mask.is_floating_point())):
            raise RuntimeError(f"paged attention takes bool or additive masks [{batch}, heads, {n}, {length} columns], "
                               f"got {mask.dtype} {list(mask.shape)}")
        mask = mask[..., :length].expand(batch, -1, n, -1)
        real = self.real
        if real is None:
            real = torch.ones((batch, length), dtype=torch.bool, device=device)
        if first:   # padding: a column that its own query does not see
            own = mask[:, 0, :, length - n:].diagonal(dim1=-2, dim2=-1)
            real = torch.cat((real[:, :length - n], own if own.dtype == torch.bool else own == 0), 1)
        # the window counts tokens, as the pages hold them
        token = None if window is None else real.cumsum(-1)
        at = torch.arange(length, device=device) if n > 1 else None   # a single query is behind all columns
        rows = max(1, (1 << 26) // (batch * mask.size(1) * length))   # bounds what is compared at a time
        other = []
        for i in range(0, n, rows):
            cols = slice(length - n + i, min(length - n + i + rows, length))
            seen = real[:, None]
            if n > 1:
                seen = seen & (at <= at[cols, None])
            if window is not None:
                seen = seen & (token[:, None] > token[:, cols, None] - window)
            seen, m = seen[:, None], mask[:, :, i:i + rows]
            differs = m != seen if m.dtype == torch.bool else torch.where(seen, m != 0, ~(m <= _HIDDEN))
            other.append((differs & real[:, None, cols, None]).any())
        if n > 1:
            fresh = real[:, length - n:]
            other.append((fresh[:, :-1] & ~fresh[:, 1:]).any())
            if other.pop():
                raise RuntimeError("paged attention takes left-padded batches (padding before the tokens of a step)")
        if other[0] if len(other) == 1 else torch.stack(other).any():
            raise RuntimeError("paged attention takes causal masks, with the layer's sliding window and left padding; "
                               "this mask shows or hides other keys")
        self.real = real

    def reset(self) -> None:
        if self.table is not None and self.length:
            self.table.release(torch.zeros_like(self.table.lens))
        self.length, self.real, self.masks, self.open = 0, None, [], False


class PagedCacheLayer:
    """One layer's K/V pages (bf16 or fp16).  ``update`` only counts the new
    columns and hands the layer on to the attention function with their K/V;
    that one knows the mask, and writes what is no padding into the pages.
    Another attention function would see the new columns alone: the next
    update raises then."""

    is_sliding = False
    is_compileable = False
    supports_early_init = False

    def __init__(self, state: _PagedState):
        self.state = state
        self.keys = self.values = None        # no dense K/V exist
        self.k_pages = self.v_pages = None
        self.is_initialized = False
        self.length = 0

    def __repr__(self):
        return f"PagedCacheLayer(length={self.length}, capacity={self.state.capacity}, page={self.state.page})"

    def page_shape(self, key_states: torch.Tensor) -> tuple:
        b, h, _, d = key_states.shape
        return b * -(-self.state.capacity // self.state.page), h, self.state.page, d

    def holds(self, key_states: torch.Tensor) -> bool:
        """Whether the pages are those of such keys."""
        return (self.k_pages.shape == self.page_shape(key_states) and self.dtype == key_states.dtype
                and self.device == key_states.device)

    def take_back(self, n: int) -> None:
        """Undoes an update whose step was refused before anything was written;
        a step that other layers have made stays open."""
        if self.state.length != self.length:
            self.length -= n
            self.state.open = False

    # -- CacheLayerMixin protocol ------------------------------------------
    def lazy_initialization(self, key_states: torch.Tensor, value_states: torch.Tensor) -> None:
        shape = self.page_shape(key_states)
        self.dtype, self.device = key_states.dtype, key_states.device
        self.k_pages = torch.empty(shape, dtype=key_states.dtype, device=key_states.device)
        self.v_pages = torch.empty(shape, dtype=value_states.dtype, device=key_states.device)
        self.is_initialized = True

    def update(self, key_states: torch.Tensor, value_states: torch.Tensor, *args, **kwargs):
        self.state.check_closed()
        n = key_states.size(-2)
        if self.length + n > self.state.capacity:
            raise RuntimeError(f"Paged cache capacity {self.state.capacity} exceeded ({self.length + n} tokens)")
        # an empty layer takes any batch, whatever it held before
        if not self.is_initialized or (self.length == 0 and not self.holds(key_states)):
            self.lazy_initialization(key_states, value_states)
        self.length += n
        self.state.open = True
        key_states = key_states.view(key_states.shape)
        key_states.paged_layer = self
        return key_states, value_states

    def get_mask_sizes(self, query_length: int):
        self.state.check_closed()
        return self.length + query_length, 0

    def get_seq_length(self) -> int:
        return self.length

    def get_max_length(self) -> int:
        return self.state.capacity

    def reset(self) -> None:
        self.length = 0
        self.state.reset()

    def crop(self, max_length: int) -> None:
        raise RuntimeError("PagedCacheLayer cannot be cropped")

    def reorder_cache(self, beam_idx) -> None:
        raise RuntimeError("PagedCacheLayer cannot be reordered")

    batch_repeat_interleave = batch_select_indices = reorder_cache

    def offload(self):
        raise RuntimeError("PagedCacheLayer cannot be offloaded")

    prefetch = offload


class PagedCache:
    """A transformers ``Cache`` whose layers keep K/V in pages of ``page``
    tokens under one page table; ``capacity`` bounds the columns (tokens and
    padding) of a sequence."""

    def __new__(cls, capacity: int, page: int = 64):
        from transformers.cache_utils import Cache, CacheLayerMixin

        if not (16 <= page <= 4096 and page & (page - 1) == 0):
            raise RuntimeError(f"page must be a power of two in [16, 4096], got {page}")
        return Cache(layer_class_to_replicate=functools.partial(_paged_layer_class(CacheLayerMixin),
                                                               _PagedState(capacity, page)))


@functools.lru_cache(maxsize=1)
def _paged_layer_class(mixin):
    return type("PagedCacheLayerHF", (PagedCacheLayer, mixin), {"__init__": PagedCacheLayer.__init__})


# Arguments of the attention interface that hold a tensor and do not change what is attended to or how.
_IGNORED = frozenset(("position_ids", "cache_position", "token_type_ids", "input_ids", "labels", "num_items_in_batch"))


def _check_interface(module, n: int, key: torch.Tensor, attention_mask, dropout: float, arguments: dict) -> None:
    """Raises for what the attention over the pages would leave out: dropout,
    scores with sinks or biases, packed sequences, queries that see later
    keys."""
    if dropout:
        raise RuntimeError("paged attention has no dropout")
    for name, x in arguments.items():
        if isinstance(x, float) or (isinstance(x, torch.Tensor) and name not in _IGNORED):
            raise RuntimeError(f"paged attention does not take {name}")
    if key.size(2) != n:
        raise RuntimeError(f"paged attention takes queries and keys of the same tokens, got {n} and {key.size(2)}")
    causal = arguments.get("is_causal")
    if n > 1 and attention_mask is None and not (getattr(module, "is_causal", True) if causal is None else causal):
        raise RuntimeError("paged attention is causal: is_causal is False and there is no mask")


class _NoBackward(torch.autograd.Function):
    """Ties an output to the inputs it has no gradients for: a backward pass
    raises, where it would leave their part out."""

    @staticmethod
    def forward(ctx, out, *inputs):
        return out.view_as(out)

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("paged attention has no backward: run the model under torch.no_grad(), or train it without "
                           "a PagedCache")


def paged_attention_forward(module, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, attention_mask,
                            scaling: float | None = None, dropout: float = 0.0, softcap: float | None = None,
                            sliding_window: int | None = None, **kwargs):
    """HF attention interface (query [B,Hq,n,D]; key/value [B,Hkv,n,D], the new
    columns a PagedCache layer handed on) -> (out [B,n,Hq,D], None).  What
    columns of padding get is for nobody: zeros before a sequence's first
    token, attention over its earlier tokens later.  Without a PagedCache:
    dense SDPA."""
    from transformers.integrations.sdpa_attention import sdpa_attention_forward

    layer = getattr(key, "paged_layer", None)
    if layer is None:
        return sdpa_attention_forward(module, query, key, value, attention_mask, dropout=dropout, scaling=scaling,
                                      **kwargs)
    b, hq, n, d = query.shape
    state = layer.state
    try:
        _check_interface(module, n, key, attention_mask, dropout, kwargs)
        plan = state.step(layer.length, n, b, query.device, attention_mask, sliding_window)
    except Exception:
        layer.take_back(key.size(2))
        raise
    rows = lambda x: x.transpose(1, 2).reshape(b * n, x.size(1), d)  # noqa: E731  (a view of what projections give)
    paged.append(rows(key), rows(value), layer.k_pages, layer.v_pages, plan.slots)
    first = None if sliding_window is None else plan.positions - (int(sliding_window) - 1)
    out = paged.attention(rows(query), layer.k_pages, layer.v_pages, state.table.table, plan.cu_rows, plan.kv_lens,
                          d ** -0.5 if scaling is None else float(scaling), max_rows=n,
                          softcap=0.0 if softcap is None else float(softcap), first_keys=first)
    state.open = False
    if torch.is_grad_enabled() and (query.requires_grad or key.requires_grad or value.requires_grad):
        out = _NoBackward.apply(out, query, key, value)
    return out.view(b, n, hq, d), None


def register_paged(name: str = "paged") -> str:
    """Register the paged attention function with transformers under ``name``."""
    from transformers import AttentionInterface
    from transformers.masking_utils import AttentionMaskInterface, sdpa_mask

    AttentionInterface.register(name, paged_attention_forward)
    AttentionMaskInterface.register(name, sdpa_mask)
    return name

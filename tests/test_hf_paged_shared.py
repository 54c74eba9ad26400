"""PagedCache.batch_repeat_interleave on the CPU: sequences that continue one
prompt, over plain forms of the page table, the writes and the attention, in
32 bits against dense SDPA of the repeated batch (the bound of the adapter's
other CPU tests)."""

import pytest
import torch

from kv_cache_amd import hf, paged
from test_hf_paged import _left_padded, _model, _plain_append, _plain_attention, _plain_release, _plain_step, _tokens


class _Shared:
    def __init__(self, parents, cu, kv, lens, rows):
        self.before = [int(lens[p]) if 0 <= p < len(parents) and n > 0 else 0 for p, n in zip(parents.tolist(), kv.tolist())]
        self.parents, self.lens = parents.tolist(), lens.tolist()
        self.positions = torch.full((rows,), -1, dtype=torch.int32)
        for b, n in enumerate(kv.tolist()):
            for row in range(int(cu[b]), min(int(cu[b + 1]), rows)):
                p = n - (int(cu[b + 1]) - row)
                if p >= 0:
                    self.positions[row] = self.before[b] + p


def _attention(q, k_pages, v_pages, table, cu, kv, scaling, *, shared=None, first_keys=None, **kw):
    if shared is None:
        return _plain_attention(q, k_pages, v_pages, table, cu, kv, scaling, first_keys=first_keys, **kw)
    # every request alone, its parent's tokens before its own in pages of one token
    out = torch.zeros_like(q)
    flat = lambda x, b, n: x[table[b].long().clamp(min=0)].transpose(1, 2).flatten(0, 1)[:n]  # noqa: E731
    for b, n in enumerate(kv.tolist()):
        a, e = int(cu[b]), min(int(cu[b + 1]), q.shape[0])
        if a >= e:
            continue
        real = min(e - a, n)       # rows with a token, the last ones
        if real == 0:
            continue
        both = [torch.cat((flat(x, shared.parents[b], shared.before[b]), flat(x, b, n))) if shared.before[b] else flat(x, b, n)
                for x in (k_pages, v_pages)]
        m = both[0].shape[0]
        pages = [x[:, :, None] for x in both]
        out[e - real:e] = _plain_attention(q[e - real:e], *pages, torch.arange(m)[None], torch.tensor([0, real]), torch.tensor([m]),
                                           scaling, first_keys=None if first_keys is None else first_keys[e - real:e], **kw)
    return out


@pytest.fixture
def plain(monkeypatch):
    monkeypatch.setattr(paged.PageTable, "step", _plain_step)
    monkeypatch.setattr(paged.PageTable, "release", _plain_release)
    monkeypatch.setattr(paged, "append", _plain_append)
    monkeypatch.setattr(paged, "attention", _attention)
    monkeypatch.setattr(paged, "share_rows", _Shared)
    hf.register_paged()


def _dense(model):
    from transformers.cache_utils import DynamicCache

    return DynamicCache(config=model.config)


def _columns(model, impl, cache, ids, mask, widths, at=0):
    model.config._attn_implementation = impl
    out = []
    with torch.no_grad():
        for w in widths:
            kw = {}
            if mask is not None:
                m = mask[:, : at + w]
                kw = dict(attention_mask=m, position_ids=(m.cumsum(-1) - 1).clamp(min=0)[:, at: at + w])
            out.append(model(ids[:, at: at + w], past_key_values=cache, use_cache=True, **kw).logits)
            at += w
    return torch.cat(out, 1)


@pytest.mark.parametrize("sliding", [False, True])
@pytest.mark.parametrize("padded", [False, True])
@pytest.mark.parametrize("prompts,copies,n,widths", [(1, 3, 20, [1, 1, 1]), (2, 2, 17, [1, 4, 1]), (2, 3, 16, [17, 1])])
def test_continuations_of_prompts(plain, prompts, copies, n, widths, padded, sliding):
    model = _model(**(dict(use_sliding_window=True, sliding_window=11, max_window_layers=0) if sliding else {}))
    ids = _tokens(prompts, n, 1).repeat_interleave(copies, 0)
    ids = torch.cat((ids, _tokens(prompts * copies, sum(widths), 2)), 1)
    mask = None
    if padded:
        mask = torch.cat((_left_padded([n - 5 * b for b in range(prompts)], n).repeat_interleave(copies, 0),
                          torch.ones((prompts * copies, sum(widths)), dtype=torch.long)), 1)
    cache = hf.PagedCache(capacity=64, page=16)
    first = _columns(model, "paged", cache, ids[::copies], None if mask is None else mask[::copies], [n])
    cache.batch_repeat_interleave(copies)
    got = torch.cat((first.repeat_interleave(copies, 0), _columns(model, "paged", cache, ids, mask, widths, n)), 1)
    want = _columns(model, "sdpa", _dense(model), ids, mask, [n, *widths])
    real = torch.ones(ids.shape, dtype=torch.bool) if mask is None else mask.bool()
    assert (got - want)[real].abs().max() <= 1e-4 * want[real].abs().max()
    state = cache.layers[0].state
    batch = prompts * copies
    assert state.table.lens[:batch].tolist() == [sum(widths)] * batch       # their own tokens alone
    held = state.table.table[state.table.table >= 0].tolist()
    assert len(held) == len(set(held)) and len(held) + int(state.table.count) == state.table.pages
    assert all(layer.k_pages.shape[0] == state.table.pages for layer in cache.layers)
    # another batch after a reset, of another size
    cache.reset()
    again = _columns(model, "paged", cache, ids[:1], None if mask is None else mask[:1], [n, *widths])
    assert (again - want[:1])[real[:1]].abs().max() <= 1e-4 * want[real].abs().max()


def test_refusals(plain):
    model, ids = _model(), _tokens(2, 12, 3)
    cache = hf.PagedCache(capacity=32, page=16)
    _columns(model, "paged", cache, ids, None, [8])
    with pytest.raises(RuntimeError, match="positive"):
        cache.batch_repeat_interleave(0)
    cache.batch_repeat_interleave(1)
    assert cache.layers[0].state.copies == 1
    cache.batch_repeat_interleave(2)
    with pytest.raises(RuntimeError, match="repeated once"):
        cache.batch_repeat_interleave(2)
    with pytest.raises(RuntimeError, match="repeated for 4 sequences, this step has 2"):
        _columns(model, "paged", cache, ids, None, [1], 8)
    with pytest.raises(RuntimeError, match="repeated for 4 sequences, this step has 2"):
        _columns(model, "paged", cache, ids, _left_padded([9, 8], 9), [1], 8)      # with a mask too
    rows = ids.repeat_interleave(2, 0)
    got = _columns(model, "paged", cache, rows, None, [1, 3], 8)      # the refused steps left it as it was
    want = _columns(model, "sdpa", _dense(model), rows, None, [12])[:, 8:]
    assert (got - want).abs().max() <= 1e-4 * want.abs().max()
    layer = hf.PagedCacheLayer(hf._PagedState(32, 16))
    with pytest.raises(RuntimeError, match="repeated once"):
        layer.batch_repeat_interleave(2)       # before a prompt
    with pytest.raises(RuntimeError, match="quantize must be"):
        hf.PagedCache(capacity=32, page=16, quantize="int8")

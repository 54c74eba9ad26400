"""PagedCache.batch_repeat_interleave on the CPU: what it refuses, and what a
step after it asks of the page table.  Plain forms and bounds as in the
adapter's other CPU tests."""

import pytest
import torch

from kv_cache_amd import hf, paged
from test_hf_paged import _model, _tokens
from test_hf_paged_shared import _columns, _dense, plain  # noqa: F401


def test_layers_repeated_apart_are_refused(plain):  # noqa: F811
    model, ids = _model(), _tokens(2, 12, 5)
    cache = hf.PagedCache(capacity=32, page=16)
    _columns(model, "paged", cache, ids, None, [8])
    rows = ids.repeat_interleave(3, 0)
    cache.layers[0].batch_repeat_interleave(3)
    with pytest.raises(RuntimeError, match="not repeated with the others"):
        _columns(model, "paged", cache, rows, None, [1], 8)
    cache.reset()
    got = _columns(model, "paged", cache, ids, None, [8])
    cache.layers[1].batch_repeat_interleave(3)
    with pytest.raises(RuntimeError, match="not repeated with the others"):
        _columns(model, "paged", cache, rows, None, [1], 8)
    cache.layers[0].batch_repeat_interleave(3)       # all of them now: the refused step left nothing
    got = torch.cat((got.repeat_interleave(3, 0), _columns(model, "paged", cache, rows, None, [1, 3], 8)), 1)
    want = _columns(model, "sdpa", _dense(model), rows, None, [8, 4])
    assert (got - want).abs().max() <= 1e-4 * want.abs().max()


@pytest.mark.parametrize("prompts,capacity,repeats", [(1, 32, 4096), (2, 32, 2048), (1, 1 << 14, 1100)])
def test_more_than_a_step_takes_is_refused(plain, prompts, capacity, repeats):  # noqa: F811
    """4096 sequences, prompts among them, or 2^20 pages: refused before the cache changes."""
    model, ids = _model(), _tokens(prompts, 10, 7)
    cache = hf.PagedCache(capacity=capacity, page=16)
    got = _columns(model, "paged", cache, ids, None, [8])
    pool, state = cache.layers[0].k_pages.shape[0], cache.layers[0].state
    with pytest.raises(RuntimeError, match="4096 sequences, prompts among them, and 2\\^20 pages"):
        cache.batch_repeat_interleave(repeats)
    assert state.copies == 1 and state.parents is None
    assert all(layer.copies == 1 and layer.k_pages.shape[0] == pool == state.table.pages for layer in cache.layers)
    got = torch.cat((got, _columns(model, "paged", cache, ids, None, [2], 8)), 1)      # it goes on as it was
    want = _columns(model, "sdpa", _dense(model), ids, None, [10])
    assert (got - want).abs().max() <= 1e-4 * want.abs().max()
    assert state.more_pages(repeats) > 0


def test_as_many_as_a_step_takes(plain):  # noqa: F811
    model, ids = _model(), _tokens(1, 9, 8)
    cache = hf.PagedCache(capacity=16, page=16)
    _columns(model, "paged", cache, ids, None, [8])
    cache.batch_repeat_interleave(4095)
    assert cache.layers[0].state.table.lens.numel() == 4096


@pytest.mark.parametrize("prompts,copies", [(1, 3), (3, 2)])
def test_prompts_have_no_rows_in_a_step(plain, monkeypatch, prompts, copies):  # noqa: F811
    """A step asks for the rows of the model's batch alone, so that 2^20 of them fit."""
    model, ids = _model(), _tokens(prompts, 20, 9)
    cache = hf.PagedCache(capacity=48, page=16)
    _columns(model, "paged", cache, ids, None, [8])
    cache.batch_repeat_interleave(copies)
    asked, made = [], []
    step, share = paged.PageTable.step, paged.share_rows
    monkeypatch.setattr(paged.PageTable, "step", lambda t, new, rows, **kw: asked.append((new.numel(), rows)) or step(t, new, rows, **kw))
    monkeypatch.setattr(paged, "share_rows", lambda parents, cu, kv, lens, rows: made.append((cu.tolist(), kv.tolist(), lens.tolist(), rows))
                        or share(parents, cu, kv, lens, rows))
    batch = prompts * copies
    _columns(model, "paged", cache, ids.repeat_interleave(copies, 0), None, [5, 1], 8)
    assert asked == [(batch, 5 * batch), (batch, batch)]
    for (cu, kv, lens, rows), n, own in zip(made, (5, 1), (5, 6)):
        assert cu == [n * b for b in range(batch + 1)] + [n * batch] * prompts and rows == n * batch
        assert kv == lens == [own] * batch + [8] * prompts

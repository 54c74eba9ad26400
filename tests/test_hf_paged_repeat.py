"""PagedCache.batch_repeat_interleave on the CPU: what it refuses, and what a
step after it asks of the page table.  Plain forms and bounds as in the
adapter's other CPU tests."""

import pytest
import torch

from kv_cache_amd import hf
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

"""Generation from a repeated prompt on the GPU: the logits of every generated
token against a dense forward pass over the same tokens, within the bf16
tolerance of the paged cache's other model tests."""

import pytest
import torch

from kv_cache_amd import hf
from test_gpu_hf_paged import _dense, _model, _run, _tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("copies,quantize", [(4, None), (3, "fp8")])
def test_generated_logits_match_a_dense_pass(copies, quantize):
    hf.register_paged()
    model = _model()
    ids = _tokens(2, 50, 51)
    cache = hf.PagedCache(capacity=80, page=16, quantize=quantize)
    first = _run(model, "paged", cache, [ids[:, :-1]], [None])[0]
    cache.batch_repeat_interleave(copies)
    rows = ids.repeat_interleave(copies, 0)
    torch.manual_seed(0)
    with torch.no_grad():
        got = model.generate(rows, past_key_values=cache, max_new_tokens=9, do_sample=True, return_dict_in_generate=True,
                             output_logits=True)
    assert got.sequences.shape == (2 * copies, 59) and (got.sequences[:, :50] == rows).all()
    assert len({tuple(s) for s in got.sequences.tolist()}) == 2 * copies        # sampled: all different
    logits = torch.stack(got.logits, 1)                                        # of tokens 50 .. 58
    # over codes: a cache of them without a repeat
    other = _dense(model) if quantize is None else hf.PagedCache(capacity=80, page=16, quantize=quantize)
    want = _run(model, "sdpa" if quantize is None else "paged", other, [got.sequences[:, :-1]], [None])[0]
    torch.testing.assert_close(logits.float(), want[:, 49:].float(), rtol=3e-2, atol=3e-2)
    torch.testing.assert_close(first.repeat_interleave(copies, 0).float(), want[:, :49].float(), rtol=3e-2, atol=3e-2)

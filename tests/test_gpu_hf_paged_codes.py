"""The paged cache inside a transformers model on the GPU: pages of codes
against 16-bit pages of the values that the codes stand for, and sequences
that continue one prompt against dense SDPA of the repeated batch.  Logits
agree within the bf16 tolerance of the paged cache's other model tests (two
attention implementations, each rounded to bf16 in every layer)."""

import pytest
import torch

from kv_cache_amd import hf, paged
from test_gpu_hf_paged import _dense, _model, _run, _tokens

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _through_codes(x, kind):
    """K or V rows as their codes stand for."""
    rows, heads, dim = x.shape
    pages = -(-rows // 16)
    (k, ks), (v, vs) = (paged.quantized_pages(pages, heads, 16, dim, kind, DEV) for _ in range(2))
    sc = dict(k_scales=ks, v_scales=vs)
    table = torch.arange(pages, dtype=torch.int32, device=DEV)[None]
    i32 = lambda *n: torch.tensor(n, dtype=torch.int32, device=DEV)  # noqa: E731
    plain_append(x, x, k, v, torch.arange(rows, device=DEV), **sc)
    return paged.read(k, v, table, i32(0, rows), i32(rows), rows, dtype=x.dtype, **sc)[0]


plain_append = paged.append


@pytest.mark.parametrize("kind,head_dim,heads,dtype", [("fp8", 128, 4, torch.bfloat16), ("fp4", 128, 8, torch.bfloat16),
                                                       ("fp8", 64, 2, torch.float16)])
def test_codes_match_the_values_they_stand_for(monkeypatch, kind, head_dim, heads, dtype):
    hf.register_paged()
    model = _model(head_dim=head_dim, heads=heads, dtype=dtype)
    chunks = [_tokens(2, n, 10 + i) for i, n in enumerate((130, 57, 1, 1, 5, 1))]
    mask = torch.ones((2, 195), dtype=torch.long, device=DEV)
    mask[1, :20] = 0
    masks, at = [], 0
    for c in chunks:
        at += c.shape[1]
        masks.append(mask[:, :at])
    cache = hf.PagedCache(capacity=256, page=16, quantize=kind)
    got = _run(model, "paged", cache, chunks, masks)
    assert cache.layers[0].k_pages.dtype == (torch.float8_e4m3fn if kind == "fp8" else torch.uint8)
    monkeypatch.setattr(paged, "append", lambda k, v, kp, vp, slots: plain_append(_through_codes(k, kind), _through_codes(v, kind),
                                                                                  kp, vp, slots))
    want = _run(model, "paged", hf.PagedCache(capacity=256, page=16), chunks, masks)
    at = 0
    for g, w in zip(got, want):
        real = mask[:, at: at + g.shape[1]].bool()
        torch.testing.assert_close(g[real], w[real], rtol=3e-2, atol=3e-2)
        at += g.shape[1]
    monkeypatch.undo()
    cache.reset()
    again = _run(model, "paged", cache, chunks[:1], [None])      # another batch in the same cache
    assert torch.isfinite(again[0]).all()


@pytest.mark.parametrize("quantize", [None, "fp8"])
def test_continuations_of_prompts(quantize):
    hf.register_paged()
    model, copies = _model(), 6
    prompt = _tokens(2, 100, 1)
    mask = torch.ones((2, 100), dtype=torch.long, device=DEV)
    mask[1, :33] = 0
    rest = [_tokens(2 * copies, n, 20 + n) for n in (1, 7, 2)]
    cache = hf.PagedCache(capacity=160, page=16, quantize=quantize)
    first = _run(model, "paged", cache, [prompt], [mask])[0]
    cache.batch_repeat_interleave(copies)
    wide, masks = mask.repeat_interleave(copies, 0), []
    for c in rest:
        wide = torch.cat((wide, torch.ones_like(c)), 1)
        masks.append(wide)
    got = _run(model, "paged", cache, rest, masks)
    if quantize is None:
        want = _run(model, "sdpa", _dense(model), [prompt.repeat_interleave(copies, 0), *rest], [masks[0][:, :100], *masks])
    else:   # the same codes without sharing
        alone = hf.PagedCache(capacity=160, page=16, quantize=quantize)
        want = _run(model, "paged", alone, [prompt.repeat_interleave(copies, 0), *rest], [masks[0][:, :100], *masks])
    torch.testing.assert_close(first.repeat_interleave(copies, 0)[masks[0][:, :100].bool()], want[0][masks[0][:, :100].bool()],
                               rtol=3e-2, atol=3e-2)
    for g, w in zip(got, want[1:]):
        torch.testing.assert_close(g, w, rtol=3e-2, atol=3e-2)
    state = cache.layers[0].state
    assert state.table.lens.tolist() == [10] * 12 + [100, 67]


def test_generate_from_a_repeated_prompt():
    hf.register_paged()
    model, copies = _model(), 4
    model.config._attn_implementation = "paged"
    ids = _tokens(1, 50, 50)
    with torch.no_grad():
        cache = hf.PagedCache(capacity=80, page=16)
        model(ids[:, :-1], past_key_values=cache, use_cache=True)
        cache.batch_repeat_interleave(copies)
        a = model.generate(ids.repeat_interleave(copies, 0), past_key_values=cache, max_new_tokens=8, do_sample=False)
    assert a.shape == (copies, 58) and (a == a[:1]).all()       # greedy: all the same

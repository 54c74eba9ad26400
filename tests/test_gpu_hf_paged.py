"""The paged cache inside a transformers Qwen3 model (random init): prompts,
chunks and decode steps against dense SDPA on a DynamicCache, left-padded
batches included.  Logits agree within the bf16 tolerance of the int4 tests
(two attention implementations, each rounded to bf16 in every layer)."""

import pytest
import torch

from kv_cache_amd import hf

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _model(layers=2, head_dim=128, heads=4, dtype=torch.bfloat16):
    from transformers import Qwen3Config, Qwen3ForCausalLM

    torch.manual_seed(0)
    cfg = Qwen3Config(vocab_size=512, hidden_size=256, intermediate_size=512, num_hidden_layers=layers,
                      num_attention_heads=heads, num_key_value_heads=2, head_dim=head_dim, max_position_embeddings=4096,
                      rope_theta=1.0e6)
    return Qwen3ForCausalLM(cfg).to(DEV, dtype).eval()


def _tokens(b, n, seed):
    return torch.randint(1, 512, (b, n), generator=torch.Generator().manual_seed(seed)).to(DEV)


def _run(model, impl, cache, chunks, masks):
    """Logits of every chunk of tokens, fed one after the other."""
    model.config._attn_implementation = impl
    out = []
    with torch.no_grad():
        for ids, mask in zip(chunks, masks):
            kw = {}
            if mask is not None:
                kw = dict(attention_mask=mask, position_ids=(mask.long().cumsum(-1) - 1).clamp(min=0)[:, -ids.size(1):])
            out.append(model(ids, past_key_values=cache, use_cache=True, **kw).logits.float())
    return out


def _dense(model):
    from transformers.cache_utils import DynamicCache

    return DynamicCache(config=model.config)


@pytest.mark.parametrize("head_dim,heads,page,dtype", [(128, 4, 64, torch.bfloat16), (64, 2, 16, torch.float16),
                                                      (128, 8, 128, torch.bfloat16)])
def test_prompt_chunks_and_steps_match_dense(head_dim, heads, page, dtype):
    hf.register_paged()
    model = _model(head_dim=head_dim, heads=heads, dtype=dtype)
    chunks = [_tokens(2, n, 10 + i) for i, n in enumerate((130, 57, 1, 1, 5, 1))]
    cache = hf.PagedCache(capacity=256, page=page)
    got = _run(model, "paged", cache, chunks, [None] * 6)
    want = _run(model, "sdpa", _dense(model), chunks, [None] * 6)
    for g, w in zip(got, want):
        torch.testing.assert_close(g, w, rtol=3e-2, atol=3e-2)
    assert cache.get_seq_length() == 195
    state = cache.layers[0].state
    assert state.table.lens.tolist() == [195, 195]
    assert all(layer.state is state for layer in cache.layers)


def test_left_padded_batch_matches_each_alone():
    hf.register_paged()
    model = _model()
    lens, n = [40, 7, 25], 40
    alone = [_tokens(1, k + 3, 30 + k) for k in lens]
    ids = torch.zeros((3, n), dtype=torch.long, device=DEV)
    mask = torch.zeros((3, n + 3), dtype=torch.long, device=DEV)
    for b, k in enumerate(lens):
        ids[b, n - k:], mask[b, n - k:] = alone[b][0, :k], 1
    chunks = [ids] + [torch.stack([alone[b][0, k + i] for b, k in enumerate(lens)])[:, None] for i in range(3)]
    cache = hf.PagedCache(capacity=64, page=16)
    got = _run(model, "paged", cache, chunks, [mask[:, : n + i] for i in range(4)])
    state = cache.layers[0].state
    assert state.table.lens.tolist() == [k + 3 for k in lens]
    # padding takes no page: 3 + 1 + 2 of 16 tokens
    assert int(state.table.count) == 12 - sum(-(-(k + 3) // 16) for k in lens)
    for b, k in enumerate(lens):
        want = _run(model, "sdpa", _dense(model), [alone[b]], [None])[0][0]
        torch.testing.assert_close(got[0][b, n - k:], want[:k], rtol=3e-2, atol=3e-2)
        for i in range(3):
            torch.testing.assert_close(got[1 + i][b, 0], want[k + i], rtol=3e-2, atol=3e-2)


def test_generate_and_reset():
    hf.register_paged()
    model = _model()
    model.config._attn_implementation = "paged"
    ids = _tokens(2, 50, 50)
    mask = torch.ones_like(ids)
    mask[1, :20] = 0
    cache = hf.PagedCache(capacity=80, page=16)
    with torch.no_grad():
        a = model.generate(ids, attention_mask=mask, past_key_values=cache, max_new_tokens=8, do_sample=False)
        assert a.shape == (2, 58)
        cache.reset()
        assert cache.get_seq_length() == 0
        table = cache.layers[0].state.table
        assert int(table.count) == table.pages and table.lens.tolist() == [0, 0]
        b = model.generate(ids, attention_mask=mask, past_key_values=cache, max_new_tokens=8, do_sample=False)
    assert torch.equal(a, b)


def test_refusals():
    hf.register_paged()
    model = _model(layers=1)
    with pytest.raises(RuntimeError, match="power of two"):
        hf.PagedCache(capacity=64, page=20)
    cache = hf.PagedCache(capacity=16, page=16)
    with pytest.raises(RuntimeError, match="capacity 16 exceeded"):
        _run(model, "paged", cache, [_tokens(1, 17, 1)], [None])
    # padding behind the tokens
    ids, mask = _tokens(2, 12, 2), torch.ones((2, 12), dtype=torch.long, device=DEV)
    mask[1, 8:] = 0
    with pytest.raises(RuntimeError, match="left-padded"):
        _run(model, "paged", hf.PagedCache(capacity=64, page=16), [ids], [mask])


def test_without_a_paged_cache_it_is_dense():
    hf.register_paged()
    model = _model(layers=1)
    ids = _tokens(2, 33, 3)
    got = _run(model, "paged", _dense(model), [ids], [None])
    want = _run(model, "sdpa", _dense(model), [ids], [None])
    assert torch.equal(got[0], want[0])


@pytest.mark.parametrize("widths", [[1] * 8, [3, 1, 4], [8]])
def test_padding_at_any_width(widths):
    # prompts fed a column or a few at a time: the padding of a sequence takes no slot
    hf.register_paged()
    model, lens, n = _model(), [8, 3], 8
    ids, mask = _tokens(2, n + 2, 60), torch.ones((2, n + 2), dtype=torch.long, device=DEV)
    mask[1, : n - 3] = 0
    chunks, masks, at = [], [], 0
    for w in widths + [1, 1]:
        chunks.append(ids[:, at: at + w])
        at += w
        masks.append(mask[:, :at])
    cache = hf.PagedCache(capacity=32, page=16)
    got = torch.cat(_run(model, "paged", cache, chunks, masks), 1)
    assert cache.layers[0].state.table.lens.tolist() == [k + 2 for k in lens]
    want = torch.cat(_run(model, "sdpa", _dense(model), chunks, masks), 1)
    torch.testing.assert_close(got[mask.bool()], want[mask.bool()], rtol=3e-2, atol=3e-2)


def _exact(q, k, v, seen, scaling, cap):
    """[B, n, Hq, D] in 64 bits, and the weighted sum of |v|."""
    g = q.shape[1] // k.shape[1]
    q, k, v = q.double(), k.double().repeat_interleave(g, 1), v.double().repeat_interleave(g, 1)
    s = torch.matmul(q, k.transpose(2, 3).contiguous()) * scaling
    if cap:
        s = cap * torch.tanh(s / cap)
    w = torch.softmax(s.masked_fill(~seen, -torch.inf), -1).nan_to_num(0.0)
    return torch.matmul(w, v).transpose(1, 2), torch.matmul(w, v.abs()).transpose(1, 2)


@pytest.mark.parametrize("heads,dim,dt", [((8, 2), 128, torch.bfloat16), ((2, 2), 64, torch.float16)])
@pytest.mark.parametrize("window,cap,scaling", [(1, 0.0, None), (5, 20.0, 0.3), (64, 0.0, 0.05), (300, 2.0, None)])
def test_windows_caps_and_scaling(heads, dim, dt, window, cap, scaling):
    """Left-padded chunks shorter and longer than the window and single steps, straight through the interface.
    The bound counts the weight's and the output's rounding, half a step each of 2^-8 (2^-11 in fp16), and
    2^-10 of the weights for scores off by 2^-12 and sums in 32 bits."""
    gen = torch.Generator(device=DEV).manual_seed(70)
    hq, hkv = heads
    lens, first = [90, 33, 1], 90
    cache, ks, vs = hf.PagedCache(capacity=256, page=16), [], []
    real = torch.ones((3, 0), dtype=torch.bool, device=DEV)
    for n in (first, 1, 70, 1, 3):
        new = lambda h: torch.randn((3, n, h, dim), generator=gen, device=DEV).to(dt).transpose(1, 2)  # noqa: E731
        q, k, v = new(hq), new(hkv), new(hkv)
        fresh = torch.ones((3, n), dtype=torch.bool, device=DEV)
        if n == first:
            for b, m in enumerate(lens):
                fresh[b, : n - m] = False
        real = torch.cat([real, fresh], 1)
        total = real.shape[1]
        own, at = torch.arange(total - n, total, device=DEV)[:, None], torch.arange(total, device=DEV)
        seen = (real[:, None] & (at <= own) & (at > own - window))[:, None]
        ks.append(k), vs.append(v)
        key, value = cache.update(k, v, 0)
        got, _ = hf.paged_attention_forward(None, q, key, value, seen, scaling=scaling, softcap=cap or None,
                                            sliding_window=window)
        want, av = _exact(q, torch.cat(ks, 2), torch.cat(vs, 2), seen, dim ** -0.5 if scaling is None else scaling, cap)
        h = torch.finfo(dt).eps / 2
        tol = h * 1.02 * (av + want.abs()) + 2.0 ** -10 * av + 2.0 ** -24
        assert got.shape == (3, n, hq, dim)
        assert ((got.double() - want).abs() <= tol)[fresh].all()


def test_other_masks_are_refused_and_the_cache_goes_on():
    hf.register_paged()
    model = _model(layers=2)
    ids = _tokens(2, 12, 80)
    tri = torch.ones((12, 12), dtype=torch.bool, device=DEV).tril()
    blocks = tri & (torch.arange(12, device=DEV)[:, None] // 6 == torch.arange(12, device=DEV) // 6)
    cache = hf.PagedCache(capacity=32, page=16)
    for wrong in (tri | True, blocks, tri | (torch.arange(12, device=DEV) < 4)):
        with pytest.raises(RuntimeError, match="mask"):
            _run_4d(model, cache, ids, wrong[None, None].expand(2, 1, 12, 12))
        assert cache.get_seq_length() == 0
    got = _run_4d(model, cache, ids, tri[None, None].expand(2, 1, 12, 12))
    want = _run(model, "sdpa", _dense(model), [ids], [None])[0]
    torch.testing.assert_close(got, want, rtol=3e-2, atol=3e-2)


def _run_4d(model, cache, ids, mask):
    model.config._attn_implementation = "paged"
    with torch.no_grad():
        return model(ids, past_key_values=cache, use_cache=True, attention_mask=mask).logits.float()


def test_another_implementation_raises():
    model = _model(layers=1)
    with pytest.raises(RuntimeError, match="register_paged"):
        _run(model, "sdpa", hf.PagedCache(capacity=32, page=16), [_tokens(2, 12, 90), _tokens(2, 1, 91)], [None, None])


def test_a_reset_cache_takes_another_batch():
    hf.register_paged()
    model, cache = _model(layers=2), hf.PagedCache(capacity=64, page=16)
    for batch in (3, 1, 2):
        ids = _tokens(batch, 20, 100 + batch)
        got = _run(model, "paged", cache, [ids, ids[:, :1]], [None, None])
        want = _run(model, "sdpa", _dense(model), [ids, ids[:, :1]], [None, None])
        for a, b in zip(got, want):
            torch.testing.assert_close(a, b, rtol=3e-2, atol=3e-2)
        cache.reset()


def test_a_backward_pass_raises():
    hf.register_paged()
    model = _model(layers=1)
    model.config._attn_implementation = "paged"
    logits = model(_tokens(1, 9, 110), past_key_values=hf.PagedCache(capacity=32, page=16), use_cache=True).logits
    with pytest.raises(RuntimeError, match="no backward"):
        logits.float().sum().backward()


def test_steps_under_inference_mode_and_outside():
    hf.register_paged()
    model = _model(layers=1)
    model.config._attn_implementation = "paged"
    ids, mask = _tokens(2, 12, 120), torch.ones((2, 12), dtype=torch.long, device=DEV)
    mask[1, :4] = 0
    caches, out = (hf.PagedCache(capacity=32, page=16), hf.PagedCache(capacity=32, page=16)), ([], [])
    for i, (a, e) in enumerate(((0, 9), (9, 10), (10, 12))):
        for c, inside, got in zip(caches, (i % 2 == 0, False), out):
            with torch.inference_mode() if inside else torch.no_grad():
                got.append(model(ids[:, a:e], attention_mask=mask[:, :e], past_key_values=c, use_cache=True).logits.clone())
    for x, y in zip(*out):
        assert torch.equal(x, y)
    assert caches[0].layers[0].state.table.lens.tolist() == [12, 8]

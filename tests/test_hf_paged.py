"""The paged cache inside transformers models on the CPU: the adapter alone, over plain forms of the page
table, the writes and the attention, in 32 bits against dense SDPA on a DynamicCache.  Both round every
sum of at most a few hundred terms to 24 bits, through two layers: 2^-24 of the largest logit for each
of about a thousand roundings in a row, 1e-4 of it."""

import pytest
import torch

from kv_cache_amd import hf, paged


def _plain_step(t, new_lens, rows, *, padded=0, out=None):
    page, count = t.page, int(t.count)
    plan = paged.StepPlan.empty(t.lens.numel(), rows, t.lens.device)
    plan.slots.fill_(-1), plan.positions.fill_(-1), plan.failed.zero_()
    end = 0
    for b, n in enumerate(new_lens.tolist()):
        have = int(t.lens[b])
        assert 0 <= n <= padded and have + n <= t.table.shape[1] * page
        plan.cu_rows[b] = end
        end += padded
        for i in range(n):
            p = have + i
            if p % page == 0:
                count -= 1
                t.table[b, p // page] = t.free[count]
            plan.positions[end - n + i] = p
            plan.slots[end - n + i] = int(t.table[b, p // page]) * page + p % page
        t.lens[b] = plan.kv_lens[b] = have + n
    plan.cu_rows[-1] = end
    t.count.fill_(count)
    return plan


def _plain_release(t, keep):
    assert (keep == 0).all()
    t.table.fill_(-1)
    t.lens.zero_()
    t.free.copy_(torch.arange(t.pages - 1, -1, -1))
    t.count.fill_(t.pages)


def _plain_append(k, v, k_pages, v_pages, slots):
    page = k_pages.shape[2]
    at = slots[slots >= 0]
    k_pages[at // page, :, at % page] = k[slots >= 0]
    v_pages[at // page, :, at % page] = v[slots >= 0]


def _plain_attention(q, k_pages, v_pages, table, cu, kv, scaling, *, max_rows=None, softcap=0.0, slopes=None,
                     prefix_lens=None, first_keys=None, out=None, workspace=None):
    page, group = k_pages.shape[2], q.shape[1] // k_pages.shape[1]
    out = torch.zeros(q.shape, dtype=q.dtype)
    for b, n in enumerate(kv.tolist()):
        a, e = int(cu[b]), int(cu[b + 1])
        for i in range(a, e):
            p = n - (e - a) + i - a
            lo = 0 if first_keys is None else max(0, int(first_keys[i]))
            if p < lo:
                continue
            ids, j = table[b, : p // page + 1].long(), torch.arange(lo, p + 1)
            k, v = (x[ids].transpose(1, 2).flatten(0, 1)[j].repeat_interleave(group, 1) for x in (k_pages, v_pages))
            s = (q[i] * k).sum(-1) * scaling
            if softcap:
                s = softcap * torch.tanh(s / softcap)
            out[i] = (torch.softmax(s, 0)[..., None] * v).sum(0)
    return out


@pytest.fixture
def taken(monkeypatch):
    """The plain forms in place; the new lengths of every step made."""
    steps = []

    def step(t, new_lens, rows, **kw):
        steps.append(new_lens.tolist())
        return _plain_step(t, new_lens, rows, **kw)

    monkeypatch.setattr(paged.PageTable, "step", step)
    monkeypatch.setattr(paged.PageTable, "release", _plain_release)
    monkeypatch.setattr(paged, "append", _plain_append)
    monkeypatch.setattr(paged, "attention", _plain_attention)
    hf.register_paged()
    return steps


def _model(layers=2, **extra):
    from transformers import Qwen3Config, Qwen3ForCausalLM

    torch.manual_seed(0)
    # weights large enough that what a token attends to shows in its logits
    return Qwen3ForCausalLM(Qwen3Config(vocab_size=64, hidden_size=64, intermediate_size=64, num_hidden_layers=layers,
                                        num_attention_heads=4, num_key_value_heads=2, head_dim=16,
                                        initializer_range=0.3, **extra)).eval()


def _tokens(b, n, seed):
    return torch.randint(1, 64, (b, n), generator=torch.Generator().manual_seed(seed))


def _left_padded(lens, n):
    mask = torch.zeros((len(lens), n), dtype=torch.long)
    for b, k in enumerate(lens):
        mask[b, n - k:] = 1
    return mask


def _run(model, impl, cache, ids, mask, widths, **kw):
    """Logits of all columns, fed ``widths`` at a time."""
    model.config._attn_implementation = impl
    out, at = [], 0
    with torch.no_grad():
        for n in widths:
            extra = dict(kw) if mask is None else dict(attention_mask=mask[:, : at + n], **kw)
            out.append(model(ids[:, at: at + n], past_key_values=cache, use_cache=True, **extra).logits)
            at += n
    return torch.cat(out, 1)


def _dense(model):
    from transformers.cache_utils import DynamicCache

    return DynamicCache(config=model.config)


def _near(got, want, real):
    assert ((got - want).abs().amax(-1)[real] <= 1e-4 * want.abs().max()).all()


@pytest.mark.parametrize("widths", [[1] * 6, [2, 1, 1, 2], [6], [1, 5]])
def test_padding_takes_no_slot_at_any_width(taken, widths):
    # one column at a time: the padding of a sequence is not its tokens
    model, lens = _model(), [6, 3]
    ids, mask = _tokens(2, 9, 1), torch.cat([_left_padded(lens, 6), torch.ones((2, 3), dtype=torch.long)], 1)
    cache = hf.PagedCache(capacity=32, page=16)
    got = _run(model, "paged", cache, ids, mask, widths + [1, 2])
    at, want = 0, []
    for n in widths + [1, 2]:
        want.append(mask[:, at: at + n].sum(1).tolist())
        at += n
    assert taken == want
    assert cache.layers[0].state.table.lens.tolist() == [9, 6]
    _near(got, _run(model, "sdpa", _dense(model), ids, mask, widths + [1, 2]), mask.bool())


def test_a_sequence_without_a_token_in_a_single_step(taken):
    model = _model()
    ids, mask = _tokens(2, 6, 2), torch.ones((2, 6), dtype=torch.long)
    mask[1, 4] = 0
    got = _run(model, "paged", hf.PagedCache(capacity=16, page=16), ids, mask, [4, 1, 1])
    assert taken == [[4, 4], [1, 0], [1, 1]]
    _near(got, _run(model, "sdpa", _dense(model), ids, mask, [4, 1, 1]), mask.bool())


# -- masks that are not what the pages show ----------------------------------------


def _causal(lens, n, total=None, window=None):
    """bool [B, 1, n, total]: the mask of left-padded sequences, for the last n of total columns."""
    total = n if total is None else total
    own, j = torch.arange(total - n, total)[:, None], torch.arange(total)
    m = j <= own
    if window is not None:
        m &= j > own - window
    return torch.stack([m & (j >= total - k) for k in lens])[:, None]


def _as_float(m, low):
    return torch.where(m, 0.0, low)


FOREIGN = ["two_sided", "prefix", "documents", "hidden_history", "one_head", "one_row", "soft", "a_later_column",
           "integers", "two_axes", "too_narrow"]


@pytest.mark.parametrize("form", FOREIGN)
def test_masks_of_other_forms_are_refused(taken, form):
    model, ids = _model(), _tokens(2, 6, 3)
    m = _causal([6, 4], 6)
    if form == "two_sided":
        m = m | (torch.arange(6) >= 2)
    elif form == "prefix":
        m[:, :, :3, 2:3] = True
    elif form == "documents":
        m[:, :, 3:, :3] = False
    elif form == "hidden_history":
        m[1, 0, 5, 3] = False
    elif form == "one_head":
        m = m.expand(2, 4, 6, 6).clone()
        m[0, 2, 4, 1] = False
    elif form == "one_row":
        m = m[:, :, -1:]
    elif form == "soft":
        m = _as_float(m, -1.0)
    elif form == "a_later_column":
        m[0, 0, 2, 3] = True
    elif form == "integers":
        m = m.long()
    elif form == "two_axes":
        m = m[0, 0]
    elif form == "too_narrow":
        m = m[..., :5]
    cache = hf.PagedCache(capacity=16, page=16)
    model.config._attn_implementation = "paged"
    q, k = torch.randn(2, 4, 6, 16), torch.randn(2, 2, 6, 16)
    key, value = cache.update(k, k, 0)
    with pytest.raises(RuntimeError, match="mask"):
        hf.paged_attention_forward(model.model.layers[0].self_attn, q, key, value, m)
    assert taken == []


def _attend(cache, m, n, layer=0, window=None, seed=0, **kw):
    g = torch.Generator().manual_seed(seed)
    q, k = torch.randn((2, 4, n, 16), generator=g), torch.randn((2, 2, n, 16), generator=g)
    key, value = cache.update(k, k, layer)
    return hf.paged_attention_forward(None, q, key, value, m, sliding_window=window, **kw)[0]


@pytest.mark.parametrize("low", [None, -1.0e4, -1.0e9, torch.finfo(torch.float32).min, -torch.inf])
def test_causal_masks_with_left_padding_are_taken(taken, low):
    form = (lambda m: m) if low is None else (lambda m: _as_float(m, low))
    a, b = hf.PagedCache(capacity=32, page=16), hf.PagedCache(capacity=32, page=16)
    for i, (n, total) in enumerate(((6, 6), (1, 7), (3, 10))):
        m = _causal([total, total - 2], n, total)
        if n > 1 and total == n:
            m[1, 0, :2] = True       # what rows of padding see does not matter, beyond their own column
            m[1, 0, 0, 0] = m[1, 0, 1, 1] = False
        got = _attend(a, form(m), n, seed=i)
        assert torch.equal(got, _attend(b, form(m.expand(2, 4, n, total)), n, seed=i))
    assert taken[0::2] == taken[1::2] == [[6, 4], [1, 1], [3, 3]]


def test_one_column_that_hides_history_is_refused(taken):
    cache = hf.PagedCache(capacity=32, page=16)
    _attend(cache, _causal([5, 3], 5), 5)
    m = _causal([6, 4], 1, 6)
    m[0, 0, 0, 2] = False
    with pytest.raises(RuntimeError, match="mask"):
        _attend(cache, m, 1)
    cache = hf.PagedCache(capacity=32, page=16)
    _attend(cache, None, 5)
    with pytest.raises(RuntimeError, match="mask"):
        _attend(cache, m, 1)


def test_every_layers_mask_is_looked_at(taken):
    cache = hf.PagedCache(capacity=32, page=16)
    m = _causal([5, 3], 5)
    _attend(cache, m, 5, layer=0)
    chunks = m & ((torch.arange(5)[:, None] // 2) == (torch.arange(5) // 2))
    with pytest.raises(RuntimeError, match="mask"):
        _attend(cache, chunks, 5, layer=1)
    # a layer with a window, and one whose mask has another
    cache = hf.PagedCache(capacity=32, page=16)
    _attend(cache, m, 5, layer=0)
    _attend(cache, _causal([5, 3], 5, window=2), 5, layer=1, window=2)
    with pytest.raises(RuntimeError, match="mask"):
        _attend(cache, _causal([5, 3], 5, window=3), 5, layer=2, window=2)


@pytest.mark.parametrize("kinds", [["full_attention", "sliding_attention"], ["sliding_attention", "full_attention"]])
@pytest.mark.parametrize("window", [3, 7])
def test_windows_match_dense(taken, window, kinds):
    # chunks longer than the window too, in left-padded batches and without a mask
    extra = dict(use_sliding_window=True, sliding_window=window, layer_types=kinds)
    model, widths = _model(**extra), [5, 1, 4, 1]
    ids, mask = _tokens(2, 11, 4), torch.cat([_left_padded([5, 3], 5), torch.ones((2, 6), dtype=torch.long)], 1)
    for m in (mask, None):
        got = _run(model, "paged", hf.PagedCache(capacity=32, page=16), ids, m, widths)
        # a dense cache without the sliding layers' own, which keeps fewer columns
        from transformers.cache_utils import DynamicCache
        want = _run(model, "sdpa", DynamicCache(), ids, m, widths)
        _near(got, want, torch.ones((2, 11), dtype=torch.bool) if m is None else m.bool())


def test_a_window_over_padding_between_tokens_is_refused(taken):
    # the window counts columns in the mask, tokens in the pages
    cache = hf.PagedCache(capacity=32, page=16)
    _attend(cache, _causal([4, 4], 4, window=3), 4, window=3)
    m = _causal([7, 7], 3, 7, window=3)
    m[1, 0, :, 4:6] = False
    with pytest.raises(RuntimeError, match="mask"):
        _attend(cache, m, 3, window=3)
    cache = hf.PagedCache(capacity=32, page=16)
    _attend(cache, _causal([4, 4], 4), 4)
    m = _causal([7, 7], 3, 7)
    m[1, 0, :, 4:6] = False
    _attend(cache, m, 3)
    assert taken[-1] == [3, 1]


# -- arguments of the attention interface ---------------------------------------------


@pytest.mark.parametrize("name,value", [
    ("s_aux", torch.zeros(4)), ("position_bias", torch.zeros(1, 4, 6, 6)), ("head_mask", torch.ones(4)),
    ("cu_seq_lens_q", torch.tensor([0, 3, 6])), ("logit_cap", 30.0), ("is_causal", False)])
def test_arguments_that_change_scores_are_refused(taken, name, value):
    cache = hf.PagedCache(capacity=16, page=16)
    with pytest.raises(RuntimeError, match=name):
        _attend(cache, None, 6, **{name: value})
    assert taken == []


def test_arguments_that_change_nothing_are_taken(taken):
    cache = hf.PagedCache(capacity=16, page=16)
    got = _attend(cache, None, 6, position_ids=torch.arange(6)[None], cache_position=torch.arange(6), use_cache=True,
                  output_attentions=False, s_aux=None, is_causal=True, logits_to_keep=1)
    assert torch.equal(got, _attend(hf.PagedCache(capacity=16, page=16), None, 6))
    # a mask says itself what is causal, a single query is last
    _attend(cache, _causal([9, 9], 3, 9), 3, is_causal=False)
    _attend(cache, None, 1, is_causal=False)


def test_a_module_that_is_not_causal_is_refused(taken):
    class Module(torch.nn.Module):
        is_causal = False

    key, value = hf.PagedCache(capacity=16, page=16).update(*[torch.randn(2, 2, 6, 16)] * 2, 0)
    with pytest.raises(RuntimeError, match="is_causal"):
        hf.paged_attention_forward(Module(), torch.randn(2, 4, 6, 16), key, value, None)


def test_keys_of_another_sequence_are_refused(taken):
    # cross attention: queries and keys are not of the same tokens
    key, value = hf.PagedCache(capacity=16, page=16).update(*[torch.randn(2, 2, 6, 16)] * 2, 0)
    with pytest.raises(RuntimeError, match="same tokens"):
        hf.paged_attention_forward(None, torch.randn(2, 4, 3, 16), key, value, None)


def test_attention_sinks_of_a_model_are_refused(taken):
    from transformers import GptOssConfig, GptOssForCausalLM

    torch.manual_seed(0)
    model = GptOssForCausalLM(GptOssConfig(vocab_size=64, hidden_size=64, intermediate_size=64, num_hidden_layers=2,
                                           num_attention_heads=4, num_key_value_heads=2, head_dim=16, sliding_window=8,
                                           num_local_experts=2, num_experts_per_tok=1)).eval()
    with pytest.raises(RuntimeError, match="s_aux"):
        _run(model, "paged", hf.PagedCache(capacity=16, page=16), _tokens(2, 5, 5), None, [5])


# -- updates that the paged attention function did not take ------------------------------


@pytest.mark.parametrize("layers", [1, 2])
@pytest.mark.parametrize("impl", ["sdpa", "eager"])
def test_another_implementation_raises(taken, layers, impl):
    # it would see the step's own columns alone, and the pages would stay empty
    model, ids = _model(layers=layers), _tokens(2, 7, 6)
    with pytest.raises(RuntimeError, match="register_paged"):
        _run(model, impl, hf.PagedCache(capacity=16, page=16), ids, None, [6, 1])


def test_a_key_that_lost_its_layer_raises(taken):
    cache = hf.PagedCache(capacity=16, page=16)
    q, k = torch.randn(2, 4, 6, 16), torch.randn(2, 2, 6, 16)
    key, value = cache.update(k, k, 0)
    # dense over the new columns, as for any keys without a layer
    module = torch.nn.Module()
    module.num_key_value_groups = 2
    hf.paged_attention_forward(module, q, key * 1.0, value, None)
    with pytest.raises(RuntimeError, match="register_paged"):
        cache.update(k, k, 1)
    with pytest.raises(RuntimeError, match="register_paged"):
        cache.layers[0].get_mask_sizes(1)
    cache.reset()
    assert cache.layers[0].get_mask_sizes(6) == (6, 0)
    _attend(cache, None, 6)
    assert taken == [[6, 6]]


def test_a_refused_step_leaves_the_cache_as_it_was(taken):
    cache = hf.PagedCache(capacity=32, page=16)
    first = _attend(cache, _causal([5, 3], 5), 5, seed=1)
    wrong = _causal([8, 6], 3, 8)
    wrong[0, 0, 2, 4] = False
    for bad in (dict(m=wrong), dict(m=None, s_aux=torch.zeros(4))):
        with pytest.raises(RuntimeError):
            _attend(cache, n=3, **bad)
        assert cache.get_seq_length() == 5 and cache.layers[0].get_mask_sizes(3) == (8, 0)
    with pytest.raises(RuntimeError, match="exceeded"):
        _attend(cache, None, 28)
    got = _attend(cache, _causal([8, 6], 3, 8), 3, seed=2)
    other = hf.PagedCache(capacity=32, page=16)
    assert torch.equal(first, _attend(other, _causal([5, 3], 5), 5, seed=1))
    assert torch.equal(got, _attend(other, _causal([8, 6], 3, 8), 3, seed=2))
    assert taken == [[5, 3], [3, 3]] * 2


def test_a_refused_first_step_binds_the_cache_to_nothing(taken):
    # its batch, heads and dtype were never taken
    cache = hf.PagedCache(capacity=32, page=16)
    wrong = _causal([6, 6], 6) | True
    with pytest.raises(RuntimeError, match="mask"):
        _attend(cache, wrong, 6)
    k = torch.randn(3, 1, 4, 8, dtype=torch.float64)
    key, value = cache.update(k, k, 0)
    out, _ = hf.paged_attention_forward(None, torch.randn(3, 2, 4, 8, dtype=torch.float64), key, value, None)
    assert out.shape == (3, 4, 2, 8) and taken == [[4, 4, 4]]


def test_a_refused_first_step_of_another_batch(taken):
    cache = hf.PagedCache(capacity=32, page=16)
    with pytest.raises(RuntimeError, match="mask"):
        _attend(cache, _causal([6, 6], 6) | True, 6)
    k = torch.randn(3, 2, 4, 16)
    key, value = cache.update(k, k, 0)
    hf.paged_attention_forward(None, torch.randn(3, 4, 4, 16), key, value, _causal([4, 1, 3], 4))
    assert taken == [[4, 1, 3]]


def test_a_step_that_fails_in_a_later_layer_has_to_be_reset(taken):
    # the layers before hold the step's columns already
    cache = hf.PagedCache(capacity=32, page=16)
    m = _causal([5, 3], 5)
    _attend(cache, m, 5, layer=0)
    with pytest.raises(RuntimeError, match="mask"):
        _attend(cache, m | True, 5, layer=1)
    for layer in (0, 1):
        with pytest.raises(RuntimeError, match="reset"):
            _attend(cache, m, 5, layer=layer)
    cache.reset()
    _attend(cache, m, 5, layer=0)
    _attend(cache, m, 5, layer=1)
    assert taken == [[5, 3]] * 2


@pytest.mark.parametrize("n", [1, 5, 6])
def test_layers_that_step_apart_are_refused(taken, n):
    # one plan serves all layers of a step: a layer that left one out is behind
    cache = hf.PagedCache(capacity=32, page=16)
    _attend(cache, None, 5, layer=0)
    _attend(cache, None, 1, layer=0)
    with pytest.raises(RuntimeError, match="together"):
        _attend(cache, None, n, layer=1)
    assert taken == [[5, 5], [1, 1]]


# -- gradients ---------------------------------------------------------------------------


def test_a_backward_pass_raises(taken):
    # the pages hold no graph: gradients through them would be left out of those of the parameters
    model, ids = _model(), _tokens(2, 6, 7)
    model.config._attn_implementation = "paged"
    want = _run(model, "paged", hf.PagedCache(capacity=16, page=16), ids, None, [6])
    got = model(ids, past_key_values=hf.PagedCache(capacity=16, page=16), use_cache=True).logits
    assert torch.equal(got, want)
    with pytest.raises(RuntimeError, match="no backward"):
        got.sum().backward()


def test_steps_under_inference_mode_and_outside(monkeypatch):
    # what the state keeps between steps is not written in place
    monkeypatch.setattr(paged.PageTable, "step", lambda t, new, rows, padded: new.tolist())
    state, at = hf._PagedState(32, 16), 0
    steps = [(_causal([5, 3], 5), 5), (_causal([6, 4], 1, 6), 1), (None, 1), (_causal([9, 7], 2, 9), 2)]
    for i, (m, n) in enumerate(steps):
        at += n
        with torch.inference_mode(i % 2 == 0):
            got = state.step(at, n, 2, "cpu", m, None)
        assert got == ([5, 3] if i == 0 else [n, n])
    assert state.real.tolist() == [[True] * 9, [False] * 2 + [True] * 7]

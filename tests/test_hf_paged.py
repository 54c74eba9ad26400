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

"""Requests that continue another request's tokens: the plan against lists,
and the attention against 64 bits over each request's parent's tokens and its
own laid out as one request, within the bound of the paged attention."""

import random

import pytest
import torch

from kv_cache_amd import paged
from test_gpu_paged import DEV, DT, HEADS, _case, _i32, _reference, _within
from test_gpu_paged_codes import _coded

pytestmark = pytest.mark.gpu
KINDS = ["none", "fp8", "fp4"]


# -- the plan -----------------------------------------------------------------------


def _plan(parents, rows, kv, lens, total):
    """(positions, places by parent) of every row, from lists."""
    n, cu = len(parents), [0]
    for m in rows:
        cu.append(cu[-1] + m)
    positions, heirs = [-1] * total, [[] for _ in range(n)]
    for b in range(n):
        p = parents[b]
        real = 0 <= p < n and p != b and lens[p] > 0 and kv[b] > 0
        for i in range(rows[b]):
            own = kv[b] - rows[b] + i
            if own >= 0:
                positions[cu[b] + i] = own + (lens[p] if real else 0)
                if real:
                    heirs[p].append(cu[b] + i)
    return positions, heirs


@pytest.mark.parametrize("requests,most,total", [(1, 3, 4), (2, 1, 2), (33, 1, 40), (64, 5, 400), (65, 3, 300), (255, 1, 200),
                                                 (257, 2, 300), (400, 2, 900), (512, 1, 600), (512, 20, 9000), (513, 1, 600), (1000, 2, 2500),
                                                 (1025, 1, 1200), (4096, 1, 4096), (4095, 3, 13000), (7, 3000, 22000)])
def test_share_rows(requests, most, total):
    rng = random.Random(requests)
    few = [rng.randrange(requests) for _ in range(3)]
    parents = [rng.choice([-1, b, rng.randint(-9, requests + 9), *few, few[0]]) for b in range(requests)]
    rows = [rng.choice([0, 1, 1, rng.randint(0, most)]) for _ in range(requests)]
    while sum(rows) > total:
        rows[rng.randrange(requests)] = 0
    lens = [rng.choice([0, rng.randint(1, 5000)]) for _ in range(requests)]
    kv = [rng.choice([m, m, m + 7, max(0, m - 1), 0]) for m in rows]
    cu = [0]
    for m in rows:
        cu.append(cu[-1] + m)
    got = paged.share_rows(_i32(parents), _i32(cu), _i32(kv), _i32(lens), total)
    positions, heirs = _plan(parents, rows, kv, lens, total)
    assert got.positions.tolist() == positions
    words = got.buffer.tolist()
    rank, order = words[total: 2 * total], words[2 * total: 3 * total]
    start = words[3 * total: 3 * total + requests + 1]
    for a in range(requests):
        assert order[start[a]: start[a + 1]] == heirs[a]     # by request, then by row
    assert start[requests] == sum(map(len, heirs))
    place = {r: i for i, r in enumerate(order[: start[requests]])}
    assert rank == [place.get(r, -1 if r < cu[-1] else -2) for r in range(total)]
    again = paged.share_rows(_i32(parents), _i32(cu), _i32(kv), _i32(lens), total, out=got)
    assert again is got and got.buffer.tolist() == words


def test_rows_out_of_order_stay_in_bounds():
    # cu_rows that does not ascend: nothing is written outside the plan, and attention stays in bounds
    total, n = 30, 3
    plan = paged.SharedRows(n, total, DEV)
    words = plan.buffer.numel()
    room = torch.full((words + 200,), 77, dtype=torch.int32, device=DEV)
    plan.buffer, plan.positions = room[:words], room[:total]
    c = _case([50, 60, 70], [10, 10, 10], 8, 2, 128, 16, "bf16", seed=17)
    for cu in ([0, 30, 0, 30], [30, 0, 30, 0], [-5, 10, 20, 1000]):
        paged.share_rows(_i32([2, 0, 1]), _i32(cu), _i32([50, 60, 70]), _i32([50, 60, 70]), total, out=plan)
        assert (room[words:] == 77).all()
        out = paged.attention(**{**c, "cu_rows": _i32(cu)}, shared=plan)
        torch.cuda.synchronize()
    assert out.shape == (30, 8, 128)


# -- attention ----------------------------------------------------------------------


def _whole(c, parents, lens):
    """The case with every request's parent's tokens before its own: one 16-bit page table of pages of 16 tokens."""
    kv, cu = c["kv_lens"].tolist(), c["cu_rows"].tolist()
    page = c["k_pages"].shape[2]
    flat = [c[x].transpose(1, 2).flatten(0, 1) for x in ("k_pages", "v_pages")]

    def tokens(b, n):
        at = torch.arange(n, device=DEV)
        ids = c["table"][b].long()[at // page]
        ok = (ids >= 0) & (ids < c["k_pages"].shape[0])
        return ids.clamp(0, c["k_pages"].shape[0] - 1) * page + at % page, ok

    out, table, at, lengths, holes = [], [], 0, [], []
    width = max(-(-(k + max(lens)) // 16) for k in kv) + 1
    for b in range(len(kv)):
        p = parents[b]
        real = 0 <= p < len(kv) and p != b and lens[p] > 0 and kv[b] > 0
        got = ([tokens(p, lens[p])] if real else []) + [tokens(b, kv[b])]
        ids, ok = torch.cat([g[0] for g in got]), torch.cat([g[1] for g in got])
        n = ids.numel()
        pad = -n % 16
        lengths.append(n)
        out.append([torch.cat([f[ids], torch.zeros((pad, *f.shape[1:]), dtype=f.dtype, device=DEV)]) for f in flat])
        need = (n + pad) // 16
        table.append(list(range(at, at + need)) + [-1] * (width - need))
        at += need
        holes.append(ok)
    pages = [torch.cat([o[i] for o in out]).unflatten(0, (-1, 16)).transpose(1, 2).contiguous() for i in range(2)]
    rows_before = [lengths[b] - kv[b] for b in range(len(kv))]
    return dict(query=c["query"], k_pages=pages[0], v_pages=pages[1], table=_i32(table), cu_rows=_i32(cu),
                kv_lens=_i32(lengths), scaling=c["scaling"]), rows_before


def _check(parents, kv, rows, hq, hkv, dim, page, dt, kind="none", seed=0, lens=None, spare_rows=0, **form):
    """Parents' rows may be 0; kv are the tokens of each request itself."""
    c = _case(kv, rows, hq, hkv, dim, page, dt, seed=seed)
    if kind == "none":
        two, ref = c, c
    else:
        two, ref = _coded(c, kind)
    hints = {k: form.pop(k) for k in ("max_rows", "workspace") if k in form}
    lens = kv if lens is None else lens
    total = sum(rows)
    if spare_rows:
        two = {**two, "query": torch.cat([two["query"], torch.full((spare_rows, hq, dim), float("nan"), device=DEV).to(DT[dt])])}
    plan = paged.share_rows(_i32(parents), two["cu_rows"], two["kv_lens"], _i32(lens), total + spare_rows)
    out = torch.full_like(two["query"], 7.0)
    paged.attention(**two, **form, **hints, shared=plan, out=out)
    whole, before = _whole(ref, parents, lens)
    want, tol = _reference(whole, **form)
    cu = c["cu_rows"].tolist()
    for b in range(len(kv)):   # rows before a request's own first token get zeros
        none = max(0, rows[b] - kv[b])
        want[cu[b]: cu[b] + none], tol[cu[b]: cu[b] + none] = 0.0, 0.0
    _within(out[:total], want, tol)
    assert (out[total:] == 7.0).all()
    return out[:total]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hq,hkv,dim", HEADS)
def test_single_tokens(hq, hkv, dim, kind):
    # request 3 is everybody's parent but for two; lengths around the tiles' ends
    kv = [1, 17, 33, 333, 64, 2, 16, 127, 300, 15, 31, 1]
    parents = [3, 3, 3, -1, 3, 3, -1, 3, 3, 3, 3, 99]
    rows = [1, 1, 1, 0, 1, 1, 1, 1, 1, 1, 1, 1]
    _check(parents, kv, rows, hq, hkv, dim, 16, "bf16", kind, seed=1, max_rows=1)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("hq,hkv,dim", [(8, 2, 128), (6, 2, 64), (40, 1, 64), (2, 2, 128)])
def test_chunks_of_several_parents(hq, hkv, dim, dt, kind):
    kv = [700, 5, 33, 64, 260, 129, 300, 90, 1]
    rows = [0, 5, 2, 64, 0, 65, 9, 90, 1]
    parents = [-1, 0, 4, 0, -1, 4, -1, 0, 4]
    _check(parents, kv, rows, hq, hkv, dim, 32, dt, kind, seed=2)


@pytest.mark.parametrize("length", [1, 15, 16, 17, 63, 64, 65, 255, 256, 257, 1000, 5000])
def test_lengths_of_the_parent(length):
    kv = [length, 3, 40, 700]
    for rows in ([0, 1, 1, 1], [0, 3, 20, 40]):
        _check([-1, 0, 0, 0], kv, rows, 8, 2, 128, 16, "bf16", seed=3)


@pytest.mark.parametrize("kind", KINDS)
def test_many_children(kind):
    rng = random.Random(5)
    n = 150
    parents = [-1, -1, -1] + [rng.choice([0, 0, 1, 2, -1]) for _ in range(n - 3)]
    kv = [900, 77, 2100] + [rng.randint(1, 60) for _ in range(n - 3)]
    rows = [0, 0, 1] + [min(k, rng.choice([0, 1, 1, 4])) for k in kv[3:]]
    _check(parents, kv, rows, 8, 2, 128, 16, "bf16", kind, seed=5)
    # everybody behind one: more than a tile of heirs
    _check([7] * n, kv, rows, 4, 2, 64, 16, "bf16", kind, seed=6)


@pytest.mark.parametrize("kind", ["none", "fp8"])
@pytest.mark.parametrize("form", ["cap", "bias", "cap_bias", "window", "documents", "prefix"])
@pytest.mark.parametrize("dt,dim", [("bf16", 128), ("fp16", 64)])
def test_forms(form, dt, dim, kind):
    kv, rows = [300, 1, 77, 150, 33, 40], [0, 1, 77, 140, 2, 1]
    parents = [-1, 0, 0, 0, 0, -1]
    f = {}
    if "cap" in form:
        f["softcap"] = 5.0
    if "bias" in form:
        f["slopes"] = torch.tensor([2.0 ** -i for i in range(8)], device=DEV)
    at = torch.cat([torch.arange(n - m, n) + (300 if p == 0 else 0) for n, m, p in zip(kv, rows, parents)])
    if form == "window":     # windows that end in the parent, at its end, in the own tokens
        f["first_keys"] = (at - 63).int().to(DEV)
    if form == "documents":
        f["first_keys"] = (at // 37 * 37).int().to(DEV)
        f["first_keys"][0], f["first_keys"][5], f["first_keys"][9] = -2 ** 31, 2 ** 31 - 1, 10 ** 6
    if form == "prefix":
        f["prefix_lens"] = _i32([3, 50, 350, 440, 333, 1000])
    _check(parents, kv, rows, 8, 2, dim, 16, dt, kind, seed=8, **f)


def test_parents_that_are_none():
    # a parent without tokens, the request itself, out of range; a request that was not served; a parent's parent
    kv = [40, 30, 0, 25, 20, 60]
    rows = [1, 2, 3, 4, 5, 6]
    parents = [1, 99, 0, 3, -7, 0]
    lens = [40, 0, 0, 25, 20, 60]
    out = _check(parents, kv, rows, 8, 2, 128, 16, "bf16", seed=9, lens=lens)
    assert (out[3:6] == 0).all()    # request 2 has no tokens


def test_padded_rows_and_rows_behind_the_last_request():
    # more rows than tokens: zeros before a request's own first one, whatever its parent holds
    kv, rows = [200, 3, 40, 0, 9], [0, 40, 40, 40, 40]
    out = _check([-1, 0, 0, 0, -1], kv, rows, 8, 2, 128, 16, "bf16", seed=10, spare_rows=11)
    assert (out[:37] == 0).all() and (out[80:120] == 0).all() and (out[37:40] != 0).any()


def test_a_parent_that_steps_too():
    # its own rows are causal, its children see all of it
    _check([-1, 0, 0], [500, 20, 1], [9, 5, 1], 8, 2, 128, 16, "bf16", seed=11)


def test_longer_tokens_than_a_table_row_and_holes():
    c = _case([90, 30], [0, 2], 8, 2, 128, 16, "bf16", seed=12)
    table = c["table"].clone()
    table[0, 2] = -1
    plan = paged.share_rows(_i32([-1, 0]), c["cu_rows"], c["kv_lens"], _i32([90, 30]), 2)
    got = paged.attention(**{**c, "table": table}, shared=plan)
    # the hidden page as a document that starts behind it, in two pieces: keys 0..31 and 48.. of the parent
    k = c["k_pages"][c["table"][0, :6].clamp(min=0).long()].transpose(1, 2).flatten(0, 1)[:90]
    v = c["v_pages"][c["table"][0, :6].clamp(min=0).long()].transpose(1, 2).flatten(0, 1)[:90]
    own = [c[x][c["table"][1, :2].long()].transpose(1, 2).flatten(0, 1)[:30] for x in ("k_pages", "v_pages")]
    kk, vv = (torch.cat([x[:32], x[48:], y]) for x, y in ((k, own[0]), (v, own[1])))
    n = kk.shape[0]
    pages = [torch.zeros((1, 2, 256, 128), device=DEV).bfloat16() for _ in range(2)]
    pages[0][0, :, :n], pages[1][0, :, :n] = kk.transpose(0, 1), vv.transpose(0, 1)
    want, tol = _reference(dict(query=c["query"], k_pages=pages[0], v_pages=pages[1], table=_i32([[0]]), cu_rows=_i32([0, 2]),
                                kv_lens=_i32([n]), scaling=c["scaling"]))
    _within(got, want, tol)
    # lengths past the table row are read as the row's end
    plan = paged.share_rows(_i32([-1, 0]), c["cu_rows"], c["kv_lens"], _i32([10 ** 6, 30]), 2)
    full = c["table"].clone()
    full[0] = full[0, 0]
    assert torch.isfinite(paged.attention(**{**c, "table": full}, shared=plan, first_keys=_i32([0, 0]))).all()


def test_infinities_and_nan_in_masked_places():
    kv, rows = [250, 60, 4], [0, 60, 1]
    c = _case(kv, rows, 4, 2, 128, 16, "bf16", seed=14)
    put = lambda x, t, d, y: c[x][int(c["table"][0, t // 16])].__setitem__((slice(None), t % 16, d), y)  # noqa: E731
    put("v_pages", 10, 3, float("nan"))
    put("v_pages", 200, 5, float("inf"))
    put("k_pages", 40, 5, float("nan"))
    first = torch.full((61,), 41, dtype=torch.int32)
    first[7], first[60] = 201, 0
    parents, lens = [-1, 0, 0], kv
    plan = paged.share_rows(_i32(parents), c["cu_rows"], c["kv_lens"], _i32(lens), 61)
    got = paged.attention(**c, shared=plan, first_keys=first.to(DEV))
    whole, _ = _whole(c, parents, lens)
    want, tol = _reference(whole, first_keys=first.to(DEV))
    _within(got, want, tol)
    assert torch.isfinite(got[7]).all() and torch.isinf(got[8, :, 5]).all() and torch.isnan(got[60]).any()


def test_workspace_hints_and_strides():
    parents, kv, rows = [-1, 0, 0, 0], [3000, 20, 31, 7], [0, 1, 9, 3]
    c = _case(kv, rows, 8, 2, 128, 16, "bf16", seed=19)
    plan = paged.share_rows(_i32(parents), c["cu_rows"], c["kv_lens"], _i32(kv), 13)
    whole, _ = _whole(c, parents, kv)
    want, tol = _reference(whole)
    ws = paged.attention_workspace(13, 13, 4, c["table"].shape[1], 16, 8, 2, 128, DEV, shared=True)
    a = paged.attention(**c, shared=plan, workspace=ws)
    ws.fill_(float("nan"))
    assert torch.equal(paged.attention(**c, shared=plan, workspace=ws), a) and torch.equal(paged.attention(**c, shared=plan), a)
    for hint in (0, 1, 2, 1000):
        _within(paged.attention(**c, shared=plan, max_rows=hint), want, tol)
    q = torch.empty((8, 13, 131), dtype=torch.bfloat16, device=DEV)[..., 1:129].transpose(0, 1)
    q.copy_(c["query"])
    wide = torch.zeros((13, 8, 256), dtype=torch.bfloat16, device=DEV)
    paged.attention(**{**c, "query": q}, shared=plan, out=wide[..., 128:])
    _within(wide[..., 128:], want, tol)
    assert (wide[..., :128] == 0).all()


def test_refusals():
    c = _case([30, 5], [2, 1], 8, 2, 128, 16, "bf16", seed=20)
    args = (_i32([-1, 0]), c["cu_rows"], c["kv_lens"], _i32([30, 5]))
    plan = paged.share_rows(*args, 3)
    with pytest.raises(RuntimeError, match="cu_rows"):
        paged.share_rows(_i32([-1, 0, 0]), *args[1:], 3)
    with pytest.raises(RuntimeError, match="parents"):
        paged.share_rows(args[0].long(), *args[1:], 3)
    with pytest.raises(RuntimeError, match="parents must be CUDA"):
        paged.share_rows(args[0].cpu(), *args[1:], 3)
    with pytest.raises(RuntimeError, match="out must be"):
        paged.share_rows(*args, 4, out=plan)
    with pytest.raises(RuntimeError, match="1 to 2"):
        paged.share_rows(*args, 0)
    other = paged.share_rows(*args, 9)
    with pytest.raises(RuntimeError, match="shared must be"):
        paged.attention(**c, shared=other)
    ws = torch.empty(100, device=DEV)
    with pytest.raises(RuntimeError, match="workspace"):
        paged.attention(**c, shared=plan, workspace=ws)


# -- a run of them together ------------------------------------------------------------


@pytest.mark.parametrize("kind", ["none", "fp8"])
def test_samples_of_a_prompt_served_in_a_graph(kind):
    """A prompt is written once; its samples start empty and grow token by token in a replayed step (plan, gathering,
    write, attention), one ends and another starts in its place; releases leave the parent's pages alone."""
    hq, hkv, dim, page, n = 8, 2, 128, 16, 5
    g = torch.Generator(device=DEV).manual_seed(22)
    new = lambda h, rows: torch.randn((rows, h, dim), generator=g, device=DEV).bfloat16()  # noqa: E731
    table = paged.PageTable(n, 700, 80, page, DEV)
    sc = {}
    if kind == "none":
        kp, vp = (torch.full((80, hkv, page, dim), float("nan"), device=DEV).bfloat16() for _ in range(2))
    else:
        (kp, ks), (vp, vs) = (paged.quantized_pages(80, hkv, page, dim, kind, DEV) for _ in range(2))
        sc = dict(k_scales=ks, v_scales=vs)
    plan = table.step(_i32([0, 0, 203, 0, 0]), 203)   # request 2 is the prompt
    paged.append(new(hkv, 203), new(hkv, 203), kp, vp, plan.slots, **sc)
    parents = _i32([2, 2, -1, 2, -1])
    one = _i32([1, 1, 0, 1, 1])
    buf = [new(hkv, 4), new(hkv, 4), new(hq, 4)]
    step, shared = paged.StepPlan.empty(n, 4, DEV), paged.SharedRows(n, 4, DEV)
    ws = paged.attention_workspace(4, 1, n, table.table.shape[1], page, hq, hkv, dim, DEV, shared=True)
    out = torch.empty_like(buf[2])

    def run():
        table.step(one, 4, out=step)
        paged.share_rows(parents, step.cu_rows, step.kv_lens, table.lens, 4, out=shared)
        paged.append(buf[0], buf[1], kp, vp, step.slots, **sc)
        paged.attention(buf[2], kp, vp, table.table, step.cu_rows, step.kv_lens, dim ** -0.5, max_rows=1, shared=shared,
                        out=out, workspace=ws, **sc)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            run()
    torch.cuda.current_stream().wait_stream(side)
    lens = [0, 0, 203, 0, 0]
    for i in range(40):
        for t, h in zip(buf, (hkv, hkv, hq)):
            t.copy_(new(h, 4))
        graph.replay() if i % 7 != 2 else run()
        lens = [m + (b != 2) for b, m in enumerate(lens)]
        assert table.lens.tolist() == lens
        assert shared.positions.tolist() == [lens[0] + 202, lens[1] + 202, lens[3] + 202, lens[4] - 1]
        if i % 5 == 0 or i > 35:   # against every request's tokens read back
            cu = _i32([0, *torch.tensor(lens).cumsum(0).tolist()])
            k, v = paged.read(kp, vp, table.table, cu, table.lens, sum(lens), **sc)
            k, v = (x.split(lens) for x in (k, v))
            for row, b in enumerate((0, 1, 3, 4)):
                both = [torch.cat([x[2], x[b]]) if b != 4 else x[b] for x in (k, v)]
                m = both[0].shape[0]
                pages = [torch.zeros((1, hkv, 512, dim), device=DEV).bfloat16() for _ in range(2)]
                for p, x in zip(pages, both):
                    p[0, :, :m] = x.transpose(0, 1)
                want, tol = _reference(dict(query=buf[2][row:row + 1], k_pages=pages[0], v_pages=pages[1], table=_i32([[0]]),
                                            cu_rows=_i32([0, 1]), kv_lens=_i32([m]), scaling=dim ** -0.5))
                _within(out[row:row + 1], want, tol)
        if i == 20:
            table.release(_i32([999, 0, 999, 999, 999]))   # request 1 ends; its row starts anew
            lens[1] = 0
    held = set(table.table[2, :13].tolist())
    table.release(_i32([0, 0, 999, 0, 0]))
    assert set(table.table[2, :13].tolist()) == held and int(table.count) == 80 - 13


def test_the_same_as_without_sharing():
    """Requests whose table rows hold the parent's pages themselves, at a page's end, give the same within rounding."""
    kv = [256, 40, 3, 100]
    c = _case(kv, [0, 1, 3, 40], 8, 2, 128, 16, "bf16", seed=30)
    table = torch.full((4, 40), -1, dtype=torch.int32, device=DEV)
    for b in range(1, 4):
        own = -(-kv[b] // 16)
        table[b, :16], table[b, 16:16 + own] = c["table"][0, :16], c["table"][b, :own]
    plain = paged.attention(**{**c, "table": table, "kv_lens": _i32([0, 296, 259, 356])})
    plan = paged.share_rows(_i32([-1, 0, 0, 0]), c["cu_rows"], c["kv_lens"], _i32(kv), 44)
    shared = paged.attention(**c, shared=plan)
    want, tol = _reference(_whole(c, [-1, 0, 0, 0], kv)[0])
    _within(plain, want, tol)
    _within(shared, want, tol)


def test_two_streams_at_once():
    cases = []
    for i in range(2):
        kv, rows = [1500 + 700 * i, 3, 40, 9], [0, 1, 2, 1]
        c = _case(kv, rows, 8, 2, 128, 16, "bf16", seed=50 + i)
        cases.append((c, paged.share_rows(_i32([-1, 0, 0, 0]), c["cu_rows"], c["kv_lens"], _i32(kv), 4)))
    want = [paged.attention(**c, shared=p) for c, p in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, (c, p) in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                got[i].append(paged.attention(**c, shared=p))
    torch.cuda.synchronize()
    for w, many in zip(want, got):
        assert all(torch.equal(w, y) for y in many)


@pytest.mark.parametrize("unit", [2624, 3008])
def test_a_chunk_and_one_key(unit):
    """A request of one key more than a chunk whose reciprocal, rounded, times the chunk is below one: 512 workgroups of
    `unit` keys, as 31 requests of two chunks and one of a chunk and that key, 8 KV heads."""
    kv = [2 * unit] * 31 + [unit + 1]
    c = _case(kv, [1] * 32, 8, 8, 64, 64, "bf16", seed=60)
    for b in range(32):     # the last key's value shows in the output
        c["v_pages"][int(c["table"][b, (kv[b] - 1) // 64]), :, (kv[b] - 1) % 64] = 512.0
    plan = paged.share_rows(_i32([-1] * 32), c["cu_rows"], c["kv_lens"], c["kv_lens"], 32)
    want, tol = _reference(c)
    _within(paged.attention(**c, shared=plan, max_rows=1), want, tol)

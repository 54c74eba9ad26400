"""Quantised pages of the paged K/V cache on the GPU: the writes code for code
against a search for the nearest one in 64 bits, reads bit for bit, and the
attention against 64 bits of the values that the codes stand for, within the
bound of the 16-bit pages (a code times its scale is a 16-bit value)."""

import math
import random

import pytest
import torch

from kv_cache_amd import paged
from test_gpu_paged import DEV, DT, HEADS, FORMS, _case, _i32, _pages, _reference, _within

pytestmark = pytest.mark.gpu
KINDS = ["fp8", "fp4"]
MOST = {("fp8", torch.bfloat16): 1.875 * 2.0 ** 127, ("fp8", torch.float16): 61440.0,
        ("fp4", torch.bfloat16): 1.5 * 2.0 ** 127, ("fp4", torch.float16): 49152.0}


def _values_of(kind):
    """What every code stands for, from its bits (64 bits)."""
    bits, man, bias = {"fp8": (8, 3, 7), "fp4": (4, 1, 1)}[kind]
    out = []
    for c in range(1 << bits):
        low = c & ((1 << (bits - 1)) - 1)
        e, f = low >> man, (low & ((1 << man) - 1)) / (1 << man)
        x = f * 2.0 ** (1 - bias) if e == 0 else (1 + f) * 2.0 ** (e - bias)
        out.append(math.nan if kind == "fp8" and low == 127 else -x if c >> (bits - 1) else x)
    return torch.tensor(out, dtype=torch.float64)


def _power(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _oracle(x, kind):
    """(codes one to an entry, scale bytes) of [..., D], by search: the least scale under which the largest magnitude
    is within half a step of a code, and each value's nearest code."""
    x = x.cpu()
    dtype, x = x.dtype, x.cpu().double().reshape(*x.shape[:-1], -1, 32)
    odd = ~torch.isfinite(x).all(-1)
    x = torch.where(odd[..., None], 0.0, x.clamp(-MOST[kind, dtype], MOST[kind, dtype]))
    edge, amax = {"fp8": 464.0, "fp4": 7.0}[kind], x.abs().amax(-1)
    e = torch.full(amax.shape, -100)
    for t in range(-100, 128):
        e = torch.where(amax > edge * 2.0 ** t, t + 1, e)
    x = x / _power(e)[..., None]
    val = _values_of(kind)
    half = len(val) // 2
    mags = val[:half].nan_to_num(math.inf)                # ascending
    off = (x.abs()[..., None] - mags).abs()
    best = off.amin(-1, keepdim=True)
    ties = off == best                                      # of two nearest the even code
    even = ties & (torch.arange(half) % 2 == 0)
    code = torch.where(even.any(-1), even.int().argmax(-1), ties.int().argmax(-1))
    code = code + half * torch.signbit(x).long()
    return code.reshape(*code.shape[:-2], -1), torch.where(odd, 255, e + 127)


def _stand_for(codes, scales, kind, dtype):
    """The 16-bit values that codes (one to an entry) and scale bytes stand for."""
    x = _values_of(kind)[codes.long()].reshape(*scales.shape, 32)
    s = torch.where(scales.long() == 255, math.nan, _power(scales.long() - 127))
    return (x * s[..., None]).reshape(codes.shape).to(dtype)


def _unpack(pages, kind):
    raw = pages.view(torch.uint8).cpu().long()
    return torch.stack([raw & 15, raw >> 4], -1).flatten(-2) if kind == "fp4" else raw


def _pack(codes, kind):
    codes = codes.to(torch.uint8).to(DEV)
    if kind == "fp4":
        return codes[..., 0::2] | codes[..., 1::2] << 4
    return codes.view(torch.float8_e4m3fn)


def _coded(c, kind):
    """The case over codes of its pages, and the case of the 16-bit pages that they stand for."""
    two, ref = dict(c), dict(c)
    for name in ("k", "v"):
        x = c[name + "_pages"]
        codes, scales = _oracle(x, kind)
        two[name + "_pages"] = _pack(codes, kind)
        two[name + "_scales"] = scales.to(torch.uint8).to(DEV)
        ref[name + "_pages"] = _stand_for(codes, scales, kind, x.dtype).to(DEV)
    return two, ref


def _check(c, kind, **form):
    two, ref = _coded(c, kind)
    hints = {k: form.pop(k) for k in ("max_rows", "workspace") if k in form}
    want, tol = _reference(ref, **form)
    got = paged.attention(**two, **form, **hints)
    _within(got, want, tol)
    return got


# -- writes and reads -----------------------------------------------------------------


def _same_codes(pages, codes, kind):
    """Code for code, but for the sign of zero."""
    val = _values_of(kind)
    a, b = val[_unpack(pages, kind)], val[codes.cpu().long()]
    assert torch.equal(a.nan_to_num(9e9), b.nan_to_num(9e9))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,heads,dim,page,dt,layout", [
    (1, 1, 64, 16, "bf16", "plain"), (37, 8, 128, 16, "fp16", "plain"), (300, 3, 64, 64, "bf16", "heads_first"),
    (300, 2, 128, 32, "bf16", "token_major"), (65, 5, 96, 128, "fp16", "unaligned"), (9, 7, 32, 16, "bf16", "plain")])
def test_append_and_read(rows, heads, dim, page, dt, layout, kind):
    rng, dtype = random.Random(rows), DT[dt]
    pages = -(-rows // page) + 3
    g = torch.Generator(device=DEV).manual_seed(3)
    make = lambda *s: (torch.randn(s, generator=g, device=DEV) * torch.exp2(torch.randn(s, generator=g, device=DEV) * 3)).to(dtype)  # noqa: E731
    if layout == "heads_first":
        k, v = (make(heads, rows, dim).transpose(0, 1) for _ in range(2))
    elif layout == "unaligned":
        k, v = (make(rows, heads, dim + 3)[..., 1:1 + dim] for _ in range(2))
    else:
        k, v = (make(rows, heads, dim) for _ in range(2))
    kp, ks = paged.quantized_pages(pages, heads, page, dim, kind, DEV)
    vp, vs = paged.quantized_pages(pages, heads, page, dim, kind, DEV)
    if layout == "token_major":
        wide = torch.zeros((2, pages, page, heads, kp.shape[3] + 16), dtype=torch.uint8, device=DEV)
        kp, vp = (x.transpose(1, 2)[..., :kp.shape[3]].view(kp.dtype) for x in wide)
    for t in (kp, vp, ks, vs):
        t.view(torch.uint8).fill_(7)
    at = rng.sample(range(pages * page), rows)
    at[0] = -1 if rows > 1 else at[0]
    if rows > 2:
        at[2] = pages * page + 5   # outside the cache: skipped
    paged.append(k, v, kp, vp, torch.tensor(at, device=DEV), k_scales=ks, v_scales=vs)
    for new, p, s in ((k, kp, ks), (v, vp, vs)):
        want_c = torch.full((pages, heads, page, dim), 7, dtype=torch.long)
        if kind == "fp4":
            want_c[..., 1::2] = 0
        want_s = torch.full((pages, heads, page, dim // 32), 7)
        codes, scales = _oracle(new, kind)
        for r, slot in enumerate(at):
            if 0 <= slot < pages * page:
                want_c[slot // page, :, slot % page], want_s[slot // page, :, slot % page] = codes[r], scales[r]
        _same_codes(p, want_c, kind)
        assert torch.equal(s.cpu().long(), want_s)
    # two requests of all tokens of the pool, read back
    table = torch.tensor([list(range(pages))[::-1], list(range(pages))], dtype=torch.int32, device=DEV)
    total = pages * page
    out = paged.read(kp, vp, table, _i32([0, total - 3, 2 * total - 3]), _i32([total, total]), 2 * total - 3, k_scales=ks,
                     v_scales=vs, dtype=dtype)
    for got, p, s in zip(out, (kp, vp), (ks, vs)):
        x = _stand_for(_unpack(p, kind), s.cpu(), kind, dtype)
        whole = torch.cat([x.flip(0).transpose(1, 2).flatten(0, 1)[3:], x.transpose(1, 2).flatten(0, 1)])
        assert torch.equal(got.cpu().nan_to_num(7777.0), whole.nan_to_num(7777.0))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_values_at_the_edges(dt, kind):
    dtype, big = DT[dt], torch.finfo(DT[dt]).max
    tiny = torch.finfo(dtype).smallest_normal / 4
    rows = []
    for top in (464.0, 465.0, 466.0, 448.0, 7.0, 7.03125, 6.0, 1.0, 0.0, big, big * 0.9, 61440.0, 49152.0, 57344.0, tiny,
                2.0 ** -14, math.inf, math.nan, -math.inf):
        x = torch.zeros(64)
        x[0], x[33] = top, -top     # and values half way between codes, of every exponent
        steps = _values_of(kind)[: 127 if kind == "fp8" else 8]
        mid = (steps[1:] + steps[:-1]) / 2
        part = mid[torch.linspace(0, len(mid) - 1, 31).long()].float()
        x[1:32], x[34:64] = part, -part[1:]
        rows.append(x)
    x = torch.stack(rows).to(dtype)[:, None].expand(-1, 2, -1).contiguous().to(DEV)
    n = x.shape[0]
    kp, ks = paged.quantized_pages(3, 2, 16, 64, kind, DEV)
    vp, vs = paged.quantized_pages(3, 2, 16, 64, kind, DEV)
    paged.append(x, -x, kp, vp, torch.arange(n, device=DEV), k_scales=ks, v_scales=vs)
    table = torch.tensor([[0, 1, 2]], dtype=torch.int32, device=DEV)
    out = paged.read(kp, vp, table, _i32([0, n]), _i32([n]), n, k_scales=ks, v_scales=vs, dtype=dtype)
    for new, got, p, s in ((x, out[0], kp, ks), (-x, out[1], vp, vs)):
        codes, scales = _oracle(new, kind)
        flat = lambda t: t.transpose(1, 2).flatten(0, 1)[:n]  # noqa: E731
        assert torch.equal(flat(s).cpu().long(), scales)
        _same_codes(flat(p), codes, kind)
        want = _stand_for(codes, scales, kind, dtype)
        assert torch.equal(got.cpu().nan_to_num(0.5, 1e30, -1e30), want.nan_to_num(0.5, 1e30, -1e30))
        # finite stays finite, blocks with what is not become NaN
        odd = ~torch.isfinite(new.reshape(n, 2, 2, 32)).all(-1, keepdim=True).expand(-1, -1, -1, 32).reshape(n, 2, 64)
        assert torch.equal(torch.isnan(got), odd) and torch.isfinite(got[~odd]).all()
        # half a step: 2^-4 (fp8) or 2^-2 (fp4; 1/2 between 4 and 6 is a quarter of 4) of the value, or half the least one
        err, y = (got.double() - new.double()).abs()[~odd], new.double().abs()[~odd]
        scale = _power(scales.clamp(max=254).to(DEV) - 127).repeat_interleave(32, -1)[~odd]
        step = (2.0 ** -4, 2.0 ** -10) if kind == "fp8" else (2.0 ** -2, 2.0 ** -2)
        fits = y <= MOST[kind, dtype]
        # reading into fp16 rounds values below 2^-14 by up to 2^-25
        assert (err <= torch.maximum(step[0] * y, step[1] * scale) + (2.0 ** -25 if dt == "fp16" else 0.0))[fits].all()


@pytest.mark.parametrize("kind", ["none", "fp8", "fp4"])
def test_read_of_tokens_that_are_not_there(kind):
    c = _case([30, 0, 70, 5], [0, 0, 0, 0], 2, 2, 64, 16, "bf16", seed=31)
    two = c if kind == "none" else _coded(c, kind)[0]
    # more rows than tokens, a request without tokens, a page outside the pool, rows behind the last request
    table = two["table"].clone()
    table[2, 1] = 10 ** 9
    rows = [33, 2, 70, 1]
    cu = [0, 33, 35, 105, 106]
    sc = {} if kind == "none" else dict(k_scales=two["k_scales"], v_scales=two["v_scales"])
    wide = torch.full((2, 110, 2, 80), 3.0, device=DEV, dtype=torch.bfloat16)
    out = tuple(w[..., :64] for w in wide)
    got = paged.read(two["k_pages"], two["v_pages"], table, _i32(cu), two["kv_lens"], 110, **sc, out=out)
    assert got[0] is out[0] and (wide[..., 64:] == 3.0).all() and (wide[:, 106:] == 3.0).all()
    ref = c if kind == "none" else _coded(c, kind)[1]
    for g, pages in zip(got, (ref["k_pages"], ref["v_pages"])):
        assert (g[:3] == 0).all() and (g[33:35] == 0).all() and (g[35 + 16:35 + 32] == 0).all()
        x = pages[table[0, :2].long()].transpose(1, 2).flatten(0, 1)[:30]
        assert torch.equal(g[3:33], x)
        x = pages[table[2, :5].clamp(0, 0 + pages.shape[0] - 1).long()].transpose(1, 2).flatten(0, 1)[:70]
        assert torch.equal(g[35:51], x[:16]) and torch.equal(g[67:105], x[32:])
        assert torch.equal(g[105], pages[table[3, 0].long(), :, 4])
    assert rows[0] == 33
    none = paged.read(two["k_pages"], two["v_pages"], table, _i32([0] * 5), two["kv_lens"], 0, **sc)
    assert none[0].shape == (0, 2, 64)


# -- attention ----------------------------------------------------------------------


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("hq,hkv,dim", HEADS)
def test_single_tokens(hq, hkv, dim, dt, kind):
    kv = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 0, 200, 256, 257, 700]
    _check(_case(kv, [1] * len(kv), hq, hkv, dim, 16, dt, seed=1), kind, max_rows=1)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("hq,hkv,dim", HEADS)
def test_chunks(hq, hkv, dim, dt, kind):
    kv, rows = [1, 5, 33, 64, 129, 300, 431, 0], [1, 5, 2, 64, 65, 9, 130, 0]
    _check(_case(kv, rows, hq, hkv, dim, 32, dt, seed=2), kind)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [16, 64, 256, 4096])
def test_pages(page, kind):
    _check(_case([1, 100, 515, 1025], [1, 40, 3, 1], 4, 2, 128, page, "bf16", seed=3), kind)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hq,hkv,dim,dt", [(8, 2, 128, "bf16"), (3, 1, 64, "fp16"), (40, 2, 64, "bf16")])
def test_split_keys(hq, hkv, dim, dt, kind):
    for kv, rows in (([5000], [1]), ([3001, 70, 2048], [2, 70, 1]), ([2500, 2600], [40, 3]), ([4097], [130])):
        _check(_case(kv, rows, hq, hkv, dim, 16, dt, seed=4), kind)


@pytest.mark.parametrize("kind", KINDS)
def test_many_requests(kind):
    rng = random.Random(7)
    kv = [rng.choice([0, 1, rng.randint(1, 90)]) for _ in range(300)]
    kv[250] = 3000
    rows = [min(n, rng.choice([0, 1, 1, 1, 20])) for n in kv]
    _check(_case(kv, rows, 4, 2, 64, 16, "bf16", seed=7), kind)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dt,dim", [("bf16", 128), ("fp16", 64)])
@pytest.mark.parametrize("form", FORMS)
def test_forms(form, dt, dim, kind):
    kv, rows = [1, 77, 300, 513, 40], [1, 77, 140, 2, 1]
    c = _case(kv, rows, 8, 2, dim, 16, dt, seed=8)
    f = {}
    if "cap" in form:
        f["softcap"] = 5.0
    if "bias" in form:
        f["slopes"] = torch.tensor([2.0 ** -i for i in range(8)], device=DEV)
    if "prefix" in form:
        f["prefix_lens"] = _i32([3, 50, 299, 0, 1000])
    at = torch.cat([torch.arange(n - m, n) for n, m in zip(kv, rows)])
    if "documents" in form:
        f["first_keys"] = (at // 37 * 37).int().to(DEV)
    if form == "window":
        f["first_keys"] = (at - 63).int().to(DEV)
    _check(c, kind, **f)


@pytest.mark.parametrize("kind", KINDS)
def test_rows_that_see_nothing(kind):
    c = _case([50, 200, 5], [50, 3, 1], 4, 2, 128, 16, "bf16", seed=11)
    first = torch.zeros(54, dtype=torch.int32)
    first[3:7], first[51], first[53] = 50, 10 ** 6, 5
    got = _check(c, kind, first_keys=first.to(DEV))
    assert (got[3:7] == 0).all() and (got[51] == 0).all() and (got[53] == 0).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("rows", [[60, 1], [2, 1], [200, 1]])
def test_nan_in_masked_places(rows, dt, kind):
    """The pages' own: blocks of NaN behind the last token, in V of tokens that some rows see, in K and V of hidden ones."""
    kv = [max(rows[0], 90) + 5, 400]
    c = _case(kv, rows, 4, 2, 128, 16, dt, seed=14)

    def put(pages, b, t, d, x):
        pages[int(c["table"][b, t // 16]), :, t % 16, d] = x

    put(c["v_pages"], 0, kv[0] - 1, 5, float("inf"))
    put(c["v_pages"], 0, kv[0] - 2, 70, float("nan"))
    got = _check(c, kind)
    assert torch.isnan(got[rows[0] - 1, :, :32]).all() and torch.isfinite(got[: rows[0] - 2]).all()
    put(c["k_pages"], 1, 3, 0, float("nan"))
    put(c["k_pages"], 1, 70, 1, float("inf"))
    put(c["v_pages"], 1, 70, 0, float("nan"))
    put(c["v_pages"], 1, 3, 0, float("-inf"))
    first = torch.zeros(sum(rows), dtype=torch.int32)
    first[-1] = 71
    got = _check(c, kind, first_keys=first.to(DEV))
    assert torch.isfinite(got[-1]).all()
    # every code and scale byte behind the last tokens, NaN codes among them
    two, ref = _coded(_case(kv, rows, 4, 2, 128, 16, dt, seed=14), kind)
    for b, n in enumerate(kv):
        if n % 16 == 0:
            continue   # nothing lies behind its last token
        last = int(two["table"][b, (n - 1) // 16])
        for name in ("k_pages", "v_pages", "k_scales", "v_scales"):
            t = two[name].view(torch.uint8)[last, :, n % 16:]
            t.copy_(torch.randint(256, t.shape, device=DEV, dtype=torch.uint8))
    want, tol = _reference(ref)
    _within(paged.attention(**two), want, tol)


@pytest.mark.parametrize("kind", KINDS)
def test_table_entries_outside_the_pool(kind):
    c = _case([200, 90, 40], [30, 1, 40], 8, 2, 128, 16, "bf16", seed=15)
    c["table"][0, 3], c["table"][1, 0], c["table"][2, 2] = -1, 10 ** 9, c["k_pages"].shape[0]
    _check(c, kind)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128])
def test_strides(kind, dim):
    c = _case([77, 300, 1], [40, 1, 1], 8, 2, dim, 16, "bf16", seed=18)
    two, ref = _coded(c, kind)
    want, tol = _reference(ref)
    # a token-major pool with both in one row; scales of both in one tensor
    p, width = two["k_pages"].shape[0], two["k_pages"].shape[3]
    pool = torch.zeros((p, 16, 2, 2, width), dtype=torch.uint8, device=DEV)
    sc = torch.zeros((p, 2, 2, 16, dim // 32), dtype=torch.uint8, device=DEV)
    odd = dict(two)
    for i, n in enumerate(("k", "v")):
        view = pool[:, :, i].transpose(1, 2).view(two["k_pages"].dtype)
        view.view(torch.uint8).copy_(two[n + "_pages"].view(torch.uint8))
        s = sc[:, i]
        s.copy_(two[n + "_scales"])
        odd[n + "_pages"], odd[n + "_scales"] = view, s
    _within(paged.attention(**odd), want, tol)


@pytest.mark.parametrize("kind", KINDS)
def test_workspace_and_hints(kind):
    two, ref = _coded(_case([3000, 20], [1, 60], 8, 2, 128, 16, "bf16", seed=19), kind)
    ws = paged.attention_workspace(61, 61, 2, two["table"].shape[1], 16, 8, 2, 128, DEV)
    a = paged.attention(**two, workspace=ws)
    ws.fill_(float("nan"))
    assert torch.equal(paged.attention(**two, workspace=ws), a) and torch.equal(paged.attention(**two), a)
    want, tol = _reference(ref)
    for hint in (0, 1, 2, 1000):
        _within(paged.attention(**two, max_rows=hint), want, tol)


def test_offsets_past_32_bits():
    """Pages far into a pool of more than 2^32 bytes."""
    pages, page = (1 << 32) // (2 * 4096 * 64) + 9, 4096
    kp, ks = paged.quantized_pages(pages, 2, page, 64, "fp8", DEV)
    vp, vs = paged.quantized_pages(pages, 2, page, 64, "fp8", DEV)
    g = torch.Generator(device=DEV).manual_seed(5)
    k, v, q = (torch.randn((40, h, 64), generator=g, device=DEV).bfloat16() for h in (2, 2, 4))
    slots = (pages - 1) * page + 100 + torch.arange(40, device=DEV)
    paged.append(k, v, kp, vp, slots, k_scales=ks, v_scales=vs)
    table = torch.full((1, 1), pages - 1, dtype=torch.int32, device=DEV)
    back = paged.read(kp, vp, table, _i32([0, 40]), _i32([140]), 40, k_scales=ks, v_scales=vs)
    for x, y in ((k, back[0]), (v, back[1])):
        codes, scales = _oracle(x, "fp8")
        assert torch.equal(y.cpu(), _stand_for(codes, scales, "fp8", torch.bfloat16))
    got = paged.attention(q, kp, vp, table, _i32([0, 40]), _i32([140]), 0.125, k_scales=ks, v_scales=vs,
                          first_keys=_i32([100] * 40))
    small = dict(query=q, k_pages=torch.zeros((1, 2, 64, 64), device=DEV).bfloat16(), table=_i32([[0]]), cu_rows=_i32([0, 40]),
                 kv_lens=_i32([40]), scaling=0.125)
    small["v_pages"] = small["k_pages"].clone()
    small["k_pages"][0, :, :40], small["v_pages"][0, :, :40] = back[0].transpose(0, 1), back[1].transpose(0, 1)
    want, tol = _reference(small)
    _within(got, want, tol)


def test_refusals():
    two, _ = _coded(_case([30], [2], 8, 2, 128, 16, "bf16", seed=20), "fp8")
    q = two["query"]
    for change, msg in ((dict(query=q.float()), "query must be"), (dict(query=q[..., :64]), "query must be"),
                        (dict(k_scales=None), "k_scales"), (dict(v_scales=two["v_scales"][..., :2]), "k_scales and v_scales"),
                        (dict(k_scales=two["k_scales"].int()), "k_scales and v_scales"),
                        (dict(k_pages=two["k_pages"][..., :64], v_pages=two["v_pages"][..., :64]), "k_scales and v_scales"),
                        (dict(v_pages=two["v_pages"].view(torch.uint8)), "one shape, dtype"),
                        (dict(v_pages=two["v_pages"].transpose(1, 2).contiguous().transpose(1, 2)), "same strides"),
                        (dict(k_pages=two["k_pages"].float(), v_pages=two["v_pages"].float()), "float8_e4m3fn or uint8"),
                        (dict(scaling=0.0), "scaling")):
        with pytest.raises(RuntimeError, match=msg):
            paged.attention(**{**two, **change})
    k = q[:, :2]
    pages = [two[n] for n in ("k_pages", "v_pages")]
    sc = dict(k_scales=two["k_scales"], v_scales=two["v_scales"])
    slots = torch.tensor([1, 2], device=DEV)
    with pytest.raises(RuntimeError, match="k_scales"):
        paged.append(k, k, *pages, slots)
    with pytest.raises(RuntimeError, match="must be bfloat16 or float16"):
        paged.append(k.float(), k.float(), *pages, slots, **sc)
    with pytest.raises(RuntimeError, match="as many rows"):
        paged.append(k, k[:1], *pages, slots, **sc)
    with pytest.raises(RuntimeError, match="as many rows"):
        paged.append(k, k.half(), *pages, slots, **sc)
    args = (*pages, two["table"], two["cu_rows"], two["kv_lens"], 2)
    for change, msg in ((dict(k_scales=None), "k_scales"), (dict(dtype=torch.float32), "dtype must be"),
                        (dict(out=(k, k[:1])), "out must be"), (dict(out=(k.float(), k.float())), "out must be")):
        with pytest.raises(RuntimeError, match=msg):
            paged.read(*args, **{**sc, **change})
    with pytest.raises(RuntimeError, match="16-byte aligned"):
        wide = torch.zeros((2, 2, 131), device=DEV, dtype=torch.bfloat16)[..., :128]
        paged.read(*args, **sc, out=(wide, wide))
    with pytest.raises(RuntimeError, match="not read as"):
        half = torch.zeros((4, 2, 16, 128), device=DEV, dtype=torch.bfloat16)
        paged.read(half, half, *args[2:], dtype=torch.float16)


# -- a run of them together ------------------------------------------------------------


@pytest.mark.parametrize("kind", KINDS)
def test_a_served_step_captured_and_replayed(kind):
    """Requests grow token by token: plan, write, attend and read captured once, replayed while they grow."""
    hq, hkv, dim, page, n = 8, 2, 128, 16, 3
    g = torch.Generator(device=DEV).manual_seed(22)
    new = lambda h, rows: torch.randn((rows, h, dim), generator=g, device=DEV).bfloat16()  # noqa: E731
    table = paged.PageTable(n, 700, 140, page, DEV)
    (kp, ks), (vp, vs) = (paged.quantized_pages(140, hkv, page, dim, kind, DEV) for _ in range(2))
    sc = dict(k_scales=ks, v_scales=vs)
    lens = [40, 600, 7]
    plan = table.step(_i32(lens), sum(lens))
    k, v = new(hkv, sum(lens)), new(hkv, sum(lens))
    paged.append(k, v, kp, vp, plan.slots, **sc)
    kept = [[x[a:b] for a, b in ((0, 40), (40, 640), (640, 647))] for x in (k, v)]
    one, buf = _i32([1] * n), [new(hkv, n), new(hkv, n), new(hq, n)]
    step = paged.StepPlan.empty(n, n, DEV)
    ws = paged.attention_workspace(n, 1, n, table.table.shape[1], page, hq, hkv, dim, DEV)
    out, back = torch.empty_like(buf[2]), (torch.empty_like(buf[0]), torch.empty_like(buf[0]))

    def run():
        table.step(one, n, out=step)
        paged.append(buf[0], buf[1], kp, vp, step.slots, **sc)
        paged.attention(buf[2], kp, vp, table.table, step.cu_rows, step.kv_lens, dim ** -0.5, max_rows=1, out=out,
                        workspace=ws, **sc)
        paged.read(kp, vp, table.table, step.cu_rows, step.kv_lens, n, out=back, **sc)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            run()
    torch.cuda.current_stream().wait_stream(side)
    for i in range(5):
        for t, h in zip(buf, (hkv, hkv, hq)):
            t.copy_(new(h, n))
        graph.replay() if i != 2 else run()
        torch.cuda.synchronize()
        for x, t in zip(kept, buf):
            x[:] = [torch.cat([old, t[b:b + 1]]) for b, old in enumerate(x)]
        values = [[_stand_for(*_oracle(y, kind), kind, torch.bfloat16).to(DEV) for y in x] for x in kept]
        for b in range(n):
            assert torch.equal(back[0][b], values[0][b][-1]) and torch.equal(back[1][b], values[1][b][-1])
            rows = len(values[0][b])
            pages = [torch.zeros((1, hkv, 4096, dim), device=DEV).bfloat16() for _ in range(2)]
            for p, x in zip(pages, values):
                p[0, :, :rows] = x[b].transpose(0, 1)
            want, tol = _reference(dict(query=buf[2][b:b + 1], k_pages=pages[0], v_pages=pages[1], table=_i32([[0]]),
                                        cu_rows=_i32([0, 1]), kv_lens=_i32([rows]), scaling=dim ** -0.5))
            _within(out[b:b + 1], want, tol)
    assert table.lens.tolist() == [n + 5 for n in lens]


def test_two_streams_at_once():
    cases = [_coded(_case([2000 + 300 * i, 31], [1, 5], 8, 2, 128, 16, "bf16", seed=40 + i), k) for i, k in enumerate(KINDS)]
    want = [paged.attention(**two) for two, _ in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, (two, _) in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                got[i].append(paged.attention(**two))
    torch.cuda.synchronize()
    for w, many in zip(want, got):
        assert all(torch.equal(w, y) for y in many)


def test_pages_made_of_other_types_are_refused():
    with pytest.raises(RuntimeError, match="kind must be"):
        paged.quantized_pages(2, 2, 16, 64, "int8", DEV)
    with pytest.raises(RuntimeError, match="multiple of 32"):
        paged.quantized_pages(2, 2, 16, 40, "fp8", DEV)
    assert _pages(1, 1, 16, 64, torch.bfloat16, 0).dtype == torch.bfloat16

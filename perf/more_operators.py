"""The paged cache in 8 and 4 bits, and attention over a prefix that requests share, as a serving
program calls them, and what they are measured on.

Kinds, by ``case["kind"]``:

* ``store``  -- the K and V rows of a step quantised into their slots (``paged.append`` into pages of
  codes with scales), and tokens of the requests read back as rows (``paged.read``).
* ``attend`` -- the step's rows over quantised pages (``paged.attention`` with scales): single tokens,
  drafts, chunks and whole prompts of requests of different lengths.
* ``shared`` -- requests that continue the tokens of another request, their parent: the step's rows
  gathered by parent (``paged.share_rows``) and the attention that reads a parent's keys once for
  all of them (``paged.attention`` with ``shared``), over 16-bit or quantised pages.

Codes are fp8 (e4m3) or fp4 (e2m1, two to a byte, the even channel in the low half), with one scale
2^(byte - 127) for each 32 channels of a token's head: the smallest, from 2^-100 on, under which the
largest magnitude rounds to a finite code.  A block with an infinity or NaN has the scale byte 255
and reads as NaN.

The inputs are those of the framework's benchmark: 16 or 32 query heads over 8 KV heads (or 8 over
4), K and V from N(0, 1) with four channels scaled by 8, queries from N(0, 1).  The pages of every
request lie in random order in the pool; what a page holds behind its request's last token is left
over from others.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
BLOCK = 32


def listed():
    return [
        # The new K and V rows of eight single tokens, read back: latency only.
        dict(name="store_8_fp8", kind="store", batch=8, tokens=700, new=1, back=1, kv_heads=8, head_dim=128, page=16,
             code="fp8", dtype="bf16"),
        # A chunk of four prompts stored, and their whole histories read back (to move the requests elsewhere).
        dict(name="store_4x2047_fp8", kind="store", batch=4, tokens=9001, new=2047, back=9001, kv_heads=8, head_dim=128,
             page=64, code="fp8", dtype="bf16"),
        # The same in 4 bits with small heads, an odd number of requests and tokens.
        dict(name="store_7x501_fp4", kind="store", batch=7, tokens=6007, new=501, back=6007, kv_heads=4, head_dim=64,
             page=32, code="fp4", dtype="fp16"),
        # One short request's single token: the smallest attention call, latency only.
        dict(name="token_b1_t500_fp8", kind="attend", batch=1, q_heads=16, kv_heads=8, head_dim=128, tokens=500,
             spread=0.0, new=1, chunks=1, page=16, cap=0.0, bias=False, window=0, code="fp8", dtype="bf16"),
        # Single tokens of 32 long requests of different lengths: the ordinary large decode step, 8 bits.
        dict(name="token_b32_t32768_fp8", kind="attend", batch=32, q_heads=32, kv_heads=8, head_dim=128, tokens=32768,
             spread=0.5, new=1, chunks=32, page=64, cap=0.0, bias=False, window=0, code="fp8", dtype="bf16"),
        # The same in 4 bits, an odd number of requests and tokens.
        dict(name="token_b29_t32001_fp4", kind="attend", batch=29, q_heads=32, kv_heads=8, head_dim=128, tokens=32001,
             spread=0.5, new=1, chunks=29, page=32, cap=0.0, bias=False, window=0, code="fp4", dtype="bf16"),
        # Five drafted tokens for each of seven requests, scores capped and biased.
        dict(name="draft5_b7_t9000_fp8", kind="attend", batch=7, q_heads=32, kv_heads=8, head_dim=128, tokens=9000,
             spread=0.7, new=5, chunks=7, page=16, cap=30.0, bias=True, window=0, code="fp8", dtype="fp16"),
        # The last chunk of a long prompt: the largest call.
        dict(name="chunk_2048x65536_fp8", kind="attend", batch=1, q_heads=32, kv_heads=8, head_dim=128, tokens=65536,
             spread=0.0, new=2048, chunks=1, page=64, cap=0.0, bias=False, window=0, code="fp8", dtype="bf16"),
        # A step that mixes one chunk with 15 single tokens under a window, small heads, 4 bits.
        dict(name="mixed_b16_t6000_fp4", kind="attend", batch=16, q_heads=8, kv_heads=4, head_dim=64, tokens=6000,
             spread=0.9, new=509, chunks=1, page=32, cap=0.0, bias=False, window=4096, code="fp4", dtype="bf16"),
        # Four samples of one short prompt: the smallest call, latency only.
        dict(name="shared_4_of_500", kind="shared", parents=1, children=4, alone=0, q_heads=16, kv_heads=8, head_dim=128,
             prefix=500, tokens=40, new=1, page=16, cap=0.0, bias=False, code="none", dtype="bf16"),
        # 64 requests behind one long instruction prompt.
        dict(name="shared_64_of_32768", kind="shared", parents=1, children=64, alone=0, q_heads=32, kv_heads=8,
             head_dim=128, prefix=32768, tokens=600, new=1, page=64, cap=0.0, bias=False, code="none", dtype="bf16"),
        # Three documents, five drafted tokens for each of their requests and of some of nobody's, 8 bits, scores biased.
        dict(name="shared_3x27_drafts_fp8", kind="shared", parents=3, children=27, alone=4, q_heads=32, kv_heads=8,
             head_dim=128, prefix=15013, tokens=901, new=5, page=32, cap=0.0, bias=True, code="fp8", dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


HEADS = [(16, 8, 128), (32, 8, 128), (32, 8, 128), (8, 4, 64), (6, 2, 64), (8, 1, 128)]


def draw(rng):
    """Another case of the same ranges, no larger than the listed ones."""
    kind = rng.choice(["store", "attend", "attend", "shared", "shared"])
    page, half = rng.choice([16, 32, 64, 128]), rng.choice(["bf16", "bf16", "fp16"])
    code = rng.choice(["fp8", "fp8", "fp4"])
    q_heads, kv_heads, head_dim = rng.choice(HEADS)
    if kind == "store":
        tokens = _log(rng, 1, 9001)
        return dict(kind=kind, batch=_log(rng, 1, max(1, 36000 // tokens)), tokens=tokens, new=_log(rng, 1, min(tokens, 2047)),
                    back=_log(rng, 1, tokens), kv_heads=kv_heads, head_dim=head_dim, page=page, code=code, dtype=half)
    if kind == "shared":
        parents, new = rng.randint(1, 4), rng.choice([1, 1, 1, rng.randint(2, 9), _log(rng, 10, 300)])
        children = _log(rng, 1, max(1, min(64, 2048 // new)))
        prefix = _log(rng, 1, 32768)
        # rows x keys of the padded batch stay below the largest listed cases'
        most = max(1, (1 << 29) // (children * new * q_heads))
        return dict(kind=kind, parents=parents, children=children, alone=rng.choice([0, 0, 3]), q_heads=q_heads,
                    kv_heads=kv_heads, head_dim=head_dim, prefix=min(prefix, most),
                    tokens=max(new, _log(rng, 1, min(2000, most))), new=new, page=page, cap=rng.choice([0.0, 0.0, 30.0]),
                    bias=rng.choice([False, False, True]), code=rng.choice(["none", "none", "fp8", "fp4"]), dtype=half)
    form = rng.choice(["token", "token", "draft", "chunk", "prompt", "mixed"])
    tokens = _log(rng, 1, 131072) if form == "token" else _log(rng, 64, 16384)
    new = {"token": 1, "draft": rng.randint(2, 9), "prompt": tokens}.get(form) or min(tokens, _log(rng, 16, 2048))
    if form == "prompt":
        tokens = new = min(tokens, 6000)
    most = max(1, min(32, (1 << 30) // (tokens * max(1, new) * q_heads), (1 << 20) // tokens))
    batch = _log(rng, 1, most)
    return dict(kind=kind, batch=batch, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim, tokens=tokens,
                spread=rng.choice([0.0, 0.3, 0.9]), new=new, chunks=1 if form == "mixed" else batch, page=page,
                cap=rng.choice([0.0, 0.0, 30.0, 50.0]), bias=rng.choice([False, False, True]),
                window=rng.choice([0, 0, _log(rng, 8, tokens + 8)]), code=code, dtype=half)


# -- inputs ---------------------------------------------------------------------


def _lengths(case):
    """(tokens in the cache, rows of the step) of every request, by the case alone: lengths spread below
    ``tokens``, ``new`` rows for the first ``chunks`` requests and one for the others."""
    less = case.get("spread", 0.3)
    kv = [max(1, int(case["tokens"] * (1.0 - less * (b * 0.6180339887 % 1.0)))) for b in range(case["batch"])]
    rows = [min(n, case["new"]) if b < case.get("chunks", case["batch"]) else 1 for b, n in enumerate(kv)]
    return kv, rows


def _family(case):
    """(parent, tokens, rows) of every request of a shared case: first the parents, which do not step, then their
    children in turn, then requests of nobody."""
    par = [-1] * case["parents"] + [i % case["parents"] for i in range(case["children"])] + [-1] * case["alone"]
    kv = [max(1, case["prefix"] - case["prefix"] // 5 * i) for i in range(case["parents"])]
    kv += [max(1, int(case["tokens"] * (1.0 - 0.9 * (b * 0.6180339887 % 1.0)))) for b in range(case["children"] + case["alone"])]
    rows = [0] * case["parents"] + [min(n, case["new"]) for n in kv[case["parents"]:]]
    return par, kv, rows


def _gen(seed, salt):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 64 + salt)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _pages_of(lens, page, seed):
    """A page table for requests of ``lens`` tokens, their pages in random order, and the pool's size."""
    need = [-(-n // page) for n in lens]
    pool = sum(need) + 3
    order = torch.randperm(pool, generator=_gen(seed, 1), device=DEV).to(torch.int32)
    at = torch.arange(max(need), device=DEV)[None, :]
    need_t = torch.tensor(need, device=DEV)[:, None]
    first = need_t.cumsum(0) - need_t
    return torch.where(at < need_t, order[(first + at).clamp(max=pool - 1)], -1), pool


def _values(shape, dtype, seed, salt):
    g = _gen(seed, salt)
    x = torch.randn(shape, generator=g, device=DEV, dtype=torch.float32 if math.prod(shape) < 1 << 28 else dtype)
    x[..., torch.randperm(shape[-1], generator=g, device=DEV)[:4]] *= 8.0
    return x.to(dtype)


def _cache(case, pool, seed, salt):
    """A layer's pages of K or V and their scales (None for 16-bit pages), full of other tokens."""
    shape = (pool, case["kv_heads"], case["page"], case["head_dim"])
    x = _values(shape, DTYPES[case["dtype"]], seed, salt)
    if case["code"] == "none":
        return x, None
    some = max(1, (1 << 27) // math.prod(shape[1:]))
    parts = [_quantise(y, case["code"]) for y in x.split(some)]
    return torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts])


def prepare(case, seed):
    dtype, dim = DTYPES[case["dtype"]], case["head_dim"]
    if case["kind"] == "shared":
        par, kv, rows = _family(case)
        slot = torch.randperm(len(kv), generator=torch.Generator().manual_seed(int(seed))).tolist()   # requests in any order
        back = sorted(range(len(kv)), key=slot.__getitem__)
        par, kv, rows = [slot[par[b]] if par[b] >= 0 else -1 for b in back], [kv[b] for b in back], [rows[b] for b in back]
    else:
        par, (kv, rows) = None, _lengths(case)
    table, pool = _pages_of(kv, case["page"], seed)
    k, ks = _cache(case, pool, seed, 2)
    v, vs = _cache(case, pool, seed, 3)
    state = dict(case=case, table=table, kv_lens=_ints(kv), cu=_ints([0] + rows).cumsum(0).to(torch.int32), k_pages=k,
                 k_scales=ks, v_pages=v, v_scales=vs, rows=sum(rows), max_rows=max(rows))
    if case["kind"] == "store":
        new = (sum(rows), case["kv_heads"], dim)
        back = [min(n, case["back"]) for n in kv]
        at = torch.cat([torch.arange(n - m, n, device=DEV) for n, m in zip(kv, rows)])
        of = torch.repeat_interleave(torch.arange(len(kv), device=DEV), torch.tensor(rows, device=DEV))
        state["slots"] = table[of, at // case["page"]].long() * case["page"] + at % case["page"]
        if len(state["slots"]) > 3:
            state["slots"][1] = -1   # padding
        state.update(k=_values(new, dtype, seed, 4), v=_values(new, dtype, seed, 5), back=sum(back),
                     back_cu=_ints([0] + back).cumsum(0).to(torch.int32))
        return state
    state["q"] = torch.randn((sum(rows), case["q_heads"], dim), generator=_gen(seed, 4), device=DEV).to(dtype)
    state["scaling"], state["slopes"], state["first"] = dim ** -0.5, None, None
    if case["bias"]:   # the usual geometric slopes
        state["slopes"] = torch.exp2(-8.0 * (torch.arange(case["q_heads"], device=DEV) + 1) / case["q_heads"]).float()
    if par is not None:
        state["parents"], state["lens"] = _ints(par), state["kv_lens"].clone()
    elif case["window"]:
        at = torch.cat([torch.arange(n - m, n, device=DEV) for n, m in zip(kv, rows)])
        state["first"] = (at - (case["window"] - 1)).to(torch.int32)
    return state


# -- the operators ----------------------------------------------------------------


def run(state):
    if own:
        return {"store": _own_store, "attend": _own_attend, "shared": _own_shared}[state["case"]["kind"]](state)
    return {"store": _plain_store, "attend": _plain_attend, "shared": _plain_shared}[state["case"]["kind"]](state)


def _own_store(s):
    from kv_cache_amd import paged

    paged.append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["slots"], k_scales=s["k_scales"], v_scales=s["v_scales"])
    return paged.read(s["k_pages"], s["v_pages"], s["table"], s["back_cu"], s["kv_lens"], s["back"],
                      k_scales=s["k_scales"], v_scales=s["v_scales"], dtype=DTYPES[s["case"]["dtype"]])


def _own_attend(s):
    from kv_cache_amd import paged

    return paged.attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["cu"], s["kv_lens"], s["scaling"],
                           max_rows=s["max_rows"], softcap=s["case"]["cap"], slopes=s["slopes"], first_keys=s["first"],
                           k_scales=s["k_scales"], v_scales=s["v_scales"])


def _own_shared(s):
    from kv_cache_amd import paged

    shared = paged.share_rows(s["parents"], s["cu"], s["kv_lens"], s["lens"], s["rows"])
    out = paged.attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["cu"], s["kv_lens"], s["scaling"],
                          max_rows=s["max_rows"], softcap=s["case"]["cap"], slopes=s["slopes"], shared=shared,
                          k_scales=s["k_scales"], v_scales=s["v_scales"])
    return out, shared.positions


# The largest values that a code and the rows' dtype both hold, the largest code, its exponent, and the fraction of
# the next power of two up to which a magnitude still rounds to it (464 = 0.90625 * 2^9, 7 = 0.875 * 2^3).
LIMITS = {("fp8", torch.bfloat16): 1.875 * 2.0 ** 127, ("fp8", torch.float16): 61440.0,
          ("fp4", torch.bfloat16): 1.5 * 2.0 ** 127, ("fp4", torch.float16): 49152.0}
CODES = {"fp8": (448.0, 9, 0.90625), "fp4": (6.0, 3, 0.875)}


def _power(e):
    """2^e in 32 bits, from its bits: the GPU's exp2 may be off by one of them, which moves halves."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _quantise(x, code):
    """(codes, scale bytes) of values [..., dim]."""
    most, exponent, share = CODES[code]
    y = x.float().reshape(*x.shape[:-1], -1, BLOCK)
    odd = ~torch.isfinite(y).all(-1, keepdim=True)
    y = torch.where(odd, 0.0, y.clamp(-LIMITS[code, x.dtype], LIMITS[code, x.dtype]))
    part, power = torch.frexp(y.abs().amax(-1, keepdim=True))
    e = (power - exponent + (part > share).to(power.dtype)).clamp(min=-100)
    e = torch.where(part == 0, -100, e)
    y = (y * _power(-e)).clamp(-most, most).reshape(x.shape)
    scales = torch.where(odd, 255, e + 127).squeeze(-1).to(torch.uint8)
    if code == "fp8":
        return y.to(torch.float8_e4m3fn), scales
    a = y.abs()   # half-way magnitudes go to the even code
    c = (a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
    c = c.to(torch.uint8) | (torch.signbit(y).to(torch.uint8) << 3)
    return c[..., 0::2] | (c[..., 1::2] << 4), scales


def _dequantise(codes, scales):
    """The values that codes stand for, in 32 bits."""
    if scales is None:
        return codes.float()
    if codes.dtype == torch.uint8:
        steps = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
        steps = torch.cat([steps, -steps])
        x = steps[torch.stack([codes & 15, codes >> 4], -1).long()].reshape(*codes.shape[:-1], -1)
    else:
        x = codes.float()
    scale = torch.where(scales == 255, math.nan, _power(scales.clamp(max=254).int() - 127))
    return (x.reshape(*scales.shape, BLOCK) * scale[..., None]).reshape(x.shape)


def _plain_store(s):
    page, code, at = s["case"]["page"], s["case"]["code"], s["slots"]
    kept = at >= 0
    row = torch.arange(s["back"], device=DEV)
    cu, kv = s["back_cu"].long(), s["kv_lens"].long()
    b = torch.searchsorted(cu, row, right=True) - 1
    pos = kv[b] - (cu[b + 1] - row)
    slot = s["table"][b, pos // page].long() * page + pos % page
    out = []
    for new, pages, scales in ((s["k"], s["k_pages"], s["k_scales"]), (s["v"], s["v_pages"], s["v_scales"])):
        codes, bytes_ = _quantise(new[kept], code)
        pages.view(torch.uint8)[at[kept] // page, :, at[kept] % page] = codes.view(torch.uint8)
        scales[at[kept] // page, :, at[kept] % page] = bytes_
        back = pages.view(torch.uint8)[slot // page, :, slot % page].view(pages.dtype)
        out.append(_dequantise(back, scales[slot // page, :, slot % page]).to(new.dtype))
    return tuple(out)


def _keys(pages, scales, ids):
    """[requests, heads, tokens, dim] in 32 bits of the pages ``ids`` [requests, width]."""
    x = _dequantise(pages.view(torch.uint8)[ids].view(pages.dtype) if scales is not None else pages[ids],
                    None if scales is None else scales[ids])
    n, width, heads, page, dim = x.shape
    return x.transpose(1, 2).reshape(n, heads, width * page, dim)


def _weigh(s, q, k, v, pos, key, seen):
    """(maximum, sum, weighted values) of rows q [b, kv heads, G, rows, dim] over keys: positions ``pos`` [b, rows] of
    the rows and ``key`` of the keys, which of them are ``seen`` [b, rows, keys]."""
    case = s["case"]
    n, heads, group, rows, dim = q.shape
    score = torch.matmul(q.reshape(n, heads, group * rows, dim), k.transpose(2, 3)).mul_(s["scaling"])
    score = score.view(n, heads, group, rows, -1)
    if case["cap"]:
        score = torch.tanh_(score.div_(case["cap"])).mul_(case["cap"])
    if s["slopes"] is not None:
        away = (pos[:, :, None] - key).abs().float()[:, None, None]
        score -= s["slopes"].view(1, heads, group, 1, 1) * away
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    score = score.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = score.sum(-1, keepdim=True)
    o = torch.matmul(score.view(n, heads, group * rows, -1), v).view(n, heads, group, rows, dim)
    return top, total, o


def _rows_of(q, row, heads):
    """[b, kv heads, G, rows, dim] in 32 bits of the rows ``row`` [b, rows]."""
    n, most = row.shape
    return q.float()[row].reshape(n, most, heads, -1, q.shape[2]).permute(0, 2, 3, 1, 4)


def _plain_attend(s):
    case, q, page = s["case"], s["q"], s["case"]["page"]
    cu, kv = s["cu"].long(), s["kv_lens"].long()
    rows = cu[1:] - cu[:-1]
    ids = s["table"].clamp(min=0).long()
    j = torch.arange(ids.shape[1] * page, device=DEV)
    i = torch.arange(s["max_rows"], device=DEV)[None, :]
    row = (cu[:-1, None] + i).clamp(max=q.shape[0] - 1)
    real = i < rows[:, None]
    pos = (kv - rows)[:, None] + i
    seen = (j <= pos[:, :, None]) & real[:, :, None]
    if s["first"] is not None:
        seen &= j >= s["first"].long()[row][:, :, None]
    k, v = _keys(s["k_pages"], s["k_scales"], ids), _keys(s["v_pages"], s["v_scales"], ids)
    _, total, o = _weigh(s, _rows_of(q, row, case["kv_heads"]), k, v, pos, j, seen)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 3, 1, 2, 4).reshape(-1, *q.shape[1:])
    out = torch.empty_like(q)
    out[row[real]] = o[real.reshape(-1)].to(q.dtype)
    return out


def _plain_shared(s):
    case, q, page, heads = s["case"], s["q"], s["case"]["page"], s["case"]["kv_heads"]
    cu, own_lens, par, lens = s["cu"].long(), s["kv_lens"].long(), s["parents"].long(), s["lens"].long()
    rows = cu[1:] - cu[:-1]
    before = torch.where(par >= 0, lens[par.clamp(min=0)], 0)
    b = torch.repeat_interleave(torch.arange(len(rows), device=DEV), rows, output_size=s["rows"])
    positions = before[b] + own_lens[b] - (cu[b + 1] - torch.arange(s["rows"], device=DEV))
    most, width = s["max_rows"], -(-case["tokens"] // page)
    # their own keys, request by request (parents' rows are none; their length in own keys does not count)
    step = (rows > 0).nonzero().squeeze(1)
    ids = s["table"][step, :width].clamp(min=0).long()
    i = torch.arange(most, device=DEV)[None, :]
    row = (cu[:-1][step, None] + i).clamp(max=q.shape[0] - 1)
    real = i < rows[step, None]
    j = torch.arange(ids.shape[1] * page, device=DEV)
    pos = (own_lens - rows)[step, None] + i
    k, v = _keys(s["k_pages"], s["k_scales"], ids), _keys(s["v_pages"], s["v_scales"], ids)
    mine = _weigh(s, _rows_of(q, row, heads), k, v, pos, j, (j <= pos[:, :, None]) & real[:, :, None])
    mine = [x.permute(0, 3, 1, 2, 4).reshape(len(step) * most, *q.shape[1:2], -1)[real.reshape(-1)] for x in mine]
    # the parents' keys, all rows of a parent together
    family, of = torch.unique(par, return_inverse=True)   # -1 first, if there is one
    heirs = torch.zeros(len(family), dtype=torch.long, device=DEV).index_add(0, of, rows)
    order = torch.argsort(of[b], stable=True)
    start = heirs.cumsum(0) - heirs
    i = torch.arange(s["rows"], device=DEV)[None, :]
    row = order[(start[:, None] + i).clamp(max=s["rows"] - 1)]
    real = (i < heirs[:, None]) & (family >= 0)[:, None]
    ids = s["table"][family.clamp(min=0)].clamp(min=0).long()
    n = torch.where(family >= 0, lens[family.clamp(min=0)], 0)
    j = torch.arange(ids.shape[1] * page, device=DEV)
    k, v = _keys(s["k_pages"], s["k_scales"], ids), _keys(s["v_pages"], s["v_scales"], ids)
    seen = (j < n[:, None])[:, None, :] & real[:, :, None]
    theirs = _weigh(s, _rows_of(q, row, heads), k, v, positions[row], j, seen)
    full = [torch.full((s["rows"], q.shape[1], 1), -math.inf, device=DEV), torch.zeros((s["rows"], q.shape[1], 1), device=DEV),
            torch.zeros(q.shape, device=DEV)]
    for x, y in zip(full, theirs):
        x[row[real]] = y.permute(0, 3, 1, 2, 4).reshape(-1, *x.shape[1:])[real.reshape(-1)]
    top = torch.maximum(mine[0], full[0])
    a, c = (mine[0] - top).exp(), (full[0] - top).exp()
    out = (mine[2] * a + full[2] * c) / (mine[1] * a + full[1] * c)
    return out.to(q.dtype), positions.to(torch.int32)


# -- what a pass cannot do without ------------------------------------------------


def _token_bytes(case):
    """Bytes of one token's K and V of a layer."""
    per = {"none": 2.0, "fp8": 1.0 + 1.0 / BLOCK, "fp4": 0.5 + 1.0 / BLOCK}[case["code"]]
    return 2 * case["kv_heads"] * case["head_dim"] * per


def work(case):
    if case["kind"] == "store":
        kv, rows = _lengths(case)
        back = sum(min(n, case["back"]) for n in kv)
        wide = 4 * case["kv_heads"] * case["head_dim"]
        return {"bytes": (sum(rows) + back) * (wide + _token_bytes(case)), "flops": 0}
    dim = case["head_dim"]
    if case["kind"] == "shared":
        par, kv, rows = _family(case)
        keys, total = sum(kv), sum(rows)
        pairs = sum(m * (n if p < 0 else n + kv[p]) - m * (m - 1) // 2 for p, n, m in zip(par, kv, rows))
    else:
        kv, rows = _lengths(case)
        less = case["window"] or case["tokens"]
        keys, total = sum(min(n, m + less - 1) for n, m in zip(kv, rows)), sum(rows)
        pairs = sum(min(p + 1, less) for n, m in zip(kv, rows) for p in range(n - m, n))
    return {"bytes": keys * _token_bytes(case) + total * case["q_heads"] * dim * 4, "flops": 4 * dim * case["q_heads"] * pairs}


# -- from the definitions, in 64 bits ---------------------------------------------


def _table_of(code):
    """What each code stands for, from its bits: sign, exponent, fraction."""
    bits, man, bias = {"fp8": (8, 3, 7), "fp4": (4, 1, 1)}[code]
    got = []
    for c in range(1 << bits):
        sign, low = c >> (bits - 1), c & ((1 << (bits - 1)) - 1)
        e, f = low >> man, low & ((1 << man) - 1)
        x = (f / 2 ** man) * 2.0 ** (1 - bias) if e == 0 else (1 + f / 2 ** man) * 2.0 ** (e - bias)
        got.append(math.nan if code == "fp8" and low == 127 else -x if sign else x)
    return torch.tensor(got, dtype=torch.float64, device=DEV)


def _double_power(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _doubles(pages, scales, ids, head, case):
    """One head's tokens of the pages ``ids``, in 64 bits."""
    dim = case["head_dim"]
    if scales is None:
        return pages[ids, head].double().reshape(-1, dim)
    raw = pages.view(torch.uint8)[ids, head].reshape(-1, pages.shape[-1]).long()
    if case["code"] == "fp4":
        raw = torch.stack((raw % 16, raw // 16), 2).reshape(-1, dim)
    x = _table_of(case["code"])[raw]
    return x * _double_power(scales[ids, head].reshape(-1, dim // BLOCK).double() - 127).repeat_interleave(BLOCK, 1)


def _exact_store(case, s):
    """What is nearest to each value under its block's scale: by search over all codes."""
    codes = _table_of(case["code"])
    codes = codes[~torch.isnan(codes)].unique()
    out = []
    kv, rows = _lengths(case)
    for new, pages, scales in ((s["k"], s["k_pages"], s["k_scales"]), (s["v"], s["v_pages"], s["v_scales"])):
        x = new.double().reshape(*new.shape[:2], -1, BLOCK)
        largest = x.abs().amax(-1, keepdim=True)
        edge = 464.0 if case["code"] == "fp8" else 7.0
        e = torch.ceil(torch.log2(largest.clamp(min=2.0 ** -120) / edge))
        e = torch.where(largest <= edge * _double_power(e - 1), e - 1, e).clamp(min=-100)
        e = torch.where(largest > edge * _double_power(e), e + 1, e)
        scale = _double_power(e)
        y = x / scale
        hi = torch.searchsorted(codes, y.contiguous()).clamp(1, len(codes) - 1)
        lo = hi - 1
        up, down = codes[hi] - y, y - codes[lo]
        # positions count from zero outwards, so that even fractions are even positions
        even = ((hi - len(codes) // 2) % 2) == 0
        y = torch.where((up < down) | ((up == down) & even), codes[hi], codes[lo])
        stored = (y * scale).reshape(new.shape)
        out.append([])
        start = 0
        for b, (n, m) in enumerate(zip(kv, rows)):
            ids = s["table"][b, : -(-n // case["page"])].long()
            whole = torch.stack([_doubles(pages, scales, ids, h, case)[:n] for h in range(case["kv_heads"])], 1)
            kept = (s["slots"][start:start + m] >= 0)[:, None, None]
            whole[n - m:] = torch.where(kept, stored[start:start + m], whole[n - m:])
            out[-1].append(whole[n - min(n, case["back"]):])
            start += m
    return tuple(torch.cat(x) for x in out)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "store":
        return _exact_store(case, s)
    heads, group, page = case["kv_heads"], case["q_heads"] // case["kv_heads"], case["page"]
    cu, kv = s["cu"].tolist(), s["kv_lens"].tolist()
    par = s["parents"].tolist() if case["kind"] == "shared" else [-1] * len(kv)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    for h in range(heads):
        kept = {}
        for b, n in enumerate(kv):
            m = cu[b + 1] - cu[b]
            if m == 0:
                continue
            both = []
            for a in ([par[b]] if par[b] >= 0 else []) + [b]:
                if a not in kept:
                    ids = s["table"][a, : -(-kv[a] // page)].long()
                    kept[a] = [_doubles(s[x + "_pages"], s[x + "_scales"], ids, h, case)[:kv[a]] for x in "kv"]
                both.append(kept[a])
            if par[b] >= 0 or len(kept) > 1:
                kept.pop(b)
            k, v = (torch.cat(x) for x in zip(*both))
            total = k.shape[0]
            j = torch.arange(total, device=DEV)
            for at in range(0, m, 1024):
                r = torch.arange(at, min(m, at + 1024), device=DEV)
                p = (total - m + r)[:, None]
                hide = j > p
                if s["first"] is not None:
                    hide |= j < s["first"][cu[b] + r].long()[:, None]
                for g in range(h * group, (h + 1) * group):
                    x = torch.mm(s["q"][cu[b] + r, g].double(), k.t()) * s["scaling"]
                    if case["cap"]:
                        x = case["cap"] * torch.tanh(x / case["cap"])
                    if s["slopes"] is not None:
                        x = x - s["slopes"][g].double() * (p - j).abs()
                    x[hide] = -math.inf
                    out[cu[b] + r, g] = torch.mm(torch.softmax(x, -1), v)
    return (out, None) if case["kind"] == "shared" else out

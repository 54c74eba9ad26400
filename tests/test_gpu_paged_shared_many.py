"""Attention over shared prefixes at the sizes that choose its other paths:
two requests a lane (65 to 128), rounds of 256 requests (more than 128), rows
placed by a launch of their own (more than 4096), eight (row, head)s a joining
workgroup (more than 16384).  Against 64 bits, within the bound of the paged
attention."""

import random

import pytest
import torch

from kv_cache_amd import paged
from test_gpu_paged import DEV, _case, _i32, _reference, _within
from test_gpu_paged_codes import _coded
from test_gpu_paged_shared import _check, _whole

pytestmark = pytest.mark.gpu


def _requests(n, parents_at, seed, most=40):
    """n requests, their parents at the given places; half of them no one's children, some without rows."""
    rng = random.Random(seed)
    parents = [rng.choice([-1, n + 3, *parents_at, *parents_at, *parents_at]) for _ in range(n)]
    kv = [rng.randint(1, most) for _ in range(n)]
    rows = [min(k, rng.choice([0, 1, 1, 1, 3])) for k in kv]
    return parents, kv, rows


@pytest.mark.parametrize("kind", ["none", "fp8"])
@pytest.mark.parametrize("n", [65, 100, 127, 128, 129])
def test_two_requests_a_lane(n, kind):
    parents, kv, rows = _requests(n, (3, 64, n - 1), n)
    for p, k in ((3, 5000), (64, 700), (n - 1, 65)):       # split keys, in the lane's first and second request
        parents[p], kv[p], rows[p] = -1, k, 0
    rows[64] = 2
    _check(parents, kv, rows, 4, 2, 128, 16, "bf16", kind, seed=n, max_rows=3)


@pytest.mark.parametrize("n,dim,kind", [(256, 64, "none"), (257, 128, "none"), (300, 64, "fp4"), (300, 128, "fp8"), (600, 128, "none"),
                                        (600, 64, "fp8")])
def test_rounds_of_requests(n, dim, kind):
    # parents and heirs in different rounds of 256; the longest of both kinds behind a round's end
    places = sorted({0, 255, n - 1, n // 2, min(n - 2, 256)})
    parents, kv, rows = _requests(n, places, n + dim)
    for i, p in enumerate(places):
        parents[p], kv[p], rows[p] = -1, (3000, 1, 63, 257, 1500)[i], i % 2
    alone = n - 3                                          # its own keys are split
    parents[alone], kv[alone], rows[alone] = -1, 4000, 3
    _check(parents, kv, rows, 4, 2, dim, 16, "bf16", kind, seed=n, max_rows=3)


def test_all_behind_the_last_request():
    # 700 heirs of one parent: tiles of rows beside token tiles, both split
    n = 701
    kv, rows = [1 + b % 5 for b in range(n)], [b % 4 != 3 for b in range(n)]
    kv[-1], rows[-1] = 2500, 0
    _check([n - 1] * (n - 1) + [-1], kv, [int(r) for r in rows], 8, 2, 64, 16, "fp16", seed=70, max_rows=1)


def test_as_many_requests_as_there_are():
    n = 4096
    rng = random.Random(9)
    parents = [rng.choice([7, 2000, 4095, -1]) for _ in range(n)]
    kv, rows = [1 + b % 3 for b in range(n)], [int(b % 5 != 1) for b in range(n)]
    for p, k in ((7, 900), (2000, 33), (4095, 300)):
        parents[p], kv[p], rows[p] = -1, k, 0
    _check(parents, kv, rows, 2, 1, 64, 16, "bf16", seed=71, max_rows=1)


@pytest.mark.parametrize("dim,kind", [(128, "none"), (64, "none"), (128, "fp8")])
def test_many_rows_and_heads(dim, kind):
    # 3 children of 300 rows, 32 heads: 28 800 (row, head)s, a parent of several chunks
    _check([-1, 0, 0, 0], [2000, 300, 310, 299], [0, 300, 300, 297], 32, 8, dim, 16, "bf16", kind, seed=72)


@pytest.mark.parametrize("form", [{}, {"softcap": 5.0}])
def test_more_rows_than_one_launch_places(form):
    # 4600 rows in all, heirs of two parents in turn; one child has more rows than tokens
    kv, rows = [1500, 950, 900, 1300, 70, 700, 1], [0, 950, 900, 1300, 0, 1400, 50]
    parents = [-1, 0, 4, 0, -1, 4, 0]
    out = _check(parents, kv, rows, 8, 2, 64, 16, "bf16", seed=73, **form)
    assert (out[3150:3850] == 0).all() and (out[4550:4599] == 0).all()


def test_rows_out_of_order_write_nothing_outside():
    """cu_rows that does not ascend: what is around the output and the workspace stays as it was."""
    total, n = 30, 3
    c = _case([50, 60, 700], [10, 10, 10], 8, 2, 128, 16, "bf16", seed=17)
    ws = paged.attention_workspace(total, total, n, c["table"].shape[1], 16, 8, 2, 128, DEV, shared=True)
    words = ws.numel()
    room = torch.full((words + 4096,), 3.0, device=DEV)
    held = torch.full((total + 8, 8, 128), 7.0, dtype=torch.bfloat16, device=DEV)
    for cu in ([0, 30, 0, 30], [30, 0, 30, 0], [-5, 10, 20, 1000], [10, 10, 10, 25]):
        plan = paged.share_rows(_i32([2, 0, 1]), _i32(cu), c["kv_lens"], c["kv_lens"], total)
        paged.attention(**{**c, "cu_rows": _i32(cu)}, shared=plan, out=held[4:-4], workspace=room[:words])
        assert (room[words:] == 3.0).all()
        assert (held[:4] == 7.0).all() and (held[-4:] == 7.0).all()
    assert (held[4:14] != 7.0).any()


def test_the_workspace_of_16_bit_pages_serves_codes():
    """A call over codes in a workspace of exactly attention_workspace's size, with nothing written behind it."""
    for kind, rows in (("fp8", 1), ("fp4", 1), ("fp4", 7), ("fp8", 40)):
        kv = [3000, 900, 2500, 40, 700]
        c, ref = _coded(_case(kv, [rows] * 5, 8, 2, 64, 16, "bf16", seed=18), kind)
        ws = paged.attention_workspace(5 * rows, rows, 5, c["table"].shape[1], 16, 8, 2, 64, DEV)
        room = torch.full((ws.numel() + 4096,), float("nan"), device=DEV)
        want, tol = _reference(ref)
        _within(paged.attention(**c, max_rows=rows, workspace=room[:ws.numel()]), want, tol)
        assert torch.isnan(room[ws.numel():]).all()


def test_a_captured_step_of_many_requests():
    """300 children in a replayed step, each replay against the eager call: the plan's launches and both of the attention."""
    n = 301
    rng = random.Random(4)
    kv = [700] + [rng.randint(1, 30) for _ in range(n - 1)]
    c = _case(kv, [0] + [1] * (n - 1), 8, 2, 64, 16, "bf16", seed=74)
    parents = _i32([-1] + [0] * (n - 1))
    shared = paged.SharedRows(n, n - 1, DEV)
    ws = paged.attention_workspace(n - 1, 1, n, c["table"].shape[1], 16, 8, 2, 64, DEV, shared=True)
    out = torch.empty_like(c["query"])

    def run(to, plan, work):
        paged.share_rows(parents, c["cu_rows"], c["kv_lens"], c["kv_lens"], n - 1, out=plan)
        return paged.attention(**c, max_rows=1, shared=plan, out=to, workspace=work)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            run(out, shared, ws)
    torch.cuda.current_stream().wait_stream(side)
    lens = torch.tensor(kv, device=DEV)
    for i in range(6):
        c["query"].copy_(torch.randn_like(c["query"].float()))
        c["kv_lens"].copy_((lens - (i * torch.arange(n, device=DEV)) % lens).int())     # shorter ones, 1 at least
        out.fill_(7.0)
        graph.replay()
        want = run(torch.empty_like(out), paged.SharedRows(n, n - 1, DEV), None)
        assert torch.equal(out, want)
    k = c["kv_lens"].tolist()
    whole, _ = _whole(c, [-1] + [0] * (n - 1), k)
    _within(out, *_reference(whole))


@pytest.mark.parametrize("hq,hkv,dim,kind", [(64, 1, 64, "none"), (128, 1, 128, "fp8"), (16, 16, 64, "fp4"), (33, 1, 128, "none")])
def test_heads_of_a_kv_head(hq, hkv, dim, kind):
    # more heads a KV head than a token tile has rows; none shared
    _check([-1, 0, 0, 5, 0, -1], [700, 9, 40, 33, 1, 90], [0, 1, 7, 2, 1, 3], hq, hkv, dim, 16, "bf16", kind, seed=75)

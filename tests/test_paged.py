"""Paged K/V cache on the CPU: the C entry points' refusals (no kernel is
launched), the size function, and the wrappers' checks."""

import ctypes

import pytest
import torch

from kv_cache_amd import _lib, paged

lib = _lib.load()
P = ctypes.c_void_p(256)
S2, S3 = _lib.strides(256, 64), _lib.strides(4096, 1024, 64)


def _plan(table=P, ld=8, requests=2, width=8, pages=16, page=16, rows=4, padded=0, new=P):
    return lib.qkv_paged_plan(new, table, ld, P, P, P, requests, width, pages, page, rows, padded, P, P, P, P, P, None)


def _release(keep=P, ld=8, requests=2, width=8, pages=16, page=16):
    return lib.qkv_paged_release(keep, P, ld, P, P, P, requests, width, pages, page, None)


def _append(key=P, kp=P, ks=S3, pages=4, page=16, heads=4, dim=64, rows=3, slots=P):
    return lib.qkv_paged_append(key, S2, P, S2, kp, ks, P, S3, pages, page, heads, dim, slots, rows, None)


def _attend(q=P, kp=P, ks=S3, pages=4, page=16, ld=8, width=8, requests=2, rows=4, max_rows=4, hq=4, hkv=4, dim=64,
            scaling=1.0, cap=0.0, ws=P, ws_bytes=0, out=P, os=S2, dtype=0):
    return lib.qkv_paged_attention(q, S2, kp, P, ks, pages, page, P, ld, width, requests, P, P, rows, max_rows,
                                   hq, hkv, dim, scaling, cap, None, None, None, ws, ws_bytes, out, os, dtype, None)


NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("call,msg", [
    (lambda: _plan(new=None), "null pointer"), (lambda: _plan(table=None), "null pointer"),
    (lambda: _plan(ld=7), "bad sizes"), (lambda: _plan(requests=0), "bad sizes"), (lambda: _plan(pages=0), "bad sizes"),
    (lambda: _plan(rows=0), "bad sizes"), (lambda: _plan(rows=5, padded=2), "requests * padded"),
    (lambda: _plan(page=24), "power of two"), (lambda: _plan(page=8), "power of two"),
    (lambda: _plan(page=8192), "power of two"), (lambda: _plan(requests=4097), "at most 4096 requests"),
    (lambda: _plan(pages=(1 << 20) + 1), "at most 1048576 pages"), (lambda: _plan(rows=(1 << 20) + 1), "at most 1048576 rows"),
    (lambda: _plan(width=(1 << 26) + 1, ld=1 << 27), "2^30"),
    (lambda: _release(keep=None), "null pointer"), (lambda: _release(width=9), "bad sizes"),
    (lambda: _release(page=17), "power of two"),
    (lambda: _append(key=None), "null pointer"), (lambda: _append(slots=None), "null pointer"),
    (lambda: _append(rows=-1), "bad sizes"), (lambda: _append(dim=60), "multiple of 8"),
    (lambda: _append(page=15), "power of two"), (lambda: _append(kp=ctypes.c_void_p(264)), "16-byte aligned"),
    (lambda: _append(ks=_lib.strides(4096, 1024, 60)), "16-byte aligned"),
    (lambda: _attend(q=None), "null pointer"), (lambda: _attend(out=None), "null pointer"),
    (lambda: _attend(dtype=2), "is not bf16"), (lambda: _attend(dtype=9), "is not bf16"),
    (lambda: _attend(dim=96), "unsupported sizes"), (lambda: _attend(page=20), "unsupported sizes"),
    (lambda: _attend(hq=6), "unsupported sizes"), (lambda: _attend(hq=129, hkv=1), "unsupported sizes"),
    (lambda: _attend(ld=7), "unsupported sizes"), (lambda: _attend(rows=-1), "unsupported sizes"),
    (lambda: _attend(scaling=0.0), "scaling must be in"), (lambda: _attend(scaling=-1.0), "scaling must be in"),
    (lambda: _attend(scaling=NAN), "scaling must be in"), (lambda: _attend(scaling=INF), "scaling must be in"),
    (lambda: _attend(cap=-1.0), "softcap"), (lambda: _attend(cap=NAN), "softcap"), (lambda: _attend(cap=INF), "softcap"),
    (lambda: _attend(scaling=1e-30), "scaling must be in"), (lambda: _attend(cap=1e-30), "softcap"),
    (lambda: _attend(width=(1 << 26) + 1, ld=1 << 27), "unsupported sizes"),
    (lambda: _attend(kp=ctypes.c_void_p(264)), "16-byte aligned"), (lambda: _attend(out=ctypes.c_void_p(260)), "16-byte aligned"),
    (lambda: _attend(os=_lib.strides(256, 60)), "16-byte aligned"),
    (lambda: _attend(ks=_lib.strides(4096, 1020, 64)), "16-byte aligned"),
    (lambda: _attend(ks=_lib.strides(4096, 1024, (1 << 26) + 8)), "within 2^30"),
    (lambda: _attend(width=100, ld=100), "workspace"),
    (lambda: _attend(width=100, ld=100, ws=ctypes.c_void_p(264), ws_bytes=1 << 40), "workspace"),
])
def test_refusals(call, msg):
    assert call() in (-1, -3)
    assert msg in lib.qkv_last_error().decode()


def test_nothing_to_do():
    assert _append(rows=0, key=None, slots=None) == 0
    assert _attend(rows=0, q=None, out=None) == 0


def test_workspace_bytes():
    f = lib.qkv_paged_attention_workspace_bytes
    assert f(32, 1, 32, 32, 16, 32, 8, 128) == 0          # 512 keys a request at most: never split
    assert f(4, 4, 2, 8, 16, 6, 4, 64) == -1
    assert f(4, 4, 2, 8, 16, 4, 4, 96) == -1
    small, large = f(1, 1, 1, 64, 16, 16, 8, 128), f(32, 1, 32, 2048, 16, 32, 8, 128)
    assert 0 < small < large
    # more of anything never needs less, so that one workspace serves every smaller call
    base = dict(rows=32, max_rows=4, requests=32, width=128, page=16, q_heads=32, kv_heads=8, head_dim=128)
    for name, values in (("rows", (1, 4, 32, 64, 1000, 10**6)), ("requests", (1, 3, 32, 200)), ("width", (8, 17, 64, 1000, 8192))):
        sizes = [f(*{**base, name: v}.values()) for v in values]
        assert sizes == sorted(sizes), (name, sizes)


def _tensors(rows=4, requests=2):
    return dict(query=torch.zeros(rows, 4, 64, dtype=torch.bfloat16), k_pages=torch.zeros(4, 4, 16, 64, dtype=torch.bfloat16),
                v_pages=torch.zeros(4, 4, 16, 64, dtype=torch.bfloat16), table=torch.zeros(requests, 8, dtype=torch.int32),
                cu_rows=torch.zeros(requests + 1, dtype=torch.int32), kv_lens=torch.zeros(requests, dtype=torch.int32),
                scaling=1.0)


def test_wrappers_refuse_cpu_tensors():
    t = _tensors()
    with pytest.raises(RuntimeError, match="must be CUDA"):
        paged.attention(**t)
    with pytest.raises(RuntimeError, match="must be CUDA"):
        paged.append(t["query"], t["query"], t["k_pages"], t["v_pages"], torch.zeros(4, dtype=torch.int64))
    i32 = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="table must be CUDA"):
        paged.plan_step(i32, t["table"], i32, i32, i32[:1], 16, 4)
    with pytest.raises(RuntimeError, match="table must be CUDA"):
        paged.release_pages(i32, t["table"], i32, i32, i32[:1], 16)
    with pytest.raises(RuntimeError, match="must be bfloat16 or float16"):
        paged.attention(**{**t, "k_pages": t["k_pages"].float()})
    for page in (8, 17, 8192):
        with pytest.raises(RuntimeError, match="power of two"):
            paged.PageTable(2, 100, 10, page, "cpu")


def test_step_plan_buffers():
    p = paged.StepPlan.empty(3, 5, "cpu")
    assert [t.shape[0] for t in p] == [4, 3, 5, 5, 1]
    assert [t.dtype for t in p] == [torch.int32, torch.int32, torch.int64, torch.int32, torch.int32]
    p.slots.fill_(-1)
    p.positions.fill_(7)
    assert (p.slots == -1).all() and (p.positions == 7).all()


def test_grids_have_less_than_2_32_threads():
    for call in (lambda: _attend(rows=1 << 30, max_rows=1 << 30), lambda: _append(rows=1 << 30, heads=64)):
        with pytest.raises(RuntimeError, match="too many rows"):
            _lib.check(call())

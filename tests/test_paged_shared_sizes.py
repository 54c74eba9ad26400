"""Sizes of the attention over shared prefixes on the CPU: no workspace is
asked for what the call refuses, and one a word short is refused."""

import pytest

from kv_cache_amd import _lib
from test_paged_codes import P, _codes, _shared

lib = _lib.load()
ARGS = dict(rows=4, max_rows=4, requests=2, width=8, page=16, q_heads=4, kv_heads=4, head_dim=64)


def _bytes(shared=True, **kw):
    f = lib.qkv_paged_attention_shared_workspace_bytes if shared else lib.qkv_paged_attention_workspace_bytes
    return f(*{**ARGS, **kw}.values())


@pytest.mark.parametrize("sizes", [dict(requests=4097), dict(rows=(1 << 20) + 1), dict(rows=1 << 20, q_heads=64),
                                   dict(rows=1 << 20, q_heads=64, kv_heads=64), dict(rows=1 << 30, max_rows=1 << 30),
                                   dict(rows=1 << 19, q_heads=128, kv_heads=1, head_dim=128), dict(requests=1 << 20)])
def test_no_workspace_for_refused_sizes(sizes):
    s = {**ARGS, **sizes}
    call = dict(rows=s["rows"], max_rows=s["max_rows"], requests=s["requests"], hq=s["q_heads"], hkv=s["kv_heads"], dim=s["head_dim"])
    assert _shared(**call) == -3 and "too many rows or requests" in lib.qkv_last_error().decode()
    assert _bytes(**sizes) == -1


@pytest.mark.parametrize("sizes", [dict(), dict(requests=4096), dict(rows=1 << 20), dict(rows=(1 << 20) - 1, q_heads=64, kv_heads=8),
                                   dict(rows=0), dict(width=8192, head_dim=128, q_heads=32, kv_heads=8, rows=64, requests=64)])
def test_a_workspace_of_that_size_and_one_short(sizes):
    s = {**ARGS, **sizes}
    call = dict(rows=s["rows"], max_rows=s["max_rows"], requests=s["requests"], hq=s["q_heads"], hkv=s["kv_heads"], dim=s["head_dim"],
                width=s["width"], ld=s["width"])
    need = _bytes(**sizes)
    if s["rows"] == 0:
        assert need >= 0 and _shared(**call) == 0
        return
    assert need > 0 and _shared(**call, ws_bytes=need - 4) == -1
    assert f"hold {need} bytes" in lib.qkv_last_error().decode()


@pytest.mark.parametrize("code", [1, 2])
@pytest.mark.parametrize("max_rows", [1, 4, 32])
def test_the_workspace_of_16_bit_pages_holds_that_of_codes(max_rows, code):
    sizes = dict(rows=32, max_rows=max_rows, requests=32, width=128, q_heads=32, kv_heads=8, head_dim=128)
    call = dict(rows=32, max_rows=max_rows, requests=32, width=128, ld=128, hq=32, hkv=8, dim=128)
    assert _codes(code=code, ws=P, ws_bytes=64, **call) == -1     # too short: the message says what codes need
    need = int(lib.qkv_last_error().decode().split(" hold ")[1].split()[0])
    assert 64 < need <= _bytes(shared=False, **sizes)
    assert _codes(code=code, ws=P, ws_bytes=need - 4, **call) == -1
    assert _codes(code=code, ws=None, ws_bytes=need, **call) == -1

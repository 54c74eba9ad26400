"""Quantised pages and shared prefixes on the CPU: the C entry points'
refusals (no kernel is launched), the size functions, the wrappers' checks, and
that no kernel of theirs spills vector registers."""

import ctypes
import re
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from kv_cache_amd import _lib, paged

lib = _lib.load()
P, ODD = ctypes.c_void_p(256), ctypes.c_void_p(264)
S2, S3 = _lib.strides(256, 64), _lib.strides(4096, 1024, 64)


def _append(key=P, value=P, kp=P, vp=P, ps=S3, ks=P, ss=S2, code=1, pages=4, page=16, heads=4, dim=64, slots=P, rows=3, dtype=0):
    return lib.qkv_paged_append_codes(key, S2, value, S2, kp, vp, ps, ks, P, ss, code, pages, page, heads, dim, slots, rows,
                                      dtype, None)


def _read(kp=P, ps=S3, ks=P, ss=S2, code=1, pages=4, page=16, heads=4, dim=64, table=P, ld=8, width=8, requests=2, cu=P, rows=3,
          key=P, ks2=S2, dtype=0):
    return lib.qkv_paged_read(kp, P, ps, ks, P, ss, code, pages, page, heads, dim, table, ld, width, requests, cu, P, rows, key,
                              ks2, P, S2, dtype, None)


def _args(pages=4, page=16, ld=8, width=8, requests=2, rows=4, max_rows=4, hq=4, hkv=4, dim=64, scaling=1.0, cap=0.0, ws=P,
          ws_bytes=0, out=P, os=S2, dtype=0):
    return (pages, page, P, ld, width, requests, P, P, rows, max_rows, hq, hkv, dim, scaling, cap, None, None, None, ws, ws_bytes,
            out, os, dtype, None)


def _codes(q=P, kp=P, ps=S3, ks=P, ss=S2, code=1, **kw):
    return lib.qkv_paged_attention_codes(q, S2, kp, P, ps, ks, P, ss, code, *_args(**kw))


def _shared(q=P, kp=P, ps=S3, ks=None, ss=None, code=0, plan=P, **kw):
    return lib.qkv_paged_attention_shared(q, S2, kp, P, ps, ks, ks, ss, code, plan, *_args(**{"ws_bytes": 1 << 40, **kw}))


def _share(parents=P, cu=P, requests=2, rows=4, shared=P):
    return lib.qkv_paged_share(parents, cu, P, P, requests, rows, shared, None)


@pytest.mark.parametrize("call,msg", [
    (lambda: _append(key=None), "null pointer"), (lambda: _append(value=None), "null pointer"),
    (lambda: _append(slots=None), "null pointer"), (lambda: _append(ks=None), "null pointer"),
    (lambda: _append(kp=None), "null pointer"), (lambda: _append(ss=None), "null pointer"),
    (lambda: _append(code=0), "is not fp8"), (lambda: _append(code=3), "is not fp8"), (lambda: _append(dtype=2), "is not bf16"),
    (lambda: _append(rows=-1), "bad sizes"), (lambda: _append(dim=40), "multiple of 32"), (lambda: _append(page=24), "power of two"),
    (lambda: _append(kp=ODD), "16-byte aligned"), (lambda: _append(ps=_lib.strides(4096, 1024, 40)), "16-byte aligned"),
    (lambda: _append(rows=1 << 30, heads=64), "too many rows"), (lambda: _append(heads=65536, dim=65536), "too many channels"),
    (lambda: _read(table=None), "null pointer"), (lambda: _read(cu=None), "null pointer"), (lambda: _read(key=None), "null pointer"),
    (lambda: _read(ks=None), "null pointer"), (lambda: _read(code=-1), "is not 0"), (lambda: _read(code=3), "is not 0"),
    (lambda: _read(dtype=2), "is not bf16"), (lambda: _read(ld=7), "bad sizes of the table"),
    (lambda: _read(requests=0), "bad sizes of the table"), (lambda: _read(width=(1 << 26) + 1, ld=1 << 27), "bad sizes of the table"),
    (lambda: _read(key=ODD), "16-byte aligned"), (lambda: _read(ks2=_lib.strides(256, 60)), "16-byte aligned"),
    (lambda: _read(code=0, ps=_lib.strides(4096, 1024, 60)), "16-byte aligned"), (lambda: _read(page=8), "power of two"),
    (lambda: _codes(q=None), "null pointer"), (lambda: _codes(ks=None), "null pointer"), (lambda: _codes(ss=None), "null pointer"),
    (lambda: _codes(code=0), "is not fp8"), (lambda: _codes(code=9), "is not fp8"), (lambda: _codes(dtype=2), "is not bf16"),
    (lambda: _codes(dim=96), "unsupported sizes"), (lambda: _codes(hq=6), "unsupported sizes"),
    (lambda: _codes(scaling=float("nan")), "scaling must be in"), (lambda: _codes(cap=-1.0), "softcap"),
    (lambda: _codes(kp=ODD), "16-byte aligned"), (lambda: _codes(ps=_lib.strides(4096, 1024, 72)), "16-byte aligned"),
    (lambda: _codes(ks=ctypes.c_void_p(258)), "4-byte aligned"), (lambda: _codes(ss=_lib.strides(256, 30)), "4-byte aligned"),
    (lambda: _codes(width=100, ld=100), "workspace"), (lambda: _codes(rows=1 << 30, max_rows=1 << 30), "too many rows"),
    (lambda: _shared(plan=None), "null pointer"), (lambda: _shared(code=1), "null pointer"), (lambda: _shared(code=5), "is not 0"),
    (lambda: _shared(requests=4097), "too many rows or requests"), (lambda: _shared(rows=(1 << 20) + 1), "too many rows or requests"),
    (lambda: _shared(ws_bytes=64), "workspace"), (lambda: _shared(ws=None), "workspace"), (lambda: _shared(ws=ODD), "workspace"),
    (lambda: _share(parents=None), "null pointer"), (lambda: _share(cu=None), "null pointer"), (lambda: _share(shared=None), "null pointer"),
    (lambda: _share(requests=0), "1 to 4096 requests"), (lambda: _share(requests=4097), "1 to 4096 requests"),
    (lambda: _share(rows=0), "1 to 4096 requests"), (lambda: _share(rows=(1 << 20) + 1), "1 to 4096 requests"),
])
def test_refusals(call, msg):
    assert call() in (-1, -3)
    assert msg in lib.qkv_last_error().decode()


def test_nothing_to_do():
    assert _append(rows=0, key=None, value=None, slots=None) == 0
    assert _read(rows=0, key=None) == 0
    assert _codes(rows=0, q=None, out=None) == 0
    assert _shared(rows=0, q=None, out=None) == 0


def test_sizes():
    assert lib.qkv_paged_share_words(5, 3) == 3 * 5 + 4 * 3 + 1
    assert lib.qkv_paged_share_words(0, 3) == -1 and lib.qkv_paged_share_words(5, 4097) == -1
    f = lib.qkv_paged_attention_shared_workspace_bytes
    assert f(4, 4, 2, 8, 16, 6, 4, 64) == -1 and f(4, 4, 2, 8, 16, 4, 4, 96) == -1
    base = dict(rows=32, max_rows=4, requests=32, width=128, page=16, q_heads=32, kv_heads=8, head_dim=128)
    for name, values in (("rows", (1, 4, 32, 64, 1000, 10**5)), ("requests", (1, 3, 32, 200)), ("width", (8, 17, 64, 1000, 8192))):
        sizes = [f(*{**base, name: v}.values()) for v in values]
        assert sizes == sorted(sizes) and sizes[0] > 0, (name, sizes)
    # the workspace of a call over 16-bit pages serves one over codes
    g = lib.qkv_paged_attention_workspace_bytes
    need = g(*base.values())
    assert _codes(**{"rows": 32, "max_rows": 1, "requests": 32, "width": 128, "ld": 128, "hq": 32, "hkv": 8, "dim": 128,
                     "ws_bytes": need - 4, "ws": None}) == -1
    one = g(*{**base, "max_rows": 1}.values())
    assert one > 0


def test_wrappers_refuse_cpu_tensors():
    codes, scales = paged.quantized_pages(4, 4, 16, 64, "fp8", "cpu")
    assert codes.shape == (4, 4, 16, 64) and scales.shape == (4, 4, 16, 2)
    half, _ = paged.quantized_pages(4, 4, 16, 64, "fp4", "cpu")
    assert half.shape == (4, 4, 16, 32) and half.dtype == torch.uint8
    q, i32 = torch.zeros((4, 4, 64), dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int32)
    sc = dict(k_scales=scales, v_scales=scales)
    with pytest.raises(RuntimeError, match="must be CUDA"):
        paged.append(q, q, codes, codes, torch.zeros(4, dtype=torch.int64), **sc)
    with pytest.raises(RuntimeError, match="must be CUDA"):
        paged.attention(q, codes, codes, i32[None], i32, i32, 1.0, **sc)
    with pytest.raises(RuntimeError, match="must be CUDA"):
        paged.read(codes, codes, i32[None], i32, i32, 4, **sc)
    with pytest.raises(RuntimeError, match="must be CUDA"):
        paged.share_rows(i32, i32, i32, i32, 3)
    with pytest.raises(RuntimeError, match="must be CUDA"):
        paged.SharedRows(3, 4, "cpu") and paged.share_rows(i32, i32, i32, i32, 4, out=paged.SharedRows(3, 4, "cpu"))


def test_no_vector_registers_are_spilled(tmp_path):
    """The kernels over codes and over shared prefixes keep everything in registers: where lanes part, a spill can be
    stored for some lanes only and read back for all."""
    tools = [Path(p) / t for p in ("/opt/rocm/llvm/bin",) for t in ("llvm-objdump", "llvm-readelf")]
    if not all(t.exists() for t in tools):
        pytest.skip("llvm tools are not installed")
    shutil.copy(_lib.LIB_PATH, tmp_path / "lib.so")
    subprocess.run([tools[0], "--offloading", "lib.so"], cwd=tmp_path, capture_output=True, check=True)
    seen = {}
    for part in tmp_path.glob("lib.so.*gfx950"):
        notes = subprocess.run([tools[1], "--notes", part], capture_output=True, text=True, check=True).stdout
        for kernel in notes.split("- .agpr_count")[1:]:
            name, spills = re.search(r"\.symbol:\s+(\S+)\.kd", kernel), re.search(r"\.vgpr_spill_count:\s+(\d+)", kernel)
            seen[name.group(1)] = int(spills.group(1))
    mine = {n: s for n, s in seen.items() if "paged_shared" in n or "codes" in n or "share_" in n or "read_kernel" in n
            or re.search(r"paged_(rows|token)_kernelILi\d+ELb[01]ELb[01]ELi[12]E", n)}
    assert len(mine) > 80, sorted(seen)
    assert not [n for n, s in mine.items() if s]

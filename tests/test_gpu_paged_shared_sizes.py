"""Attention over shared prefixes refuses sizes before it allocates for them."""

import pytest
import torch

from kv_cache_amd import paged
from test_gpu_paged import DEV, _i32

pytestmark = pytest.mark.gpu


def test_refused_sizes_allocate_nothing():
    rows, heads, dim = 1 << 20, 64, 64       # 2^26 rows times heads
    q, out = (torch.zeros((1, heads, dim), dtype=torch.bfloat16, device=DEV).expand(rows, heads, dim) for _ in range(2))
    pages = torch.zeros((1, heads, 16, dim), dtype=torch.bfloat16, device=DEV)
    cu, kv = _i32([0, rows]), _i32([16])
    plan = paged.share_rows(_i32([-1]), cu, kv, kv, rows)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    held = torch.cuda.memory_allocated()
    with pytest.raises(RuntimeError, match="too many rows or requests"):
        paged.attention(q, pages, pages, _i32([[0]]), cu, kv, 1.0, shared=plan, out=out)
    assert torch.cuda.max_memory_allocated() - held < 1 << 20
    with pytest.raises(RuntimeError, match="sizes that attention does not take"):
        paged.attention_workspace(rows, rows, 1, 1, 16, heads, heads, dim, DEV, shared=True)

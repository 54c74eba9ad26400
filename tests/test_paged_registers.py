"""No kernel of the paged cache spills vector registers, whatever its pages
hold: where lanes part, a spill can be stored for some lanes only and read
back for all.  Read from the notes of the built library; no kernel runs."""

import re
import shutil
import subprocess
from pathlib import Path

import pytest

from kv_cache_amd import _lib

TOOLS = [Path("/opt/rocm/llvm/bin") / t for t in ("llvm-objdump", "llvm-readelf")]
# kernels of paged.hip, paged_codes.hip, paged_attention*.hip, paged_shared*.hip, by the start of their names
KERNELS = ("plan", "plan_rows", "release", "append", "append_codes", "read", "share", "share_few", "share_rows", "paged_token",
           "paged_rows", "paged_join", "paged_shared", "paged_shared_join")


def test_no_paged_kernel_spills_vector_registers(tmp_path):
    if not all(t.exists() for t in TOOLS):
        pytest.skip("llvm tools are not installed")
    shutil.copy(_lib.LIB_PATH, tmp_path / "lib.so")
    subprocess.run([TOOLS[0], "--offloading", "lib.so"], cwd=tmp_path, capture_output=True, check=True)
    seen = {}
    for part in tmp_path.glob("lib.so.*gfx950"):
        notes = subprocess.run([TOOLS[1], "--notes", part], capture_output=True, text=True, check=True).stdout
        for kernel in notes.split("- .agpr_count")[1:]:
            name = re.search(r"\.symbol:\s+(\S+)\.kd", kernel).group(1)
            short = re.match(r"_ZN3qkv12_GLOBAL__N_1\d+([a-z_0-9]+?)_kernel", name)
            if short and short.group(1) in KERNELS:
                size = lambda f: int(re.search(rf"\.{f}:\s+(\d+)", kernel).group(1))  # noqa: E731
                seen[name] = short.group(1), size("vgpr_spill_count"), size("private_segment_fixed_size")
    assert {k for k, _, _ in seen.values()} == set(KERNELS)
    # 2 head dims x 2 dtypes x 2 score forms x 3 kinds of pages, the rows kernel once, the others for one and two column sets
    count = lambda kind: sum(k == kind for k, _, _ in seen.values())  # noqa: E731
    assert (count("paged_rows"), count("paged_token"), count("paged_shared")) == (24, 48, 48)
    assert not {n: s for n, s in seen.items() if s[1] or s[2]}

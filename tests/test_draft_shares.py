"""How a tree call's work is divided where its tiles are short (no GPU): a workgroup for each tile, whatever share a cut is worth."""
import os
import shutil
import subprocess

import pytest

from cuda_attn import _native

HERE = os.path.dirname(os.path.abspath(__file__))
REPO = os.path.dirname(HERE)


def test_share_count(tmp_path):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc not found")
    exe = tmp_path / "share_count_check"
    build = subprocess.run([hipcc, "--offload-arch=gfx950", "-O2", "-std=c++17", "-Xclang", "-target-feature", "-Xclang",
                            "-packed-fp32-ops", "-I", os.path.join(REPO, "phantom-a100_amd", "csrc"),
                            os.path.join(HERE, "native", "share_count_check.cpp"), "-o", str(exe)],
                           capture_output=True, text=True, timeout=300)
    assert build.returncode == 0, build.stdout + build.stderr
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0 and run.stdout.strip().endswith("ok"), run.stdout + run.stderr


@pytest.mark.parametrize("dtype,d,seqs,heads,new,capacity,rows,wgs", [
    ("f16", 64, 14, 4, 256, 208, 128, 505),     # tiles of 464 units: (14 * 256 / 32 + 14) * 4 of them and one
    ("f16", 64, 32, 4, 24, 200, 32, 512),       # 448 tiles of 456 units, as many as are resident with 128 units each
    ("f16", 128, 2, 1, 4, 300, 16, 18),         # (8 / 4 + 2) * 1 tiles of 556 units, 128 each: 17 and one
    ("i8", 128, 32, 8, 48, 8192, 256, 256),
    ("f16", 64, 4, 4, 40, 700, 32, 512)])       # (160 / 8 + 4) * 4 tiles of 956 units, 128 each: more than are resident
def test_workgroups_of_short_calls(dtype, d, seqs, heads, new, capacity, rows, wgs):
    """4 query heads a key/value head; the workgroups by the workspace that a call asks for."""
    c = _native.PagedCacheArgs(256, 256, None, None, 256, 256, 40000, 1, heads, d, seqs, capacity, capacity, _native.DTYPE_F16)
    if dtype == "i8":
        c.dtype, c.k_scale, c.v_scale = _native.DTYPE_I8, 256, 256
    need = _native.lib().pa_paged_tree_attn_workspace(c, _native.DTYPE_F16, seqs * new, 4 * heads, None, 0)
    size = lambda n: -(-n * 16 // 256) * 256 + n * 2 * rows * (d + 2) * 4  # noqa: E731
    assert need == size(wgs), [n for n in range(1, 600) if size(n) == need]

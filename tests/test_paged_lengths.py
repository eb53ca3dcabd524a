"""The lengths that a paged call counts its work by, at the largest sizes (host arithmetic, no GPU)."""
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
REPO = os.path.dirname(HERE)


def test_lengths_at_the_largest_sizes(tmp_path):
    """Built with the host compiler's check of signed overflow, which ends the program at the first one."""
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc not found")
    exe = tmp_path / "paged_length_check"
    build = subprocess.run([hipcc, "--offload-arch=gfx950", "-O1", "-std=c++17", "-Xclang", "-target-feature", "-Xclang",
                            "-packed-fp32-ops", "-Xarch_host", "-fsanitize=signed-integer-overflow", "-Xarch_host",
                            "-fsanitize-trap=signed-integer-overflow", "-I", os.path.join(REPO, "phantom-a100_amd", "csrc"),
                            os.path.join(HERE, "native", "paged_length_check.cpp"), "-o", str(exe)],
                           capture_output=True, text=True, timeout=300)
    assert build.returncode == 0, build.stdout + build.stderr
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0 and run.stdout.strip().endswith("ok"), (run.returncode, run.stdout + run.stderr)

"""States of the gated scan after a wait that ran out: tests/cpp/gated_waits_states_test.cu, built here with the test hooks and short waits."""
import os
import shutil
import subprocess

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_states_behind_rows_that_never_came(tmp_path):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.isfile(nvcc):
        pytest.skip("nvcc is not available on this machine")
    exe = str(tmp_path / "gated_waits_states_test")
    r = subprocess.run([nvcc, "-std=c++17", "-O2", "-gencode", "arch=compute_100a,code=sm_100a", "-DTB200_TEST_HOOKS", "-DTB200_SPIN_LIMIT=65536",
                        "-I" + os.path.join(ROOT, "include"), "-I" + os.path.join(ROOT, "thrust_b200", "csrc"), os.path.join(ROOT, "tests", "cpp", "gated_waits_states_test.cu"), "-o", exe],
                       capture_output=True, text=True, timeout=900)
    assert r.returncode == 0, r.stdout + r.stderr
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr

"""Rows of no channels: every entry point says what it needs and has nothing to do (no GPU is needed here).  In a process of its own, since a
division by zero would end this one."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PREAMBLE = """
import ctypes as C
from thrust_b200 import _lib
lib, BUF, F32, I32 = _lib.load(), 256, 8, 4
def sized(fn, before, after):
    need = C.c_size_t(0)
    assert getattr(lib, fn)(*before, None, C.byref(need), None) == 0 and need.value >= 256, fn
    return need
"""
# an address that is never read; no kernel is launched where there is nothing to write
CALLS = {
    "embedding": "assert lib.tb200_embedding(BUF, 4, 0, BUF, I32, 10, 0, F32, 1.0, BUF, None) == 0",
    "embedding_grad": """
for n in (0, 1, 10, 100000):
    for accumulate in (0, 1):
        args = (BUF, 0, BUF, I32, n, 4, 0, F32, F32, 1.0, accumulate, BUF)
        need = sized('tb200_embedding_grad', args, ())
        assert lib.tb200_embedding_grad(*args, BUF, C.byref(need), None) == 0""",
    "gated_scan": """
args = (BUF, 0, BUF, 0, None, None, 0, 2, 10, 0, F32, BUF, BUF)
need = sized('tb200_gated_scan', args, ())
assert lib.tb200_gated_scan(*args, BUF, C.byref(need), None) == 0""",
    "gated_scan_grad": """
args = (BUF, 0, BUF, 0, BUF, 0, BUF, 0, None, None, None, 0, 2, 10, 0, F32, BUF, BUF, BUF)
need = sized('tb200_gated_scan_grad', args, ())
assert lib.tb200_gated_scan_grad(*args, BUF, C.byref(need), None) == 0""",
    "gated_step": "assert lib.tb200_gated_step(BUF, 0, BUF, 0, BUF, 4, None, 0, 2, 0, F32, BUF, None) == 0",
    "expert_dispatch": "sized('tb200_expert_dispatch', (BUF, 0, BUF, I32, 10, 2, 4, 0, F32, BUF, BUF, BUF, BUF), ())",
    "expert_combine": "assert lib.tb200_expert_combine(BUF, 0, BUF, None, 10, 2, 0, F32, BUF, None) == 0",
}


@pytest.mark.parametrize("name", sorted(CALLS))
def test_rows_of_no_channels(name):
    r = subprocess.run([sys.executable, "-c", PREAMBLE + CALLS[name]], cwd=ROOT, capture_output=True, text=True, timeout=300, env=dict(os.environ, CUDA_VISIBLE_DEVICES=""))
    assert r.returncode == 0, "exit %d\n%s%s" % (r.returncode, r.stdout, r.stderr)

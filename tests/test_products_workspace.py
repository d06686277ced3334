"""The products refuse a workspace that is not 16-byte aligned, before anything reaches a GPU (no GPU is needed here)."""
import ctypes

import pytest

from thrust_b200 import _lib

BUF, I32, F32, BF16 = 256, 4, 8, 11       # an address that is never read


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("off", [1, 4, 8])
def test_workspaces_off_16_bytes_are_refused(t, off):
    lib, need = _lib.load(), ctypes.c_size_t(1 << 30)
    assert lib.tb200_expert_product(BUF, 7, BUF, I32, BUF, 63, 9, 0, None, None, 0, 0, 100, 3, 7, 9, t, BUF, None, BUF + off, ctypes.byref(need), None) == 1
    assert lib.tb200_expert_product_grad(BUF, 9, BUF, 7, BUF, I32, BUF, 63, 9, 0, 100, 3, 7, 9, t, F32, 0, BUF, BUF, None, BUF + off, ctypes.byref(need), None) == 1

"""The operators on rows refuse what they cannot take before anything reaches a GPU (no GPU is needed here)."""
import ctypes

import pytest
import torch

import thrust_b200 as tb
from thrust_b200 import _lib

BUF = 256       # an address that is never read: every call below is refused, or has nothing to do


def test_host_tensors_are_refused():
    x, ids = torch.zeros(2, 4), torch.zeros(2, 1, dtype=torch.int64)
    for call in (lambda: tb.embedding(x, ids), lambda: tb.embedding_grad(x, ids[:, 0], 3), lambda: tb.gated_scan(x, x), lambda: tb.gated_scan_grad(x, x, x, x),
                 lambda: tb.gated_step(x, x, x), lambda: tb.expert_dispatch(x, ids, 2), lambda: tb.expert_combine(x, tb.ExpertPlan(ids.int(), None, None))):
        with pytest.raises(ValueError, match="CUDA device"):
            call()


def test_c_calls_refuse_wrong_arguments():
    lib, size = _lib.load(), ctypes.c_size_t(0)
    ref = ctypes.byref(size)
    f32, f64, i32, u8 = 8, 9, 4, 1
    big = ctypes.byref(ctypes.c_size_t(1 << 20))
    # types
    assert lib.tb200_embedding(BUF, 4, 8, BUF, i32, 2, 8, f64, 1.0, BUF, None) == 801
    assert lib.tb200_embedding(BUF, 4, 8, BUF, u8, 2, 8, f32, 1.0, BUF, None) == 801
    assert lib.tb200_gated_scan(BUF, 8, BUF, 8, None, BUF, u8, 1, 4, 8, f32, BUF, BUF, BUF, big, None) == 801
    assert lib.tb200_expert_dispatch(BUF, 8, BUF, f32, 2, 1, 4, 8, f32, BUF, BUF, BUF, BUF, None, ref, None) == 801
    # strides shorter than a row, missing buffers, sizes past their limits
    assert lib.tb200_embedding(BUF, 4, 7, BUF, i32, 2, 8, f32, 1.0, BUF, None) == 1
    assert lib.tb200_embedding(None, 4, 8, BUF, i32, 2, 8, f32, 1.0, BUF, None) == 1
    assert lib.tb200_embedding(BUF, 4, 8, BUF, i32, 1 << 31, 8, f32, 1.0, BUF, None) == 1
    assert lib.tb200_embedding_grad(BUF, 8, BUF, i32, 2, 1 << 31, 8, f32, f32, 1.0, 0, BUF, None, ref, None) == 1
    assert lib.tb200_gated_scan(BUF, 7, BUF, 8, None, None, 0, 1, 4, 8, f32, BUF, BUF, BUF, big, None) == 1
    assert lib.tb200_gated_scan(BUF, 8, BUF, 8, None, None, 0, 3, 4, 8, f32, BUF, BUF, BUF, big, None) == 1       # 4 rows are no 3 sequences
    assert lib.tb200_gated_scan(BUF, 8, BUF, 8, None, None, 0, 1, 4, 8, f32, None, BUF, BUF, big, None) == 1
    assert lib.tb200_gated_scan_grad(BUF, 8, BUF, 8, BUF, 8, BUF, 8, None, None, None, 0, 1, 4, 8, f32, BUF, BUF, None, BUF, big, None) == 1
    assert lib.tb200_gated_step(BUF, 8, BUF, 8, None, 3, BUF, i32, 2, 8, f32, BUF, None) == 1
    assert lib.tb200_expert_dispatch(BUF, 8, BUF, i32, 2, 1, 1025, 8, f32, BUF, BUF, BUF, BUF, None, ref, None) == 1
    assert lib.tb200_expert_dispatch(BUF, 8, BUF, i32, 1 << 30, 1, 4, 8, f32, BUF, BUF, BUF, BUF, None, ref, None) == 1
    assert lib.tb200_expert_combine(BUF, 8, BUF, None, 2, 33, 8, f32, BUF, None) == 1
    assert lib.tb200_expert_combine(BUF, 7, BUF, None, 2, 2, 8, f32, BUF, None) == 1
    assert lib.tb200_expert_combine_grad(BUF, 8, BUF, 8, BUF, None, BUF, 2, 2, 8, f32, BUF, BUF, None) == 1


def test_c_calls_say_how_much_workspace_they_need():
    lib, size = _lib.load(), ctypes.c_size_t(0)
    ref = ctypes.byref(size)
    before = 0
    for n in (0, 1, 1000, 50000, 1 << 20, (1 << 31) - 1):
        assert lib.tb200_embedding_grad(None, 8, None, 4, n, 1000, 8, 11, 8, 1.0, 0, None, None, ref, None) == 0
        assert size.value >= max(256, before, 4 * n)
        before = size.value
        size.value -= 1
        assert lib.tb200_embedding_grad(BUF, 8, BUF, 4, n, 1000, 8, 11, 8, 1.0, 0, BUF, BUF, ref, None) == 1
    for offsets, need in ((None, 256), (BUF, 256 + 4 * 1000)):
        assert lib.tb200_gated_scan(None, 8, None, 8, None, offsets, 4, 1, 1000, 8, 11, None, None, None, ref, None) == 0 and size.value >= need
        assert lib.tb200_gated_scan_grad(None, 8, None, 8, None, 8, None, 8, None, None, offsets, 4, 1, 1000, 8, 11, None, None, None, None, ref, None) == 0 and size.value >= need
        size.value -= 1
        assert lib.tb200_gated_scan(BUF, 8, BUF, 8, None, offsets, 4, 1, 1000, 8, 11, BUF, BUF, BUF, ref, None) == 1
    for n in (0, 1, 1000, 1 << 20):
        assert lib.tb200_expert_dispatch(None, 8, None, 4, n, 8, 64, 8, 11, None, None, None, None, None, ref, None) == 0 and size.value >= 256
        size.value = 255
        assert lib.tb200_expert_dispatch(BUF, 8, BUF, 4, n, 8, 64, 8, 11, BUF, BUF, BUF, BUF, BUF, ref, None) == 1
    assert lib.tb200_expert_dispatch(None, 8, None, 4, 8, 8, 64, 8, 11, None, None, None, None, None, None, None) == 1


def test_nothing_to_do():
    lib = _lib.load()
    assert lib.tb200_embedding(None, 4, 8, None, 4, 0, 8, 8, 1.0, None, None) == 0
    assert lib.tb200_gated_scan(None, 8, None, 8, None, None, 0, 0, 0, 8, 8, None, None, BUF, ctypes.byref(ctypes.c_size_t(1 << 20)), None) == 0
    assert lib.tb200_gated_step(None, 8, None, 8, None, 0, None, 4, 0, 8, 8, None, None) == 0
    assert lib.tb200_expert_combine(None, 8, None, None, 0, 2, 8, 8, None, None) == 0

"""Gradients of products without inputs or without outputs: no operand is read, so none is laid out anew (the workspace has no room for it) and none need be there."""
import ctypes

import pytest
import torch

from thrust_b200 import _lib

I32, F32, BF16 = 4, 8, 11
HEADER = 256


def grad(n, experts, i, o, t, d=None, rows=None, offsets=None, w=None, drows=None, dw=None, db=None, ws=None, need=None, stream=None):
    """Rows whose distances are not whole 16-byte pieces, which would have to be laid out anew."""
    dstride, rstride = odd(o), odd(i)
    return _lib.load().tb200_expert_product_grad(d, dstride, rows, rstride, offsets, I32, w, i * o, o, 0, n, experts, i, o, t, F32, 0, drows, dw, db, ws, ctypes.byref(need), stream)


def odd(width):
    return width + (3 if width % 2 == 0 else 2)


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("n, experts, i, o", [(100, 3, 7, 0), (100, 3, 0, 7), (100000, 1, 7, 0), (100000, 1, 0, 9), (5000, 2, 130, 0), (0, 2, 7, 9)])
def test_no_room_for_what_is_not_read(t, n, experts, i, o):
    need = ctypes.c_size_t(0)
    assert grad(n, experts, i, o, t, need=need) == 0
    assert need.value == HEADER


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, t", [(torch.float32, F32), (torch.bfloat16, BF16)])
@pytest.mark.parametrize("n, experts", [(100, 3), (5000, 1)])
def test_operands_that_are_not_read_may_be_null(tb, dtype, t, n, experts):
    ws = torch.full((1 << 20,), 255, dtype=torch.uint8, device="cuda")
    offsets = torch.linspace(0, n - 2, experts + 1, device="cuda").int()
    stream = torch.cuda.current_stream().cuda_stream
    # no outputs: the gradient of rows is zero
    drows, need = torch.full((n, 7), 5.0, dtype=dtype, device="cuda"), ctypes.c_size_t(ws.numel())
    assert grad(n, experts, 7, 0, t, offsets=offsets.data_ptr(), drows=drows.data_ptr(), ws=ws.data_ptr(), need=need, stream=stream) == 0
    torch.cuda.synchronize()
    assert drows.abs().max() == 0
    # no inputs: what is left is the gradient of bias
    d, db = torch.ones(n, 12, dtype=dtype, device="cuda"), torch.empty(experts, 9, device="cuda")
    room = ctypes.c_size_t(0)
    assert grad(n, experts, 0, 9, t, d=d.data_ptr(), offsets=offsets.data_ptr(), db=db.data_ptr(), need=room, stream=stream) == 0 and room.value <= ws.numel()
    assert grad(n, experts, 0, 9, t, d=d.data_ptr(), offsets=offsets.data_ptr(), db=db.data_ptr(), ws=ws.data_ptr(), need=need, stream=stream) == 0
    assert torch.equal(db, offsets.diff().float()[:, None].expand(experts, 9))


@pytest.mark.gpu
@pytest.mark.parametrize("n, experts", [(100, 3), (5000, 1), (0, 2)])
def test_a_gradient_of_bias_alone_leaves_a_status(tb, n, experts):
    """As the other calls' kernels, its own clear what is in the workspace."""
    ws = torch.full((1 << 20,), 255, dtype=torch.uint8, device="cuda")
    offsets = torch.linspace(0, n, experts + 1, device="cuda").int()
    stream, status, need = torch.cuda.current_stream().cuda_stream, ctypes.c_uint(7), ctypes.c_size_t(ws.numel())
    d, db = torch.ones(n + 1, 12, device="cuda"), torch.empty(experts, 9, device="cuda")
    assert grad(n, experts, 0, 9, F32, d=d.data_ptr(), offsets=offsets.data_ptr(), db=db.data_ptr(), ws=ws.data_ptr(), need=need, stream=stream) == 0
    assert _lib.load().tb200_workspace_status(ws.data_ptr(), stream, ctypes.byref(status)) == 0 and status.value == 0
    assert torch.equal(db, offsets.diff().float()[:, None].expand(experts, 9))

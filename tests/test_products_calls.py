"""The router and the experts' products refuse what they cannot take before anything reaches a GPU (no GPU is needed here)."""
import ctypes

import pytest
import torch

import thrust_b200 as tb
from thrust_b200 import _lib

BUF = 256       # an address that is never read: every call below is refused, or has nothing to do
I32, I64, U8, F32, F64, F16, BF16 = 4, 6, 1, 8, 9, 10, 11


def test_host_tensors_are_refused():
    x, ids, w = torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int32), torch.zeros(2, 8, 6)
    offsets = torch.tensor([0, 2, 4])
    for call in (lambda: tb.expert_route(x, 2), lambda: tb.expert_route_grad(x[:, :2], ids, x), lambda: tb.expert_product(x, offsets, w),
                 lambda: tb.expert_activation_grad(x, x, "silu"), lambda: tb.expert_product_grad(x[:, :6], x, offsets, w)):
        with pytest.raises(ValueError, match="CUDA device"):
            call()


def route(lib, logits=BUF, stride=8, n=4, experts=8, t=F32, bias=None, choices=2, scores=0, groups=1, kept=1, best=1, ids=BUF, weights=BUF):
    return lib.tb200_expert_route(logits, stride, n, experts, t, bias, choices, scores, groups, kept, best, 1, 1.0, ids, weights, None)


def test_router_refuses_wrong_arguments():
    lib = _lib.load()
    assert route(lib, t=F64) == 801 and route(lib, t=I32) == 801
    for wrong in ({"stride": 7}, {"experts": 0}, {"experts": 1025, "stride": 2000}, {"choices": 0}, {"choices": 9}, {"experts": 64, "stride": 64, "choices": 33}, {"scores": 2}, {"groups": 0},
                  {"groups": 3}, {"groups": 2, "kept": 3}, {"groups": 2, "kept": 0}, {"experts": 64, "stride": 64, "groups": 64}, {"best": 0}, {"best": 3}, {"logits": None}, {"ids": None},
                  {"weights": None}, {"n": 1 << 30}):
        assert route(lib, **wrong) == 1, wrong
    assert route(lib, n=0, logits=None, ids=None, weights=None) == 0
    grad = lambda d=BUF, ids=BUF, x=BUF, stride=8, n=4, experts=8, choices=2, t=F32, scores=0, to=BUF: lib.tb200_expert_route_grad(  # noqa: E731
        d, ids, x, stride, n, experts, choices, t, scores, 1, 1.0, to, None)
    assert grad(t=F64) == 801
    for wrong in ({"d": None}, {"ids": None}, {"x": None}, {"to": None}, {"stride": 7}, {"choices": 9}, {"scores": 5}, {"n": 1 << 31}):
        assert grad(**wrong) == 1, wrong
    assert grad(n=0, d=None, ids=None, x=None, to=None) == 0


def product(lib, rows=BUF, rstride=8, offsets=BUF, ot=I32, w=BUF, each=48, stride=6, inside=0, bias=None, res=None, resstride=0, act=0, n=4, experts=2, i=8, o=6, t=F32, out=BUF,
            before=None, ws=BUF, size=1 << 30):
    need = ctypes.c_size_t(size)
    return lib.tb200_expert_product(rows, rstride, offsets, ot, w, each, stride, inside, bias, res, resstride, act, n, experts, i, o, t, out, before, ws, ctypes.byref(need), None)


def product_grad(lib, d=BUF, dstride=6, rows=BUF, rstride=8, offsets=BUF, ot=I32, w=BUF, each=48, stride=6, inside=0, n=4, experts=2, i=8, o=6, t=F32, gt=F32, drows=BUF, dw=BUF, db=None,
                 ws=BUF, size=1 << 30):
    need = ctypes.c_size_t(size)
    return lib.tb200_expert_product_grad(d, dstride, rows, rstride, offsets, ot, w, each, stride, inside, n, experts, i, o, t, gt, 0, drows, dw, db, ws, ctypes.byref(need), None)


def test_products_refuse_wrong_arguments():
    lib = _lib.load()
    assert product(lib, t=F64) == 801 and product(lib, ot=U8) == 801 and product_grad(lib, t=F64) == 801 and product_grad(lib, ot=F32) == 801
    assert product_grad(lib, t=BF16, gt=F16) == 801 and product_grad(lib, t=F32, gt=BF16) == 801
    both = ({"rstride": 7}, {"offsets": None}, {"w": None}, {"rows": None}, {"each": 47}, {"stride": 5}, {"inside": 1, "stride": 7}, {"experts": 0}, {"experts": 1025}, {"i": 1 << 24, "rstride": 1 << 24},
            {"o": 1 << 24, "stride": 1 << 24}, {"n": 1 << 31}, {"size": 255})
    for wrong in both + ({"out": None}, {"act": 3}, {"act": 4}, {"act": 7}, {"act": -1}, {"act": 5, "o": 5, "stride": 5}, {"res": BUF, "resstride": 5}):
        assert product(lib, **wrong) == 1, wrong
    for wrong in both + ({"d": None}, {"dstride": 5}, {"drows": None}, {"dw": None}):
        assert product_grad(lib, **wrong) == 1, wrong
    act = lambda d=BUF, stride=6, before=BUF, a=1, n=4, width=6, t=F32, to=BUF: lib.tb200_expert_activation_grad(d, stride, before, a, n, width, t, to, None)  # noqa: E731
    assert act(t=F64) == 801
    for wrong in ({"d": None}, {"before": None}, {"to": None}, {"stride": 5}, {"a": 0}, {"a": 3}, {"a": 4}, {"n": 1 << 31}, {"width": 1 << 24, "stride": 1 << 24}):
        assert act(**wrong) == 1, wrong
    assert act(n=0, d=None, before=None, to=None) == 0 and act(width=0, d=None, before=None, to=None) == 0
    assert product(lib, n=0, rows=None, offsets=None, w=None, out=None) == 0 and product(lib, o=0, stride=0, offsets=None, out=None) == 0
    assert product_grad(lib, n=0, o=0, dstride=0, stride=0, d=None, rows=None, offsets=None, w=None, drows=None, dw=None) == 0


def test_products_say_how_much_workspace_they_need():
    lib, need = _lib.load(), ctypes.c_size_t(0)
    ask = lambda t, i, o, rstride, each, stride, inside=0, act=0, at=None: lib.tb200_expert_product(  # noqa: E731
        at, rstride, None, I32, None, each, stride, inside, None, None, 0, act, 100, 3, i, o, t, None, None, None, ctypes.byref(need), None)
    assert ask(F32, 8, 12, 8, 96, 12) == 0 and need.value == 256
    assert ask(F32, 7, 9, 7, 63, 9) == 0 and need.value >= 256 + 100 * 8 * 4 + 3 * 7 * 12 * 4        # both laid out anew
    assert ask(BF16, 64, 32, 64, 64 * 32, 32) == 0 and need.value == 256
    assert ask(BF16, 7, 32, 7, 7 * 32, 32) == 0 and need.value >= 256 + 100 * 8 * 2              # rows laid out anew
    assert ask(BF16, 64, 9, 64, 64 * 9, 9) == 0 and need.value >= 256 + 3 * 64 * 16 * 2           # the matrices
    assert ask(BF16, 64, 24, 64, 64 * 24, 24, 0, 5) == 0 and need.value >= 256 + 3 * 64 * 32 * 2      # halves of 12 outputs
    assert ask(BF16, 64, 24, 64, 64 * 24, 64, 1, 5) == 0 and need.value == 256                    # halves along the other axis
    assert ask(BF16, 64, 32, 64, 64 * 32, 32, at=258) == 0 and need.value >= 256 + 100 * 64 * 2   # rows that begin in the middle of a piece
    assert lib.tb200_expert_product(None, 8, None, I32, None, 48, 6, 0, None, None, 0, 0, 4, 2, 8, 6, F32, None, None, None, None, None) == 1
    for n, out in ((1, 8), (100000, 64), (100000, 4096)):
        assert lib.tb200_expert_product_grad(None, out, None, 8, None, I32, None, 8 * out, out, 0, n, 2, 8, out, BF16, F32, 0, None, None, BUF, None, ctypes.byref(need), None) == 0
        assert need.value >= 256

"""Results do not get worse with the length of a contraction: sums of numbers of one sign, which the matrix instructions make too small, always."""
import pytest
import torch

from layers_util import STORE, TINY, U

pytestmark = pytest.mark.gpu
# What a matrix instruction adds to its sum are 16 products, each cut off at a bit of the sum, and so is the sum: 17 U of it at most.  A group is 8 instructions for each of its
# stages; its sum is half as large on average as at the end.  Groups' sums are added up rounded to nearest, U each.
GROUP = {torch.float16: 32, torch.bfloat16: 128}      # stages of 128


def limit(dtype, length):
    stages = -(-length // 128)
    return STORE[dtype] + (8 * min(GROUP[dtype], stages) / 2 * 17 + -(-stages // GROUP[dtype])) * U


def inputs(dtype, *shape):
    """Around 1 / sqrt(length), so that results are around 1"""
    g = torch.Generator(device="cuda").manual_seed(sum(shape))
    return lambda length, *shape: ((0.5 + torch.rand(*shape, generator=g, device="cuda")) * length ** -0.5).to(dtype)


def check(got, want, length):
    assert bool(((got.double() - want).abs() <= limit(got.dtype, length) * want + TINY[got.dtype]).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("counts", [[1 << 20], [3, (1 << 19) + 77, 0, 200000]])
@pytest.mark.parametrize("i, o", [(64, 40), (24, 264)])
def test_gradients_of_matrices(tb, dtype, counts, i, o):
    make = inputs(dtype, sum(counts), i, o)
    offsets = torch.tensor([0] + counts, device="cuda").cumsum(0)
    x, d, w = make(max(counts), sum(counts), i), make(max(counts), sum(counts), o), make(1, len(counts), i, o)
    dw = tb.expert_product_grad(d, x, offsets, w)[1]
    at = offsets.tolist()
    for e, c in enumerate(counts):
        check(dw[e], x[at[e]:at[e + 1]].double().t() @ d[at[e]:at[e + 1]].double(), c)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lies", ["in_out", "out_in"])
@pytest.mark.parametrize("n, k", [(9, 1 << 19), (200, 1 << 19), (300, 20008), (70, 4096), (70, 4104)])
def test_products_of_long_rows(tb, dtype, lies, n, k):
    make = inputs(dtype, n, k)
    x, w = make(k, n, k), make(k, 1, k, 160) if lies == "in_out" else make(k, 1, 160, k).transpose(1, 2)
    offsets = torch.tensor([0, n], device="cuda")
    want = x.double() @ w[0].double()
    check(tb.expert_product(x, offsets, w), want, k)
    check(tb.expert_product(x, offsets, w, None, "gated_silu", keep=True)[1], want, k)
    # the same sums as a gradient of rows, by the same matrix the other way round
    check(tb.expert_product_grad(x, make(1, n, 160), offsets, w.transpose(1, 2))[0], want, k)


# 32 bits by multiply-adds.  A rounding is off by at most 2^-24 of the sum, 2^-24 / 3^0.5 of it in the norm, in either direction.  1024 of them while a sum grows evenly are a walk of
# (1024 / 3)^0.5 such steps, 6.4e-7; one of up to 512 sums of so many adds 4.5e-7; twice both together is 1.6e-6.  A chain of 500000 would be 1.4e-5, of 65536 5e-6.
LIMIT_32 = 1.6e-6


@pytest.mark.parametrize("experts, n, i, o", [(256, 500000, 64, 64), (1024, 65536, 200, 136), (1024, 66000, 33, 50), (300, 500000, 8, 300)])
def test_all_rows_of_one_of_many_experts(tb, experts, n, i, o):
    """The rows of an expert on average are few, those of one are all."""
    make = inputs(torch.float32, n, i, o)
    offsets = torch.zeros(experts + 1, dtype=torch.int32, device="cuda")
    offsets[experts // 2 + 1:] = n
    x, d, w = make(1, n, i), make(1, n, o), make(1, experts, i, o)
    dw = tb.expert_product_grad(d, x, offsets, w)[1]
    want = x.double().t() @ d.double()
    assert float((dw[experts // 2].double() - want).norm()) <= LIMIT_32 * float(want.norm())
    assert float(dw[:experts // 2].abs().max()) == 0 and float(dw[experts // 2 + 1:].abs().max()) == 0


@pytest.mark.parametrize("lies", ["in_out", "out_in"])
@pytest.mark.parametrize("activation", [None, "gated_silu"])
@pytest.mark.parametrize("n, k", [(5, 300000), (60, 70001), (200, 1024), (3, 1025), (3, 2049)])
def test_few_long_rows(tb, lies, activation, n, k):
    make = inputs(torch.float32, n, k)
    x, w = make(k, n, k), make(k, 3, k, 70) if lies == "in_out" else make(k, 3, 70, k).transpose(1, 2)
    offsets = torch.tensor([0, n // 2, n // 2, n], device="cuda")
    want = torch.cat([x[:n // 2].double() @ w[0].double(), x[n // 2:].double() @ w[2].double()])
    got = tb.expert_product(x, offsets, w, None, "gated_silu", keep=True)[1] if activation else tb.expert_product(x, offsets, w)
    assert float((got.double() - want).norm()) <= LIMIT_32 * float(want.norm())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("o", [8, 5])
def test_bias_of_one_of_many_experts(tb, dtype, o):
    """Two parts of 4000000 rows, of either 250000 a warp: 244 sums of 1024 each, as above, and the sixteen warps' walks are not one another's: a quarter of a single
    one's.  (Chains of 250000: (250000 / 3)^0.5 2^-24 / 3^0.5 / 4 = 2.5e-6.)"""
    n, experts = 4000000, 1024
    make = inputs(torch.float32, n, o)
    offsets = torch.zeros(experts + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = 7
    offsets[100:] = n - 3
    d = make(1, n, o).to(dtype)
    d[:7], d[-3:] = float("nan"), float("nan")
    db = tb.expert_product_grad(d, make(1, n, 8).to(dtype), offsets, make(1, experts, 8, o).to(dtype), bias=True)[2]
    want = d[7:-3].double().sum(0)
    assert float((db[99].double() - want).norm()) <= LIMIT_32 / 4 * float(want.norm())
    assert float(db[100:].abs().max()) == 0 and float(db[1:99].abs().max()) == 0

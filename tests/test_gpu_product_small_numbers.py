"""32-bit rows and matrices of very small numbers, as planes of 16 bits: how far results are off does not depend on how large the numbers are, nor on which kernel they come to."""
import pytest
import torch

pytestmark = pytest.mark.gpu


# The norm's bound of long sums in 32 bits, 1.9e-6, holds for any scale; the planes end at 2^-148 of half a step, which of numbers around 2^-126 are 2.4e-7.
@pytest.mark.parametrize("of", ["rows", "weight"])
@pytest.mark.parametrize("lies", ["in_out", "out_in"])
@pytest.mark.parametrize("power", [0, -100, -110, -114, -118, -122, -126])
def test_scale_does_not_matter(tb, of, lies, power):
    g = torch.Generator(device="cuda").manual_seed(power % 97)
    rand = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    counts, i, o = [90, 0, 300, 131], 264, 200
    n, offsets = sum(counts), torch.tensor([0] + counts, device="cuda").cumsum(0)
    x, d = rand(n, i), rand(n, o)
    w = rand(4, i, o) if lies == "in_out" else rand(4, o, i).transpose(1, 2)
    small = torch.tensor(power, device="cuda")
    x, d, w = (torch.ldexp(x, small), d, w) if of == "rows" else (x, torch.ldexp(d, small), torch.ldexp(w, small))
    out, (dx, dw, _) = tb.expert_product(x, offsets, w), tb.expert_product_grad(d, x, offsets, w)
    at = offsets.tolist()
    for e, c in enumerate(counts):
        r = slice(at[e], at[e + 1])
        for got, want in ((out[r], x[r].double() @ w[e].double()), (dw[e], x[r].double().t() @ d[r].double())):
            assert float((got.double() - want).norm()) <= 1.9e-6 * float(want.norm())
        if of == "rows":
            want = d[r].double() @ w[e].double().t()
            assert float((dx[r].double() - want).norm()) <= 1.9e-6 * float(want.norm())


def test_every_number_of_32_bits(tb):
    """Through a matrix of one: what three planes hold of a number, exactly down to 2^-123, to 2^-148 below."""
    g = torch.Generator(device="cuda").manual_seed(3)
    bits = torch.randint(0, 0x7f800000, (120000,), generator=g, device="cuda", dtype=torch.int32)
    bits[:2000] = torch.arange(2000, device="cuda", dtype=torch.int32)
    bits[2000:4000] = 0x7f7fffff - torch.arange(2000, device="cuda", dtype=torch.int32)
    bits[4000:6000] = 0x00800000 - 1000 + torch.arange(2000, device="cuda", dtype=torch.int32)
    bits[1::2] |= -0x80000000
    x = torch.zeros(120000, 128, device="cuda")
    x[:, 5] = bits.view(torch.float32)
    w = torch.zeros(1, 128, 128, device="cuda")
    w[0, 5] = 1.0
    out = tb.expert_product(x, torch.tensor([0, 120000], device="cuda"), w)[:, :1]
    x = x[:, 5:6]
    exact = x.abs() >= 2.0 ** -123
    assert torch.equal(out[exact], x[exact])
    assert float((out.double() - x.double()).abs()[~exact].max()) <= 2.0 ** -148


def test_large_numbers_beside_others(tb):
    """The largest numbers times numbers below one, whose products are finite."""
    top = torch.finfo(torch.float32).max
    x = torch.zeros(200, 128, device="cuda")
    x[:, 0] = torch.linspace(0.05, 1.0, 200, device="cuda") * top
    x[:, 1] = -x[:, 0] / 2
    w = torch.zeros(1, 128, 130, device="cuda")
    w[0, 0], w[0, 1] = torch.linspace(0.0, 0.9999, 130, device="cuda"), torch.linspace(0.3, 0.9, 130, device="cuda")
    offsets = torch.tensor([0, 200], device="cuda")
    want = x.double() @ w[0].double()
    error = 1e-6 * (x.double().abs() @ w[0].double().abs())
    assert bool(((tb.expert_product(x, offsets, w).double() - want).abs() <= error).all())

"""Products of many 32-bit rows of 128 channels and more, which go to the tensor cores as planes of 16 bits: everything that the products of fewer rows or channels are tested for.
And offsets that are cut off, of any type, where tiles are a pair's."""
import pytest
import torch

import products_util as ref
import test_gpu_expert_layer as whole
from test_gpu_product import ACTIVATIONS, TYPES, check, check_grad, inputs, rand

pytestmark = pytest.mark.gpu
F32 = torch.float32


@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("lies", ["in_out", "out_in"])
@pytest.mark.parametrize("i, o", [(128, 256), (200, 144), (130, 262), (257, 514), (1001, 136)])
def test_epilogue(tb, activation, lies, i, o):
    g = torch.Generator(device="cuda").manual_seed(21)
    x, offsets, w = inputs(g, [200, 70, 1, 0, 333], 1, 3, i, o, F32, lies)
    width = o // 2 if ref.halves(activation)[1] else o
    wide = rand(g, x.shape[0], width + 24)
    for bias, residual in ((None, None), (rand(g, 5, o), wide[:, 8:8 + width]), (None, wide[:, 3:3 + width])):
        out = check(tb, x, offsets, w, bias, activation, residual)
        assert out[0].abs().max() == 0 and out[-3:].abs().max() == 0


@pytest.mark.parametrize("lies", ["in_out", "out_in"])
@pytest.mark.parametrize("i, o", [(128, 264), (136, 128), (131, 300), (512, 129)])
def test_gradients_added_to_what_is_there(tb, lies, i, o):
    g = torch.Generator(device="cuda").manual_seed(22)
    x, offsets, w = inputs(g, [270, 0, 300, 9, 128], 2, 4, i, o, F32, lies, torch.int64)
    d = rand(g, x.shape[0], o)
    assert check_grad(tb, d, x, offsets, w)[1][1].abs().max() == 0
    into = rand(g, 5, i, o) if lies == "in_out" else rand(g, 5, o, i).transpose(1, 2)
    kept = into[1].clone()
    got = check_grad(tb, d, x, offsets, w, into=into)
    assert got[1] is into and torch.equal(into[1], kept)


@pytest.mark.parametrize("shift, pad", [(0, 8), (8, 16), (1, 3), (3, 8), (4, 4)])
def test_strides_and_alignment(tb, shift, pad):
    g = torch.Generator(device="cuda").manual_seed(23)
    i, o = 136, 200
    x, offsets, _ = inputs(g, [140, 0, 97, 150], 2, 2, i, o, F32, "in_out")
    n = x.shape[0]
    x = rand(g, n, i + pad + shift)[:, shift:shift + i]
    d = rand(g, n, o + pad + shift)[:, shift:shift + o]
    for w in (rand(g, 4, i, o + pad + shift)[:, :, shift:shift + o], rand(g, 4, o, i + pad + shift)[:, :, shift:shift + i].transpose(1, 2), rand(g, 4, i + 3, o)[:, 1:1 + i],
              rand(g, 4 * i * o + 40)[8 + shift:8 + shift + 4 * i * o].view(4, i, o), rand(g, 4, i * o + 64 + shift)[:, :i * o].view(4, i, o)):
        check(tb, x, offsets, w, None, "gated_silu")
        check_grad(tb, d, x, offsets, w)


@pytest.mark.parametrize("counts", [[0, 261, 100, 0, 90, 300], [128, 129, 100, 127, 3, 144]])
@pytest.mark.parametrize("i, o", [(160, 192), (133, 150), (128, 256)])
def test_nothing_of_others_reaches_a_result(tb, counts, i, o):
    g = torch.Generator(device="cuda").manual_seed(24)
    x, offsets, w = inputs(g, counts, 3, 6, i, o, F32, "in_out")
    d, b = rand(g, x.shape[0], o), rand(g, 6, o)
    out, grads = tb.expert_product(x, offsets, w, b, "gelu"), tb.expert_product_grad(d, x, offsets, w, bias=True)
    x, d, w, b, at = x.clone(), d.clone(), w.clone(), b.clone(), offsets.tolist()
    for r in list(range(at[0])) + list(range(at[-1], x.shape[0])):
        x[r], d[r] = float("nan"), float("inf")
    for e, c in enumerate(counts):
        if c == 0:
            w[e], b[e] = float("nan"), float("inf")
    assert torch.equal(tb.expert_product(x, offsets, w, b, "gelu"), out)
    assert all(torch.equal(p, q) for p, q in zip(tb.expert_product_grad(d, x, offsets, w, bias=True), grads))
    for bad in (2, 5):      # the rows of one expert, then of two: the others' results are as they were
        x[at[bad]:at[bad + 1]], d[at[bad]:at[bad + 1]] = float("nan"), float("nan")
        keep = ~x.isnan().any(1)
        keep[:at[0]], keep[at[-1]:] = True, True
        others = [e for e in range(6) if e not in (2, bad)]
        assert torch.equal(tb.expert_product(x, offsets, w, b, "gelu")[keep], out[keep])
        dx, dw, db = tb.expert_product_grad(d, x, offsets, w, bias=True)
        assert torch.equal(dx[keep], grads[0][keep]) and torch.equal(dw[others], grads[1][others]) and torch.equal(db[others], grads[2][others])
        assert dw[bad].isnan().all() and db[bad].isnan().all()


@pytest.mark.parametrize("dtype", TYPES)
def test_offsets_are_cut_off(tb, dtype):
    g = torch.Generator(device="cuda").manual_seed(25)
    x, _, w = inputs(g, [200, 300], 0, 0, 128, 136, dtype, "in_out")
    d = rand(g, 500, 136, dtype=dtype)
    for at in ([-5, 120, 100000], [500, 500, 500], [0, 0, 0], [0, 500, 500], [-7, -7, -7], [310, 2 ** 40, 2 ** 41]):
        offsets = torch.tensor(at, device="cuda")
        check(tb, x, offsets, w)
        check_grad(tb, d, x, offsets, w)


def test_same_bits(tb):
    g = torch.Generator(device="cuda").manual_seed(26)
    x, offsets, w = inputs(g, [300, 20, 0, 1000], 0, 0, 333, 517, F32, "in_out")
    d = rand(g, x.shape[0], 517)
    out, grads = tb.expert_product(x, offsets, w), tb.expert_product_grad(d, x, offsets, w, bias=True)
    for _ in range(5):
        assert torch.equal(tb.expert_product(x, offsets, w), out)
        assert all(torch.equal(p, q) for p, q in zip(tb.expert_product_grad(d, x, offsets, w, bias=True), grads))


@pytest.mark.parametrize("tokens", [500, 3000])
def test_the_whole_layer(tb, monkeypatch, tokens):
    """As that of fewer channels: the ten roundings of 32 bits and 32-bit sums of up to 750 terms."""
    monkeypatch.setattr(whole, "DIM", 160)
    monkeypatch.setattr(whole, "HIDDEN", 200)
    whole.test_layer_and_gradients(tb, dtype=F32, tokens=tokens)

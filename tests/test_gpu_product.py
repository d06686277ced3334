"""The experts' products and their gradients against plain 64-bit forms: every type, both layouts of the weights, ragged experts, odd sizes and strides."""
import pytest
import torch

import products_util as ref
from products_util import near

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
ACTIVATIONS = [None, "silu", "gelu", "gated_silu", "gated_gelu"]


def rand(g, *shape, dtype=torch.float32, scale=1.0):
    return (scale * torch.randn(*shape, generator=g, device="cuda")).to(dtype)


def inputs(g, counts, head, tail, i, o, dtype, lies, ids=torch.int32):
    n = head + sum(counts) + tail
    offsets = torch.tensor([head] + counts, device="cuda").cumsum(0).to(ids)
    x = rand(g, n, i, dtype=dtype)
    w = rand(g, len(counts), i, o, dtype=dtype, scale=i ** -0.5) if lies == "in_out" else rand(g, len(counts), o, i, dtype=dtype, scale=i ** -0.5).transpose(1, 2)
    return x, offsets, w


def check(tb, x, offsets, w, bias=None, activation=None, residual=None):
    out, before = tb.expert_product(x, offsets, w, bias, activation, residual, keep=True)
    want, wbefore, error, ebefore = ref.product(x, offsets, w, bias, activation, residual)
    near(before, wbefore, ebefore)
    near(out, want, error)
    assert torch.equal(tb.expert_product(x, offsets, w, bias, activation, residual), out)
    return out


def check_grad(tb, dout, x, offsets, w, dtype=None, into=None):
    want = ref.product_grad(dout, x, offsets, w, into)
    got = tb.expert_product_grad(dout, x, offsets, w, bias=True, dtype=dtype, out=None if into is None else into, accumulate=into is not None)
    assert got[1].stride() == w.stride() or not (w.is_contiguous() or w.transpose(1, 2).is_contiguous())
    for v, r, e in zip(got, want[:3], want[3:]):
        near(v, r, e)
    return got


# rows of the experts: none, one, around the tiles' heights of 16, 32, 64, 128 and 256
RAGGED = [[0, 1, 15, 16, 17, 0, 31, 33], [63, 64, 65, 1, 0], [127, 128, 129], [255, 256, 257, 513], [700], [0, 0, 3, 0], [0], [1]]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lies", ["in_out", "out_in"])
@pytest.mark.parametrize("counts", RAGGED, ids=lambda c: "-".join(map(str, c)))
def test_ragged_experts(tb, dtype, lies, counts):
    g = torch.Generator(device="cuda").manual_seed(1)
    x, offsets, w = inputs(g, counts, 3, 5, 128, 192, dtype, lies)
    check(tb, x, offsets, w)
    check_grad(tb, rand(g, x.shape[0], 192, dtype=dtype), x, offsets, w)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lies", ["in_out", "out_in"])
@pytest.mark.parametrize("i, o", [(8, 8), (16, 136), (64, 128), (72, 264), (200, 120), (1, 1), (7, 9), (63, 129), (65, 2), (1000, 40), (128, 1001), (2056, 16)])
@pytest.mark.parametrize("counts", [[5, 0, 20], [130, 0, 75, 301]], ids=["few", "many"])
def test_sizes(tb, dtype, lies, i, o, counts):
    g = torch.Generator(device="cuda").manual_seed(2)
    x, offsets, w = inputs(g, counts, 0, 2, i, o, dtype, lies, torch.int64)
    check(tb, x, offsets, w, rand(g, len(counts), o, dtype=dtype), "silu")
    check_grad(tb, rand(g, x.shape[0], o, dtype=dtype), x, offsets, w)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("lies", ["in_out", "out_in"])
@pytest.mark.parametrize("o", [64, 144, 262, 514])
def test_epilogue(tb, dtype, activation, lies, o):
    g = torch.Generator(device="cuda").manual_seed(3)
    for counts in ([9, 0, 30], [200, 70, 1]):
        x, offsets, w = inputs(g, counts, 1, 3, 96, o, dtype, lies)
        width = o // 2 if ref.halves(activation)[1] else o
        wide = rand(g, x.shape[0], width + 24, dtype=dtype)
        for bias, residual in ((None, None), (rand(g, len(counts), o, dtype=dtype), wide[:, 8:8 + width])):
            out = check(tb, x, offsets, w, bias, activation, residual)
            assert out[0].abs().max() == 0 and out[-3:].abs().max() == 0


@pytest.mark.parametrize("dtype", TYPES)
def test_activations_far_out(tb, dtype):
    """Arguments of all sizes, through a matrix of one."""
    x = torch.cat([torch.linspace(-60, 60, 2001, device="cuda"), torch.tensor([0.0, -0.0, 1e-6, -1e-6, 300.0, -300.0, 60000.0, -60000.0], device="cuda")]).to(dtype)[:, None]
    offsets = torch.tensor([0, x.shape[0]], device="cuda")
    for activation in ("silu", "gelu"):
        check(tb, x, offsets, torch.ones(1, 1, 1, dtype=dtype, device="cuda"), None, activation)
    for activation in ("gated_silu", "gated_gelu"):
        check(tb, x, offsets, torch.tensor([[[1.0, 0.5]]], dtype=dtype, device="cuda"), None, activation)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("activation", ACTIVATIONS[1:])
@pytest.mark.parametrize("n, width", [(1, 1), (3, 8), (130, 72), (17, 333), (1000, 1024), (0, 16)])
def test_activation_grad(tb, dtype, activation, n, width):
    g = torch.Generator(device="cuda").manual_seed(4)
    before = rand(g, n, width * (2 if ref.halves(activation)[1] else 1), dtype=dtype, scale=3.0)
    if n > 100:
        before[:50] *= 8
    for dout in (rand(g, n, width, dtype=dtype), rand(g, n, width + 8, dtype=dtype)[:, 8:], rand(g, n, width + 3, dtype=dtype)[:, 2:2 + width]):
        got = tb.expert_activation_grad(dout, before, activation)
        want, error = ref.activation_grad(dout, before, activation)
        near(got, want, error)


@pytest.mark.parametrize("activation", ACTIVATIONS[1:])
def test_activation_grad_against_differences(tb, activation):
    g = torch.Generator(device="cuda").manual_seed(5)
    gated = ref.halves(activation)[1]
    x, d = 2 * torch.randn(40, 32, generator=g, device="cuda", dtype=torch.float64), torch.randn(40, 16 if gated else 32, generator=g, device="cuda", dtype=torch.float64)
    name = ref.halves(activation)[0]
    f = lambda x: ref.act(x[:, :16], name)[0] * x[:, 16:] if gated else ref.act(x, name)[0]  # noqa: E731
    got = tb.expert_activation_grad(d.float(), x.float(), activation).double()
    h = 1e-5
    for c in (0, 5, 15, 16, 31):
        e = torch.zeros_like(x)
        e[:, c] = h
        slope = ((f(x.float().double() + e) - f(x.float().double() - e)) * d.float().double()).sum(1) / (2 * h)
        # a third derivative of at most 2 (times d) leaves h^2 / 3, the difference of rounded values 2^-50 / h
        torch.testing.assert_close(got[:, c], slope, rtol=1e-5, atol=1e-6)


def test_product_grad_against_differences(tb):
    """The whole way, by rows, weight and bias, in 32 bits."""
    g = torch.Generator(device="cuda").manual_seed(6)
    x, offsets, w = inputs(g, [5, 0, 12], 1, 2, 24, 20, torch.float32, "in_out")
    b, d = rand(g, 3, 20), rand(g, x.shape[0], 10)
    out, before = tb.expert_product(x, offsets, w, b, "gated_gelu", keep=True)
    dbefore = tb.expert_activation_grad(d, before, "gated_gelu")
    dx, dw, db = tb.expert_product_grad(dbefore, x, offsets, w, bias=True)
    f = lambda x, w, b: (ref.product(x, offsets, w, b, "gated_gelu")[0] * d.double()).sum()  # noqa: E731
    x64, w64, b64, h = x.double(), w.double(), b.double(), 1e-5
    for t, got, which in ((x64, dx, [(1, 0), (3, 7), (17, 23), (0, 4), (19, 2)]), (w64, dw, [(0, 0, 0), (2, 23, 19), (1, 3, 3), (0, 11, 10)]), (b64, db, [(0, 0), (2, 19), (1, 5)])):
        for at in which:
            t[at] += h
            up = f(x64, w64, b64)
            t[at] -= 2 * h
            down = f(x64, w64, b64)
            t[at] += h
            assert abs(float(got[at]) - float(up - down) / (2 * h)) < 1e-4 * (1 + abs(float(got[at])))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lies", ["in_out", "out_in"])
def test_gradient_types_and_accumulation(tb, dtype, lies):
    g = torch.Generator(device="cuda").manual_seed(7)
    x, offsets, w = inputs(g, [70, 0, 300, 9], 0, 4, 80, 264, dtype, lies)
    d = rand(g, x.shape[0], 264, dtype=dtype)
    for to in {dtype, torch.float32}:
        got = check_grad(tb, d, x, offsets, w, dtype=to)
        assert got[1].dtype == to and got[1][1].abs().max() == 0
        into = rand(g, 4, 80, 264, dtype=to) if lies == "in_out" else rand(g, 4, 264, 80, dtype=to).transpose(1, 2)
        kept = into[1].clone()
        got = check_grad(tb, d, x, offsets, w, into=into)
        assert got[1] is into and torch.equal(into[1], kept)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shift, pad", [(0, 8), (8, 16), (1, 3), (3, 8), (4, 4)])
def test_strides_and_alignment(tb, dtype, shift, pad):
    g = torch.Generator(device="cuda").manual_seed(8)
    counts, i, o = [40, 0, 7, 150], 72, 136
    x, offsets, _ = inputs(g, counts, 2, 2, i, o, dtype, "in_out")
    n = x.shape[0]
    x = rand(g, n, i + pad + shift, dtype=dtype)[:, shift:shift + i]
    d = rand(g, n, o + pad + shift, dtype=dtype)[:, shift:shift + o]
    for w in (rand(g, 4, i, o + pad + shift, dtype=dtype)[:, :, shift:shift + o], rand(g, 4, o, i + pad + shift, dtype=dtype)[:, :, shift:shift + i].transpose(1, 2),
              rand(g, 4, i + 3, o, dtype=dtype)[:, 1:1 + i], rand(g, 4 * i * o + 40, dtype=dtype)[8 + shift:8 + shift + 4 * i * o].view(4, i, o),
              rand(g, 4, i * o + 64 + shift, dtype=dtype)[:, :i * o].view(4, i, o)):
        check(tb, x, offsets, w, None, "gated_silu")
        check_grad(tb, d, x, offsets, w)


@pytest.mark.parametrize("dtype", TYPES)
def test_nothing_of_others_reaches_a_result(tb, dtype):
    """NaNs and infinities in the rows of no expert, of other experts, and in the matrices of experts without rows."""
    g = torch.Generator(device="cuda").manual_seed(9)
    for counts in ([5, 0, 37, 2, 0, 70], [0, 261, 100, 0, 90, 300]):
        for i, o in ((96, 160), (33, 50)):
            x, offsets, w = inputs(g, counts, 3, 6, i, o, dtype, "in_out")
            d, b = rand(g, x.shape[0], o, dtype=dtype), rand(g, 6, o, dtype=dtype)
            out = tb.expert_product(x, offsets, w, b, "gelu")
            grads = tb.expert_product_grad(d, x, offsets, w, bias=True)
            x2, w2, d2, b2 = x.clone(), w.clone(), d.clone(), b.clone()
            at = offsets.tolist()
            for r in list(range(at[0])) + list(range(at[-1], x.shape[0])):
                x2[r], d2[r] = float("nan"), float("inf")
            for e, c in enumerate(counts):
                if c == 0:
                    w2[e], b2[e] = float("nan"), float("inf")
            assert torch.equal(tb.expert_product(x2, offsets, w2, b2, "gelu"), out)
            for p, q in zip(tb.expert_product_grad(d2, x2, offsets, w2, bias=True), grads):
                assert torch.equal(p, q)
            # one expert's rows are NaN: the others' results are as they were
            bad = next(e for e, c in enumerate(counts) if c and e > 1)
            x2[at[bad]:at[bad + 1]], d2[at[bad]:at[bad + 1]] = float("nan"), float("nan")
            keep = torch.ones(x.shape[0], dtype=torch.bool, device="cuda")
            keep[at[bad]:at[bad + 1]] = False
            others = [e for e in range(6) if e != bad]
            assert torch.equal(tb.expert_product(x2, offsets, w2, b2, "gelu")[keep], out[keep])
            dx, dw, db = tb.expert_product_grad(d2, x2, offsets, w2, bias=True)
            assert torch.equal(dx[keep], grads[0][keep]) and torch.equal(dw[others], grads[1][others]) and torch.equal(db[others], grads[2][others])
            assert dw[bad].isnan().all() and db[bad].isnan().all()


@pytest.mark.parametrize("dtype", TYPES)
def test_offsets_are_cut_off(tb, dtype):
    g = torch.Generator(device="cuda").manual_seed(10)
    x, _, w = inputs(g, [50, 50], 0, 0, 64, 64, dtype, "in_out")
    d = rand(g, 100, 64, dtype=dtype)
    for at in ([-5, 20, 1000], [100, 100, 100], [0, 0, 0], [0, 100, 100], [-7, -7, -7], [10, 2 ** 40, 2 ** 41]):
        offsets = torch.tensor(at, device="cuda")
        check(tb, x, offsets, w)
        check_grad(tb, d, x, offsets, w)


def test_nothing_to_do(tb):
    e = lambda *shape: torch.ones(*shape, device="cuda", dtype=torch.bfloat16)  # noqa: E731
    offsets = torch.tensor([0, 0, 0], device="cuda")
    assert tb.expert_product(e(0, 8), offsets, e(2, 8, 16)).shape == (0, 16)
    dx, dw, db = tb.expert_product_grad(e(0, 16), e(0, 8), offsets, e(2, 8, 16), bias=True)
    assert dx.shape == (0, 8) and dw.abs().max() == 0 and db.abs().max() == 0
    # no inputs: what is left is the bias; no outputs: nothing
    offsets = torch.tensor([1, 3, 5], device="cuda")
    out = tb.expert_product(e(6, 0), offsets, e(2, 0, 4), 3 * e(2, 4))
    assert torch.equal(out, 3 * e(6, 4) * torch.tensor([0, 1, 1, 1, 1, 0], device="cuda")[:, None])
    dx, dw, db = tb.expert_product_grad(e(6, 4), e(6, 0), offsets, e(2, 0, 4), bias=True)
    assert dx.shape == (6, 0) and dw.shape == (2, 0, 4) and torch.equal(db, torch.full((2, 4), 2.0, device="cuda"))
    assert tb.expert_product(e(6, 3), offsets, e(2, 3, 0)).shape == (6, 0)
    dx, dw, db = tb.expert_product_grad(e(6, 0), e(6, 3), offsets, e(2, 3, 0), bias=True)
    assert dx.abs().max() == 0 and dw.shape == (2, 3, 0) and db.shape == (2, 0)


@pytest.mark.parametrize("dtype", TYPES)
def test_many_experts_and_many_tiles(tb, dtype):
    g = torch.Generator(device="cuda").manual_seed(11)
    counts = torch.randint(0, 9, (1024,), generator=g, device="cuda").tolist()
    x, offsets, w = inputs(g, counts, 0, 0, 64, 72, dtype, "out_in")
    check(tb, x, offsets, w)
    check_grad(tb, rand(g, x.shape[0], 72, dtype=dtype), x, offsets, w)
    counts = (torch.randint(0, 900, (30,), generator=g, device="cuda")).tolist()
    x, offsets, w = inputs(g, counts, 0, 77, 320, 1100, dtype, "in_out")
    check(tb, x, offsets, w, None, "gated_gelu")
    check_grad(tb, rand(g, x.shape[0], 1100, dtype=dtype), x, offsets, w)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_long_contractions(tb, dtype):
    g = torch.Generator(device="cuda").manual_seed(12)
    x, offsets, w = inputs(g, [20, 3], 0, 0, 8192, 96, dtype, "out_in")
    check(tb, x, offsets, w, None, "gated_silu")
    x, offsets, w = inputs(g, [5001], 0, 0, 64, 40, dtype, "in_out")
    check_grad(tb, rand(g, 5001, 40, dtype=dtype), x, offsets, w, dtype=torch.float32)


def test_same_bits(tb):
    g = torch.Generator(device="cuda").manual_seed(13)
    x, offsets, w = inputs(g, [300, 20, 0, 1000], 0, 0, 512, 512, torch.bfloat16, "in_out")
    d = rand(g, x.shape[0], 512, dtype=torch.bfloat16)
    out, grads = tb.expert_product(x, offsets, w), tb.expert_product_grad(d, x, offsets, w, bias=True, dtype=torch.float32)
    for _ in range(5):
        assert torch.equal(tb.expert_product(x, offsets, w), out)
        for p, q in zip(tb.expert_product_grad(d, x, offsets, w, bias=True, dtype=torch.float32), grads):
            assert torch.equal(p, q)


@pytest.mark.parametrize("i, o", [(128, 256), (65, 100)])
def test_streams_and_graphs(tb, i, o):
    g = torch.Generator(device="cuda").manual_seed(14)
    x, offsets, w = inputs(g, [130, 0, 20, 77], 0, 3, i, o, torch.bfloat16, "in_out")
    d = rand(g, x.shape[0], o, dtype=torch.bfloat16)
    run = lambda: (*tb.expert_product(x, offsets, w, None, "gated_silu", keep=True), *tb.expert_product_grad(d, x, offsets, w, bias=True))  # noqa: E731
    want = run()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    results = []
    for s in streams * 4:      # at the same time, each with its own workspace
        with torch.cuda.stream(s):
            results.append(run())
    torch.cuda.synchronize()
    for r in results:
        assert all(torch.equal(p, q) for p, q in zip(r, want))
    with torch.cuda.stream(streams[0]):
        run()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=streams[0]):
            got = run()
    x.copy_(rand(g, *x.shape, dtype=torch.bfloat16))
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, run()))


def test_refusals(tb):
    e = lambda *shape, dtype=torch.bfloat16: torch.ones(*shape, device="cuda", dtype=dtype)  # noqa: E731
    offsets = torch.tensor([0, 4, 8], device="cuda")
    x, w, d = e(8, 16), e(2, 16, 32), e(8, 32)
    for call in (lambda: tb.expert_product(x.double(), offsets, w.double()), lambda: tb.expert_product(x, offsets, w.float()), lambda: tb.expert_product(x, offsets[:2], w),
                 lambda: tb.expert_product(x, offsets.float(), w), lambda: tb.expert_product(x, offsets, w[0]), lambda: tb.expert_product(e(8, 15), offsets, w),
                 lambda: tb.expert_product(x, offsets, w, activation="tanh"), lambda: tb.expert_product(x, offsets, e(2, 16, 31), activation="gated_silu"),
                 lambda: tb.expert_product(x, offsets, w, e(2, 31)), lambda: tb.expert_product(x, offsets, w, e(2, 32, dtype=torch.float32)),
                 lambda: tb.expert_product(x, offsets, w, None, None, e(8, 31)), lambda: tb.expert_product(x, offsets, w, None, "gated_silu", e(8, 32)),
                 lambda: tb.expert_product(x, offsets, w[:1].expand(2, 16, 32)), lambda: tb.expert_product(x, offsets, e(2, 16, 64)[:, :, ::2]),
                 lambda: tb.expert_product(x, offsets, w.cpu()), lambda: tb.expert_product(x, offsets.cpu(), w), lambda: tb.expert_product(x.t(), offsets, w),
                 lambda: tb.expert_product_grad(e(8, 31), x, offsets, w), lambda: tb.expert_product_grad(d, x, offsets, w, accumulate=True),
                 lambda: tb.expert_product_grad(d, x, offsets, w, dtype=torch.float16), lambda: tb.expert_product_grad(d, x, offsets, w, out=e(2, 32, 16)),
                 lambda: tb.expert_product_grad(d, x, offsets, w, out=e(2, 32, 16).transpose(1, 2)), lambda: tb.expert_activation_grad(d, d, None),
                 lambda: tb.expert_activation_grad(d, d, "gated_silu"), lambda: tb.expert_activation_grad(d, d.float(), "silu"),
                 lambda: tb.expert_activation_grad(d, e(8, 64)[:, ::2], "silu")):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("dtype", TYPES)
def test_graphs_side_by_side(tb, dtype):
    """Two graphs captured on one stream, with operands that are laid out anew, replayed at the same time."""
    g = torch.Generator(device="cuda").manual_seed(15)
    capture, streams, graphs, results, wants = torch.cuda.Stream(), [torch.cuda.Stream(), torch.cuda.Stream()], [], [], []
    for counts in ([700, 0, 900, 811], [1500, 33, 640, 2]):
        x, offsets, w = inputs(g, counts, 0, 3, 333, 517, dtype, "in_out")
        d = rand(g, x.shape[0], 517, dtype=dtype)
        wants.append((tb.expert_product(x, offsets, w), *tb.expert_product_grad(d, x, offsets, w, bias=True)))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=capture):
            results.append((tb.expert_product(x, offsets, w), *tb.expert_product_grad(d, x, offsets, w, bias=True)))
        graphs.append((graph, x, offsets, w, d))
    for _ in range(10):
        for s, (graph, *_) in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for got, want in zip(results, wants):
        assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("dtype", TYPES)
def test_long_sums_in_32_bits(tb, dtype):
    """32-bit results do not get worse with the length of the contraction.  The matrix instructions cut off what they add up to, 2^-24 of it on average, and what
    they add up to is two thirds of the result on average: 48 of them between sums that are rounded (24 by rows) are 1.9e-6; without those sums 30000 rows
    would be 7e-5."""
    g = torch.Generator(device="cuda").manual_seed(16)
    x, offsets, w = inputs(g, [30000], 0, 0, 72, 136, dtype, "in_out")
    d = rand(g, 30000, 136, dtype=dtype)
    want = x.double().t() @ d.double()
    got = tb.expert_product_grad(d, x, offsets, w, dtype=torch.float32)[1][0].double()
    assert float((got - want).norm()) <= 1.9e-6 * float(want.norm())
    if dtype == torch.float32:
        x, offsets, w = inputs(g, [400], 0, 0, 6000, 128, dtype, "out_in")
        want = x.double() @ w[0].double()
        assert float((tb.expert_product(x, offsets, w).double() - want).norm()) <= 1.9e-6 * float(want.norm())


def test_numbers_at_the_ends_of_32_bits(tb):
    """As three planes of 16 bits: the largest and the smallest numbers, and infinities, which leave what is not finite and stay in their rows."""
    x = torch.zeros(200, 128, device="cuda")
    x[:, 0] = 1.0
    x[0, 0], x[1, 0], x[2, 0], x[3, 0], x[4, 0] = torch.finfo(torch.float32).max, -3.3961e38, 1e-30, 1.1754944e-38, 1 + 2.0 ** -23
    x[5, 3], x[6, 3] = float("inf"), float("-inf")
    w = torch.zeros(1, 128, 128, device="cuda")
    w[0, 0] = 1.0
    w[0, 3] = 0.5
    offsets = torch.tensor([0, 200], device="cuda")
    out = tb.expert_product(x, offsets, w)
    assert torch.equal(out[:5], x[:5, :1].expand(5, 128)) and torch.equal(out[7:], torch.ones(193, 128, device="cuda"))
    assert not out[5:7].isfinite().any()

"""The router and its gradient against plain 64-bit forms: scores, biases, groups, closed experts, ties, and choices near a border."""
import math

import pytest
import torch

import products_util as ref
from layers_util import STORE, U

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def check(tb, logits, choices, **how):
    experts, weights = tb.expert_route(logits, choices, **{k if k != "kind" else "scores": v for k, v in how.items()})
    want, w = ref.route(logits, choices, **how)
    assert experts.dtype == torch.int32 and weights.dtype == torch.float32
    assert torch.equal(experts.cpu(), want), "at %s" % torch.nonzero(experts.cpu() != want)[:3].tolist()
    # exponentials of rounded differences d: (2 + |d|) 2u each, at most exp(-|d|) of the largest, sums of up to 1024 of them in 37 additions, two quotients
    torch.testing.assert_close(weights.cpu().double(), w, rtol=100 * U, atol=1e-37)
    return experts, weights


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("n, e, k", [(1, 1, 1), (3, 2, 2), (50, 7, 3), (40, 32, 32), (33, 33, 4), (64, 60, 8), (100, 128, 8), (30, 200, 6), (20, 257, 5), (9, 600, 32), (7, 1024, 10)])
def test_choices(tb, dtype, kind, biased, n, e, k):
    g = torch.Generator(device="cuda").manual_seed(1)
    logits = torch.randn(n, e, generator=g, device="cuda").to(dtype)
    bias = 0.1 * torch.randn(e, generator=g, device="cuda") if biased else None
    for renormalize, scale in ((True, 1.0), (False, 2.5)):
        check(tb, logits, k, kind=kind, bias=bias, renormalize=renormalize, scale=scale)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("best", [1, 2])
@pytest.mark.parametrize("e, groups, kept, k", [(8, 8, 3, 2), (64, 4, 2, 6), (256, 8, 4, 8), (96, 32, 5, 7), (14, 2, 1, 7), (1024, 16, 3, 16), (30, 3, 3, 4)])
def test_groups(tb, dtype, kind, biased, best, e, groups, kept, k):
    g = torch.Generator(device="cuda").manual_seed(2)
    logits = torch.randn(60, e, generator=g, device="cuda").to(dtype)
    logits[::3] = torch.where(torch.rand(20, e, generator=g, device="cuda") < 0.5, -math.inf, logits[::3])
    bias = 0.2 * torch.randn(e, generator=g, device="cuda") if biased else None
    check(tb, logits, k, kind=kind, bias=bias, groups=groups, group_choices=kept, group_best=best)


@pytest.mark.parametrize("kind", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
def test_closed_experts_and_rows_without_any(tb, kind, biased):
    g = torch.Generator(device="cuda").manual_seed(3)
    logits = torch.randn(12, 40, generator=g, device="cuda")
    logits[1] = -math.inf
    logits[2] = math.nan
    logits[3, 3:] = -math.inf
    logits[4, ::2] = math.nan
    logits[5, 7] = math.inf
    logits[6, 5:9] = math.inf
    logits[7] = torch.finfo(torch.float32).min
    logits[8, 1:] = torch.finfo(torch.float32).min
    logits[9] = 0.0
    logits[9, ::2] = -0.0
    bias = 0.1 * torch.randn(40, generator=g, device="cuda") if biased else None
    if biased:
        bias[10], bias[11] = -math.inf, math.nan
    rows = [r for r in range(12) if r != 7 or kind == "softmax"]      # (the sigmoid of row 7 vanishes in 64 bits)
    for renormalize in (True, False):
        experts, weights = check(tb, logits[rows], 6, kind=kind, bias=bias, renormalize=renormalize)
        assert (experts[1:3] == -1).all() and (weights[1:3] == 0).all()
        assert (experts[3] >= 0).sum() == 3
    # quotients of scores that vanish
    low = torch.full((1, 8), -300.0, device="cuda")
    low[0, 3] += math.log(3.0)
    experts, weights = tb.expert_route(low, 2, "sigmoid")
    assert experts.tolist() == [[3, 0]]
    torch.testing.assert_close(weights, torch.tensor([[0.75, 0.25]], device="cuda"), rtol=3e-5, atol=0)      # (-300 + log 3 is rounded to 2^-16)
    experts, weights = tb.expert_route(logits[7:8], 4, "sigmoid")
    assert experts.tolist() == [[0, 1, 2, 3]] and weights.tolist() == [[0.25] * 4]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["softmax", "sigmoid"])
def test_ties_go_to_the_lower_index(tb, dtype, kind):
    g = torch.Generator(device="cuda").manual_seed(4)
    logits = torch.randint(-2, 3, (64, 96), generator=g, device="cuda").to(dtype) / 2
    levels = torch.randint(0, 3, (96,), generator=g, device="cuda").float() / 4
    for bias in (None, torch.zeros(96, device="cuda"), levels):
        check(tb, logits, 8, kind=kind, bias=bias)
        check(tb, logits, 8, kind=kind, bias=bias, groups=8, group_choices=3, group_best=1)
        check(tb, logits, 8, kind=kind, bias=bias, groups=8, group_choices=3, group_best=2)


@pytest.mark.parametrize("kind", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups", [1, 4])
def test_choices_nearer_than_32_bits_tell(tb, kind, groups):
    """Biases that make up for the scores to a few parts in 10^8: 32-bit sums of the two are equal or the wrong way round, 64-bit ones tell."""
    g = torch.Generator(device="cuda").manual_seed(5)
    n, e = 200, 48
    logits = torch.randn(1, e, generator=g, device="cuda").expand(n, e) + 1e-6 * torch.randn(n, e, generator=g, device="cuda")
    score = ref.scores(logits[:1], kind)[0][0]
    bias = (1.0 - score).float()
    experts, _ = check(tb, logits, 6, kind=kind, bias=bias, groups=groups, group_choices=(groups + 1) // 2)
    assert len({tuple(r) for r in experts.tolist()}) > 20


def test_strides_streams_and_graphs(tb):
    g = torch.Generator(device="cuda").manual_seed(6)
    wide = torch.randn(500, 150, generator=g, device="cuda")
    logits = wide[:, 11:75]
    d = torch.randn(500, 4, generator=g, device="cuda")
    want, w = check(tb, logits, 4)
    assert torch.equal(tb.expert_route(logits.contiguous(), 4)[1], w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            experts, weights = tb.expert_route(logits, 4)
            dlogits = tb.expert_route_grad(d, experts, logits)
    wide.copy_(torch.randn(500, 150, generator=g, device="cuda"))
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    want, w = check(tb, logits, 4)
    assert torch.equal(experts, want) and torch.equal(weights, w) and torch.equal(dlogits, tb.expert_route_grad(d, want, logits))


def near_grad(got, want, dweights, scale):
    """Products and sums of up to 64 weights times gradients: 40 roundings of what is at most scale times the largest gradient, twice"""
    size = scale * dweights.double().abs().amax(1, keepdim=True)
    bound = 200 * U * size + STORE[got.dtype] * want.abs() + 2.0 ** -24 * (got.dtype == torch.float16)
    assert ((got.double() - want).abs() <= bound).all(), float(((got.double() - want).abs() - bound).max())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
@pytest.mark.parametrize("n, e, k", [(1, 1, 1), (5, 3, 2), (70, 64, 6), (33, 33, 4), (40, 200, 8), (9, 1000, 32), (20, 1024, 3)])
def test_gradient(tb, dtype, kind, renormalize, n, e, k):
    g = torch.Generator(device="cuda").manual_seed(7)
    logits = (2 * torch.randn(n, e, generator=g, device="cuda")).to(dtype)
    if e > 10:
        logits = torch.where(torch.rand(n, e, generator=g, device="cuda") < 0.1, -math.inf, logits)
        logits[-1, 2:] = -math.inf
        logits[0, 1] = math.nan
    experts, _ = tb.expert_route(logits, k, kind)
    d = torch.randn(n, k, generator=g, device="cuda")
    want = ref.route_grad(d, experts, logits, kind, renormalize, 1.5)
    got = tb.expert_route_grad(torch.where(experts < 0, math.nan, d), experts, logits, kind, renormalize, 1.5)
    assert got.dtype == dtype
    near_grad(got, want, d, 1.5)
    assert (got[~(logits > -math.inf)] == 0).all()


@pytest.mark.parametrize("kind", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
def test_gradient_of_the_same_expert_twice_and_of_none(tb, kind, renormalize):
    g = torch.Generator(device="cuda").manual_seed(8)
    logits = torch.randn(6, 16, generator=g, device="cuda")
    logits[4] = -math.inf
    experts = torch.tensor([[3, 3, 1], [-1, 5, 5], [-1, -1, -1], [16, 2, -7], [0, 1, 2], [7, 7, 7]], dtype=torch.int32, device="cuda")
    d = torch.randn(6, 3, generator=g, device="cuda")
    got = tb.expert_route_grad(d, experts, logits, kind, renormalize)
    near_grad(got, ref.route_grad(d, experts, logits, kind, renormalize), d, 1.0)
    assert (got[2] == 0).all() and (got[4] == 0).all()


@pytest.mark.parametrize("kind", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
def test_gradient_against_differences(tb, kind, renormalize):
    g = torch.Generator(device="cuda").manual_seed(9)
    logits, d = torch.randn(8, 12, generator=g, device="cuda"), torch.randn(8, 3, generator=g, device="cuda")
    experts, _ = tb.expert_route(logits, 3, kind, renormalize=renormalize)
    got = tb.expert_route_grad(d, experts, logits, kind, renormalize).double()

    def f(x):
        s = torch.softmax(x, 1) if kind == "softmax" else torch.sigmoid(x)
        w = torch.gather(s, 1, experts.long())
        return ((w / w.sum(1, keepdim=True) if renormalize else w) * d.double()).sum(1)
    h = 1e-5
    for c in range(12):
        x = logits.double().clone()
        x[:, c] += h
        up = f(x)
        x[:, c] -= 2 * h
        torch.testing.assert_close(got[:, c], (up - f(x)) / (2 * h), rtol=1e-5, atol=1e-6)


def test_nothing_to_do(tb):
    experts, weights = tb.expert_route(torch.empty(0, 8, device="cuda"), 2)
    assert experts.shape == weights.shape == (0, 2)
    assert tb.expert_route_grad(weights, experts, torch.empty(0, 8, device="cuda")).shape == (0, 8)


def test_refusals(tb):
    x = torch.zeros(4, 8, device="cuda")
    d, e = torch.zeros(4, 2, device="cuda"), torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    for call in (lambda: tb.expert_route(x, 0), lambda: tb.expert_route(x, 9), lambda: tb.expert_route(x, 2, "cosine"), lambda: tb.expert_route(x.double(), 2),
                 lambda: tb.expert_route(torch.zeros(4, 1025, device="cuda"), 2), lambda: tb.expert_route(x[0], 2), lambda: tb.expert_route(x, 2, groups=3),
                 lambda: tb.expert_route(x, 2, groups=4, group_choices=5), lambda: tb.expert_route(x, 2, groups=4, group_best=3), lambda: tb.expert_route(x.t(), 2),
                 lambda: tb.expert_route(x, 2, bias=torch.zeros(7, device="cuda")), lambda: tb.expert_route(x, 2, bias=torch.zeros(8, device="cuda").half()),
                 lambda: tb.expert_route(x, 2, bias=torch.zeros(8)), lambda: tb.expert_route_grad(d, e.long(), x), lambda: tb.expert_route_grad(d[:3], e, x),
                 lambda: tb.expert_route_grad(d.half(), e, x), lambda: tb.expert_route_grad(d, e[0], x)):
        with pytest.raises(ValueError):
            call()

"""Router, dispatch, two products and combination together, forward and back, as a layer of a model has them, against the same in 64 bits by autograd."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DIM, HIDDEN, EXPERTS, CHOICES = 96, 160, 12, 3


def layer(tb, x, router, bias, w1, w2, b2, keep=False):
    """What a program calls; keep: with what the way back needs."""
    logits = x @ router
    experts, weights = tb.expert_route(logits, CHOICES, "sigmoid", bias, groups=4, group_choices=2, scale=1.5)
    rows, plan = tb.expert_dispatch(x, experts, EXPERTS)
    made = tb.expert_product(rows, plan.offsets, w1, None, "gated_silu", keep=keep)
    hidden, before = made if keep else (made, None)
    out = tb.expert_product(hidden, plan.offsets, w2, b2)
    y = tb.expert_combine(out, plan, weights)
    return (y, (logits, experts, weights, rows, plan, before, hidden, out)) if keep else y


def back(tb, dy, kept, x, router, w1, w2):
    logits, experts, weights, rows, plan, before, hidden, out = kept
    dout, dweights = tb.expert_combine_grad(dy, out, plan, weights)
    dhidden, dw2, db2 = tb.expert_product_grad(dout, hidden, plan.offsets, w2, bias=True, dtype=torch.float32)
    dbefore = tb.expert_activation_grad(dhidden, before, "gated_silu")
    drows, dw1, _ = tb.expert_product_grad(dbefore, rows, plan.offsets, w1, dtype=torch.float32)
    dlogits = tb.expert_route_grad(dweights, experts, logits, "sigmoid", scale=1.5)
    return tb.expert_dispatch_grad(drows, plan) + dlogits @ router.t(), x.t() @ dlogits, dw1, dw2, db2


def reference(x, router, w1, w2, b2, experts):
    """In 64 bits, token by token and choice by choice; the choice is given."""
    score = torch.sigmoid(x @ router)
    y = torch.zeros(x.shape[0], DIM, dtype=torch.float64, device="cuda")
    chosen = experts >= 0
    w = torch.where(chosen, torch.gather(score, 1, experts.clamp(min=0).long()), 0.0)
    w = 1.5 * w / w.sum(1, keepdim=True).clamp(min=1e-300)
    for e in range(EXPERTS):
        t, c = torch.nonzero(experts == e, as_tuple=True)
        h = x[t] @ w1[e]
        h = torch.nn.functional.silu(h[:, :HIDDEN]) * h[:, HIDDEN:]
        y = y.index_add(0, t, (h @ w2[e] + b2[e]) * w[t, c][:, None])
    return y


def inputs(tokens, dtype):
    g = torch.Generator(device="cuda").manual_seed(1)
    rand = lambda *shape, scale=1.0: (scale * torch.randn(*shape, generator=g, device="cuda")).to(dtype)  # noqa: E731
    return (rand(tokens, DIM), rand(DIM, EXPERTS, scale=DIM ** -0.5), 0.1 * torch.randn(EXPERTS, generator=g, device="cuda"), rand(EXPERTS, DIM, 2 * HIDDEN, scale=DIM ** -0.5),
            rand(EXPERTS, DIM, HIDDEN, scale=HIDDEN ** -0.5).transpose(1, 2), rand(EXPERTS, DIM, scale=0.1)), rand(tokens, DIM)


# Each of the five tensors between input and output is rounded once on the way there and once on the way back: ten halves of a step, of values that are sums of many, so
# that they add up like steps of a walk at most: eps / 2 * 10, in the norm.  32-bit sums of up to 480 terms add less than that of 32 bits.
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tokens", [1, 7, 500, 3000])
def test_layer_and_gradients(tb, dtype, tokens):
    (x, router, bias, w1, w2, b2), dy = inputs(tokens, dtype)
    y, kept = layer(tb, x, router, bias, w1, w2, b2, keep=True)
    assert torch.equal(layer(tb, x, router, bias, w1, w2, b2), y)
    leaves = [t.double().detach().requires_grad_() for t in (x, router, w1, w2, b2)]
    want = reference(*leaves, kept[1])
    want.backward(dy.double())
    tolerance = 10 * torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 2e-5
    for got, ref in zip((y, *back(tb, dy, kept, x, router, w1, w2)), (want.detach(), *(t.grad for t in leaves))):
        assert float((got.double() - ref).norm()) <= tolerance * float(ref.norm()) + 1e-12


def test_one_token_at_a_time(tb):
    """Tokens by themselves take the kernels for few rows, all together those for many."""
    (x, router, bias, w1, w2, b2), _ = inputs(600, torch.bfloat16)
    y = layer(tb, x, router, bias, w1, w2, b2)
    for t in (0, 1, 17, 599):
        one = layer(tb, x[t:t + 1], router, bias, w1, w2, b2)
        assert float((one.double() - y[t:t + 1].double()).norm()) <= 6 * 2.0 ** -8 * float(y[t].double().norm())


def test_padding_tokens_reach_nothing(tb):
    (x, router, bias, w1, w2, b2), dy = inputs(300, torch.float32)
    logits = x @ router
    logits[::5] = -math.inf
    experts, weights = tb.expert_route(logits, CHOICES, "sigmoid", bias)
    assert (experts[::5] == -1).all() and (weights[::5] == 0).all()
    x[::5] = math.nan
    rows, plan = tb.expert_dispatch(x, experts, EXPERTS)
    out, before = tb.expert_product(rows, plan.offsets, w1, None, "gated_silu", keep=True)
    assert int(plan.offsets[-1]) == 240 * CHOICES and out.isfinite().all() and (out[240 * CHOICES:] == 0).all()
    y = tb.expert_combine(out, plan, weights)
    assert y.isfinite().all() and (y[::5] == 0).all()
    d = torch.randn_like(out)
    d[240 * CHOICES:] = math.nan
    for t in tb.expert_product_grad(tb.expert_activation_grad(d, before, "gated_silu"), rows, plan.offsets, w1):
        assert t is None or t.isfinite().all()

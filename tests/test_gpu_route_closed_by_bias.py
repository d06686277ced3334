"""Experts that the bias closes are never chosen and keep their share of the softmax, in the weights and in their gradient; those that their logit closes have none."""
import pytest
import torch

import products_util as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("experts, choices", [(8, 3), (60, 8), (256, 6), (700, 4)])
@pytest.mark.parametrize("closed", [float("-inf"), float("nan")])
def test_softmax_goes_over_what_the_logits_leave_open(tb, dtype, experts, choices, closed):
    g = torch.Generator(device="cuda").manual_seed(experts)
    n = 120
    logits = torch.randn(n, experts, generator=g, device="cuda").to(dtype)
    logits[:, 1::4] = float("-inf")
    logits[3:6] = float("-inf")
    bias = 0.1 * torch.randn(experts, generator=g, device="cuda")
    bias[::2] = closed
    ids, weights = tb.expert_route(logits, choices, "softmax", bias, renormalize=False)
    is_open = (torch.arange(experts, device="cuda") % 2 == 1) & (torch.arange(experts, device="cuda") % 4 != 1)
    chosen = ids >= 0
    assert bool(is_open[ids[chosen].long()].all()) and bool((chosen.sum(1) == min(choices, int(is_open.sum()))).logical_or(torch.isneginf(logits).all(1)).all())
    # the share of every expert with a logit, chosen or closed by the bias, is in the sum; an exponential, its argument, a sum of 700 and a quotient: below 2^-20 of a weight
    x = logits.double()
    share = torch.exp(x) / torch.exp(x).sum(1, keepdim=True).clamp(min=1e-300)
    want = torch.where(chosen, torch.gather(share, 1, ids.clamp(min=0).long()), 0.0)
    assert bool(((weights.double() - want).abs() <= 2.0 ** -20 * want).all())
    assert torch.equal(ids.cpu(), ref.route(logits, choices, "softmax", bias, renormalize=False)[0])
    # its gradient, the same function's along a direction, by differences of 64-bit numbers
    dweights = torch.randn(n, choices, generator=g, device="cuda")
    grad = tb.expert_route_grad(dweights, ids, logits, "softmax", renormalize=False).double()
    along = torch.where(torch.isneginf(x), 0.0, torch.randn(n, experts, generator=g, device="cuda").double())

    def value(h):
        e = torch.exp(x + h * along)
        return (torch.where(chosen, torch.gather(e / e.sum(1, keepdim=True).clamp(min=1e-300), 1, ids.clamp(min=0).long()), 0.0) * dweights.double()).sum(1)
    h = 1e-5
    slope = (value(h) - value(-h)) / (2 * h)
    # a third derivative along a direction of up to 4 a logit leaves h^2 times some hundred; each of the gradients is rounded to dtype
    error = 1e-7 + 2 * torch.finfo(dtype).eps * (grad * along).abs().sum(1) + (2.0 ** -24 if dtype == torch.float16 else 0.0) * along.abs().sum(1)
    assert bool((((grad * along).sum(1) - slope).abs() <= error).all())

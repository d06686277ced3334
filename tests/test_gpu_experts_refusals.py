"""expert_combine_grad needs the weights, although expert_combine does not: a refusal like the others."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_no_weights_to_differentiate(tb):
    x, ids = torch.ones(6, 8, device="cuda"), torch.zeros(6, 2, dtype=torch.int64, device="cuda")
    rows, plan = tb.expert_dispatch(x, ids, 4)
    assert torch.equal(tb.expert_combine(rows, plan), 2 * x)
    with pytest.raises(ValueError, match="weights"):
        tb.expert_combine_grad(x, rows, plan, None)

"""Rows of no channels through the Python calls: shapes and plans come out as for any rows."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [0, 5, 9000])
def test_rows_of_no_channels(tb, n):
    ids = torch.arange(2 * n, device="cuda").view(n, 2) % 3
    none, state = torch.empty(n, 0, device="cuda"), torch.empty(n, 0, device="cuda")
    assert tb.embedding(torch.empty(4, 0, device="cuda"), ids[:, 0].contiguous()).shape == (n, 0)
    assert tb.embedding_grad(none, ids[:, 0].contiguous(), 4).shape == (4, 0)
    h, last = tb.gated_scan(none, none)
    assert h.shape == (n, 0) and last.shape == (1, 0)
    dx, dgate, dh0 = tb.gated_scan_grad(none, none, none, none)
    assert dx.shape == dgate.shape == (n, 0) and dh0.shape == (1, 0)
    assert tb.gated_step(none, none, state).shape == (n, 0)
    rows, plan = tb.expert_dispatch(none, ids, 3)
    assert rows.shape == (2 * n, 0) and plan.offsets[-1] == 2 * n and int((plan.slots >= 0).sum()) == 2 * n
    assert tb.expert_combine(rows, plan).shape == (n, 0) and tb.expert_dispatch_grad(rows, plan).shape == (n, 0)
    drows, dweights = tb.expert_combine_grad(none, rows, plan, torch.ones(n, 2, device="cuda"))
    assert drows.shape == (2 * n, 0) and dweights.shape == (n, 2) and not dweights.any()

"""embedding_grad with nothing to write, waited for: what an earlier call left in the workspace's header is not its status."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,dim", [(0, 8), (5, 0)])
@pytest.mark.parametrize("n", [0, 3])
@pytest.mark.parametrize("accumulate", [False, True])
def test_nothing_to_write(tb, rows, dim, n, accumulate):
    tokens, dout = torch.zeros(n, dtype=torch.int64, device="cuda"), torch.ones(n, dim, device="cuda")
    tb.embedding_grad(torch.ones(3, 8, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda"), 5)
    kept = tb.workspaces.at(tb.workspaces.key("embedding_grad"))
    kept.buf.fill_(1)                      # as a wait that ran out in that call would leave it
    into = torch.empty(rows, dim, device="cuda") if accumulate else None
    assert tb.embedding_grad(dout, tokens, rows, out=into, accumulate=accumulate, sync=True).shape == (rows, dim)
    tb.workspaces.clear()                  # in a workspace of its own, whatever lies in it
    assert tb.embedding_grad(dout, tokens, rows, out=into, accumulate=accumulate, sync=True).shape == (rows, dim)

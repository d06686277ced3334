"""The gated recurrence over many windows of few channels, where a cluster's carries are all there is between one part of a sequence and the next."""
import pytest
import torch

import layers_util as lu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,dim,dtype", [(16385, 8, torch.float32), (9001, 5, torch.bfloat16), (9001, 64, torch.bfloat16)])
@pytest.mark.parametrize("packed", [False, True])
def test_many_windows(tb, rows, dim, dtype, packed):
    g = torch.Generator(device="cuda").manual_seed(rows + dim)
    rand = lambda *shape: torch.randn(*shape, generator=g, device="cuda")   # noqa: E731
    # states are kept for a few or for thousands of rows
    x, gate = rand(rows, dim).to(dtype), (rand(rows, dim) + torch.arange(dim, device="cuda") % 9).to(dtype)
    cut = torch.tensor([0, 3, rows // 2, rows // 2 + 1, rows - 7, rows], device="cuda") if packed else None
    sequences = 5 if packed else 1
    h0, dlast, dh = rand(sequences, dim), rand(sequences, dim), rand(rows, dim).to(dtype)
    h, last = tb.gated_scan(x, gate, h0, cut)
    want, want_last, e, e_last = lu.gated_scan(x, gate, h0, cut)
    lu.near(h, want, e)
    lu.near(last, want_last, e_last)
    dx, dgate, dh0 = tb.gated_scan_grad(dh, x, gate, h, h0, dlast, cut)
    wx, wg, w0, ex, eg, e0 = lu.gated_scan_grad(dh, x, gate, h, h0, dlast, cut)
    lu.near(dx, wx, ex)
    lu.near(dgate, wg, eg)
    lu.near(dh0, w0, e0)

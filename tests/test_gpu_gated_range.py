"""The gated recurrence over the whole range of its gates: every quarter from -100 to 100, the ends of the range of 32-bit exponentials (about 87.3
and 88.7) closely, infinities and NaN; with tiles and without, packed and not, forward, backward and one token at a time.

A gate's two factors may be taken as zero below 2^-126, the smallest normal number: a result of up to 150 rows, in which a factor meets a difference
of at most 12 and a sum of at most 150 terms of at most 6, is off by no more than 2 * 150 * 12 * 900 * 2^-126 < 1e-31 for that (FLUSHED)."""
import pytest
import torch

import layers_util as lu

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
FLUSHED = 1e-31
GATES = [q / 4 for q in range(-400, 401)] + [s * (87 + q / 32) for s in (1, -1) for q in range(0, 64)] + [float("inf"), -float("inf"), 3e4, -3e4]


def _normal(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


def _gates(rows, dim, dtype, by_row):
    """All of GATES along the channels; by_row: another one in each row, so that states meet all of them."""
    c = torch.arange(dim, device="cuda")[None] + (37 * torch.arange(rows, device="cuda")[:, None] if by_row else torch.zeros(rows, 1, dtype=torch.long, device="cuda"))
    return torch.tensor(GATES, device="cuda")[c % len(GATES)].to(dtype)


def _inputs(dim, dtype, packed, by_row):
    rows = 150
    x, gate, dh = _normal((rows, dim), dtype, 1), _gates(rows, dim, dtype, by_row), _normal((rows, dim), dtype, 2)
    offsets = torch.tensor([0, 1, 70, 70, 133, 150], device="cuda") if packed else None
    sequences = 5 if packed else 1
    return x, gate, dh, offsets, _normal((sequences, dim), torch.float32, 3), _normal((sequences, dim), torch.float32, 4)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [1000, 937])          # rows of whole 16-byte pieces, and others
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("by_row", [False, True])
def test_scan_and_its_gradient(tb, dtype, dim, packed, by_row):
    assert dim >= len(GATES)
    x, gate, dh, offsets, h0, dlast = _inputs(dim, dtype, packed, by_row)
    h, last = tb.gated_scan(x, gate, h0, offsets)
    want, want_last, e, e_last = lu.gated_scan(x, gate, h0, offsets)
    lu.near(h, want, e + FLUSHED)
    lu.near(last, want_last, e_last + FLUSHED)
    dx, dgate, dh0 = tb.gated_scan_grad(dh, x, gate, h, h0, dlast, offsets)
    wx, wg, w0, ex, eg, e0 = lu.gated_scan_grad(dh, x, gate, h, h0, dlast, offsets)
    lu.near(dx, wx, ex + FLUSHED)
    lu.near(dgate, wg, eg + FLUSHED)
    lu.near(dh0, w0, e0 + FLUSHED)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [1000, 937])
def test_one_row(tb, dtype, dim):
    """A sequence of one token, by the scan and by the step."""
    x, gate, state = _normal((1, dim), dtype, 5), _gates(1, dim, dtype, False), _normal((1, dim), torch.float32, 6)
    want, want_last, e, e_last = lu.gated_scan(x, gate, state)
    h, last = tb.gated_scan(x, gate, state)
    lu.near(h, want, e + FLUSHED)
    lu.near(last, want_last, e_last + FLUSHED)
    h = tb.gated_step(x, gate, state)
    lu.near(h, want, e + FLUSHED)
    lu.near(state, want_last, e_last + FLUSHED)


@pytest.mark.parametrize("dtype", TYPES)
def test_closed_gates_replace_the_state(tb, dtype):
    """Where 1 - sigmoid is 1 to 32 bits the scan stores x itself, and all of the gradient goes to x."""
    gate = torch.tensor([-20.0, -50, -87, -87.25, -87.5, -88, -88.5, -88.75, -89, -95, -100, -1000], device="cuda").to(dtype).repeat(200, 4)
    x, dh = _normal(tuple(gate.shape), dtype, 7), _normal(tuple(gate.shape), dtype, 8)
    h, _ = tb.gated_scan(x, gate)
    dx, _, _ = tb.gated_scan_grad(dh, x, gate, h)
    assert torch.allclose(h.float(), x.float(), rtol=2.0 ** -8, atol=1e-6) and torch.allclose(dx.float(), dh.float(), rtol=2.0 ** -8, atol=1e-6)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 61])
@pytest.mark.parametrize("packed", [False, True])
def test_gates_that_are_nan(tb, dtype, dim, packed):
    """A NaN gate makes NaNs of its channel from its row to the end of its sequence, backward from its row to the beginning, and nothing else."""
    x, gate, dh = (_normal((150, dim), dtype, seed) for seed in (9, 10, 11))
    offsets = torch.tensor([0, 60, 150], device="cuda") if packed else None
    end = 60 if packed else 150
    h, last = tb.gated_scan(x, gate, None, offsets)
    clean = tb.gated_scan_grad(dh, x, gate, h, None, None, offsets)
    bad = gate.clone()
    bad[40, 5] = float("nan")
    hb, lb = tb.gated_scan(x, bad, None, offsets)
    nan = torch.zeros(150, dim, dtype=torch.bool, device="cuda")
    nan[40:end, 5] = True
    assert torch.equal(hb.isnan(), nan) and torch.equal(hb[~nan], h[~nan])
    assert lb[0, 5].isnan() and int(lb.isnan().sum()) == 1
    dx, dgate, dh0 = tb.gated_scan_grad(dh, x, bad, h, None, None, offsets)
    nan.zero_()
    nan[:41, 5] = True
    for got, fine in zip((dx, dgate), clean):
        assert torch.equal(got.isnan(), nan) and torch.equal(got[~nan], fine[~nan])
    assert dh0[0, 5].isnan() and int(dh0.isnan().sum()) == 1
    state = torch.zeros(150, dim, device="cuda")
    step = tb.gated_step(x, bad, state)
    assert step[40, 5].isnan() and int(step.isnan().sum()) == 1 and int(state.isnan().sum()) == 1

"""Rows sent to experts and back, and both gradients, against plain forms in 64 bits."""
import pytest
import torch

import layers_util as lu

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _normal(shape, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _ids(n, choices, experts, seed, ids=torch.int64, dropped=0.1, skew=2.0):
    """Different experts for each token while there are enough of them, the first ones more often; some ids that are none."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    score = torch.rand(n, max(experts, choices), generator=g, device="cuda") + skew * torch.rand(max(experts, choices), generator=g, device="cuda")
    e = torch.topk(score, choices, dim=1).indices % experts
    u = torch.rand(n, choices, generator=g, device="cuda")
    e = torch.where(u < dropped / 2, -1, torch.where(u < dropped, experts + 5, e))
    if dropped and n > 2:
        e[n // 2] = -1                 # a token that goes nowhere
    return e.to(ids)


def _check_plan(plan, ids, experts):
    slots, sources, offsets = lu.plan(ids, experts)
    assert plan.slots.reshape(-1).tolist() == slots and plan.sources.tolist() == sources and plan.offsets.tolist() == offsets
    assert plan.slots.dtype == plan.sources.dtype == plan.offsets.dtype == torch.int32 and plan.slots.shape == ids.shape


SIZES = [(1, 1, 1, 1), (1, 8, 64, 64), (3, 2, 5, 33), (33, 4, 64, 256), (64, 8, 8, 100), (257, 1, 3, 257), (300, 6, 1024, 64), (1000, 3, 7, 1000), (1025, 2, 256, 128), (2048, 8, 100, 40),
         (5, 32, 40, 2048), (20011, 4, 129, 24), (40000, 8, 513, 16)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,choices,experts,dim", SIZES)
def test_there_and_back(tb, dtype, n, choices, experts, dim):
    ids = _ids(n, choices, experts, 1, torch.int32 if n % 2 else torch.int64)
    x, weights = _normal((n, dim), dtype, 2), _normal((n, choices), torch.float32, 3)
    rows, plan = tb.expert_dispatch(x, ids, experts)
    _check_plan(plan, ids, experts)
    sources = plan.sources.long()
    want = torch.where((sources >= 0)[:, None], x[sources.clamp(min=0) // choices], torch.zeros((), dtype=dtype, device="cuda"))
    assert torch.equal(rows, want)
    y = _normal((n * choices, dim), dtype, 4)
    lu.near(tb.expert_combine(y, plan, weights), *lu.combine(y, plan.slots, weights))
    lu.near(tb.expert_combine(y, plan), *lu.combine(y, plan.slots))
    lu.near(tb.expert_dispatch_grad(y, plan), *lu.combine(y, plan.slots))
    dout = _normal((n, dim), dtype, 5)
    drows, dweights = tb.expert_combine_grad(dout, y, plan, weights)
    wr, ww, er, ew = lu.combine_grad(dout, y, plan.slots, weights)
    lu.near(drows, wr, er)
    lu.near(dweights, ww, ew)


@pytest.mark.parametrize("n,choices,experts", [(7, 2, 4), (5000, 3, 16)])
@pytest.mark.parametrize("kind", ["all of one expert", "nothing kept", "ids far out of range"])
def test_lopsided_plans(tb, n, choices, experts, kind):
    ids = torch.full((n, choices), {"all of one expert": experts - 1, "nothing kept": -1, "ids far out of range": 2 ** 32}[kind], device="cuda")
    x = _normal((n, 72), torch.bfloat16, 6)
    rows, plan = tb.expert_dispatch(x, ids, experts)
    _check_plan(plan, ids, experts)
    if kind == "all of one expert":
        assert torch.equal(rows, x.repeat_interleave(choices, 0))
    else:
        assert not rows.any() and not tb.expert_combine(torch.full_like(rows, float("nan")), plan).any()
        drows, dweights = tb.expert_combine_grad(x, torch.full_like(rows, float("nan")), plan, torch.full((n, choices), float("nan"), device="cuda"))
        assert not drows.any() and not dweights.any()


def test_dropped_assignments_read_nothing(tb):
    """NaN weights and rows of what was dropped, and NaNs behind the last row in use."""
    ids = _ids(400, 4, 9, 7, dropped=0.4)
    x = _normal((400, 136), torch.float32, 8)
    rows, plan = tb.expert_dispatch(x, ids, 9)
    gone = plan.slots < 0
    weights = torch.where(gone, float("nan"), _normal((400, 4), torch.float32, 9))
    y = _normal((1600, 136), torch.float32, 10)
    y[int(plan.offsets[-1]):] = float("nan")
    fine = torch.where(gone, 0.0, weights)
    out, (drows, dweights) = tb.expert_combine(y, plan, weights), tb.expert_combine_grad(x, y, plan, weights)
    lu.near(out, *lu.combine(y, plan.slots, weights))
    assert not out[gone.all(1)].any() and int(gone.all(1).sum()) > 0
    wr, ww, er, ew = lu.combine_grad(x, y, plan.slots, fine)
    lu.near(drows, wr, er)
    lu.near(dweights, ww, ew)


def test_slots_out_of_range_are_left_out(tb):
    y, x = _normal((6, 40), torch.float32, 11), _normal((3, 40), torch.float32, 12)
    plan = tb.ExpertPlan(torch.tensor([[0, 6], [-7, 3], [2 ** 31 - 1, 5]], dtype=torch.int32, device="cuda"), None, torch.tensor([0, 6], dtype=torch.int32, device="cuda"))
    weights = torch.ones(3, 2, device="cuda")
    assert torch.equal(tb.expert_combine(y, plan, weights), torch.stack([y[0], y[3], y[5]]))
    dweights = tb.expert_combine_grad(x, y, plan, weights)[1]
    assert dweights[0, 1] == dweights[1, 0] == dweights[2, 0] == 0


def test_empty(tb):
    ids = torch.empty(0, 2, dtype=torch.int64, device="cuda")
    rows, plan = tb.expert_dispatch(torch.empty(0, 8, device="cuda"), ids, 3)
    assert rows.shape == (0, 8) and plan.offsets.tolist() == [0, 0, 0, 0]
    assert tb.expert_combine(rows, plan).shape == (0, 8)
    drows, dweights = tb.expert_combine_grad(rows, rows, plan, torch.empty(0, 2, device="cuda"))
    assert drows.shape == (0, 8) and dweights.shape == (0, 2)


def test_strided_and_misaligned_rows(tb):
    wide = _normal((200, 300), torch.bfloat16, 13)
    ids, weights = _ids(50, 4, 6, 14), _normal((50, 4), torch.float32, 15)
    for a, w in ((0, 128), (1, 128), (8, 257), (3, 96)):
        x, y = wide[:100:2, a:a + w], wide[:, a:a + w]
        rows, plan = tb.expert_dispatch(x, ids, 6)
        assert torch.equal(rows, tb.expert_dispatch(x.contiguous(), ids, 6)[0])
        lu.near(tb.expert_combine(y, plan, weights), *lu.combine(y, plan.slots, weights))
        drows, dweights = tb.expert_combine_grad(x, y, plan, weights)
        wr, ww, er, ew = lu.combine_grad(x, y, plan.slots, weights)
        lu.near(drows, wr, er)
        lu.near(dweights, ww, ew)


def test_gradients_against_differences(tb):
    """out is linear in the rows and in the weights, so a step of one gives each derivative exactly, but for 64-bit rounding."""
    ids = _ids(4, 2, 3, 16, dropped=0.3)
    x, c = _normal((4, 3), torch.float32, 17), _normal((4, 3), torch.float32, 18)
    weights = _normal((4, 2), torch.float32, 19)
    rows, plan = tb.expert_dispatch(x, ids, 3)
    drows, dweights = tb.expert_combine_grad(c, rows, plan, weights)
    dx = tb.expert_dispatch_grad(drows, plan)
    source = plan.sources.long()

    def loss(x, weights, rows=None):
        if rows is None:
            rows = torch.where((source >= 0)[:, None], x[source.clamp(min=0) // 2], 0.0)
        return float((lu.combine(rows, plan.slots, weights)[0] * c.double()).sum())

    def slope(f, at):
        out = torch.zeros_like(at)
        for i in range(at.numel()):
            up, down = at.clone(), at.clone()
            up.view(-1)[i] += 1
            down.view(-1)[i] -= 1
            out.view(-1)[i] = (f(up) - f(down)) / 2
        return out

    xd, wd, rd = x.double(), weights.double(), rows.double()
    assert torch.allclose(slope(lambda v: loss(v, wd), xd), dx.double(), atol=1e-5)
    assert torch.allclose(slope(lambda v: loss(xd, v), wd), dweights.double(), atol=1e-5)
    assert torch.allclose(slope(lambda v: loss(xd, wd, v), rd), drows.double(), atol=1e-5)


def test_rows_past_32_bits(tb):
    n, choices, dim = 140000, 8, 2048          # 2.29 billion elements
    ids = torch.arange(n * choices, device="cuda").view(n, choices) % 16
    x = torch.zeros(n, dim, dtype=torch.bfloat16, device="cuda")
    x[-3:] = _normal((3, dim), torch.bfloat16, 20)
    rows, plan = tb.expert_dispatch(x, ids, 16)
    per = n * choices // 16
    assert torch.equal(plan.offsets, torch.arange(17, dtype=torch.int32, device="cuda") * per)
    # expert 15 has the last choice of every second token
    assert torch.equal(rows[-2:], x[[n - 3, n - 1]]) and torch.equal(rows[per - 1], x[n - 2])
    out = tb.expert_combine(rows, plan)
    assert torch.equal(out[-3:].float(), 8 * x[-3:].float()) and not out[:-3].any()
    weights = torch.full((n, choices), 0.5, device="cuda")
    drows, dweights = tb.expert_combine_grad(x, rows, plan, weights)
    assert torch.equal(drows[-2:].float(), x[[n - 3, n - 1]].float() / 2)
    lu.near(dweights[-3:], (x[-3:].double() ** 2).sum(1, keepdim=True).expand(3, 8), 2049 * lu.U * (x[-3:].double() ** 2).sum(1, keepdim=True).expand(3, 8))
    assert not dweights[:-3].any()


def test_another_stream_and_a_graph(tb):
    ids, x, weights = _ids(700, 4, 20, 21), _normal((700, 192), torch.bfloat16, 22), _normal((700, 4), torch.float32, 23)
    kept = {}

    def work():
        kept["rows"], kept["plan"] = tb.expert_dispatch(x, ids, 20)
        kept["out"] = tb.expert_combine(kept["rows"], kept["plan"], weights)
        kept["grad"] = tb.expert_combine_grad(x, kept["rows"], kept["plan"], weights)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        work()
    for seed in (24, 25):
        ids.copy_(_ids(700, 4, 20, seed))
        graph.replay()
        _check_plan(kept["plan"], ids, 20)
        lu.near(kept["out"], *lu.combine(kept["rows"], kept["plan"].slots, weights))
        wr, ww, er, ew = lu.combine_grad(x, kept["rows"], kept["plan"].slots, weights)
        lu.near(kept["grad"][0], wr, er)
        lu.near(kept["grad"][1], ww, ew)
    del graph


def test_refusals(tb):
    x, ids = _normal((6, 8), torch.float32, 26), torch.zeros(6, 2, dtype=torch.int64, device="cuda")
    rows, plan = tb.expert_dispatch(x, ids, 4)
    w = torch.ones(6, 2, device="cuda")
    for call in (lambda: tb.expert_dispatch(x.double(), ids, 4), lambda: tb.expert_dispatch(x, ids.float(), 4), lambda: tb.expert_dispatch(x[:5], ids, 4),
                 lambda: tb.expert_dispatch(x, ids, 0), lambda: tb.expert_dispatch(x, ids, 1025), lambda: tb.expert_dispatch(x, ids[:, 0], 4), lambda: tb.expert_dispatch(x, ids.t(), 4),
                 lambda: tb.expert_dispatch(x, ids[:, :0], 4), lambda: tb.expert_dispatch(x, torch.zeros(6, 33, dtype=torch.int64, device="cuda"), 4),
                 lambda: tb.expert_dispatch(x.cpu(), ids, 4), lambda: tb.expert_dispatch(x, ids.cpu(), 4), lambda: tb.expert_combine(rows[:-1], plan),
                 lambda: tb.expert_combine(rows, plan, w[:, :1]), lambda: tb.expert_combine(rows, plan, w.half()), lambda: tb.expert_combine(rows, plan._replace(slots=plan.slots.long())),
                 lambda: tb.expert_combine_grad(x[:5], rows, plan, w), lambda: tb.expert_combine_grad(x.half(), rows, plan, w),
                 lambda: tb.expert_combine_grad(x, rows, plan._replace(offsets=plan.offsets[:1]), w), lambda: tb.expert_combine_grad(x, rows, plan, w.double())):
        with pytest.raises(ValueError):
            call()

"""The gated recurrence, its gradient and its step, against plain forms in 64 bits."""
import pytest
import torch

import layers_util as lu

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _normal(shape, dtype, seed, shift=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") + shift).to(dtype)


def _inputs(shape, dtype, seed, fused=False):
    """x and a gate whose channels keep their state for a few or for thousands of tokens, perhaps halves of one tensor."""
    d = shape[-1]
    gate = _normal(shape, dtype, seed + 1) + (torch.arange(d, device="cuda") % 7 - 0.0).to(dtype)
    x = _normal(shape, dtype, seed)
    if fused:
        both = torch.cat([x, gate], dim=-1)
        return both[..., :d], both[..., d:]
    return x, gate


def _check(tb, x, gate, h0, offsets):
    h, last = tb.gated_scan(x, gate, h0, offsets)
    want, want_last, e, e_last = lu.gated_scan(x, gate, h0, offsets)
    lu.near(h, want, e)
    lu.near(last, want_last, e_last)
    return h


def _check_grad(tb, x, gate, h, h0, offsets, seed, with_last):
    dh = _normal(tuple(x.shape), x.dtype, seed)
    sequences = x.shape[0] if x.dim() == 3 else 1 if offsets is None else offsets.numel() - 1
    dlast = _normal((sequences, x.shape[-1]), torch.float32, seed + 1) if with_last else None
    dx, dgate, dh0 = tb.gated_scan_grad(dh, x, gate, h, h0, dlast, offsets)
    wx, wg, w0, ex, eg, e0 = lu.gated_scan_grad(dh, x, gate, h, h0, dlast, offsets)
    lu.near(dx, wx, ex)
    lu.near(dgate, wg, eg)
    lu.near(dh0, w0, e0)


SHAPES = [(1, 1, 1), (2, 2, 3), (1, 33, 64), (3, 31, 100), (1, 64, 7), (5, 65, 128), (2, 127, 66), (1, 129, 257), (7, 256, 64), (1, 1000, 130), (2, 1025, 320), (1, 2500, 64),
          (300, 3, 32), (1, 4099, 36), (16, 513, 72)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_equal_lengths(tb, dtype, shape):
    x, gate = _inputs(shape, dtype, 1, fused=shape[1] % 2 == 0)
    h0 = _normal((shape[0], shape[2]), torch.float32, 3) if shape[0] % 2 else None
    h = _check(tb, x, gate, h0, None)
    _check_grad(tb, x, gate, h, h0, None, 4, shape[0] % 3 != 2)


PACKED = [([0, 1], 1, 8), ([0, 0, 0], 3, 64), ([2, 5, 5, 9], 12, 33), ([0, 64, 128, 192], 192, 64), ([0, 63, 64, 65, 200], 200, 128), ([0, 1, 2, 3, 4, 5, 300], 300, 65),
          ([0, 0, 700, 700, 700, 1500, 1500], 1500, 96), ([10, 2000], 2100, 64), (list(range(0, 900, 9)), 895, 40), ([0, 255, 257, 1024, 1025, 2600], 2600, 320)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offsets,rows,dim", PACKED)
@pytest.mark.parametrize("initial", [False, True])
def test_packed_sequences(tb, dtype, offsets, rows, dim, initial):
    x, gate = _inputs((rows, dim), dtype, 5, fused=not initial)
    at = torch.tensor(offsets, dtype=torch.int32 if initial else torch.int64, device="cuda")
    h0 = _normal((len(offsets) - 1, dim), torch.float32, 7) if initial else None
    h = _check(tb, x, gate, h0, at)
    _check_grad(tb, x, gate, h, h0, at, 8, initial)


def test_rows_without_offsets_are_one_sequence(tb):
    x, gate = _inputs((300, 48), torch.float32, 9)
    h, last = tb.gated_scan(x, gate)
    g, l2 = tb.gated_scan(x[None], gate[None])
    assert torch.equal(h, g[0]) and torch.equal(last, l2) and last.shape == (1, 48)


def test_empty(tb):
    x = torch.empty(0, 16, device="cuda")
    h0 = _normal((3, 16), torch.float32, 10)
    zeros = torch.zeros(4, dtype=torch.int64, device="cuda")
    h, last = tb.gated_scan(x, x, h0, zeros)
    assert h.shape == (0, 16) and torch.equal(last, h0)
    assert torch.equal(tb.gated_scan(x, x, None, zeros)[1], torch.zeros(3, 16, device="cuda"))
    dx, dgate, dh0 = tb.gated_scan_grad(x, x, x, x, None, h0, zeros)
    assert dx.shape == dgate.shape == (0, 16) and torch.equal(dh0, h0)
    x3 = torch.empty(3, 0, 16, device="cuda")
    assert torch.equal(tb.gated_scan(x3, x3, h0)[1], h0)
    x = _normal((5, 16), torch.float32, 11)        # rows that are no sequence's
    h, last = tb.gated_scan(x, x, None, zeros[:1])
    assert not h.any() and last.shape == (0, 16)


def test_sequences_do_not_see_one_another(tb):
    """NaNs and infinities in one sequence, and in rows outside all of them, stay there; others have the bits that they have alone."""
    x, gate = _inputs((900, 70), torch.float32, 12)
    at = torch.tensor([4, 300, 301, 301, 650, 890], device="cuda")
    h0, dlast = _normal((5, 70), torch.float32, 14), _normal((5, 70), torch.float32, 15)
    dh = _normal((900, 70), torch.float32, 16)
    h, last = tb.gated_scan(x, gate, h0, at)
    clean = tb.gated_scan_grad(dh, x, gate, h, h0, dlast, at)
    x2, gate2, h02, dh2, dlast2, h2 = (t.clone() for t in (x, gate, h0, dh, dlast, h))
    for t in (x2, gate2, dh2):
        t[:4] = float("nan")
        t[890:] = float("inf")
        t[300] = float("nan")
        t[400:402] = float("inf")
    h2[300] = float("nan")
    h02[3], dlast2[3], h02[1] = float("inf"), float("nan"), float("nan")
    hb, lb = tb.gated_scan(x2, gate2, h02, at)
    got = tb.gated_scan_grad(dh2, x2, gate2, h2, h02, dlast2, at)
    fine = torch.ones(900, dtype=torch.bool)
    fine[300], fine[301:650] = False, False
    assert torch.equal(hb[fine], h[fine]) and torch.equal(lb[[0, 2, 4]], last[[0, 2, 4]])
    assert torch.equal(got[0][fine], clean[0][fine]) and torch.equal(got[1][fine], clean[1][fine]) and torch.equal(got[2][[0, 2, 4]], clean[2][[0, 2, 4]])
    assert hb[300].isnan().all() and lb[1].isnan().all() and got[0][300].isnan().all()


def test_closed_and_open_gates(tb):
    """sigmoid of +inf, -inf and very large values: the state is kept, or replaced, and nothing becomes NaN."""
    for dtype in TYPES:
        x, gate = _inputs((2, 70, 40), dtype, 17)
        gate[:, 10:20], gate[:, 20:30], gate[:, 30:40], gate[:, 40:50] = float("inf"), -float("inf"), 3e4, -3e4
        h0 = _normal((2, 40), torch.float32, 18)
        h = _check(tb, x, gate, h0, None)
        assert torch.equal(h[:, 20:30], x[:, 20:30]) and torch.equal(h[:, 40:50], x[:, 40:50])
        dh = _normal((2, 70, 40), dtype, 19)
        dx, dgate, dh0 = tb.gated_scan_grad(dh, x, gate, h, h0)
        assert not (dx.isnan().any() or dgate.isnan().any() or dh0.isnan().any()) and not dgate[:, 10:50].any() and not dx[:, 10:20].any()


def test_offsets_out_of_range_are_cut_off(tb):
    x, gate = _inputs((100, 24), torch.float32, 20)
    h, last = tb.gated_scan(x, gate, None, torch.tensor([-5, 40, 1000], device="cuda"))
    g, l2 = tb.gated_scan(x, gate, None, torch.tensor([0, 40, 100], device="cuda"))
    assert torch.equal(h, g) and torch.equal(last, l2)


def test_gradient_against_differences(tb):
    x, gate = _inputs((2, 9, 3), torch.float32, 21)
    h0, dh, dlast = _normal((2, 3), torch.float32, 23), _normal((2, 9, 3), torch.float32, 24), _normal((2, 3), torch.float32, 25)
    h, _ = tb.gated_scan(x, gate, h0)
    got = tb.gated_scan_grad(dh, x, gate, h, h0, dlast)

    def loss(x, gate, h0):
        h, last = lu.gated_scan(x, gate, h0)[:2]
        return float((h * dh.double()).sum() + (last * dlast.double()).sum())

    base, step = [t.double() for t in (x, gate, h0)], 1e-4
    for k in range(3):
        for i in range(0, base[k].numel(), 2):
            sides = []
            for sign in (1, -1):
                args = [t.clone() for t in base]
                args[k].view(-1)[i] += sign * step
                sides.append(loss(*args))
            # the central difference is off by step^2 / 6 times a third derivative of at most about 10; the gradient by 32-bit rounding
            assert abs((sides[0] - sides[1]) / (2 * step) - float(got[k].reshape(-1)[i])) <= 1e-5


def test_strided_and_misaligned_rows(tb):
    wide = _normal((130, 400), torch.bfloat16, 26)
    for a, b in ((0, 128), (1, 129), (3, 131), (8, 200)):
        x, gate = wide[:, a:a + 96], wide[:, b:b + 96]
        h = _check(tb, x, gate, None, None)
        _check_grad(tb, x, gate, h, None, None, 27, True)
    x, gate = wide[::2, :96], wide[::2, 100:196]
    h = _check(tb, x, gate, None, None)
    _check_grad(tb, x, gate, wide[:65, 200:296].copy_(h), None, None, 28, False)


def test_sequences_past_32_bits(tb):
    rows, dim = (1 << 20) + 40000, 2048        # 2.23 billion elements
    x = torch.zeros(rows, dim, dtype=torch.bfloat16, device="cuda")
    gate = torch.zeros(rows, dim, dtype=torch.bfloat16, device="cuda")
    tail = 300
    x[-tail:], gate[-tail:] = _normal((tail, dim), torch.bfloat16, 29), _normal((tail, dim), torch.bfloat16, 30)
    x[rows - tail - 1] = 1.0
    at = torch.tensor([0, rows - tail, rows], device="cuda")
    h, last = tb.gated_scan(x, gate, None, at)
    want, want_last, e, e_last = lu.gated_scan(x[-tail:], gate[-tail:])
    lu.near(h[-tail:], want, e)
    lu.near(last[1:], want_last, e_last)
    assert not h[:rows - tail - 1].any() and bool((last[0] == 0.5).all())
    dx, dgate, dh0 = tb.gated_scan_grad(x, x, gate, h, None, None, at)
    wx, wg, w0, ex, eg, e0 = lu.gated_scan_grad(x[-tail:], x[-tail:], gate[-tail:], h[-tail:])
    lu.near(dx[-tail:], wx, ex)
    lu.near(dgate[-tail:], wg, eg)
    lu.near(dh0[1:], w0, e0)
    assert bool((dx[rows - tail - 3] == 0.125).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,pool,dim", [(1, 1, 1), (3, 5, 33), (64, 64, 128), (5, 9, 2048), (130, 300, 1001)])
def test_step(tb, dtype, n, pool, dim):
    x, gate = _inputs((n, dim), dtype, 31, fused=True)
    state = _normal((pool, dim), torch.float32, 33)
    slots = torch.randperm(pool, generator=torch.Generator(device="cuda").manual_seed(34), device="cuda")[:n]
    slots[::4] = torch.tensor([-1, pool], device="cuda").repeat(n)[:slots[::4].numel()]
    used = (slots >= 0) & (slots < pool)
    before = state.clone()
    h = tb.gated_step(x, gate, state, slots if n % 2 else slots.int())
    want, last, e, e_last = lu.gated_scan(x[used][:, None], gate[used][:, None], before[slots[used]])
    lu.near(h[used], want[:, 0], e[:, 0])
    lu.near(state[slots[used]], last, e_last)
    assert not h[~used].any()
    rest = torch.ones(pool, dtype=torch.bool, device="cuda")
    rest[slots[used]] = False
    assert torch.equal(state[rest], before[rest])


def test_steps_make_a_scan(tb):
    x, gate = _inputs((3, 50, 64), torch.float32, 35)
    state = torch.zeros(3, 64, device="cuda")
    h, last = tb.gated_scan(x, gate)
    for t in range(50):
        got = tb.gated_step(x[:, t].contiguous(), gate[:, t], state)
        assert torch.allclose(got, h[:, t], rtol=1e-5, atol=1e-6)
    assert torch.allclose(state, last, rtol=1e-5, atol=1e-6)


def test_unused_places_read_nothing(tb):
    x = torch.full((2, 40), float("nan"), device="cuda")
    state = torch.full((3, 40), float("nan"), device="cuda")
    assert not tb.gated_step(x, x, state, torch.tensor([-1, 2 ** 32 + 1], device="cuda")).any()


def test_another_stream_and_a_graph(tb):
    x, gate = _inputs((2, 600, 192), torch.bfloat16, 36)
    state = _normal((2, 192), torch.float32, 37)
    dh, kept = _normal((2, 600, 192), torch.bfloat16, 38), {}

    def work():
        kept["h"], kept["last"] = tb.gated_scan(x, gate)
        kept["grad"] = tb.gated_scan_grad(dh, x, gate, kept["h"])
        kept["step"] = tb.gated_step(x[:, 0], gate[:, 0], state)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        work()
    for seed in (39, 40):
        a, b = _inputs((2, 600, 192), torch.bfloat16, seed)
        x.copy_(a)
        gate.copy_(b)
        graph.replay()
        want, want_last, e, e_last = lu.gated_scan(x, gate)
        lu.near(kept["h"], want, e)
        lu.near(kept["last"], want_last, e_last)
        wx, wg, w0, ex, eg, e0 = lu.gated_scan_grad(dh, x, gate, kept["h"])
        lu.near(kept["grad"][0], wx, ex)
        lu.near(kept["grad"][1], wg, eg)
        lu.near(kept["grad"][2], w0, e0)
    del graph


def test_refusals(tb):
    x, h0 = _normal((2, 5, 8), torch.float32, 41), _normal((2, 8), torch.float32, 42)
    flat, at = x.view(10, 8), torch.tensor([0, 10], device="cuda")
    for call in (lambda: tb.gated_scan(x.double(), x.double()), lambda: tb.gated_scan(x, x.bfloat16()), lambda: tb.gated_scan(x, x[:, :4]), lambda: tb.gated_scan(x.cpu(), x.cpu()),
                 lambda: tb.gated_scan(x, x, h0[:1]), lambda: tb.gated_scan(x, x, h0.bfloat16()), lambda: tb.gated_scan(x, x, None, at), lambda: tb.gated_scan(x[0, 0], x[0, 0]),
                 lambda: tb.gated_scan(flat, flat, None, at.float()), lambda: tb.gated_scan(flat, flat, None, at[:0]), lambda: tb.gated_scan(flat, flat, None, at.cpu()),
                 lambda: tb.gated_scan(x.transpose(0, 1), x.transpose(0, 1)), lambda: tb.gated_scan(x[:, :3], x[:, :3]), lambda: tb.gated_scan(flat.t(), flat.t()),
                 lambda: tb.gated_scan(flat[:1].expand(4, 8), flat[:4]), lambda: tb.gated_scan(x, x, out=x[0]),
                 lambda: tb.gated_scan_grad(x, x, x, x[:, :4]), lambda: tb.gated_scan_grad(x, x, x, x, None, h0[0]), lambda: tb.gated_scan_grad(x, x, x.half(), x),
                 lambda: tb.gated_step(x, x, h0), lambda: tb.gated_step(flat, flat, h0), lambda: tb.gated_step(flat, flat, h0.half(), at), lambda: tb.gated_step(flat, flat, h0, at),
                 lambda: tb.gated_step(flat[:2], flat[:2], h0, at.float()), lambda: tb.gated_step(flat[:2], flat[:2], h0[:, :4], at)):
        with pytest.raises(ValueError):
            call()


def test_copies_that_never_come(tmp_path):
    """tests/cpp/gated_waits_test.cu, built here with the test hooks and short waits: the wait runs out, the kernel ends, the results are NaNs and the
    status says so; the next call is right again."""
    import os
    import shutil
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.isfile(nvcc):
        pytest.skip("nvcc is not available on this machine")
    exe = str(tmp_path / "gated_waits_test")
    r = subprocess.run([nvcc, "-std=c++17", "-O2", "-gencode", "arch=compute_100a,code=sm_100a", "-DTB200_TEST_HOOKS", "-DTB200_SPIN_LIMIT=65536",
                        "-I" + os.path.join(root, "include"), "-I" + os.path.join(root, "thrust_b200", "csrc"), os.path.join(root, "tests", "cpp", "gated_waits_test.cu"), "-o", exe],
                       capture_output=True, text=True, timeout=900)
    assert r.returncode == 0, r.stdout + r.stderr
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr

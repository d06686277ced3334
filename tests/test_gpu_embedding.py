"""Rows looked up by token and the gradient of the table, against plain forms in 64 bits."""
import pytest
import torch

import layers_util as lu

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _tokens(n, rows, seed, ids=torch.int64, padding=0.1, skew=3.0):
    """Small ids more often than large ones, some outside the table on either side."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    tok = (torch.rand(n, generator=g, device="cuda") ** skew * rows).long().clamp(max=max(0, rows - 1))
    odd = torch.rand(n, generator=g, device="cuda")
    tok = torch.where(odd < padding / 2, -1, torch.where(odd < padding, rows + 3, tok))
    return tok.to(ids)


def _normal(shape, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,rows,dim", [(1, 1, 1), (3, 10, 7), (64, 1000, 64), (33, 5, 100), (257, 70000, 257), (1000, 300, 1000), (2049, 513, 2048), (5, 9, 8200)])
def test_lookup(tb, dtype, n, rows, dim):
    weight, tokens = _normal((rows, dim), dtype, 1), _tokens(n, rows, 2, torch.int32 if n % 2 else torch.int64)
    got = tb.embedding(weight, tokens, 1.7)
    want = lu.embedding(weight, tokens, float(torch.tensor(1.7)))
    lu.near(got, want, lu.U * want.abs())
    assert got.dtype == dtype


def test_lookup_of_strided_and_misaligned_tables(tb):
    wide = _normal((50, 300), torch.bfloat16, 3)
    tokens = _tokens(77, 50, 4).view(7, 11)
    for part in (wide[:, 8:136], wide[:, 1:129], wide[:, 5:262], wide[::2, :64]):
        got = tb.embedding(part, tokens)
        want = lu.embedding(part, tokens, 1.0)
        assert got.shape == (7, 11, part.shape[1]) and torch.equal(got.double(), want)


def test_absent_tokens_read_nothing(tb):
    weight = torch.full((4, 64), float("nan"), device="cuda")
    tokens = torch.tensor([-1, 4, 2 ** 31 - 1, -2 ** 31], device="cuda")
    assert torch.equal(tb.embedding(weight, tokens), torch.zeros(4, 64, device="cuda"))
    tokens = torch.tensor([-1, 2 ** 32, 2 ** 40 + 1, -2 ** 63], device="cuda")       # low halves that would be rows
    assert torch.equal(tb.embedding(weight, tokens), torch.zeros(4, 64, device="cuda"))
    dout = torch.full((4, 64), float("nan"), device="cuda")
    assert torch.equal(tb.embedding_grad(dout, tokens, 4), torch.zeros(4, 64, device="cuda"))
    # values of a row that is there pass as they are
    weight[1] = float("inf")
    assert torch.equal(tb.embedding(weight, torch.tensor([1], device="cuda"), -2.0), torch.full((1, 64), -float("inf"), device="cuda"))


def test_empty_lookups(tb):
    weight = _normal((4, 64), torch.float32, 5)
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    assert tb.embedding(weight, none).shape == (0, 64)
    assert torch.equal(tb.embedding(weight[:0], torch.tensor([0, 1], device="cuda")), torch.zeros(2, 64, device="cuda"))
    assert torch.equal(tb.embedding_grad(weight[:0], none, 3), torch.zeros(3, 64, device="cuda"))
    into = weight.clone()
    tb.embedding_grad(weight[:0], none, 4, out=into, accumulate=True)
    assert torch.equal(into, weight)
    assert tb.embedding_grad(weight, torch.tensor([0, 1, 2, 3], device="cuda"), 0).shape == (0, 64)


@pytest.mark.parametrize("dtype,out", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32),
                                       (torch.float16, torch.float16), (torch.float32, torch.bfloat16)])
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("n,rows,dim", [(1, 1, 1), (2, 300, 64), (31, 2, 100), (64, 1, 512), (129, 5000, 257), (1000, 255, 1000), (1025, 256, 64), (4097, 65536, 40),
                                        (5000, 3, 1024), (40000, 70000, 65), (50001, 20, 128)])
def test_gradient(tb, dtype, out, accumulate, n, rows, dim):
    dout, tokens = _normal((n, dim), dtype, 6), _tokens(n, rows, 7, torch.int32 if n % 2 else torch.int64)
    into = _normal((rows, dim), out, 8) if accumulate else None
    scale = float(torch.tensor(0.3))
    want, error = lu.embedding_grad(dout, tokens, rows, scale, into)
    got = tb.embedding_grad(dout, tokens, rows, 0.3, dtype=out, out=into, accumulate=accumulate, sync=True)
    assert got.dtype == out and (into is None or got is into)
    lu.near(got, want, error)


@pytest.mark.parametrize("n", [1, 31, 32, 33, 34, 66, 99, 32 * 33, 33 * 33, 33 * 33 + 1, 33 * 33 * 2, 33 * 66, 33 * 33 * 33])
@pytest.mark.parametrize("shift", [0, 31])
def test_each_row_is_summed_or_cleared(tb, n, shift):
    """Tokens that all differ, so that each row of the result is one row of dout or zero: whether a row occurs is searched for 33 parts at a time, and
    these numbers of places are where such a search comes out even."""
    rows = n + 70
    tokens = torch.randperm(n, generator=torch.Generator(device="cuda").manual_seed(n), device="cuda") + shift
    dout = 1.0 + torch.rand(n, 8, generator=torch.Generator(device="cuda").manual_seed(n + 1), device="cuda")
    want = torch.zeros(rows, 8, device="cuda")
    want[tokens] = dout
    for _ in range(3):
        assert torch.equal(tb.embedding_grad(dout, tokens, rows), want)


@pytest.mark.parametrize("n", [2, 31, 33, 127, 129, 4095, 4736, 4737, 6001, 8191, 8192, 8193])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_places_of_a_token_are_added_in_their_order(tb, n, index):
    """Each token occurs four times or so and some are no rows: the sums of so few are taken one after another in 32 bits, so that any other order shows."""
    rows = n // 4 + 1
    g = torch.Generator(device="cuda").manual_seed(n)
    tokens = ((torch.randperm(n, generator=g, device="cuda") % (rows + 3)) - 1).to(index)      # -1 and some behind the last row
    dout = _normal((n, 12), torch.float32, n + 1)
    on_host, want = dout.cpu(), torch.zeros(rows, 12)
    for i, token in enumerate(tokens.tolist()):
        if 0 <= token < rows:
            want[token] += on_host[i]
    assert torch.equal(tb.embedding_grad(dout, tokens, rows).cpu(), want)


@pytest.mark.parametrize("n,rows,dim", [(20000, 50, 320), (3001, 3001, 72)])
def test_gradient_gives_the_same_bits(tb, n, rows, dim):
    dout, tokens = _normal((n, dim), torch.float32, 9), _tokens(n, rows, 10)
    first = tb.embedding_grad(dout, tokens, rows)
    for _ in range(3):
        assert torch.equal(tb.embedding_grad(dout, tokens, rows), first)


def test_gradient_of_strided_rows(tb):
    wide = _normal((400, 300), torch.bfloat16, 11)
    tokens = _tokens(200, 30, 12)
    for part in (wide[::2, 16:144], wide[::2, 1:129], wide[:200, 3:260]):
        got = tb.embedding_grad(part, tokens, 30, dtype=torch.float32)
        lu.near(got, *lu.embedding_grad(part, tokens, 30, 1.0))


def test_gradient_against_differences(tb):
    """The loss is linear in the table, so a step of one gives the derivative: exactly, but for 64-bit rounding."""
    rows, dim = 5, 3
    weight, c = _normal((rows, dim), torch.float32, 13), _normal((9, dim), torch.float32, 14)
    tokens = _tokens(9, rows, 15)
    loss = lambda w: float((lu.embedding(w, tokens, 0.5) * c.double()).sum())   # noqa: E731
    got = tb.embedding_grad(c, tokens, rows, 0.5)
    for v in range(rows):
        for d in range(dim):
            up, down = weight.double().clone(), weight.double().clone()
            up[v, d] += 1
            down[v, d] -= 1
            assert abs((loss(up) - loss(down)) / 2 - float(got[v, d])) <= 1e-5


def test_tables_past_32_bits(tb):
    rows, dim = (1 << 20) + 60000, 2048       # 2.27 billion elements
    weight = torch.zeros(rows, dim, dtype=torch.bfloat16, device="cuda")
    weight[-5:] = _normal((5, dim), torch.bfloat16, 16)
    tokens = torch.tensor([rows - 1, 0, rows - 5, rows, rows - 3], device="cuda")
    assert torch.equal(tb.embedding(weight, tokens).double(), lu.embedding(weight, tokens, 1.0))
    dout = _normal((5, dim), torch.bfloat16, 17)
    tb.embedding_grad(dout, tokens, rows, out=weight.zero_(), accumulate=True)
    assert torch.equal(weight[rows - 1], dout[0]) and torch.equal(weight[rows - 5], dout[2]) and torch.equal(weight[rows - 3], dout[4])
    assert torch.equal(weight[0], dout[1]) and not weight[1:rows - 5].any()
    got = tb.embedding_grad(dout, tokens, rows, out=weight.fill_(1))
    assert torch.equal(got[rows - 1], dout[0]) and torch.equal(got[rows - 5], dout[2]) and not got[1:rows - 5].any()


def test_another_stream_and_a_graph(tb):
    weight, dout = _normal((300, 128), torch.bfloat16, 18), _normal((700, 128), torch.bfloat16, 19)
    tokens = _tokens(700, 300, 20)
    rows, grad = torch.empty(700, 128, dtype=torch.bfloat16, device="cuda"), torch.empty(300, 128, device="cuda")

    def work():
        tb.embedding(weight, tokens, out=rows)
        tb.embedding_grad(dout, tokens, 300, dtype=torch.float32, out=grad)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(rows.double(), lu.embedding(weight, tokens, 1.0))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        work()
    for seed in (21, 22):
        tokens.copy_(_tokens(700, 300, seed))
        graph.replay()
        assert torch.equal(rows.double(), lu.embedding(weight, tokens, 1.0))
        lu.near(grad, *lu.embedding_grad(dout, tokens, 300, 1.0))
    del graph


def test_refusals(tb):
    weight, tokens = _normal((4, 8), torch.float32, 23), torch.tensor([0, 1], device="cuda")
    for call in (lambda: tb.embedding(weight.double(), tokens), lambda: tb.embedding(weight, tokens.float()), lambda: tb.embedding(weight.cpu(), tokens),
                 lambda: tb.embedding(weight, tokens.cpu()), lambda: tb.embedding(weight.t(), tokens), lambda: tb.embedding(weight[0], tokens),
                 lambda: tb.embedding(weight, tokens, out=torch.empty(2, 7, device="cuda")), lambda: tb.embedding(weight[:1].expand(4, 8), tokens),
                 lambda: tb.embedding(weight, tokens, out=torch.empty(2, 8, device="cuda", dtype=torch.bfloat16)),
                 lambda: tb.embedding_grad(weight, tokens, 4), lambda: tb.embedding_grad(weight[:2], tokens, 1 << 31), lambda: tb.embedding_grad(weight[:2], tokens, -1),
                 lambda: tb.embedding_grad(weight[:2], tokens, 4, accumulate=True), lambda: tb.embedding_grad(weight[:2], tokens, 4, dtype=torch.float64),
                 lambda: tb.embedding_grad(weight[:2], tokens, 4, out=torch.empty(5, 8, device="cuda")),
                 lambda: tb.embedding_grad(weight[:2], tokens, 4, dtype=torch.bfloat16, out=torch.empty(4, 8, device="cuda"))):
        with pytest.raises(ValueError):
            call()

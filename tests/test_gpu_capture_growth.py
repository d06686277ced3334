"""A captured call goes on using the workspace that it was captured with: it stays when a later call on the same stream needs a larger one."""
import weakref

import pytest
import torch

import layers_util as lu

pytestmark = pytest.mark.gpu


def _data(n, rows, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(0, rows, (n,), generator=g, device="cuda"), torch.randn(n, 64, generator=g, device="cuda")


def _grown(tb, side, tag, small, large):
    """Captures small(), calls large() on the same stream, and returns the graph and whether the small call's buffer is still there."""
    with torch.cuda.stream(side):
        small()                             # the workspace exists before the capture
        before = tb.workspaces.at(tb.workspaces.key(tag)).buf.data_ptr()
        held = weakref.ref(tb.workspaces.at(tb.workspaces.key(tag)).buf)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        small()
    with torch.cuda.stream(side):
        large()
        assert tb.workspaces.at(tb.workspaces.key(tag)).buf.data_ptr() != before      # it was too small
    side.synchronize()
    return graph, held() is not None


@pytest.mark.parametrize("what", ["embedding_grad", "sort", "pairs"])
def test_workspace_of_a_graph_stays(tb, what):
    tb.workspaces.clear()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    if what == "embedding_grad":
        tokens, dout = _data(9000, 300, 1)
        big_tokens, big_dout = _data(200000, 300, 2)
        out = torch.empty(300, 64, device="cuda")
        small, large = (lambda: tb.embedding_grad(dout, tokens, 300, out=out)), (lambda: tb.embedding_grad(big_dout, big_tokens, 300))
        tag = "embedding_grad"
    else:
        keys, many = torch.empty(600000, dtype=torch.int32, device="cuda"), torch.randint(0, 1 << 30, (5000000,), device="cuda", dtype=torch.int32)
        keys.random_(0, 1 << 30)
        places = torch.arange(5000000, device="cuda", dtype=torch.int32)
        if what == "sort":
            small, large = (lambda: tb.sort(keys, sync=False)), (lambda: tb.sort(many, sync=False))
        else:
            small, large = (lambda: tb.sort_by_key(keys, places[:600000], sync=False)), (lambda: tb.sort_by_key(many, places, sync=False))
        tag = "sort_keys_alt" if what == "sort" else "sort_vals_alt"
    graph, there = _grown(tb, side, tag, small, large)
    assert there
    # memory that was given back since would be found among these
    others = [torch.full((1 << 20,), 7, dtype=torch.uint8, device="cuda") for _ in range(64)]
    if what == "embedding_grad":
        t, d = _data(9000, 300, 3)
        tokens.copy_(t)
        dout.copy_(d)
        graph.replay()
        lu.near(out, *lu.embedding_grad(d, t, 300, 1.0))
    else:
        keys.random_(0, 1 << 30)
        want = torch.sort(keys).values
        graph.replay()
        assert torch.equal(keys, want)
    assert all(bool((o == 7).all()) for o in others)
    del graph
    tb.workspaces.clear()


def test_workspace_without_a_graph_is_given_back(tb):
    tb.workspaces.clear()
    tokens, dout = _data(9000, 300, 4)
    tb.embedding_grad(dout, tokens, 300)
    held = weakref.ref(tb.workspaces.at(tb.workspaces.key("embedding_grad")).buf)
    tokens, dout = _data(200000, 300, 5)
    tb.embedding_grad(dout, tokens, 300)
    assert held() is None
    tb.workspaces.clear()

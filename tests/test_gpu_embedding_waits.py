"""The embedding's gradient where a wait of the sort before its sums runs out: the result is NaN throughout, the status is 1, a call that waits for its result
raises, and the next call is right.  In a library of its own, built here with the test hooks and a limit of 65536 polls."""
import ctypes as C
import os
import shutil
import subprocess

import pytest

import layers_util as lu

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F32, I64 = 8, 6
GRID, GENERAL = 200003, 600011      # places that the sort of one resident grid takes, and that the general one takes


@pytest.fixture(scope="module")
def short(tmp_path_factory):
    from thrust_b200 import _lib
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.isfile(nvcc):
        pytest.skip("nvcc is not available on this machine")
    path = str(tmp_path_factory.mktemp("waits") / "libwaits.so")
    r = subprocess.run([nvcc, "-std=c++17", "-shared", "-O2", "-gencode", "arch=compute_100a,code=sm_100a", "-Xcompiler", "-fPIC,-fvisibility=hidden", "--threads", "3",
                        "--expt-relaxed-constexpr", "-DTB200_TEST_HOOKS", "-DTB200_SPIN_LIMIT=65536", "-I" + os.path.join(ROOT, "include"), "-I" + os.path.join(ROOT, "thrust_b200", "csrc"),
                        *[os.path.join(ROOT, "thrust_b200", "csrc", f) for f in ("abi_embedding.cu", "abi_reduce.cu", "abi_util.cu")], "-o", path],
                       capture_output=True, text=True, timeout=900)
    assert r.returncode == 0, r.stdout + r.stderr
    lib = _lib.load_partial(path)
    lib.tb200_test_hooks.argtypes = [C.c_uint]
    lib.tb200_test_hooks.restype = C.c_int
    yield lib
    lib.tb200_test_hooks(0)


def _data(n, rows=3000, dim=8):
    import torch
    g = torch.Generator(device="cuda").manual_seed(n)
    return torch.randint(-1, rows + 1, (n,), generator=g, device="cuda"), torch.randn(n, dim, generator=g, device="cuda"), rows


@pytest.mark.parametrize("n", [GRID, GENERAL])
@pytest.mark.parametrize("announced", [False, True])
@pytest.mark.parametrize("accumulate", [0, 1])
def test_the_result_says_that_the_sort_gave_up(short, n, announced, accumulate):
    import torch
    tokens, dout, rows = _data(n)
    out = torch.zeros(rows, dout.shape[1], device="cuda")
    need = C.c_size_t(0)
    args = (dout.data_ptr(), dout.shape[1], tokens.data_ptr(), I64, n, rows, dout.shape[1], F32, F32, 1.0, accumulate, out.data_ptr())
    assert short.tb200_embedding_grad(*args, None, C.byref(need), None) == 0
    ws = torch.full((need.value,), 0xff, dtype=torch.uint8, device="cuda")      # positions that an earlier call has left there might be any
    torch.cuda.synchronize()
    for withheld in (1, 0):
        assert short.tb200_test_hooks(withheld) == 0
        out.zero_()
        torch.cuda.synchronize()
        if announced:
            assert short.tb200_workspace_watch(ws.data_ptr()) == 0
        assert short.tb200_embedding_grad(*args, ws.data_ptr(), C.byref(need), None) == 0
        head = C.create_string_buffer(16)
        assert short.tb200_workspace_read(ws.data_ptr(), 16, head, None) == 0
        status = C.c_uint(7)
        assert short.tb200_workspace_status(ws.data_ptr(), None, C.byref(status)) == 0
        assert head.raw[:4] == bytes([withheld, 0, 0, 0]) and status.value == withheld
        if withheld:
            assert bool(out.isnan().all())
        else:
            lu.near(out, *lu.embedding_grad(dout, tokens, rows, 1.0))


@pytest.mark.parametrize("n", [GRID, GENERAL])
def test_a_call_that_waits_raises(tb, short, monkeypatch, n):
    from thrust_b200 import _lib, api
    tokens, dout, rows = _data(n)
    monkeypatch.setattr(_lib, "_lib", short)
    api.workspaces.clear()
    for _ in range(2):                     # the first call makes the workspace, the second one is announced
        assert short.tb200_test_hooks(1) == 0
        with pytest.raises(api.Tb200Error, match="status 1"):
            tb.embedding_grad(dout, tokens, rows, sync=True)
        assert bool(tb.embedding_grad(dout, tokens, rows).isnan().all())
        assert short.tb200_test_hooks(0) == 0
        lu.near(tb.embedding_grad(dout, tokens, rows, sync=True), *lu.embedding_grad(dout, tokens, rows, 1.0))

"""GPU tests of Sample where the rows of a call decide how it runs: rows of 40960 tokens or more are
cut over work-groups while they are at most vocabulary / 1024 and at most 128. Beyond 131072 tokens
it is the second that counts."""
import ctypes

import pytest
import torch

from my_pytchon_opencl_lib_amd import _native
from test_sample_gpu import check, gen

pytestmark = pytest.mark.gpu

VOCAB = 262144


def new_stream():
    """A stream that nothing used before (torch's own come from a pool of 32, in turn)."""
    s = ctypes.c_void_p()
    _native.call("migemm_stream_create", ctypes.byref(s))
    return torch.cuda.ExternalStream(s.value)


@pytest.mark.parametrize("rows,uses", [(128, True), (129, False), (200, False)])
def test_a_capture_needs_a_workspace_up_to_128_rows(nncl, rows, uses):
    print(rows, flush=True)
    x = torch.randn(rows, VOCAB, generator=gen(rows), device="cuda")
    u = torch.rand(rows, generator=gen(1), device="cuda")
    stream = new_stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    if uses:
        with pytest.raises(_native.MigemmRuntimeError, match="WORKSPACE"):
            with torch.cuda.graph(graph, stream=stream):
                nncl.Sample(x, u)
        torch.cuda.synchronize()
        nncl.reserve_workspace(stream, rows * 34 << 10)  # what the header names
        graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = nncl.Sample(x, u, 0.9, 0, 0.95)
    for i in range(3):
        u.copy_(torch.rand(rows, generator=gen(50 + i), device="cuda"))
        expect = nncl.Sample(x, u, 0.9, 0, 0.95)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], expect[0]) and torch.equal(got[1], expect[1])


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
def test_128_rows_and_129_give_the_same_bits(nncl, kind):
    x = (2 * torch.randn(129, VOCAB, generator=gen(3), device="cuda")).to(kind)
    u = torch.rand(129, generator=gen(4), device="cuda")
    for f in ((1.0, 0, 1.0, 0.0), (0.8, 50, 0.95, 0.0), (1.5, 0, 0.9, 0.01), (0.0, 0, 1.0, 0.0)):
        print(kind, f, flush=True)
        whole, cut = nncl.Sample(x, u, *f), nncl.Sample(x[:128], u[:128], *f)
        assert torch.equal(whole[0][:128], cut[0]) and torch.equal(whole[1][:128], cut[1])
        check(nncl, x[126:], u[126:], *f)

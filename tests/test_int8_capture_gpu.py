"""GPU tests of which LinearInt8 calls use the stream's workspace, as the header states it: a capture
on a stream without one fails where rows * ceil(K / 4096) > 3, and there alone."""
import pytest
import torch

from my_pytchon_opencl_lib_amd import _native

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,k", [(1, 100), (1, 12288), (3, 4096), (1, 12289), (1, 14336),
                                    (2, 4097), (3, 4100), (4, 64)])
def test_capture_needs_a_workspace_where_the_header_says(nncl, rows, k, kind):
    print("capture", rows, k, kind, flush=True)
    g = torch.Generator(device="cuda").manual_seed(k)
    x = torch.randn(rows, k, generator=g, device="cuda").to(kind)
    w8, ws = nncl.QuantizeRows(torch.randn(96, k, generator=g, device="cuda"))
    stream = torch.cuda.Stream()
    # (torch hands out streams again: this one may have a workspace)
    _native.call("migemm_workspace_release", stream.cuda_stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    if rows * -(-k // 4096) > 3:
        with pytest.raises(_native.MigemmRuntimeError, match="WORKSPACE"):
            with torch.cuda.graph(graph, stream=stream):
                nncl.LinearInt8(x, w8, ws)
        torch.cuda.synchronize()
        nncl.reserve_workspace(stream, 1 << 20)
        graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        y = nncl.LinearInt8(x, w8, ws)
    for seed in range(3):
        x.copy_(torch.randn(rows, k, generator=g, device="cuda"))
        expect = nncl.LinearInt8(x, w8, ws)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, expect)

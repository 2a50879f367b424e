"""GPU test of two graphs captured on one stream, the workspace reserved before each: each has buffers
of its own, so that they may be replayed at once on two streams, beside eager calls on the stream of
their capture."""
import pytest
import torch

from test_int8_gpu import gen
from test_sample_border_gpu import new_stream

pytestmark = pytest.mark.gpu


def test_two_graphs_of_one_stream_replayed_at_once(nncl):
    stream = new_stream()
    xs = [torch.randn(3, 131072, generator=gen(i), device="cuda") for i in range(3)]
    us = [torch.rand(3, generator=gen(10 + i), device="cuda") for i in range(3)]
    want = [nncl.Sample(x, u, 0.8, 0, 0.9) for x, u in zip(xs, us)]
    torch.cuda.synchronize()
    graphs, got = [], []
    for i in range(2):
        nncl.reserve_workspace(stream, 1 << 20)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got.append(nncl.Sample(xs[i], us[i], 0.8, 0, 0.9))
        graphs.append(graph)
    sides = [new_stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(5):
        for _ in range(8):
            for graph, side in zip(graphs, sides):
                with torch.cuda.stream(side):
                    graph.replay()
            with torch.cuda.stream(stream):
                eager = nncl.Sample(xs[2], us[2], 0.8, 0, 0.9)
        torch.cuda.synchronize()
        for a, b in zip(got + [eager], want):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])

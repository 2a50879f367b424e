"""GPU tests of a decoder's step in 8 bits as a whole: NormInt8, products with activation, gate and
residual, and Sample together, as a server calls them (examples/serve_int8.py runs them with the
cache and the attention)."""
import importlib.util
import os

import pytest
import torch

from test_int8_gpu import gen

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples",
                    "serve_int8.py")


def block(nncl, x, w, held):
    """Two norms around an inner pair of layers: gate and up in one weight, down with
    the residual."""
    rows, scales, x = nncl.NormInt8(x, w["norm"], residual=held)
    y = w["up"].forwardRows(rows, scales, x.dtype)
    x = w["down"](y, residual=x)
    rows, scales, _ = nncl.NormInt8(x, w["norm"])
    return w["head"].forwardRows(rows, scales)


def weights(nncl, width, inner, vocab):
    from my_pytchon_opencl_lib_amd.layers import LinearInt8
    return {"norm": torch.rand(width, generator=gen(1), device="cuda") + 0.5,
            "up": LinearInt8(torch.randn(2 * inner, width, generator=gen(2), device="cuda") /
                             width ** 0.5, nnclglob=nncl, activation="silu", gated=True),
            "down": LinearInt8(torch.randn(width, inner, generator=gen(3), device="cuda") /
                               inner ** 0.5, nnclglob=nncl),
            "head": LinearInt8(3 * torch.randn(vocab, width, generator=gen(4), device="cuda") /
                               width ** 0.5, nnclglob=nncl)}


def plain(x, w, held):
    """The same in 64 bits from the weights that the layers hold."""
    def full(layer):
        return layer.weight[:, :layer.in_features].double() * layer.scales.double()[:, None]

    def normed(x):
        return x / (x.square().mean(1, keepdim=True) + 1e-6).sqrt() * w["norm"].double()
    x = x.double() + held.double()
    g, u = (normed(x) @ full(w["up"]).t()).chunk(2, 1)
    x = x + (torch.nn.functional.silu(g) * u) @ full(w["down"]).t()
    return normed(x) @ full(w["head"]).t()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,width,inner,vocab", [(1, 256, 512, 1000), (5, 200, 333, 50001),
                                                    (70, 512, 1000, 4001)])
def test_step_against_the_formula(nncl, rows, width, inner, vocab, kind):
    """8 bits cost a few percent of the logits' norm (half a step of 1/127 of a row's largest value
    a term, three layers deep); a wrong gate, residual or scale changes them altogether. The
    greedy token is the logits' largest."""
    print(rows, width, inner, vocab, kind, flush=True)
    w = weights(nncl, width, inner, vocab)
    x = torch.randn(rows, width, generator=gen(5), device="cuda").to(TYPES[kind])
    held = (3 * torch.randn(rows, width, generator=gen(6), device="cuda")).to(TYPES[kind])
    logits = block(nncl, x, w, held)
    want = plain(x, w, held)
    assert float((logits.double() - want).norm() / want.norm()) < 0.06
    tokens, chances = nncl.Sample(logits, torch.rand(rows, device="cuda"), temperature=0.0)
    assert torch.equal(tokens.long(), logits.max(1).indices) and bool((chances == 1).all())


@pytest.mark.parametrize("rows", [1, 6])
def test_captured_step(nncl, rows):
    """A whole step in one graph: every replay gives the eager calls' bits for its inputs."""
    w = weights(nncl, 256, 512, 50001)
    x = torch.randn(rows, 256, generator=gen(7), device="cuda").bfloat16()
    held = torch.randn(rows, 256, generator=gen(8), device="cuda").bfloat16()
    u = torch.rand(rows, generator=gen(9), device="cuda")

    def step():
        logits = block(nncl, x, w, held)
        return logits, nncl.Sample(logits, u, 0.8, 40, 0.95, 0.01)
    stream = torch.cuda.Stream()
    nncl.reserve_workspace(stream, 64 << 20)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        logits, (tokens, chances) = step()
    for i in range(4):
        held.copy_(2 * torch.randn(rows, 256, generator=gen(20 + i), device="cuda"))
        u.copy_(torch.rand(rows, generator=gen(30 + i), device="cuda"))
        want, (t, c) = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(logits, want) and torch.equal(tokens, t) and torch.equal(chances, c)


def test_a_server_samples_what_its_logits_say(nncl):
    """examples/serve_int8.py: a request's sampled tokens are those of its rows alone, and with the
    same random numbers the same again."""
    spec = importlib.util.spec_from_file_location("serve_int8", PATH)
    serve = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(serve)
    runs = []
    for _ in range(2):
        server = serve.Server(nncl, requests=2, pages=20, dtype=torch.bfloat16)
        new, said = [[1, 2, 3], [7] * 20], []
        for i in range(6):
            logits = server.step(new)
            rows = logits[[len(new[0]) - 1, len(logits) - 1]]
            u = torch.rand(2, generator=gen(40 + i), device="cuda")
            t = torch.tensor([0.0, 0.9], device="cuda")
            chosen = server.choose(rows, u, t, topK=50)
            assert chosen[0] == int(rows[0].float().argmax())
            assert chosen[1] == server.choose(rows[1:], u[1:], 0.9, topK=50)[0]
            best = torch.topk(rows[1].float(), 50).values[-1]
            assert float(rows[1, chosen[1]]) >= float(best)
            new = [[c] for c in chosen]
            said.append(chosen)
        runs.append(said)
    assert runs[0] == runs[1]

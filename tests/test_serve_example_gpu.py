"""GPU tests of examples/serve_int8.py: layers, tables, cache and attention together.

The plain model is the same decoder with the layers' float weights, no cache and float32
attention over each request's tokens. What 8 bits cost is a few percent of the logits' norm (a
step of a scale is 1/127 of the largest of a row or page); a wrong slot, page, mask or scale
changes them altogether."""
import importlib.util
import os
import subprocess
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples",
                    "serve_int8.py")


@pytest.fixture(scope="module")
def serve():
    spec = importlib.util.spec_from_file_location("serve_int8", PATH)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def plain_logits(serve, server, tokens):
    """Logits of every token of one request, from the weights that the layers hold."""
    def full(layer):
        return (layer.weight[:, :layer.in_features].double() * layer.scales.double()[:, None])

    pos = torch.arange(len(tokens), device="cuda", dtype=torch.int32)
    angle = pos[:, None] * server.rate
    x = server.embed[tokens].double() + torch.cat([angle.sin(), angle.cos()], 1).double()
    mask = torch.ones(len(tokens), len(tokens), device="cuda").tril() > 0
    for b in server.blocks:
        y = serve.normed(x) @ full(b.qkv).t()
        q, k, v = y.unflatten(1, (b.heads + 2 * b.kvHeads, b.dim)).split(
            (b.heads, b.kvHeads, b.kvHeads), 1)
        k, v = (t.repeat_interleave(b.heads // b.kvHeads, 1) for t in (k, v))
        z = torch.einsum("ihd,jhd->hij", q, k) / b.dim ** 0.5
        p = torch.softmax(z.masked_fill(~mask, float("-inf")), -1)
        o = torch.einsum("hij,jhd->ihd", p, v).flatten(1)
        x = x + o @ full(b.out).t()
        x = x + torch.nn.functional.silu(serve.normed(x) @ full(b.up).t()) @ full(b.down).t()
    return serve.normed(x) @ full(server.head).t()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_steps_match_the_plain_model(nncl, serve, kind):
    server = serve.Server(nncl, dtype={"f32": torch.float32, "bf16": torch.bfloat16}[kind],
                          requests=3, pages=40)
    rng = torch.Generator().manual_seed(4)
    text = [torch.randint(0, 512, (90,), generator=rng).tolist() for _ in range(3)]
    at = [0, 0, 0]
    got = [[], [], []]
    for counts in ([40, 1, 0], [1, 17, 33], [1, 1, 1], [20, 1, 1], [1, 0, 40], [1, 1, 1]):
        logits = server.step([t[a:a + c] for t, a, c in zip(text, at, counts)])
        place = 0
        for r, c in enumerate(counts):
            got[r].append(logits[place:place + c])
            place, at[r] = place + c, at[r] + c
    assert server.lengths.tolist() == at
    for r in range(3):
        mine = torch.cat(got[r]).double()
        want = plain_logits(serve, server, torch.tensor(text[r][:at[r]], device="cuda"))
        far = float((mine - want).norm() / want.norm())
        print("request", r, "off by", far, flush=True)
        assert far < 0.1


def test_a_released_request_leaves_no_trace(nncl, serve):
    """A request in pages that another one used gives the bits that it gives in a new cache."""
    used = serve.Server(nncl, requests=2, pages=12)
    used.step([list(range(100)), list(range(60))])
    used.release([True, True])
    assert int(used.freeCount) == 12
    new = serve.Server(nncl, requests=2, pages=12)
    for tokens in ([[5, 6, 7], []], [[8], [1] * 20], [[9], [2]]):
        assert torch.equal(used.step(tokens), new.step(tokens))


def test_the_example_runs():
    r = subprocess.run([sys.executable, PATH], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stderr[-2000:]
    assert "request 2 said" in r.stdout and "pages free:" in r.stdout

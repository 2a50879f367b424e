"""A small decoder served in 8 bits: layers whose weights are int8, an int8 paged cache, its
tables kept on the GPU.

Each step takes any mix of prompts and single tokens: CacheTables finds pages and slots for the
new tokens, and every block runs NormInt8, a product of its rows (q, k and v in one), CacheAppend,
CacheAttention, LinearInt8 with the residual, and the same for its two inner layers, the first with
its activation. Sample chooses each request's next token. The weights are random; `main` serves
three requests of different lengths side by side, each with its own temperature and top-p, frees one
and admits another in its place.

    python examples/serve_int8.py
"""
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from my_pytchon_opencl_lib_amd import NnClGlob  # noqa: E402
from my_pytchon_opencl_lib_amd.cache import Int8Cache  # noqa: E402
from my_pytchon_opencl_lib_amd.layers import LinearInt8  # noqa: E402


def normed(x):
    """What NormInt8 holds in 8 bits, in the type of x (to compare with)."""
    return x / (x.float().square().mean(-1, keepdim=True) + 1e-6).sqrt().to(x.dtype)


class Block:
    def __init__(self, nncl, width, heads, kvHeads, inner, g):
        def layer(out, fan, activation=None):
            bound = 1 / math.sqrt(fan)
            return LinearInt8((torch.rand(out, fan, generator=g) * 2 - 1) * bound * 1.7,
                              nnclglob=nncl, activation=activation)
        self.nncl, self.heads, self.kvHeads, self.dim = nncl, heads, kvHeads, width // heads
        self.qkv = layer((heads + 2 * kvHeads) * self.dim, width)
        self.out = layer(width, width)
        self.up = layer(inner, width, "silu")
        self.down = layer(width, inner)

    def __call__(self, x, cache, step):
        h, kv = self.heads, self.kvHeads
        rows, scales, _ = self.nncl.NormInt8(x)
        y = self.qkv.forwardRows(rows, scales, x.dtype)
        q, k, v = y.unflatten(1, (h + 2 * kv, self.dim)).split((h, kv, kv), 1)
        # three slices of one product, taken by the operators as they lie
        self.nncl.CacheAppend(k, v, step["slots"], cache)
        o = self.nncl.CacheAttention(q, cache, step["table"], step["starts"],
                                     step["positions"], maxCount=step["maxCount"],
                                     maxLength=step["maxLength"])
        x = self.out(o.flatten(1), residual=x)
        rows, scales, _ = self.nncl.NormInt8(x)
        return self.down(self.up.forwardRows(rows, scales, x.dtype), residual=x)


class Server:
    """A decoder, its caches (one a layer, with one table for all) and its requests' state."""

    def __init__(self, nncl, vocab=512, width=256, heads=8, kvHeads=2, inner=512, layers=2,
                 requests=4, pages=64, pageSize=16, dtype=torch.float32, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.nncl, self.dtype, self.pageSize = nncl, dtype, pageSize
        self.embed = torch.randn(vocab, width, generator=g).to(nncl.device, dtype)
        # positions are added to the embeddings: sines of growing wavelength
        rate = torch.exp(-math.log(10000.0) * torch.arange(0, width, 2) / width)
        self.rate = rate.to(nncl.device)
        self.blocks = [Block(nncl, width, heads, kvHeads, inner, g) for _ in range(layers)]
        self.head = LinearInt8(torch.randn(vocab, width, generator=g) / math.sqrt(width),
                               nnclglob=nncl)
        self.caches = [Int8Cache(pages, kvHeads, width // heads, pageSize, nncl.device)
                       for _ in range(layers)]
        self.free, self.freeCount = self.caches[0].freePages()
        self.table = self.caches[0].blockTable(requests, pages)
        self.lengths = torch.zeros(requests, dtype=torch.int32, device=nncl.device)
        self.longest = [0] * requests  # the host's bound of each length

    def step(self, tokens):
        """tokens: a list of new token numbers for each request (empty: it rests). Returns the
        logits of every new token, packed in the requests' order."""
        counts = [len(t) for t in tokens]
        flat = torch.tensor([v for t in tokens for v in t], dtype=torch.int32)
        dev = self.nncl.device
        self.longest = [a + b for a, b in zip(self.longest, counts)]
        slots, positions, starts, self.lengths, self.freeCount = self.nncl.CacheTables(
            self.lengths, torch.tensor(counts, dtype=torch.int32).to(dev), self.table, self.free,
            self.freeCount, len(flat), self.pageSize)
        step = {"slots": slots, "positions": positions, "starts": starts, "table": self.table,
                "maxCount": max(counts), "maxLength": max(self.longest)}
        angle = positions[:, None] * self.rate
        x = self.embed[flat.to(dev)] + torch.cat([angle.sin(), angle.cos()], 1).to(self.dtype)
        for block, cache in zip(self.blocks, self.caches):
            x = block(x, cache, step)
        rows, scales, _ = self.nncl.NormInt8(x)
        return self.head.forwardRows(rows, scales, self.dtype)

    def choose(self, logits, uniforms, temperature=1.0, topK=0, topP=1.0, minP=0.0):
        """A token for each row of logits, from one random number a row, as a list."""
        return self.nncl.Sample(logits, uniforms, temperature, topK, topP, minP)[0].tolist()

    def release(self, finished):
        """Frees the requests i with finished[i]: their pages may be given out again."""
        flags = torch.tensor([int(bool(f)) for f in finished], dtype=torch.int32)
        self.nncl.CacheRelease(flags.to(self.nncl.device), self.lengths, self.table, self.free,
                               self.freeCount, self.pageSize)
        self.longest = [0 if f else n for f, n in zip(finished, self.longest)]


def main():
    server = Server(NnClGlob("cuda:0"), dtype=torch.bfloat16)
    prompts = [list(range(1, 38)), [5, 6, 7], list(range(100, 180)), []]
    said = [[] for _ in prompts]
    new = prompts
    # request 0 takes the likeliest token, the others sample
    temperature = torch.tensor([0.0, 0.8, 1.0, 1.0], device="cuda")
    topP = torch.tensor([1.0, 0.9, 0.95, 1.0], device="cuda")
    rng = torch.Generator(device="cuda").manual_seed(1)
    for i in range(12):
        if i == 6:  # request 1 is done; another comes in its place
            server.release([False, True, False, False])
            print("request 1 said", said[1])
            said[1] = []
            new[1] = list(range(200, 220))
        logits = server.step(new)
        active = [r for r, t in enumerate(new) if t]
        last, at = [], -1
        for r in active:
            at += len(new[r])
            last.append(at)
        chosen = server.choose(logits[last], torch.rand(len(active), generator=rng, device="cuda"),
                               temperature[active], topP=topP[active])
        new = [[] for _ in prompts]
        for r, token in zip(active, chosen):
            new[r] = [token]
            said[r].append(token)
    for r, s in enumerate(said):
        if s:
            print("request", r, "said", s)
    print("pages free:", int(server.freeCount), "of", server.caches[0].pages)


if __name__ == "__main__":
    main()

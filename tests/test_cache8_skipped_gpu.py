"""GPU tests of NnClGlob.CacheAppend where tokens are skipped (slot -1 or outside the pool) between
the tokens of one page: drafts that were turned down, padding inside a request. The page has one
scale over all its new tokens, as if the skipped ones were not there; every byte and scale by the
rule (PlainCache of test_cache8_gpu.py)."""
import random

import numpy as np
import pytest
import torch

from my_pytchon_opencl_lib_amd.cache import Int8Cache
from test_cache8_gpu import TYPES, PlainCache, filled, gen, ints, same_cache, say

pytestmark = pytest.mark.gpu


def append(nncl, cache, plain, slots, kind, seed):
    heads, dim = cache.kvHeads, cache.headDim
    size = torch.exp(torch.randn(len(slots), 1, 1, generator=gen(seed), device="cuda"))
    k = (size * torch.randn(len(slots), heads, dim, generator=gen(seed + 1), device="cuda"))
    v = (torch.randn(len(slots), heads, dim, generator=gen(seed + 2), device="cuda") / size)
    k, v = k.to(TYPES[kind]), v.to(TYPES[kind])
    nncl.CacheAppend(k, v, ints(slots), cache)
    plain.append(k.float().cpu().numpy(), v.float().cpu().numpy(), slots)
    same_cache(cache, plain)


def known(cache):
    plain = PlainCache(cache)
    plain.known[:] = True
    return plain


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("gap", [1, 2, 61, 62, 63, 64, 190, 255, 256, 511, 513, 1100, 5000])
def test_two_tokens_of_a_page_with_a_gap(nncl, gap, kind):
    """One work-group a token (few tokens), and chunks that the gap runs over."""
    say("gap", gap, kind)
    cache = filled(1, 40, 16, 4, gap)
    plain = known(cache)
    append(nncl, cache, plain, [5] + [-1] * gap + [6], kind, gap)
    append(nncl, cache, plain, [-1] * 3 + [7] + [10 ** 9] * gap + [8] + [-1] * gap, kind, gap)
    # the page's first slot behind the gap, another page before and behind
    append(nncl, cache, plain, [31, 33] + [64] * gap + [32] + [-1] * gap + [34, 0], kind, gap)
    # a gap between two pages is none inside either
    append(nncl, cache, plain, [40] + [-1] * gap + [16, 17], kind, gap)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("heads,dim,page,tokens", [(1, 8, 16, 400), (2, 128, 64, 300),
                                                   (4, 64, 16, 5000), (8, 64, 32, 3000),
                                                   (16, 32, 64, 4500), (16, 40, 128, 5000)])
def test_skipped_tokens_anywhere(nncl, heads, dim, page, tokens, kind):
    """Chunks of 1 to 64 tokens; pages begun anywhere, some tokens out of order, gaps of any
    length."""
    say("skipped", heads, dim, page, tokens, kind)
    rng = random.Random(tokens + page)
    pages = tokens // page + 80
    cache = filled(heads, dim, page, pages, dim)
    plain = known(cache)
    order = list(range(pages))
    rng.shuffle(order)
    slots = []
    for p in order:
        first = rng.choice([0, 0, rng.randrange(page)])
        run = list(range(p * page + first, p * page + rng.randint(first + 1, page)))
        if rng.random() < 0.3:
            rng.shuffle(run)
        share = rng.choice([0.0, 0.1, 0.5])
        for s in run:
            while rng.random() < share:
                slots.append(rng.choice([-1, -7, pages * page, 2 ** 31 - 1]))
            if rng.random() < 0.01:
                slots += [-1] * rng.choice([64, 130, 257, 600])
            slots.append(s)
    append(nncl, cache, plain, slots[:tokens], kind, page)


def test_a_page_full_of_tokens_between_skipped_ones(nncl):
    """128 tokens of a page, several skipped behind each, and none of the call past its last."""
    cache = Int8Cache(3, 2, 256, 128)
    plain = PlainCache(cache)
    slots = [s for t in range(128, 256) for s in [t] + [-1] * (t % 7)]
    append(nncl, cache, plain, slots, "f32", 1)
    append(nncl, cache, plain, [-1] * 700, "f32", 2)  # nothing at all
    assert np.array_equal(plain.scales[0][0], [0, 0])

"""GPU tests of NnClGlob.CacheAttention for steps of few tokens over long contexts, whose tiles of
all requests are cut into even shares: cuts inside contexts of any length, requests without tokens
or pages, more than 16 rows a request, hints that are wrong, and more requests than the shares
take. Compared like test_cache8_gpu.py's attention, within the same bounds."""
import random

import pytest
import torch

from test_cache8_gpu import TYPES, attention64, check_attention, filled, gen, ints, say, step_of

pytestmark = pytest.mark.gpu


def run(nncl, heads, kv, dim, page, lengths, counts, kind, hints, lose=0, seed=1):
    need = sum(-(-n // page) for n in lengths)
    cache = filled(kv, dim, page, need + 2, dim + seed)
    table, starts, positions, tokens = step_of(nncl, cache, lengths, counts, 2, page + seed)
    rng = random.Random(seed)
    for _ in range(lose):  # pages that are not there: their tokens are not seen
        row = rng.randrange(len(table))
        used = -(-lengths[row] // page)
        if used > 1:
            table[row][rng.randrange(used)] = rng.choice([-1, cache.pages, 2 ** 31 - 1])
    q = torch.randn(tokens, heads, dim, generator=gen(heads + seed), device="cuda")
    q = q.to(TYPES[kind])
    want = attention64(q, cache, table, starts, positions, dim ** -0.5)
    for count, length in hints:
        say("shares", heads, kv, dim, page, len(lengths), kind, count, length)
        got = nncl.CacheAttention(q, cache, ints(table), starts, positions, maxCount=count,
                                  maxLength=length)
        check_attention(got, want, max(lengths))
        assert not got[sum(counts):].any()
        again = nncl.CacheAttention(q, cache, ints(table), starts, positions, maxCount=count,
                                    maxLength=length)
        assert torch.equal(got, again)  # the same bits every time


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("heads,kv,dim,page,requests,most,seed", [
    (8, 2, 64, 32, 40, 1500, 1), (4, 4, 128, 64, 23, 900, 2), (2, 1, 32, 16, 70, 700, 3),
    (3, 3, 96, 128, 9, 2500, 4), (4, 2, 192, 64, 6, 1300, 5), (2, 1, 256, 16, 5, 1100, 6),
    (16, 1, 128, 16, 3, 5000, 7)])
def test_shares_of_contexts_of_any_length(nncl, heads, kv, dim, page, requests, most, seed, kind):
    rng = random.Random(seed)
    lengths = [rng.choice([1, 63, 64, 65, rng.randint(1, most)]) for _ in range(requests - 1)]
    run(nncl, heads, kv, dim, page, lengths + [most], [1] * requests, kind, [(1, most)], seed=seed)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("heads,kv,dim,page,lengths,counts", [
    (4, 1, 64, 16, [600, 5, 0, 130], [4, 3, 0, 1]),       # several tokens, up to 16 rows
    (4, 2, 128, 64, [700, 41, 260], [30, 40, 9]),         # more rows than 16: further units
    (6, 1, 96, 32, [520, 17, 1000], [1, 17, 7]),
    (2, 2, 256, 128, [900, 3], [20, 2])])
def test_shares_of_several_tokens_and_wrong_hints(nncl, heads, kv, dim, page, lengths, counts,
                                                  kind):
    run(nncl, heads, kv, dim, page, lengths, counts, kind,
        [(1, max(lengths)), (1, 100000), (2, 513), (max(counts), max(lengths))])


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("heads,kv,dim,page,lengths,counts", [
    (4, 1, 128, 64, [2100, 64, 1500], [5, 8, 6]),         # 20 to 32 rows: float32 in shares
    (8, 2, 64, 16, [1300, 900], [8, 1]),
    (2, 1, 256, 32, [1100, 30, 600], [12, 16, 9]),
    (4, 1, 96, 64, [3000, 1200], [30, 100]),              # more rows: two ranges a CU
    (8, 1, 128, 32, [1024], [64])])
def test_few_queries_over_long_contexts(nncl, heads, kv, dim, page, lengths, counts, kind):
    run(nncl, heads, kv, dim, page, lengths, counts, kind, [(max(counts), max(lengths)), (0, 0)])


@pytest.mark.parametrize("page", [16, 64])
def test_shares_with_pages_that_are_not_there(nncl, page):
    rng = random.Random(page)
    lengths = [rng.randint(1, 800) for _ in range(12)] + [0, 2, 1200]
    counts = [1] * 12 + [0, 1, 1]
    run(nncl, 4, 2, 64, page, lengths, counts, "f32", [(1, 1200)], lose=25)


@pytest.mark.parametrize("requests", [1000, 1022, 1023, 1100])
def test_shares_of_many_requests(nncl, requests):
    rng = random.Random(requests)
    lengths = [rng.randint(1, 40) for _ in range(requests - 1)] + [600]
    run(nncl, 2, 1, 32, 16, lengths, [1] * requests, "bf16", [(1, 600)], seed=requests)

"""GPU tests of NnClGlob.CacheAttention over the range of query values: a few large ones among
ordinary ones (as layers' outlier channels are), and rows of any size. Every form of the kernel (single
tokens in ranges and in shares, several tokens, prompts) holds a query as exactly as float32
does, so the bounds are those of test_cache8_gpu.py, whose A leaves out what a zero of the cache
multiplies."""
import pytest
import torch

from test_cache8_gpu import TYPES, attention64, check_attention, filled, gen, ints, say, step_of

pytestmark = pytest.mark.gpu

FORMS = [  # lengths after the step, new tokens, hints
    ([300, 20, 64], [1, 1, 1], (1, 300)),       # single tokens, ranges
    ([700, 90, 513], [1, 1, 1], (1, 700)),      # shares
    ([900, 40], [9, 2], (2, 900)),              # shares, more rows
    ([330, 40], [40, 40], (40, 330)),           # prompts
]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("dim", [32, 72, 96, 128, 256])
@pytest.mark.parametrize("lengths,counts,hints", FORMS)
@pytest.mark.parametrize("big", [1e3, 1e4, 1e6])
def test_a_large_value_over_a_channel_of_zeros(nncl, lengths, counts, hints, dim, big, kind):
    say("outlier", lengths, counts, dim, big, kind)
    cache = filled(2, dim, 16, sum(-(-n // 16) for n in lengths) + 2, dim)
    at = dim // 2 + 3
    cache.keys[..., at] = 0
    table, starts, positions, tokens = step_of(nncl, cache, lengths, counts, 0, 5)
    q = torch.randn(tokens, 4, dim, generator=gen(dim), device="cuda").to(TYPES[kind])
    q[:, :, at] = big
    got = nncl.CacheAttention(q, cache, ints(table), starts, positions, maxCount=hints[0],
                              maxLength=hints[1])
    check_attention(got, attention64(q, cache, table, starts, positions, dim ** -0.5),
                    max(lengths))
    # what a zero multiplies does not count at all
    q[:, :, at] = 0
    other = nncl.CacheAttention(q, cache, ints(table), starts, positions, maxCount=hints[0],
                                maxLength=hints[1])
    assert torch.equal(got, other)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("lengths,counts,hints", FORMS)
def test_rows_of_any_size(nncl, lengths, counts, hints, kind):
    """Each row and value of another size; scores stay below a few hundred."""
    dim = 64
    cache = filled(2, dim, 16, sum(-(-n // 16) for n in lengths) + 2, dim)
    table, starts, positions, tokens = step_of(nncl, cache, lengths, counts, 0, 5)
    g = gen(7)
    q = torch.randn(tokens, 4, dim, generator=g, device="cuda")
    q = q * torch.exp2(torch.randint(-40, 4, (tokens, 4, dim), generator=g, device="cuda"))
    q = (q * torch.exp2(torch.randint(-30, 4, (tokens, 4, 1), generator=g, device="cuda")))
    q = q.to(TYPES[kind])
    got = nncl.CacheAttention(q, cache, ints(table), starts, positions, maxCount=hints[0],
                              maxLength=hints[1])
    check_attention(got, attention64(q, cache, table, starts, positions, 1.0 / 8), max(lengths))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("lengths,counts,hints", FORMS)
@pytest.mark.parametrize("value", ["inf", "-inf", "nan"])
def test_queries_that_are_not_finite_are_seen(nncl, lengths, counts, hints, value, kind):
    """Against keys of one sign an infinite query's scores are all inf or all -inf, neither of
    which has a softmax: NaN, never zeros, in its row and no other; 0 where the row has no key."""
    dim = 64
    cache = filled(2, dim, 16, sum(-(-n // 16) for n in lengths) + 2, dim)
    cache.keys[..., 11] = cache.keys[..., 11].abs().clamp(min=1)
    table, starts, positions, tokens = step_of(nncl, cache, lengths, counts, 0, 5)
    q = torch.randn(tokens, 4, dim, generator=gen(9), device="cuda").to(TYPES[kind])
    args = dict(maxCount=hints[0], maxLength=hints[1])
    clean = nncl.CacheAttention(q, cache, ints(table), starts, positions, **args)
    bad = torch.zeros(tokens, 4, dtype=torch.bool, device="cuda")
    bad[0, 1] = bad[-1, 3] = bad[tokens // 2, 0] = True
    q[:, :, 11] = torch.where(bad, float(value), q[:, :, 11])
    got = nncl.CacheAttention(q, cache, ints(table), starts, positions, **args)
    assert torch.equal(got.isnan(), bad[:, :, None].expand_as(got))
    assert torch.equal(got[~bad], clean[~bad])
    positions[0] = -1
    got = nncl.CacheAttention(q, cache, ints(table), starts, positions, **args)
    assert not got[0].any()

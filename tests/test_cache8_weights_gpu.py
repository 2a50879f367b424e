"""GPU tests of the weights of NnClGlob.CacheAttention's bfloat16 calls, which are held in 11 bits
with a running maximum of their own over score + log2 of the value scale.

Before it is rounded to bfloat16 a result is off from y, the formula in 64 bits, by at most e: with Y
the same mean over the values' magnitudes, 2^-11 Y from the weights (2^-11 each at most; they are the
same in numerator and denominator, so that what counts is how far the values are from their mean),
what float32 scores and sums add (test_cache8_gpu.py's docstring, with Y for its V), and 2^-30 of the
row's largest Y a key for weights that are subnormal in f16 (2^-25, where the row's largest is 2^6 at
least). Rounding is monotone, so the result lies between y - e and y + e rounded.

In norm, rounding to 8 bits alone is off by 2^-8 / sqrt(3) of what 1 / mantissa averages to over
values of all sizes, 0.74: 1.66e-3. Weights of 8 bits bring that to 2.2e-3 to 2.4e-3."""
import copy

import pytest
import torch

from test_cache8_gpu import attention64, filled, gen, ints, say, step_of

pytestmark = pytest.mark.gpu

FORMS = [  # lengths after the step, new tokens, max_count, max_length
    ([400, 130], [1, 1], 1, 400),           # single tokens, ranges
    ([1700, 600, 65], [1, 1, 1], 1, 1700),  # shares
    ([900, 500], [5, 8], 8, 900),           # several tokens
    ([500, 130], [200, 130], 200, 500),     # prompts
]


def run(nncl, heads, dim, page, lengths, counts, hints, seed, change=None):
    """(result, y, y - e and y + e rounded)"""
    cache = filled(2, dim, page, sum(-(-n // page) for n in lengths) + 2, seed)
    table, starts, positions, tokens = step_of(nncl, cache, lengths, counts, 0, seed)
    q = torch.randn(tokens, heads, dim, generator=gen(seed), device="cuda").bfloat16()
    if change is not None:
        change(cache, table, q)
    got = nncl.CacheAttention(q, cache, ints(table), starts, positions, maxCount=hints[0],
                              maxLength=hints[1])
    y, a, _ = attention64(q, cache, table, starts, positions, dim ** -0.5)
    sizes = copy.deepcopy(cache)
    sizes.values.abs_()
    most = attention64(q, sizes, table, starts, positions, dim ** -0.5)[0]
    keys = max(lengths)
    part = 2 * (2 * (dim + 8) * 2.0 ** -24 * a + 2.0 ** -21) + (keys / 64 + 72) * 2.0 ** -24
    e = (2.0 ** -11 + part[..., None]) * most + keys * 2.0 ** -30 * most.amax(2, keepdim=True)
    return got, y, rounded(y - e), rounded(y + e)


def rounded(x):
    """64 bits to bfloat16 at once (a float32 between would round twice), as 64 bits."""
    _, n = torch.frexp(x)
    # 2^(n - 8), put together from its bits (a power computed on the GPU need not be exact)
    step = ((n.long().clamp(min=-125) - 8 + 1023) << 52).view(torch.float64)
    return torch.round(x / step) * step


@pytest.mark.parametrize("dim", [32, 72, 96, 128, 256])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("lengths,counts,count,length", FORMS)
def test_the_result_is_little_more_off_than_its_rounding(nncl, lengths, counts, count, length, page,
                                                         dim):
    say("weights", lengths, counts, page, dim)
    got, y, low, high = run(nncl, 8, dim, page, lengths, counts, (count, length), dim + page)
    got = got.double()
    assert bool(((low <= got) & (got <= high)).all())
    far = float((got - y).norm() / y.norm())
    say(far)
    assert far <= 2.0 ** -9 + 2.0 ** -12


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("shape", ["rising", "falling", "random", "steps", "zeros between"])
@pytest.mark.parametrize("lengths,counts,count,length", FORMS)
def test_value_scales_of_any_size_side_by_side(nncl, lengths, counts, count, length, shape, page):
    """Every result on its own, whatever sizes its row's pages have (what a row sees ends inside
    tiles, among pages of other sizes)."""
    say("scales", shape, lengths, page)

    def change(cache, table, q):
        for row in table:
            for j, p in enumerate(row):
                if 0 <= p < cache.pages:
                    s = {"rising": 2.0 ** (j - 20), "falling": 2.0 ** (20 - j),
                         "random": 2.0 ** ((j * 37 + 11) % 61 - 30),
                         "steps": 1e-6 if j % 5 else 1e6,
                         "zeros between": 0.0 if j % 3 == 0 else 0.01}[shape]
                    cache.valueScales[p] = max(s, 2.0 ** -100) if s else 0.0

    got, _, low, high = run(nncl, 4, 64, page, lengths, counts, (count, length), 3, change)
    got = got.double()
    assert bool(((low <= got) & (got <= high)).all())


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("big", [2.0 ** 10, 2.0 ** 40, 2.0 ** 90])
@pytest.mark.parametrize("lengths,counts,count,length", FORMS)
def test_a_huge_page_without_weight(nncl, lengths, counts, count, length, big, page):
    """A page whose keys no query attends to (scores 2^-290 of the others' weight) has values 2^10 to
    2^90 times the others': the others' result keeps its bits; and the other way round a page of tiny
    values that has nearly all the weight counts in full in the denominator."""
    say("huge", lengths, big, page)

    def change(cache, table, q):
        q[:, :, 0] = 8.0
        cache.keys[..., 0] = 0
        for row in table:
            if len(row) > 1 and row[1] >= 0:
                cache.keys[row[1], :, :, 0] = -127
                cache.keys[row[1], :, :, 1:] = 0
                cache.keyScales[row[1]] = 200.0 * 8 / 8 / 127  # scores of -200
                cache.valueScales[row[1]] = 0.01 * big

    got, _, low, high = run(nncl, 4, 64, page, lengths, counts, (count, length), 5, change)
    got = got.double()
    assert bool(((low <= got) & (got <= high)).all())

    def heavy(cache, table, q):
        q[:, :, 0] = 8.0
        cache.keys[..., 0] = 0
        for row in table:
            cache.keys[row[0], :, :, 0] = 127
            cache.keyScales[row[0]] = 20.0 / 127  # scores of 20 and more
            cache.valueScales[row[0]] = 0.01 / big

    got, _, low, high = run(nncl, 4, 64, page, lengths, counts, (count, length), 6, heavy)
    got = got.double()
    assert bool(((low <= got) & (got <= high)).all())

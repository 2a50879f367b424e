"""GPU tests of CacheAttention's reading of starts: tokens that belong to no request, before the
first one's and past the last one's, are written as 0 by every form of the kernel; starts that
descend leave what lies around the result as it is."""
import pytest
import torch

from my_pytchon_opencl_lib_amd import _native
from test_cache8_gpu import TYPES, attention64, check_attention, filled, gen, ints, say, step_of

pytestmark = pytest.mark.gpu

FORMS = [  # lengths after the step, new tokens, max_count, max_length
    ([130, 20], [1, 1], 1, 130),         # single tokens, whole
    ([490, 20], [1, 1], 1, 490),         # ranges
    ([700, 90, 513], [1, 1, 1], 1, 700),  # shares
    ([200, 40], [40, 40], 40, 200),      # prompts, whole
    ([1500, 40], [40, 40], 40, 1500),    # prompts, ranges
    ([600, 90], [33, 2], 0, 0),
]


def attend(q, cache, table, starts, positions, count, length, out):
    rows, columns = len(table), len(table[0])
    tokens, heads, dim = q.shape
    table = ints(table)
    _native.call("migemm_cache_attention", torch.cuda.current_stream().cuda_stream, q.data_ptr(),
                 int(q.dtype == torch.bfloat16), heads * dim, *cache.pointers, *cache.sizes,
                 table.data_ptr(), columns, starts.data_ptr(), positions.data_ptr(), rows, tokens,
                 heads, dim ** -0.5, count, length, out.data_ptr())
    torch.cuda.synchronize()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("lead", [1, 2, 9, 200])
@pytest.mark.parametrize("lengths,counts,count,length", FORMS)
def test_tokens_before_the_first_request(nncl, lengths, counts, count, length, lead, kind):
    say("lead", lead, lengths, counts, kind)
    cache = filled(2, 64, 16, sum(-(-n // 16) for n in lengths) + 2, 4)
    table, starts, positions, tokens = step_of(nncl, cache, lengths, counts, 3, 7)
    starts = starts + lead
    # (positions of the tokens that have no request look like others')
    positions = torch.cat([ints([5] * lead), positions[:-3], ints([7, 0, 300])])
    tokens += lead
    q = torch.randn(tokens, 4, 64, generator=gen(2), device="cuda").to(TYPES[kind])
    whole = torch.full((tokens + 2, 4, 64), float("nan"), device="cuda", dtype=q.dtype)
    attend(q, cache, table, starts, positions, count, length, whole[1:-1])
    got = whole[1:-1]
    assert not got[:lead].any() and not got[-3:].any()
    check_attention(got, attention64(q, cache, table, starts, positions, 0.125), max(lengths))
    assert bool(whole[0].isnan().all()) and bool(whole[-1].isnan().all())


@pytest.mark.parametrize("lengths,counts,count,length", FORMS)
def test_no_request_has_tokens(nncl, lengths, counts, count, length):
    """Starts past the step, or all at one place: zeros everywhere."""
    cache = filled(2, 64, 16, sum(-(-n // 16) for n in lengths) + 2, 4)
    table, starts, positions, tokens = step_of(nncl, cache, lengths, counts, 0, 7)
    q = torch.randn(tokens, 4, 64, generator=gen(2), device="cuda")
    for place in (0, tokens // 2, tokens, 2 ** 31 - 1, -2 ** 31):
        out = torch.full_like(q, float("nan"))
        attend(q, cache, table, torch.full_like(starts, place), positions, count, length, out)
        assert not out.any()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("lengths,counts,count,length", FORMS)
def test_starts_that_descend(nncl, lengths, counts, count, length, kind):
    """What the rows hold is not defined; what lies around them stays, and the next call is right."""
    cache = filled(2, 64, 16, sum(-(-n // 16) for n in lengths) + 2, 4)
    table, starts, positions, tokens = step_of(nncl, cache, lengths, counts, 0, 7)
    q = torch.randn(tokens, 4, 64, generator=gen(2), device="cuda").to(TYPES[kind])
    whole = torch.full((tokens + 2, 4, 64), 7.0, device="cuda", dtype=q.dtype)
    for odd in (starts.flip(0), torch.tensor([0, tokens] * 9)[:starts.numel()].to(starts)):
        attend(q, cache, table, odd.contiguous(), positions, count, length, whole[1:-1])
        assert bool((whole[0] == 7).all()) and bool((whole[-1] == 7).all())
    attend(q, cache, table, starts, positions, count, length, whole[1:-1])
    check_attention(whole[1:-1], attention64(q, cache, table, starts, positions, 0.125),
                    max(lengths))

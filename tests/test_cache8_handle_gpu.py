"""GPU tests of copies and changes of a cache.Int8Cache: the operators work on the tensors that the
handle holds, and refuse ones that do not fit it."""
import copy
import pickle

import pytest
import torch

from my_pytchon_opencl_lib_amd import ShapeError
from my_pytchon_opencl_lib_amd.cache import Int8Cache
from test_cache8_gpu import filled, gen, ints

pytestmark = pytest.mark.gpu


def contents(cache):
    return [t.clone() for t in (cache.keys, cache.values, cache.keyScales, cache.valueScales)]


@pytest.mark.parametrize("copied", [copy.deepcopy, lambda c: pickle.loads(pickle.dumps(c))],
                         ids=["deepcopy", "pickle"])
def test_a_copy_is_a_cache_of_its_own(nncl, copied):
    """A fork of a request: what is appended to the copy is in the copy alone, and reading and
    attention see it there."""
    first = filled(2, 64, 16, 4, 3)
    before = contents(first)
    other = copied(first)
    k = torch.randn(3, 2, 64, generator=gen(1), device="cuda") * 5
    slots = ints([14, 15, 16])
    nncl.CacheAppend(k, 2 * k, slots, other)
    assert all(torch.equal(a, b) for a, b in zip(before, contents(first)))
    assert not torch.equal(other.keys, first.keys)
    half = 0.51 * k.abs().max() / 127
    assert bool(((nncl.CacheRead(other, slots)[0] - k).abs() <= half).all())
    nncl.CacheAppend(k, 2 * k, slots, first)  # the same step gives the same cache
    assert all(torch.equal(a, b) for a, b in zip(contents(other), contents(first)))
    q = torch.randn(1, 4, 64, generator=gen(2), device="cuda")
    args = ints([[0, 1]]), ints([0, 1]), ints([20])
    a, b = nncl.CacheAttention(q, first, *args), nncl.CacheAttention(q, other, *args)
    assert torch.equal(a, b)
    other.valueScales.mul_(2)
    assert torch.equal(nncl.CacheAttention(q, other, *args), 2 * b)
    assert torch.equal(nncl.CacheAttention(q, first, *args), a)


def test_tensors_that_do_not_fit_are_refused(nncl):
    q = torch.zeros(2, 2, 64, device="cuda")
    for name, wrong in (("keys", lambda t: t[:3]), ("values", lambda t: t.float()),
                        ("keyScales", lambda t: t.t().contiguous().t()),
                        ("valueScales", lambda t: t.cpu()), ("keyScales", lambda t: t.double()),
                        ("values", lambda t: t.transpose(2, 3)), ("pages", lambda n: n + 1)):
        cache = Int8Cache(4, 2, 64, 16)
        setattr(cache, name, wrong(getattr(cache, name)))
        for call in (lambda: nncl.CacheAppend(q, q, ints([0, 1]), cache),
                     lambda: nncl.CacheRead(cache, ints([0, 1])),
                     lambda: nncl.CacheAttention(q, cache, ints([[0, 1]]), ints([0, 2]),
                                                 ints([0, 1]))):
            with pytest.raises(ShapeError, match="of the cache must|on one device"):
                call()

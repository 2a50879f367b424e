"""CPU tests of the handle of the 8-bit paged cache: what it hands to the kernels are the tensors
that it holds now. (Its operators on the GPU: test_cache8_handle_gpu.py.)"""
import copy
import io
import pickle

import pytest
import torch

from my_pytchon_opencl_lib_amd.cache import Int8Cache


def saved_and_loaded(cache):
    f = io.BytesIO()
    torch.save(cache, f)
    f.seek(0)
    return torch.load(f, weights_only=False)  # (written by this test)


@pytest.mark.parametrize("copied", [copy.deepcopy, lambda c: pickle.loads(pickle.dumps(c)),
                                    saved_and_loaded], ids=["deepcopy", "pickle", "torch.save"])
def test_a_copy_names_its_own_memory(copied):
    cache = Int8Cache(3, 2, 40, 16, device="cpu")
    cache.keys.random_(-127, 128)
    other = copied(cache)
    mine = (other.keys, other.values, other.keyScales, other.valueScales)
    assert other.pointers == tuple(t.data_ptr() for t in mine)
    assert not set(other.pointers) & set(cache.pointers)
    assert other.sizes == cache.sizes and torch.equal(other.keys, cache.keys)


def test_a_replaced_tensor_is_the_one_that_counts():
    cache = Int8Cache(3, 2, 40, 16, device="cpu")
    cache.values = torch.zeros_like(cache.values)
    assert cache.pointers[1] == cache.values.data_ptr()

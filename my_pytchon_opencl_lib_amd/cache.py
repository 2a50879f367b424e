"""The 8-bit paged cache of keys and values that the Cache operators of NnClGlob work on.

A page holds pageSize tokens of every kv head. Keys and values are int8 with one float32 scale
for each page and head (so a page's tokens of a head share it). A page lies as the attention
kernels read it: keys [page, head, token, width], values [page, head, width, token] (transposed,
the tokens of one feature are neighbours); width is the head size rounded up to 32 (to 64
above 128), the added features hold nothing. Which request owns which page stands in a block
table that NnClGlob.CacheTables fills on the GPU from a list of free pages.
"""
import torch

from . import _native
from .nncl_glob import ShapeError, _check_typed, _require

_INT8, _FLOAT = torch.int8, torch.float32


def width(headDim):
    return -(-headDim // 32) * 32 if headDim <= 128 else -(-headDim // 64) * 64


class Int8Cache:
    """`pages` pages of `pageSize` (16, 32, 64 or 128) tokens, for kvHeads heads of headDim (a
    multiple of 8, at most 256). Memory: 2 * pages * kvHeads * (pageSize * width + 4) bytes."""

    def __init__(self, pages, kvHeads, headDim, pageSize=64, device="cuda:0"):
        _native.load()
        self.pages, self.kvHeads = int(pages), int(kvHeads)
        self.headDim, self.pageSize = int(headDim), int(pageSize)
        _require(self.pages >= 1 and self.kvHeads >= 1, "pages and kvHeads must be at least 1")
        if not (8 <= self.headDim <= 256 and self.headDim % 8 == 0):
            raise ShapeError(f"headDim must be a multiple of 8 in 8..256 (got {self.headDim})")
        if self.pageSize not in (16, 32, 64, 128):
            raise ShapeError(f"pageSize must be 16, 32, 64 or 128 (got {self.pageSize})")
        if self.pages * self.pageSize >= 2 ** 31:
            raise ShapeError(f"{self.pages} pages of {self.pageSize} tokens exceed the int32 "
                             "slots")
        w = width(self.headDim)
        self.keys = torch.zeros((self.pages, self.kvHeads, self.pageSize, w), dtype=torch.int8,
                                device=device)
        self.values = torch.zeros((self.pages, self.kvHeads, w, self.pageSize),
                                  dtype=torch.int8, device=device)
        self.keyScales = torch.zeros((self.pages, self.kvHeads), dtype=torch.float32,
                                     device=device)
        self.valueScales = torch.zeros_like(self.keyScales)

    @property
    def pointers(self):
        """Where the four tensors are now. Nothing is remembered: a copy of a cache (deepcopy,
        pickle, torch.save) has memory of its own, and a tensor may be replaced by another."""
        return (self.keys.data_ptr(), self.values.data_ptr(), self.keyScales.data_ptr(),
                self.valueScales.data_ptr())

    @property
    def sizes(self):
        return self.pages, self.kvHeads, self.headDim, self.pageSize

    def operands(self):
        """(the four tensors, their addresses and the sizes as the C entries take them), after a
        look at the tensors: types, shapes and layout may have been changed since (the devices
        are looked at with those of a call's other operands)."""
        k, v, ks, vs = held = self.keys, self.values, self.keyScales, self.valueScales
        pages, heads, dim, page = sizes = self.sizes
        w = width(dim)
        flat = (pages, heads)
        if not (k.dtype is _INT8 and v.dtype is _INT8 and ks.dtype is _FLOAT and
                vs.dtype is _FLOAT and k.shape == (pages, heads, page, w) and
                v.shape == (pages, heads, w, page) and ks.shape == flat and vs.shape == flat and
                k.is_contiguous() and v.is_contiguous() and ks.is_contiguous() and
                vs.is_contiguous()):
            for name, t, dtype, shape in (("keys", k, _INT8, (pages, heads, page, w)),
                                          ("values", v, _INT8, (pages, heads, w, page)),
                                          ("keyScales", ks, _FLOAT, flat),
                                          ("valueScales", vs, _FLOAT, flat)):
                _check_typed(name + " of the cache", t, dtype, shape)
        return held, (k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr()) + sizes

    def freePages(self):
        """(free [pages], freeCount [1]) int32: every page free, for CacheTables."""
        dev = self.keys.device
        return (torch.arange(self.pages - 1, -1, -1, dtype=torch.int32, device=dev),
                torch.full((1,), self.pages, dtype=torch.int32, device=dev))

    def blockTable(self, requests, maxPages):
        """An empty block table [requests, maxPages]."""
        return torch.full((int(requests), int(maxPages)), -1, dtype=torch.int32,
                          device=self.keys.device)

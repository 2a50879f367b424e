"""CPU tests of the 8-bit operators' argument checks: every C entry refuses bad arguments with a
message before it touches HIP (the pointers here are never followed), and the Python operators
refuse CPU tensors. And of gemm_int8's generated code (as tests/test_codegen.py)."""
import ctypes
import os
import re
import subprocess

import pytest

from my_pytchon_opencl_lib_amd import _native
from test_codegen import CSRC, _hipcc

INVALID = _native.MIGEMM_ERR_INVALID_ARG
ALIAS = _native.MIGEMM_ERR_ALIAS
UNSUPPORTED = _native.MIGEMM_ERR_UNSUPPORTED
GIB = 1 << 40


class P(int):
    """The n-th fake buffer, far from the others."""
    def __new__(cls, n, off=0):
        return int.__new__(cls, (n + 1) * GIB + off)


@pytest.fixture(scope="module")
def lib():
    return _native.load()


def entries():
    """Valid arguments of every entry, by name; a test changes one of them. Valid calls would
    reach HIP, so none is made."""
    rows = dict(stream=None, X=P(0), type=0, ldx=50, values=P(1), ldv=64, scales=P(2), rows=7,
                cols=50)
    mat = dict(stream=None, A=P(0), lda=64, a_scales=P(1), B=P(2), ldb=64, b_scales=P(3),
               bias=P(4), C=P(5), type=0, ldc=9, M=7, N=9, K=48)
    lin = dict(stream=None, X=P(0), type=1, ldx=50, W=P(1), ldw=64, w_scales=P(2), bias=None,
               Y=P(3), ldy=9, M=7, N=9, cols=50)
    tab = dict(stream=None, lengths=P(0), counts=P(1), requests=3, table=P(2), max_pages=4,
               page_size=16, free_pages=P(3), free_count=P(4), free_capacity=9, slots=P(5),
               positions=P(6), starts=P(7), new_lengths=P(8), new_free=P(9), tokens=10)
    slo = dict(stream=None, lengths=P(0), counts=P(1), requests=3, table=P(2), max_pages=4,
               page_size=16, slots=P(5), positions=P(6), starts=P(7), tokens=10)
    rel = dict(stream=None, finished=P(0), lengths=P(1), requests=3, table=P(2), max_pages=4,
               page_size=16, free_pages=P(3), pages=9, free_count=P(4))
    cache = dict(keys=P(10), values=P(20), key_scales=P(30), value_scales=P(40), pages=9,
                 kv_heads=2, head_dim=40, page_size=32)
    app = dict(stream=None, K=P(0), V=P(1), type=0, ldk=80, ldv=80, slots=P(2), tokens=10,
               **cache)
    rea = dict(stream=None, **cache, slots=P(2), tokens=10, K=P(3), V=P(4), type=0)
    att = dict(stream=None, Q=P(0), type=0, ldq=160, **cache, table=P(1), max_pages=4,
               starts=P(2), positions=P(3), requests=3, tokens=10, heads=4, scale=0.1,
               max_count=0, max_length=0, O=P(4))
    return {"quantize_rows": rows, "matmul_int8": mat, "linear_int8": lin, "cache_tables": tab,
            "cache_slots": slo, "cache_release": rel, "cache_append": app, "cache_read": rea,
            "cache_attention": att}


def refused(lib, name, code, fragment, **change):
    args = dict(entries()[name])
    assert set(change) <= set(args), name
    args.update(change)
    status = getattr(lib, "migemm_" + name)(*args.values())
    assert status == code, (name, change, status, _native.last_error())
    assert fragment in _native.last_error(), (name, change, _native.last_error())


@pytest.mark.parametrize("name", sorted(entries()))
def test_null_pointers(lib, name):
    for arg, value in entries()[name].items():
        if isinstance(value, P) and arg not in ("bias",):
            refused(lib, name, INVALID, "null pointer", **{arg: None})


@pytest.mark.parametrize("name", [n for n, a in entries().items() if "type" in a])
def test_types(lib, name):
    for t in (-1, 2, 7):
        refused(lib, name, INVALID, "MIGEMM_BFLOAT16", type=t)


OUTPUTS = {"quantize_rows": ["values", "scales"], "matmul_int8": ["C"], "linear_int8": ["Y"],
           "cache_tables": ["table", "slots", "positions", "starts", "new_lengths", "new_free"],
           "cache_slots": ["slots", "positions", "starts"],
           "cache_release": ["lengths", "table", "free_pages", "free_count"],
           "cache_append": ["keys", "values", "key_scales", "value_scales"],
           "cache_read": ["K", "V"], "cache_attention": ["O"]}


@pytest.mark.parametrize("name", sorted(OUTPUTS))
def test_overlapping_buffers(lib, name):
    args = entries()[name]
    for out in OUTPUTS[name]:
        for other, value in args.items():
            if isinstance(value, P) and other != out:
                refused(lib, name, ALIAS, "overlap", **{out: value})


def test_product_sizes_and_strides(lib):
    for name, bad in (("matmul_int8", dict(M=0)), ("matmul_int8", dict(N=-1)),
                      ("matmul_int8", dict(K=0)), ("linear_int8", dict(cols=0)),
                      ("quantize_rows", dict(rows=0)), ("quantize_rows", dict(cols=0))):
        refused(lib, name, INVALID, "sizes must be >= 1", **bad)
    refused(lib, "matmul_int8", INVALID, "multiple of 16", K=40)
    refused(lib, "matmul_int8", UNSUPPORTED, "131071", K=131072, lda=131072, ldb=131072)
    refused(lib, "linear_int8", UNSUPPORTED, "131071", cols=131072, ldx=131072, ldw=131072)
    refused(lib, "linear_int8", UNSUPPORTED, "131071", cols=131071, ldx=131071, ldw=131072)
    for arg in ("lda", "ldb"):
        for ld in (32, 56, (1 << 23) + 16, -64):
            refused(lib, "matmul_int8", INVALID, arg, **{arg: ld})
    refused(lib, "matmul_int8", INVALID, "aligned", A=P(0, 8))
    refused(lib, "matmul_int8", INVALID, "aligned", B=P(0, 1))
    refused(lib, "linear_int8", INVALID, "aligned", W=P(0, 4))
    refused(lib, "matmul_int8", INVALID, "ldc", ldc=8)
    refused(lib, "linear_int8", INVALID, "ldx", ldx=49)
    refused(lib, "linear_int8", INVALID, "ldw", ldw=48)
    refused(lib, "linear_int8", INVALID, "ldy", ldy=(1 << 28) + 1)
    refused(lib, "quantize_rows", INVALID, "ldv", ldv=48)
    refused(lib, "quantize_rows", INVALID, "multiple of 16", ldv=72)
    refused(lib, "quantize_rows", INVALID, "aligned", values=P(1, 8))
    refused(lib, "quantize_rows", INVALID, "ldx", ldx=-50)
    refused(lib, "quantize_rows", UNSUPPORTED, "exceed one launch", rows=1 << 24)
    refused(lib, "matmul_int8", UNSUPPORTED, "exceed one launch", M=2 ** 31 - 1, N=2 ** 31 - 1,
            ldc=2 ** 28)


def test_table_sizes(lib):
    for name in ("cache_tables", "cache_slots", "cache_release"):
        refused(lib, name, INVALID, "requests", requests=0)
        refused(lib, name, INVALID, "requests", requests=(1 << 24) + 1)
        refused(lib, name, UNSUPPORTED, "page_size", page_size=48)
        refused(lib, name, UNSUPPORTED, "page_size", page_size=0)
        refused(lib, name, INVALID, "max_pages", max_pages=0)
        refused(lib, name, INVALID, "max_pages", max_pages=(1 << 26) + 1)
    for name in ("cache_tables", "cache_slots"):
        refused(lib, name, INVALID, "tokens", tokens=-1)
        refused(lib, name, INVALID, "tokens", tokens=(1 << 30) + 1)
    refused(lib, "cache_tables", INVALID, "free_capacity", free_capacity=0)
    refused(lib, "cache_release", INVALID, "pages", pages=0)


@pytest.mark.parametrize("name", ["cache_append", "cache_read", "cache_attention"])
def test_cache_shapes(lib, name):
    for dim in (0, 4, 12, 264, -8):
        refused(lib, name, UNSUPPORTED, "head_dim", head_dim=dim)
    for page in (0, 8, 24, 256):
        refused(lib, name, UNSUPPORTED, "page_size", page_size=page)
    refused(lib, name, INVALID, "pages", pages=0)
    refused(lib, name, INVALID, "kv_heads", kv_heads=0)
    refused(lib, name, INVALID, "kv_heads", kv_heads=65536)
    refused(lib, name, UNSUPPORTED, "int32", pages=1 << 26)
    refused(lib, name, INVALID, "aligned", keys=P(10, 8))
    refused(lib, name, INVALID, "aligned", values=P(10, 4))
    refused(lib, name, INVALID, "aligned", key_scales=P(30, 2))
    refused(lib, name, INVALID, "tokens", tokens=-1)
    if name == "cache_append":
        refused(lib, name, INVALID, "ldk", ldk=79)
        refused(lib, name, INVALID, "ldv", ldv=0)
    # no tokens: nothing to do, whatever the pointers are
    none = dict(entries()[name], tokens=0, **({"K": None, "V": None, "slots": None}
                                              if name != "cache_attention" else
                                              {"Q": None, "positions": None, "O": None}))
    assert getattr(lib, "migemm_" + name)(*none.values()) == 0


def test_attention_arguments(lib):
    refused(lib, "cache_attention", INVALID, "heads", heads=3)
    refused(lib, "cache_attention", INVALID, "heads", heads=0)
    for scale in (-1.0, float("nan"), float("inf")):
        refused(lib, "cache_attention", INVALID, "scale", scale=scale)
    refused(lib, "cache_attention", INVALID, "max_count", max_count=-1)
    refused(lib, "cache_attention", INVALID, "max_length", max_length=-1)
    refused(lib, "cache_attention", INVALID, "ldq", ldq=159)
    refused(lib, "cache_attention", UNSUPPORTED, "int32", tokens=1 << 30)


def test_python_operators_refuse_cpu_tensors():
    import torch
    from my_pytchon_opencl_lib_amd import NnClGlob, ShapeError
    from my_pytchon_opencl_lib_amd.cache import Int8Cache
    g = NnClGlob("cuda:0")
    x = torch.zeros(2, 16)
    i = torch.zeros(2, dtype=torch.int32)
    cache = Int8Cache(2, 1, 16, 16, device="cpu")  # (never reached by a kernel)
    k = torch.zeros(2, 1, 16)
    for call in (lambda: g.QuantizeRows(x),
                 lambda: g.MatmulInt8(x.to(torch.int8), x[:, 0], x.to(torch.int8), x[:, 0]),
                 lambda: g.LinearInt8(x, x.to(torch.int8), x[:, 0]),
                 lambda: g.CacheTables(i, i, i.view(2, 1), i, i[:1], 2, 16),
                 lambda: g.CacheSlots(i, i, i.view(2, 1), 2, 16),
                 lambda: g.CacheRelease(i, i, i.view(2, 1), i, i[:1], 16),
                 lambda: g.CacheAppend(k, k, i, cache),
                 lambda: g.CacheRead(cache, i),
                 lambda: g.CacheAttention(k, cache, i.view(2, 1), i, i)):
        with pytest.raises(ShapeError, match="no CPU fallback"):
            call()


@pytest.mark.skipif(_hipcc() is None, reason="hipcc not available")
def test_m0_only_feeds_the_lds_loads(tmp_path):
    """gemm_int8's tiles are loaded by the same inline assembly as gemm_direct's."""
    out = tmp_path / "gemm_int8.s"
    r = subprocess.run([_hipcc(), "--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang",
                        "-target-feature", "-Xclang", "-packed-fp32-ops", "-Wno-inline-asm",
                        "--cuda-device-only", "-S", os.path.join(CSRC, "gemm_int8.hip"), "-o",
                        str(out)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    lines = [l.split(";")[0].strip() for l in out.read_text().splitlines()]
    code = [l for l in lines if l and not l.startswith(".") and not l.endswith(":")]
    loads = [i for i, l in enumerate(code) if re.match(r"global_load_lds_dwordx4 ", l)]
    uses = [i for i, l in enumerate(code) if re.search(r"\bm0\b", l)]
    assert loads and [i + 1 for i in uses] == loads
    assert all(re.fullmatch(r"s_mov_b32 m0, s\d+", code[i]) for i in uses)

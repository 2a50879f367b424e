"""CPU tests of the argument checks of the operators that close a decoder's step in 8 bits: the
norm, the products with activation, gate and residual, and sampling. Every C entry refuses bad
arguments with a message before it touches HIP (the pointers here are never followed), and the
Python operators refuse CPU tensors."""
import os
import re
import subprocess

import pytest

from my_pytchon_opencl_lib_amd import _native
from test_codegen import CSRC, _hipcc
from test_serve_args import ALIAS, INVALID, UNSUPPORTED, P


@pytest.fixture(scope="module")
def lib():
    return _native.load()


def entries():
    """Valid arguments of every entry, by name; a test changes one of them. Valid calls would
    reach HIP, so none is made."""
    norm = dict(stream=None, X=P(0), ldx=50, R=P(1), ldr=50, type=0, weight=P(2), eps=1e-6, S=P(3),
                lds=50, values=P(4), ldv=64, scales=P(5), rows=7, cols=50)
    mat = dict(stream=None, A=P(0), lda=64, a_scales=P(1), B=P(2), ldb=64, b_scales=P(3),
               bias=P(4), activation=2, gated=0, residual=P(6), ldr=9, C=P(5), type=0, ldc=9, M=7,
               N=9, K=48)
    lin = dict(stream=None, X=P(0), type=1, ldx=50, W=P(1), ldw=64, w_scales=P(2), bias=P(5),
               activation=4, gated=1, residual=P(6), ldr=9, Y=P(3), ldy=9, M=7, N=9, cols=50)
    sam = dict(stream=None, logits=P(0), type=1, ld=100, rows=3, vocab=100, uniforms=P(1),
               temperatures=P(2), temperature=0.0, top_ks=P(3), top_k=0, top_ps=P(4), top_p=0.0,
               min_ps=P(5), min_p=0.0, tokens=P(6), probabilities=P(7))
    return {"norm_int8": norm, "matmul_int8_ex": mat, "linear_int8_ex": lin, "sample": sam}


OPTIONAL = {"norm_int8": ("R", "weight", "S"), "matmul_int8_ex": ("bias", "residual"),
            "linear_int8_ex": ("bias", "residual"),
            "sample": ("temperatures", "top_ks", "top_ps", "min_ps")}
OUTPUTS = {"norm_int8": ["S", "values", "scales"], "matmul_int8_ex": ["C"],
           "linear_int8_ex": ["Y"], "sample": ["tokens", "probabilities"]}


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
        if isinstance(value, P) and arg not in OPTIONAL[name]:
            refused(lib, name, INVALID, "null pointer", **{arg: None})


@pytest.mark.parametrize("name", [n for n, a in entries().items() if "type" in a])
def test_types(lib, name):
    for t in (-1, 2, 7):
        refused(lib, name, INVALID, "MIGEMM_BFLOAT16", type=t)


@pytest.mark.parametrize("name", sorted(OUTPUTS))
def test_overlapping_buffers(lib, name):
    args = entries()[name]
    for out in OUTPUTS[name]:
        for other, value in args.items():
            if isinstance(value, P) and other != out:
                refused(lib, name, ALIAS, "overlap", **{out: value})


def test_the_second_half_of_a_gated_weight_is_an_input_too(lib):
    """An output that begins where the N rows of the gate end overlaps the weight."""
    for name, out, weight in (("matmul_int8_ex", "C", "B"), ("linear_int8_ex", "Y", "W")):
        base = entries()[name][weight]
        refused(lib, name, ALIAS, "overlap", gated=1, **{out: base + 9 * 64})
    refused(lib, "matmul_int8_ex", ALIAS, "overlap", gated=1, C=P(3) + 4 * 9)
    refused(lib, "linear_int8_ex", ALIAS, "overlap", gated=1, Y=P(5) + 4 * 9)


def test_norm(lib):
    for bad in (dict(rows=0), dict(cols=0), dict(rows=-3), dict(cols=2 ** 31 - 1)):
        refused(lib, "norm_int8", INVALID, "sizes must be >= 1", **bad)
    for eps in (0.0, -1e-6, float("nan"), float("inf"), 1e-60):
        refused(lib, "norm_int8", INVALID, "eps", eps=eps)
    refused(lib, "norm_int8", INVALID, "a sum needs a residual", R=None)
    for arg in ("ldx", "ldr", "lds"):
        for ld in (49, -50, (1 << 28) + 1):
            refused(lib, "norm_int8", INVALID, arg, **{arg: ld})
    refused(lib, "norm_int8", INVALID, "ldv", ldv=48)
    refused(lib, "norm_int8", INVALID, "multiple of 16", ldv=72)
    refused(lib, "norm_int8", INVALID, "aligned", values=P(4, 8))
    refused(lib, "norm_int8", UNSUPPORTED, "exceed one launch", rows=1 << 24)
    refused(lib, "norm_int8", UNSUPPORTED, "exceed one launch", rows=1 << 23, cols=4097, ldx=4097,
            ldr=4097, lds=4097, ldv=4112)  # (512 threads a row)


def test_closings(lib):
    for name in ("matmul_int8_ex", "linear_int8_ex"):
        for act in (-1, 5):
            refused(lib, name, INVALID, "MIGEMM_ACT", activation=act)
        for gated in (-1, 2):
            refused(lib, name, INVALID, "gated", gated=gated)
        for ld in (8, -9, (1 << 28) + 1):
            refused(lib, name, INVALID, "ldr", ldr=ld)
        refused(lib, name, UNSUPPORTED, "int32 rows", gated=1, N=2 ** 30, ldr=2 ** 28,
                **{"ldc" if name == "matmul_int8_ex" else "ldy": 2 ** 28})
        for bad in (dict(M=0), dict(N=-1)):
            refused(lib, name, INVALID, "sizes must be >= 1", **bad)
    refused(lib, "matmul_int8_ex", INVALID, "multiple of 16", K=40)
    refused(lib, "matmul_int8_ex", INVALID, "aligned", A=P(0, 8))
    refused(lib, "matmul_int8_ex", INVALID, "ldc", ldc=8)
    refused(lib, "linear_int8_ex", INVALID, "ldw", ldw=48)
    refused(lib, "linear_int8_ex", INVALID, "ldx", ldx=49)
    refused(lib, "linear_int8_ex", UNSUPPORTED, "131071", cols=131071, ldx=131071, ldw=131072)


def test_sample(lib):
    for bad in (dict(rows=0), dict(vocab=0), dict(rows=-1)):
        refused(lib, "sample", INVALID, "sizes must be >= 1", **bad)
    refused(lib, "sample", UNSUPPORTED, "2^20", vocab=(1 << 20) + 1, ld=1 << 21)
    refused(lib, "sample", UNSUPPORTED, "exceed one launch", rows=1 << 22)
    for ld in (99, -100, (1 << 28) + 1):
        refused(lib, "sample", INVALID, "ld", ld=ld)
    nan, inf = float("nan"), float("inf")
    for v in (-1.0, inf, nan):
        refused(lib, "sample", INVALID, "temperature", temperatures=None, temperature=v)
    refused(lib, "sample", INVALID, "top_k", top_ks=None, top_k=-1)
    for v in (0.0, -1.0, 1.01, nan):
        refused(lib, "sample", INVALID, "top_p", top_ps=None, top_p=v)
    for v in (-0.01, 1.01, nan):
        refused(lib, "sample", INVALID, "min_p", min_ps=None, min_p=v)


def test_python_operators_refuse_cpu_tensors():
    import torch
    from my_pytchon_opencl_lib_amd import NnClGlob, ShapeError
    g = NnClGlob("cuda:0")
    x = torch.zeros(2, 16)
    for call in (lambda: g.NormInt8(x), lambda: g.NormInt8(x, residual=x),
                 lambda: g.MatmulInt8(x.to(torch.int8), x[:, 0], x.to(torch.int8), x[:, 0],
                                      activation="silu"),
                 lambda: g.LinearInt8(x, x.to(torch.int8), x[:, 0], gated=True),
                 lambda: g.Sample(x, x[:, 0])):
        with pytest.raises(ShapeError, match="no CPU fallback"):
            call()


@pytest.mark.skipif(_hipcc() is None, reason="hipcc not available")
@pytest.mark.parametrize("name", ["gemm_int8_epilogue", "gemm_int8_gated"])
def test_m0_only_feeds_the_lds_loads(tmp_path, name):
    """The closed products' tiles are loaded by the same inline assembly as the plain ones'."""
    out = tmp_path / (name + ".s")
    r = subprocess.run([_hipcc(), "--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang",
                        "-target-feature", "-Xclang", "-packed-fp32-ops", "-Wno-inline-asm",
                        "--cuda-device-only", "-S", os.path.join(CSRC, name + ".hip"), "-o",
                        str(out)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    lines = [l.split(";")[0].strip() for l in out.read_text().splitlines()]
    code = [l for l in lines if l and not l.startswith(".") and not l.endswith(":")]
    loads = [i for i, l in enumerate(code) if re.match(r"global_load_lds_dwordx4 ", l)]
    uses = [i for i, l in enumerate(code) if re.search(r"\bm0\b", l)]
    assert loads and [i + 1 for i in uses] == loads
    assert all(re.fullmatch(r"s_mov_b32 m0, s\d+", code[i]) for i in uses)

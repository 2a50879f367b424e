"""CPU tests of sample.hip's barriers: its kernels, compiled for the CPU, give the definition's tokens
in whatever order the wavefronts of a work-group run between two barriers (tests/waves). A read that
a barrier should keep apart from another wavefront's write gives something else in one of them."""
import ctypes
import os
import re
import shutil
import subprocess

import numpy as np
import pytest

from test_sample_gpu import row64

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "my_pytchon_opencl_lib_amd", "csrc")
CLANG = shutil.which("clang++", path="/opt/rocm/llvm/bin:" + os.environ.get("PATH", ""))
# the three pieces of inline assembly, in plain C++
PLAIN = [(r'asm\("v_min_f32 [^;]*;', "r = fminf(kMost, l);"),
         (r'asm\("v_fma_f64 [^;]*;', "r = fma(a, b, c);"),
         (r'asm volatile\(""[^;]*;', ";")]


@pytest.fixture(scope="module")
def sample(tmp_path_factory):
    if CLANG is None:
        pytest.skip("clang++ not available")
    out = tmp_path_factory.mktemp("waves")
    text = open(os.path.join(CSRC, "sample.hip")).read()
    for pattern, plain in PLAIN:
        text, n = re.subn(pattern, plain, text)
        assert n == 1, pattern
    (out / "sample.inc").write_text(text)
    lib = out / "sample.so"
    r = subprocess.run([CLANG, "-std=c++17", "-O1", "-shared", "-fPIC", "-w", "-ffp-contract=off",
                        "-I" + os.path.join(HERE, "waves"), "-I" + CSRC,
                        f'-DSAMPLE="{out / "sample.inc"}"', os.path.join(HERE, "waves", "sample.cpp"),
                        "-o", str(lib)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    fn = ctypes.CDLL(str(lib)).run
    fn.argtypes = [ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_int, ctypes.c_int,
                   ctypes.c_void_p, ctypes.c_float, ctypes.c_int, ctypes.c_float, ctypes.c_float,
                   ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int]

    def run(x, u, t, k, p, m, order):
        x, u = np.ascontiguousarray(x, np.float32), np.ascontiguousarray(u, np.float32)
        rows, vocab = x.shape
        tokens, chances = np.full(rows, -7, np.int32), np.full(rows, -7, np.float32)
        assert fn(x.ctypes.data, 0, vocab, rows, vocab, u.ctypes.data, t, k, p, m,
                  tokens.ctypes.data, chances.ctypes.data, order) == 0
        return tokens, chances
    return run


# (rows, vocabulary, deviation of the logits, temperature, top-k, top-p, min-p): what an answer can go
# through. Tokens gathered whole, and sorted at once; single bins; top-k's tokens weighed again; bins
# of too many tokens for the list, cut by bits; greedy; rows cut over work-groups
CASES = {"whole": (3, 1000, 2.0, 1.0, 200, 1.0, 0.0),
         "whole, top-p": (3, 3000, 3.0, 1.0, 0, 0.8, 0.0),
         "whole, min-p": (2, 3000, 2.0, 0.8, 0, 1.0, 0.02),
         "bins": (3, 9000, 1.5, 1.0, 0, 1.0, 0.0),
         "bins, top-p": (3, 9000, 1.0, 1.0, 0, 0.9, 0.0),
         "counted": (3, 5000, 1.0, 1.0, 700, 0.8, 0.0),
         "counted, crowded": (2, 7000, 1.0, 1.0, 3000, 0.9, 0.0),
         "crowded": (2, 7000, 0.01, 1.0, 0, 0.9, 0.0),
         "one bin": (2, 5000, 0.0, 1.0, 0, 0.7, 0.0),
         "hot": (2, 3000, 1.0, 30.0, 0, 0.9, 0.0),
         "greedy": (3, 3000, 1.0, 0.0, 0, 1.0, 0.0),
         "parts": (2, 40960, 2.0, 0.9, 0, 0.9, 0.0),
         "parts, counted": (2, 40963, 2.0, 0.9, 300, 0.9, 0.0),
         "parts, greedy": (2, 40963, 2.0, 0.0, 0, 0.9, 0.0)}


@pytest.mark.parametrize("order", [0, 1, 2, 3])
@pytest.mark.parametrize("case", CASES)
def test_every_order_of_wavefronts_gives_the_definition(sample, case, order):
    rows, vocab, deviation, t, k, p, m = CASES[case]
    g = np.random.default_rng(vocab)
    x = (deviation * g.standard_normal((rows, vocab))).astype(np.float32)
    u = np.linspace(0.03, 0.97, rows).astype(np.float32)
    tokens, chances = sample(x, u, t, k, p, m, order)
    for i in range(rows):
        token, chance = row64(x[i].astype(np.float64), float(u[i]), t, k, float(np.float32(p)),
                              float(np.float32(m)))
        assert tokens[i] == token, (i, tokens[i], token)
        assert abs(chances[i] - chance) <= 2.0 ** -23 * chance

"""GPU tests of rows that lie beyond 2^31 elements: NormInt8, 8-bit products with a residual, and
Sample, on rows 2^28 elements apart (the largest distance the entries take) and a gated weight whose
second half begins beyond 2^31 bytes. The bits are those of the same rows side by side. About
5 GB of device memory, freed at the end."""
import pytest
import torch

from test_int8_gpu import gen, int8

pytestmark = pytest.mark.gpu

FAR = 1 << 28
ROWS = 9  # the last one begins at element 2^31


@pytest.fixture(scope="module")
def pool():
    p = torch.empty(10 * FAR, dtype=torch.bfloat16, device="cuda")
    yield p
    del p
    torch.cuda.synchronize()
    torch.cuda.empty_cache()


def apart(pool, x):
    far = pool.as_strided((ROWS, x.shape[1]), (FAR, 1))
    far.copy_(x)
    return far


@pytest.mark.parametrize("cols", [400, 3000, 20000])
def test_norm(nncl, pool, cols):
    print("norm", cols, flush=True)
    x = torch.randn(ROWS, cols, generator=gen(cols), device="cuda").bfloat16()
    r = torch.randn(ROWS, cols, generator=gen(1), device="cuda").bfloat16()
    for got, want in ((nncl.NormInt8(apart(pool, x), residual=r), nncl.NormInt8(x, residual=r)),
                      (nncl.NormInt8(x, residual=apart(pool, r)), nncl.NormInt8(x, residual=r))):
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("n", [40, 300])
def test_residual(nncl, pool, n):
    for k in (64, 8208):
        a, b = int8(1, ROWS, k), int8(2, n, k)
        sa, sb = torch.rand(ROWS, device="cuda") * 1e-3, torch.rand(n, device="cuda")
        r = torch.randn(ROWS, n, generator=gen(3), device="cuda").bfloat16()
        want = nncl.MatmulInt8(a, sa, b, sb, None, torch.bfloat16, "silu", False, r)
        got = nncl.MatmulInt8(a, sa, b, sb, None, torch.bfloat16, "silu", False, apart(pool, r))
        assert torch.equal(got, want)


@pytest.mark.parametrize("rows", [2, 100])
def test_gated_weight(nncl, pool, rows):
    """B's rows 2^23 bytes apart: 300 rows of the gate span 2.5 GB, the other half lies behind them."""
    n, k, far = 300, 512, 1 << 23
    held = pool.view(torch.int8).as_strided((2 * n, k), (far, 1))
    b = int8(5, 2 * n, k)
    held.copy_(b)
    a = int8(6, rows, k)
    sa, sb = torch.rand(rows, device="cuda") * 1e-4, torch.rand(2 * n, device="cuda")
    want = nncl.MatmulInt8(a, sa, b, sb, activation="gelu", gated=True)
    assert torch.equal(nncl.MatmulInt8(a, sa, held, sb, activation="gelu", gated=True), want)


@pytest.mark.parametrize("vocab", [5001, 50001])
def test_sample(nncl, pool, vocab):
    x = (2 * torch.randn(ROWS, vocab, generator=gen(vocab), device="cuda")).bfloat16()
    u = torch.rand(ROWS, generator=gen(7), device="cuda")
    far = apart(pool, x)
    for f in ((1.0, 50, 0.9, 0.0), (0.7, 0, 1.0, 0.0), (0.0, 0, 1.0, 0.0), (5.0, 4000, 0.8, 0.0)):
        got, want = nncl.Sample(far, u, *f), nncl.Sample(x, u, *f)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])

"""GPU tests of the 8-bit products' gelu near zero results: x P(x) with the normal distribution P, to a
bound relative to the value. A row of B with one byte and a scale a row of A make the x of each
output one float32 product, so that the definition can be taken at the very same x.

The bound counts the kernel's roundings, u = 2^-24 each and the hardware's exponential and reciprocal
2 u: P(-a) = exp(-a^2 / 2) v q(v), v = 1 / (1 + 0.39 a). The steps to v give 3 u, times the largest
slope of log P(-a) + a^2 / 2 over log v, 2.05; Horner's rule for q, its coefficients' roundings
included, 7.1 u; the fit 2^-26.7; the exponential 2 u, three products and a difference 4 u: 19.4 u
together. The exponent a^2 / 2 log2(e) carries 3 u of itself, which the exponential multiplies by
a^2 / 2. And 2^-126 |x| where the exponential is not a normal number."""
import math

import pytest
import torch

from test_int8_gpu import gen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("m", [3, 30, 200, 1500])
def test_gelu_is_near_relative_to_its_value(nncl, m, gated):
    print(m, gated, flush=True)
    n = 254
    b = torch.zeros(2 * n if gated else n, 16, dtype=torch.int8, device="cuda")
    byte = torch.cat([torch.arange(-127, 0), torch.arange(1, 128)])
    b[:n, 0] = byte.to(torch.int8)
    a = torch.zeros(m, 16, dtype=torch.int8, device="cuda")
    a[:, 0] = 1
    sa = 0.11 * torch.rand(m, generator=gen(m), device="cuda")  # x up to 14
    sa[0], sa[1] = 0.04, 1e-6
    ones = torch.ones(len(b), device="cuda")
    bias = torch.zeros(len(b), device="cuda")
    bias[n:] = 1.0  # (a gated value is multiplied by 1)
    y = nncl.MatmulInt8(a, sa, b, ones, bias, activation="gelu", gated=gated)
    x = (byte.float()[None] * sa.cpu()[:, None]).double()
    want = 0.5 * x * torch.special.erfc(-x * math.sqrt(0.5))
    room = (19.4 + 3 * x * x / 2) * 2.0 ** -24 * want.abs() + 2.0 ** -126 * x.abs()
    assert bool(((y.double().cpu() - want).abs() <= room).all())


def test_gelu_of_values_that_are_not_finite(nncl):
    """inf and NaN as the formula gives them, in the kernels of few rows and of many."""
    for m in (3, 200):
        a = torch.zeros(m, 16, dtype=torch.int8, device="cuda")
        a[:, 0] = 1
        b = torch.zeros(4, 16, dtype=torch.int8, device="cuda")
        bias = torch.tensor([math.inf, math.nan, -3e38, 3e38], device="cuda")
        y = nncl.MatmulInt8(a, torch.ones(m, device="cuda"), b, torch.ones(4, device="cuda"), bias,
                            activation="gelu")
        assert bool((y[:, 0] == math.inf).all()) and bool(y[:, 1].isnan().all())
        assert bool((y[:, 2] == 0).all()) and torch.equal(y[:, 3], bias[3].expand(m))

"""GPU tests of what closes an 8-bit product: activation, gate and residual of NnClGlob.MatmulInt8,
LinearInt8 and layers.LinearInt8.

Against the formula in 64 bits, with every rounding counted (u = 2^-24):
  c     as the product alone: 4 u (|product| + |bias|)
  act   relu none; an error d of c becomes at most 1.13 d (the largest slope of the others);
        silu and gelu_tanh add (4 + 1.5 |z|) 2 u |act|, z = x (a + b x^2) the exponent, and
        2^-126 |x| (the hardware's reciprocal 1 / (1 + e) has no subnormals: it is 0 where it
        would be less than 2^-126), gelu 2^-21 |x| (an error of erf near -1 is absolute)
  gate  |act| d(up) + |up| d(act) + their product, and u of it
  sum   u (|value| + |residual|)
A bfloat16 result is the float32 one rounded: the same bits as the float32 result converted."""
import math

import pytest
import torch

from my_pytchon_opencl_lib_amd import ShapeError, _native
from test_int8_gpu import SIZES as PRODUCTS, TYPES, gen, int8, product64

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
SIZES = PRODUCTS + [(2040, 4090, 144), (2040, 2040, 144)]  # (128 x 256 tiles, of each kind)
ACTS = (None, "relu", "silu", "gelu", "gelu_tanh")
KAPPA = 2 * math.sqrt(2 / math.pi)


def say(*a):
    print(*a, flush=True)


def activated(x, d, act):
    """(act(x), its error for an error d of x) in 64 bits."""
    if act is None:
        return x, d
    if act == "relu":
        return torch.where(x < 0, torch.zeros_like(x), x), d
    if act == "gelu":
        return 0.5 * x * torch.special.erfc(-x * math.sqrt(0.5)), 1.13 * d + 2 ** -21 * x.abs()
    z = x if act == "silu" else KAPPA * (x + 0.044715 * x ** 3)
    y = x * torch.sigmoid(z)
    return y, 1.13 * d + (4 + 1.5 * z.abs()) * 2 * U * y.abs() + 2.0 ** -126 * x.abs()


def closed64(a, sa, b, sb, bias, act, gated, residual):
    """(result, room) by the formula."""
    c, size = product64(a, sa, b, sb, bias)
    d = 4 * U * size
    n = c.shape[1] // 2 if gated else c.shape[1]
    y, e = activated(c[:, :n], d[:, :n], act)
    if gated:
        up, du = c[:, n:], d[:, n:]
        y, e = y * up, y.abs() * du + up.abs() * e + e * du
        e = e + U * y.abs()
    if residual is not None:
        y = y + residual.double()
        e = e + U * (y.abs() + residual.double().abs()) + U * e
    return y, e + U * y.abs() + 1e-30


def check(got, *args):
    y, room = closed64(*args)
    far = (got.double() - y).abs() - room
    assert bool((far <= 0).all()), float(far.max())


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_closed_product(nncl, m, n, k, kind, gated):
    """Each kernel at ragged sizes, each activation; the sums span +-8 standard deviations."""
    say("matmul_int8", m, n, k, kind, gated)
    wide = 2 * n if gated else n
    a, b = int8(m + k, m, k), int8(n + k + 1, wide, k)
    spread = 74.0 ** 2 * k ** 0.5  # of a sum over random bytes
    sa = (torch.rand(m, generator=gen(5), device="cuda") + 0.1) * 3 / spread
    sb = torch.rand(wide, generator=gen(6), device="cuda") + 0.1
    bias = torch.randn(wide, generator=gen(7), device="cuda")
    residual = torch.randn(m, n, generator=gen(8), device="cuda").to(TYPES[kind])
    for i, act in enumerate(ACTS):
        for r in ((residual,) if act is None and not gated else (None, residual)):
            one = bias if i % 2 else None
            got = nncl.MatmulInt8(a, sa, b, sb, one, TYPES[kind], act, gated, r)
            full = nncl.MatmulInt8(a, sa, b, sb, one, torch.float32, act, gated,
                                   r.float() if r is not None else None)
            check(full, a, sa, b, sb, one, act, gated, r)
            assert got.dtype == TYPES[kind] and torch.equal(got, full.to(TYPES[kind]))
    plan = _native.last_plan()
    tall = -(-n // 16) * 32 if gated else n
    rows = (m <= 32 and tall * k <= 12 << 20 and k <= (10240 if m <= 16 else 6144)) or \
        (m <= 16 and 2048 <= tall <= 8192)
    assert plan.startswith("int8-rows" if rows else "int8-tiles"), plan


def test_every_tile_and_range_is_among_the_sizes(nncl):
    """Plans of the sizes above: all tiles, whole and in k ranges, and the kernel of few rows."""
    plans = set()
    for m, n, k in SIZES:
        for gated in (False, True):
            a, b = int8(1, m, k), int8(2, 2 * n if gated else n, k)
            nncl.MatmulInt8(a, torch.ones(m, device="cuda"), b,
                            torch.ones(b.shape[0], device="cuda"), activation="relu", gated=gated)
            plans.add((gated,) + tuple(_native.last_plan().split()[:3]))
    say(sorted(plans))
    text = [" ".join(map(str, p)) for p in plans]
    for gated in ("False", "True"):
        mine = [t for t in text if t.startswith(gated)]
        for tile in ("256x256", "128x256", "128x128", "64x128", "64x64"):
            assert any(tile in t and "int8-tiles" in t for t in mine), (gated, tile)
        assert any("int8-rows" in t for t in mine)


def test_no_activation_and_a_residual_of_zeros_is_the_product(nncl):
    for m, n, k in ((3, 40, 64), (150, 90, 400), (1000, 300, 2064)):
        a, b = int8(m, m, k), int8(n, n, k)
        sa, sb = torch.rand(m, device="cuda"), torch.rand(n, device="cuda")
        bias = torch.randn(n, device="cuda")
        plain = nncl.MatmulInt8(a, sa, b, sb, bias)
        zero = torch.zeros(m, n, device="cuda")
        assert torch.equal(nncl.MatmulInt8(a, sa, b, sb, bias, residual=zero), plain)
        assert torch.equal(nncl.MatmulInt8(a, sa, b, sb, bias, activation="relu"),
                           plain.clamp(min=0))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("m,n,k", [(1, 1500, 4096), (1, 5, 12000), (2, 100, 33), (3, 1000, 777),
                                   (4, 64, 8192), (24, 500, 100), (70, 130, 777), (600, 520, 1000)])
def test_layer_is_the_product_of_its_rows(nncl, m, n, k, gated, kind):
    say("linear_int8", m, n, k, gated, kind)
    x = torch.randn(m, k, generator=gen(m), device="cuda").to(TYPES[kind])
    wide = 2 * n if gated else n
    w8, ws = nncl.QuantizeRows(torch.randn(wide, k, generator=gen(n), device="cuda") / k ** 0.5)
    bias = torch.randn(wide, generator=gen(9), device="cuda")
    residual = torch.randn(m, n, generator=gen(10), device="cuda").to(TYPES[kind])
    x8, xs = nncl.QuantizeRows(x)
    for act in ACTS:
        y = nncl.LinearInt8(x, w8, ws, bias, act, gated, residual)
        assert _native.last_plan().startswith("int8-rows-fused") == (m * -(-k // 4096) <= 3)
        assert torch.equal(y, nncl.MatmulInt8(x8, xs, w8, ws, bias, x.dtype, act, gated, residual))
    if kind == "f32":
        check(y, x8, xs, w8, ws, bias, act, gated, residual)


def test_layer_object_more_axes_and_empty_rows(nncl):
    from my_pytchon_opencl_lib_amd.layers import LinearInt8
    w = torch.randn(80, 96, generator=gen(1), device="cuda")
    layer = LinearInt8(w, nnclglob=nncl, activation="silu", gated=True)
    assert layer.out_channels == 40
    x = torch.randn(2, 3, 96, device="cuda")
    r = torch.randn(2, 3, 40, device="cuda")
    y = layer(x, residual=r)
    assert y.shape == (2, 3, 40)
    flat = nncl.LinearInt8(x.view(6, 96), layer.weight, layer.scales, None, "silu", True,
                           r.view(6, 40))
    assert torch.equal(y.view(6, 40), flat)
    x8, xs, _ = nncl.NormInt8(x.view(6, 96))
    assert torch.equal(layer.forwardRows(x8, xs, residual=r.view(6, 40)),
                       nncl.MatmulInt8(x8, xs, layer.weight, layer.scales, None, torch.float32,
                                       "silu", True, r.view(6, 40)))
    assert layer.forwardRows(x8, xs, torch.bfloat16).dtype == torch.bfloat16
    assert layer(x[:, :0], residual=r[:, :0]).shape == (2, 0, 40)
    a = torch.zeros(0, 96, dtype=torch.int8, device="cuda")
    assert nncl.MatmulInt8(a, xs[:0], layer.weight, layer.scales, gated=True).shape == (0, 40)
    plain = LinearInt8(w, nnclglob=nncl)
    assert torch.equal(plain(x), nncl.LinearInt8(x, plain.weight, plain.scales))


@pytest.mark.parametrize("gated", [False, True])
def test_strided_residuals_and_outputs(nncl, gated):
    """A residual that is a slice (rows at odd elements), and an output with room between rows."""
    for kind, code in ((torch.float32, 0), (torch.bfloat16, 1)):
        for m, n, k in ((5, 30, 400), (150, 90, 400), (300, 515, 2064), (40, 60, 8208)):
            wide = 2 * n if gated else n
            a, b = int8(11, m, k), int8(12, wide, k)
            sa = torch.rand(m, generator=gen(1), device="cuda") * 1e-4
            sb = torch.rand(wide, generator=gen(2), device="cuda")
            big = torch.randn(m, n + 9, generator=gen(3), device="cuda").to(kind)
            part = big[:, 3:3 + n]
            want = nncl.MatmulInt8(a, sa, b, sb, None, kind, "gelu", gated, part.contiguous())
            assert torch.equal(nncl.MatmulInt8(a, sa, b, sb, None, kind, "gelu", gated, part), want)
            out = torch.full((m + 1, n + 7), 7.0, device="cuda").to(kind)
            _native.call("migemm_matmul_int8_ex", torch.cuda.current_stream().cuda_stream,
                         a.data_ptr(), k, sa.data_ptr(), b.data_ptr(), k, sb.data_ptr(), None,
                         _native.MIGEMM_ACT_GELU, int(gated), part.data_ptr(), n + 9,
                         out.data_ptr(), code, n + 7, m, n, k)
            assert torch.equal(out[:m, :n], want)
            assert bool((out[:, n:] == 7).all()) and bool((out[m] == 7).all())


@pytest.mark.parametrize("act", ACTS)
def test_values_far_out_and_not_finite(nncl, act):
    """Sums of +-1e30 give their limits, a NaN scale gives NaN through every activation (relu too),
    and in no other row or column."""
    for m in (4, 40):
        a = torch.zeros(m, 16, dtype=torch.int8, device="cuda")
        a[:, 0] = 1
        b = torch.zeros(6, 16, dtype=torch.int8, device="cuda")
        b[:, 0] = torch.tensor([1, -1, 0, 100, -100, 1], dtype=torch.int8)
        sa = torch.full((m,), 1e30, device="cuda")
        sa[0], sa[2] = 1.0, float("nan")
        y = nncl.MatmulInt8(a, sa, b, torch.ones(6, device="cuda"), activation=act)
        assert bool(y[2].isnan().all()) and bool(y[torch.arange(m) != 2].isfinite().all())
        x = b[:, 0].double()
        far = y[1].double()
        if act is None:
            assert torch.equal(far, (x.float() * 1e30).double())
        else:
            assert torch.equal(far, (x.float().clamp(min=0) * 1e30).double())
        want, room = activated(x, 0 * x, act)
        assert bool(((y[0].double() - want).abs() <= room + 2 * U * want.abs()).all())
        sb = torch.ones(6, device="cuda")
        sb[5] = float("nan")
        y = nncl.MatmulInt8(a, torch.ones(m, device="cuda"), b, sb, activation=act)
        assert torch.equal(y.isnan(), (torch.arange(6, device="cuda") == 5).expand(m, 6))


@pytest.mark.parametrize("m", [2, 30, 90, 300])
def test_replayed_graphs(nncl, m):
    """Captured calls (their workspace reserved beforehand) give the eager bits on every replay."""
    w8, ws = nncl.QuantizeRows(torch.randn(600, 4096, generator=gen(20), device="cuda"))
    stream = torch.cuda.Stream()
    nncl.reserve_workspace(stream, 64 << 20)
    x = torch.randn(m, 4096, generator=gen(m), device="cuda")
    r = torch.randn(m, 300, generator=gen(m + 1), device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        y = nncl.LinearInt8(x, w8, ws, activation="gelu_tanh", gated=True, residual=r)
    for i in range(3):
        x.copy_(torch.randn(m, 4096, generator=gen(100 * m + i), device="cuda"))
        expect = nncl.LinearInt8(x, w8, ws, activation="gelu_tanh", gated=True, residual=r)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, expect)


def test_refusals(nncl):
    x = torch.randn(4, 64, device="cuda")
    w8, ws = nncl.QuantizeRows(torch.randn(9, 64, device="cuda"))
    a8, s8 = nncl.QuantizeRows(x)
    r = torch.randn(4, 9, device="cuda")
    for call in (lambda **k: nncl.LinearInt8(x, w8, ws, **k),
                 lambda **k: nncl.MatmulInt8(a8, s8, w8, ws, **k)):
        with pytest.raises(ShapeError, match="activation must be"):
            call(activation="tanh")
        with pytest.raises(ShapeError, match="even number of rows"):
            call(gated=True)
        with pytest.raises(ShapeError, match="residual must be"):
            call(residual=r[:3])
        with pytest.raises(ShapeError, match="residual must be"):
            call(residual=r.bfloat16())
        with pytest.raises(ShapeError, match="axes"):
            call(residual=r[0])
        with pytest.raises(ShapeError, match="torch.Tensor"):
            call(residual=1.0)
        with pytest.raises(ShapeError, match="no CPU fallback"):
            call(residual=r.cpu())
        with pytest.raises(ShapeError, match="contiguous"):
            call(residual=torch.randn(9, 4, device="cuda").t())
    with pytest.raises(ShapeError, match="residual must be"):
        nncl.LinearInt8(x.view(2, 2, 64), w8, ws, residual=r)

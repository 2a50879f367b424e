"""GPU tests of the 8-bit rows and products: NnClGlob.QuantizeRows, MatmulInt8, LinearInt8 and
layers.LinearInt8.

Quantised rows are compared bit for bit with the rule in numpy's float32 (each step of it is
one correctly rounded operation). A product's integer sum is exact, so its float32 result is
off by the roundings of the conversion, the two scales and the bias alone: within
4 * 2^-24 * (|product| + |bias|) of the 64-bit value. A bfloat16 result is that float32 value
rounded: the same bits as the float32 result converted."""
import numpy as np
import pytest
import torch

from my_pytchon_opencl_lib_amd import ShapeError, _native

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
TINY = np.float32(2.0 ** -126)


def say(*a):
    print(*a, flush=True)


def quantized(x):
    """(values, scales) of float32 rows by the rule, every operation in float32."""
    x = x.astype(np.float32)
    most = np.max(np.abs(x), axis=1)
    with np.errstate(all="ignore"):
        s = (most / np.float32(127)).astype(np.float32)
        s = np.where(s < TINY, np.float32(0), s)
        s = np.where(np.isfinite(most), s, np.float32(np.nan)).astype(np.float32)
        inv = np.where(s > 0, np.float32(1) / s, np.float32(0)).astype(np.float32)
        v = np.rint((x * inv[:, None]).astype(np.float32))
    return v, s


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def product64(a, sa, b, sb, bias=None):
    """(result, |product| + |bias|) in 64 bits."""
    y = (a.double() @ b.double().t()) * sa.double()[:, None] * sb.double()[None]
    size = y.abs()
    if bias is not None:
        y = y + bias.double()
        size = size + bias.double().abs()
    return y, size


def check(got, y, size):
    tol = 4 * 2.0 ** -24 * size
    off = (got.double() - y).abs()
    assert bool((off <= tol + 1e-300).all()), float((off - tol).max())


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 16), (4, 500), (6, 513), (2, 2048),
                                       (3, 2049), (2, 4096), (3, 4100), (2, 16384), (2, 16400),
                                       (1, 40003), (1000, 777)])
def test_rows_bit_for_bit(nncl, rows, cols, kind):
    say("quantize", rows, cols, kind)
    x = (torch.randn(rows, cols, generator=gen(rows + cols), device="cuda") * 3).to(TYPES[kind])
    x[0] = 0  # a row of zeros has the scale 0
    if rows > 2:
        x[1, cols // 2] = 1e30
        x[2] *= 1e-36
    v, s = nncl.QuantizeRows(x)
    ev, es = quantized(x.float().cpu().numpy())
    assert v.shape == (rows, (cols + 15) // 16 * 16) and s.shape == (rows,)
    assert np.array_equal(s.cpu().numpy(), es)
    assert np.array_equal(v.cpu().numpy()[:, :cols], ev.astype(np.int8))
    assert not v[:, cols:].any()


def test_rows_ties_go_to_even_and_subnormal_scales_to_zero(nncl):
    x = torch.zeros(4, 300, device="cuda")
    x[0, 0] = 127.0  # scale 1: halves are ties
    x[0, 1:255] = torch.arange(-127, 127, device="cuda") + 0.5
    x[1, 7] = 127 * 1.17549435e-38  # the smallest normal scale
    x[2, 7] = 126 * 1.17549435e-38  # a subnormal one
    x[3, 299] = 3.4e38
    v, s = nncl.QuantizeRows(x)
    ev, es = quantized(x.cpu().numpy())
    assert np.array_equal(s.cpu().numpy(), es) and es[2] == 0 and es[1] > 0
    assert np.array_equal(v.cpu().numpy()[:, :300], ev.astype(np.int8))


@pytest.mark.parametrize("kind", TYPES)
def test_rows_that_are_not_finite(nncl, kind):
    """inf and NaN make their own row's scale NaN and its products NaN, and no other's."""
    x = torch.randn(6, 90, generator=gen(1), device="cuda").to(TYPES[kind])
    x[1, 3], x[3, 89], x[4, 0] = float("inf"), float("nan"), float("-inf")
    w = torch.randn(20, 90, generator=gen(2), device="cuda")
    w[5, 5] = float("nan")
    v, s = nncl.QuantizeRows(x)
    bad = torch.tensor([False, True, False, True, True, False], device="cuda")
    assert torch.equal(s.isnan(), bad)
    w8, ws = nncl.QuantizeRows(w)
    for rows in (x, x.repeat(30, 1)):
        y = nncl.LinearInt8(rows, w8, ws)
        expect = bad.repeat(rows.shape[0] // 6)[:, None] | (torch.arange(20, device="cuda") == 5)
        assert torch.equal(y.isnan(), expect)


@pytest.mark.parametrize("kind", TYPES)
def test_rows_of_a_wider_tensor_and_more_axes(nncl, kind):
    big = torch.randn(5, 7, 3 * 50 + 1, generator=gen(3), device="cuda").to(TYPES[kind])
    part = big.view(35, -1)[:, 51:101]  # strided rows that begin at an odd element
    v, s = nncl.QuantizeRows(part)
    ev, es = quantized(part.float().cpu().numpy())
    assert np.array_equal(v.cpu().numpy()[:, :50], ev.astype(np.int8))
    assert np.array_equal(s.cpu().numpy(), es)
    w8, ws = nncl.QuantizeRows(torch.randn(33, 50, generator=gen(4), device="cuda"))
    y = nncl.LinearInt8(big[..., 51:101], w8, ws)
    assert y.shape == (5, 7, 33)
    assert torch.equal(y.view(35, 33), nncl.LinearInt8(part.contiguous(), w8, ws))


def int8(seed, *shape):
    return torch.randint(-128, 128, shape, generator=gen(seed), device="cuda", dtype=torch.int8)


SIZES = [(1, 1, 16), (1, 17, 48), (2, 16, 128), (5, 100, 144), (16, 257, 4112), (17, 33, 1024),
         (32, 1000, 528), (33, 15, 272), (64, 300, 2064), (65, 64, 16), (65, 70, 4112),
         (100, 1, 8208), (130, 257, 144), (300, 300, 1040), (1000, 3000, 784), (257, 2048, 128),
         (1500, 1100, 2048), (4000, 3100, 144), (4097, 3333, 640), (16, 2048, 8208),
         (9, 8192, 2064), (3, 8193, 1600), (17, 4096, 4112),
         (128, 4090, 4112)]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_product(nncl, m, n, k, kind):
    """Each kernel at ragged sizes, over every byte value; the work around C is untouched."""
    say("matmul_int8", m, n, k, kind)
    a, b = int8(m + k, m, k), int8(n + k + 1, n, k)
    sa = torch.rand(m, generator=gen(5), device="cuda") + 0.1
    sb = torch.rand(n, generator=gen(6), device="cuda") + 0.1
    for bias in (None, torch.randn(n, generator=gen(7), device="cuda")):
        got = nncl.MatmulInt8(a, sa, b, sb, bias, dtype=TYPES[kind])
        full = nncl.MatmulInt8(a, sa, b, sb, bias)
        check(full, *product64(a, sa, b, sb, bias))
        assert torch.equal(got, full.to(TYPES[kind]))
    plan = _native.last_plan()
    rows = (m <= 32 and n * k <= 12 << 20) or (m <= 16 and 2048 <= n <= 8192)
    assert plan.startswith("int8-rows" if rows else "int8-tiles"), plan


def test_product_takes_strided_rows_and_keeps_to_its_output(nncl):
    m, n, k = 150, 90, 400
    big = int8(11, m, 1024)
    a = big[:, 208:608]  # 16-byte aligned rows 1024 apart
    b = int8(12, n, k)
    sa, sb = torch.rand(m, device="cuda"), torch.rand(n, device="cuda")
    check(nncl.MatmulInt8(a, sa, b, sb), *product64(a, sa, b, sb))
    few = a[:9]
    check(nncl.MatmulInt8(few, sa[:9].contiguous(), b, sb), *product64(few, sa[:9], b, sb))
    # C with ldc > N through the C entry: what lies between rows stays
    for rows in (150, 9):
        out = torch.full((rows, n + 13), 7.0, device="cuda")
        _native.call("migemm_matmul_int8", torch.cuda.current_stream().cuda_stream,
                     a.data_ptr(), 1024, sa.data_ptr(), b.data_ptr(), k, sb.data_ptr(), None,
                     out.data_ptr(), 0, n + 13, rows, n, k)
        check(out[:, :n], *product64(a[:rows], sa[:rows], b, sb))
        assert bool((out[:, n:] == 7).all())


@pytest.mark.parametrize("m", [3, 70])
def test_product_sums_are_exact_at_the_longest_k(nncl, m):
    """131056 products of -128 and 127 or -128: the int32 sum comes within a bit of its range."""
    k = 131056
    a = torch.full((m, k), -128, dtype=torch.int8, device="cuda")
    b = torch.full((5, k), -128, dtype=torch.int8, device="cuda")
    b[1:3] = 127
    b[4, 0] = 127
    one = torch.ones(m, device="cuda")
    got = nncl.MatmulInt8(a, one, b, torch.ones(5, device="cuda"))
    y, size = product64(a, one, b, torch.ones(5, device="cuda"))
    assert torch.equal(got, y.float())


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 11008, 4096), (1, 5, 30001), (2, 100, 33), (3, 1000, 777),
                                   (4, 64, 8192), (4, 50, 8209), (5, 64, 777), (24, 500, 100),
                                   (70, 130, 777), (600, 520, 1000), (3, 600, 4096), (1, 300, 12000),
                                   (2, 200, 4100), (9, 2050, 6000)])
def test_layer_is_the_product_of_its_rows(nncl, m, n, k, kind):
    """One launch or two, quantised by every work-group or once: the same bits as the two
    operators called one after the other, and within the rule's distance of x W^T: half a step
    of each row's and each column's scale a term."""
    say("linear_int8", m, n, k, kind)
    x = torch.randn(m, k, generator=gen(m), device="cuda").to(TYPES[kind])
    w = (torch.rand(n, k, generator=gen(n), device="cuda") * 2 - 1) / k ** 0.5
    bias = torch.randn(n, generator=gen(9), device="cuda")
    w8, ws = nncl.QuantizeRows(w)
    y = nncl.LinearInt8(x, w8, ws, bias)
    plan = _native.last_plan()
    assert plan.startswith("int8-rows-fused") == (m * -(-k // 4096) <= 3)
    x8, xs = nncl.QuantizeRows(x)
    assert torch.equal(y, nncl.MatmulInt8(x8, xs, w8, ws, bias, dtype=x.dtype))
    assert y.dtype == x.dtype
    exact = x.double() @ w.double().t() + bias.double()
    room = 0.501 * (xs.double()[:, None] * w.double().abs().sum(1)[None] +
                    ws.double()[None] * x.double().abs().sum(1)[:, None] +
                    0.501 * k * xs.double()[:, None] * ws.double()[None])
    room = room + 2.0 ** -8 * (exact.abs() + room)
    assert bool(((y.double() - exact).abs() <= room).all())


def test_layer_object_and_empty_rows(nncl):
    from my_pytchon_opencl_lib_amd.layers import Linear, LinearInt8
    lin = Linear(96, 40, nncl, seed=3)
    q = LinearInt8(lin.weight, bias=np.ones(40, dtype=np.float32), nnclglob=nncl)
    x = torch.randn(2, 3, 96, device="cuda")
    full = lin(x) + 1
    assert q(x).shape == (2, 3, 40)
    assert float((q(x) - full).norm() / full.norm()) < 0.02
    assert q(x[:, :0]).shape == (2, 0, 40)
    assert len(q.parameters()) == 3
    assert nncl.QuantizeRows(x[:0])[0].shape == (0, 96)
    assert nncl.MatmulInt8(*nncl.QuantizeRows(x[0, :0]), q.weight, q.scales).shape == (0, 40)


def test_another_stream_and_replayed_graphs(nncl):
    """Captured calls (their workspace reserved beforehand) give the eager bits on every replay
    with new inputs, eager work in between."""
    w8, ws = nncl.QuantizeRows(torch.randn(300, 512, generator=gen(20), device="cuda"))
    stream = torch.cuda.Stream()
    nncl.reserve_workspace(stream, 64 << 20)
    for m in (2, 30, 90):
        x = torch.randn(m, 512, generator=gen(m), device="cuda")
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            y = nncl.LinearInt8(x, w8, ws)
        for i in range(3):
            x.copy_(torch.randn(m, 512, generator=gen(100 * m + i), device="cuda"))
            expect = nncl.LinearInt8(x, w8, ws)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, expect)


def test_refusals(nncl):
    x = torch.randn(4, 64, device="cuda")
    w8, ws = nncl.QuantizeRows(torch.randn(8, 64, device="cuda"))
    with pytest.raises(ShapeError, match="float32 or bfloat16"):
        nncl.LinearInt8(x.half(), w8, ws)
    with pytest.raises(ShapeError, match="features"):
        nncl.LinearInt8(x[:, :40], w8, ws)
    with pytest.raises(ShapeError, match="scales must have the shape"):
        nncl.LinearInt8(x, w8, ws[:7])
    with pytest.raises(ShapeError, match="bias"):
        nncl.LinearInt8(x, w8, ws, ws[:7].contiguous())
    with pytest.raises(ShapeError, match="contiguous"):
        nncl.QuantizeRows(x.t())
    with pytest.raises(ShapeError, match="overlap"):
        nncl.QuantizeRows(x.view(-1).as_strided((8, 64), (16, 1)))
    a8, s8 = nncl.QuantizeRows(x)
    with pytest.raises(ShapeError, match="inner dimensions"):
        nncl.MatmulInt8(a8[:, :48], s8, w8, ws)
    with pytest.raises(_native.MigemmArgumentError, match="multiple of 16"):
        nncl.MatmulInt8(a8[:, :40], s8, w8[:, :40], ws)
    with pytest.raises(_native.MigemmArgumentError, match="aligned"):
        nncl.MatmulInt8(a8[:, 8:24], s8, w8[:, 8:24], ws)
    with pytest.raises(ShapeError, match="int8"):
        nncl.MatmulInt8(x, s8, w8, ws)
    with pytest.raises(ShapeError, match="dtype"):
        nncl.MatmulInt8(a8, s8, w8, ws, dtype=torch.float16)
    with pytest.raises(_native.MigemmArgumentError, match="131071"):
        nncl.MatmulInt8(torch.zeros(1, 131072, dtype=torch.int8, device="cuda"), s8[:1],
                        torch.zeros(1, 131072, dtype=torch.int8, device="cuda"), ws[:1])

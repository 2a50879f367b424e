"""GPU tests of NnClGlob.NormInt8: the residual's addition, the root-mean-square norm and its rows
in 8 bits.

Its rule is compared bit for bit with numpy: the sum is one float32 addition (rounded to bfloat16
where that is the type), the sum of squares and its root are taken in 64 bits and rounded to
float32 once, and every step after that is one correctly rounded float32 operation. (Two orders of
the 64-bit sum differ by less than n 2^-53 of it, so the rounded root differs only where it lies
that near a tie of float32: less than one row in 2^53 / (n 2^24), about 10^5 for the longest row
here; the inputs are fixed.)"""
import numpy as np
import pytest
import torch

from my_pytchon_opencl_lib_amd import ShapeError, _native
from test_int8_gpu import TYPES, gen, product64, quantized

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)


def expected(x, residual, weight, eps):
    """(values, scales, sum) by the rule."""
    total = x
    if residual is not None:
        total = (x.float().cpu() + residual.float().cpu()).to(x.dtype)
    t = total.float().cpu().numpy()
    with np.errstate(all="ignore"):
        mean = np.sum(t.astype(np.float64) ** 2, axis=1) / t.shape[1]
        q = (1.0 / np.sqrt(mean + np.float64(np.float32(eps)))).astype(np.float32)
        y = (t * q[:, None]).astype(np.float32)
        if weight is not None:
            y = (y * weight.cpu().numpy()[None]).astype(np.float32)
    v, s = quantized(y)
    return v, s, total


def check(nncl, x, residual, weight, eps=1e-6):
    v, s, total = nncl.NormInt8(x, weight, residual=residual, eps=eps)
    ev, es, et = expected(x, residual, weight, eps)
    cols = x.shape[-1]
    assert v.dtype == torch.int8 and v.shape == (x.shape[0], (cols + 15) // 16 * 16)
    assert s.shape == (x.shape[0],) and total.dtype == x.dtype and total.shape == x.shape
    assert torch.equal(total.cpu(), et.cpu())
    assert np.array_equal(s.cpu().numpy(), es, equal_nan=True)
    fine = np.isfinite(es)
    assert np.array_equal(v.cpu().numpy()[fine, :cols], ev[fine].astype(np.int8))
    assert not v[torch.from_numpy(fine).cuda(), cols:].any()


SIZES = [(1, 1), (3, 7), (5, 16), (4, 500), (9, 512), (6, 513), (2, 2048), (3, 2049), (1, 4096),
         (3, 4095), (2, 4100), (2, 16384), (2, 16400), (1, 40003), (1000, 777),
         (5, 1024), (5, 1025), (2, 4096), (2, 8192), (2, 8193), (1, 12000), (2, 16385)]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,cols", SIZES)
def test_bit_for_bit(nncl, rows, cols, kind):
    say("norm", rows, cols, kind)
    g = gen(rows * 7 + cols)
    x = torch.randn(rows, cols, generator=g, device="cuda").to(TYPES[kind])
    residual = (torch.randn(rows, cols, generator=g, device="cuda") * 5).to(TYPES[kind])
    weight = torch.randn(cols, generator=g, device="cuda")
    if rows > 2:
        x[0], residual[0] = 0, 0  # zeros: a scale of 0
        residual[1, cols // 2] = 1e30  # squares beyond float32
        x[2] *= 1e-30
        residual[2] *= 1e-30  # far below eps
    for r in (residual, None):
        for w in (weight, None):
            check(nncl, x, r, w)
    check(nncl, x, residual, weight, eps=1.5)
    check(nncl, x, residual, weight, eps=1e-30)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("cols", [90, 3000, 20000])
def test_values_that_are_not_finite_stay_in_their_row(nncl, cols, kind):
    x = torch.randn(6, cols, generator=gen(1), device="cuda").to(TYPES[kind])
    r = torch.randn(6, cols, generator=gen(2), device="cuda").to(TYPES[kind])
    x[1, 3], r[3, cols - 1], x[4, 0] = float("inf"), float("nan"), float("-inf")
    v, s, total = nncl.NormInt8(x, residual=r)
    bad = torch.tensor([False, True, False, True, True, False], device="cuda")
    assert torch.equal(s.isnan(), bad)
    assert torch.equal(total.isfinite().all(1), ~bad)
    check(nncl, x[~bad], r[~bad], None)


@pytest.mark.parametrize("kind", TYPES)
def test_rows_of_wider_tensors_and_more_axes(nncl, kind):
    """Rows that lie apart (beginning at odd elements) and more axes: the contiguous rows' bits."""
    big = torch.randn(5, 7, 151, generator=gen(3), device="cuda").to(TYPES[kind])
    more = torch.randn(5, 7, 131, generator=gen(4), device="cuda").to(TYPES[kind])
    x, r = big[..., 51:101], more[..., 3:53]
    v, s, total = nncl.NormInt8(x, residual=r)
    ev, es, et = nncl.NormInt8(x.contiguous().view(35, 50), residual=r.contiguous().view(35, 50))
    assert total.shape == (5, 7, 50) and torch.equal(total.reshape(35, 50), et)
    assert torch.equal(v, ev) and torch.equal(s, es)
    one = nncl.NormInt8(x[0, 0], residual=r[0, 0])
    assert one[2].shape == (50,) and torch.equal(one[0], ev[:1])
    assert nncl.NormInt8(x[:, :0])[0].shape == (0, 64)
    same = nncl.NormInt8(x)
    assert same[2] is x


def test_the_work_around_the_outputs_stays(nncl):
    """Sum and values with rows further apart, through the C entry."""
    for cols in (90, 3000, 20000):
        rows, p = 3, (cols + 15) // 16 * 16
        x = torch.randn(rows, cols, device="cuda")
        r = torch.randn(rows, cols, device="cuda")
        total = torch.full((rows, cols + 5), 7.0, device="cuda")
        values = torch.full((rows, p + 32), 7, dtype=torch.int8, device="cuda")
        scales = torch.full((rows + 1,), 7.0, device="cuda")
        _native.call("migemm_norm_int8", torch.cuda.current_stream().cuda_stream, x.data_ptr(),
                     cols, r.data_ptr(), cols, 0, None, 1e-6, total.data_ptr(), cols + 5,
                     values.data_ptr(), p + 32, scales.data_ptr(), rows, cols)
        v, s, t = nncl.NormInt8(x, residual=r)
        assert torch.equal(values[:, :p], v) and bool((values[:, p:] == 7).all())
        assert torch.equal(scales[:rows], s) and float(scales[rows]) == 7
        assert torch.equal(total[:, :cols], t) and bool((total[:, cols:] == 7).all())


@pytest.mark.parametrize("kind", TYPES)
def test_norm_then_product(nncl, kind):
    """The rows go into MatmulInt8 as they are: within half a step of each row's scale a term of
    the product of the 64-bit norm (the scales of the weight are exact here)."""
    g = gen(9)
    x = torch.randn(40, 600, generator=g, device="cuda").to(TYPES[kind])
    r = torch.randn(40, 600, generator=g, device="cuda").to(TYPES[kind])
    w8, ws = nncl.QuantizeRows(torch.randn(50, 600, generator=g, device="cuda"))
    v, s, total = nncl.NormInt8(x, residual=r)
    y = nncl.MatmulInt8(v, s, w8, ws)
    t = total.double()
    t = t / (t.square().mean(1, keepdim=True) + 1e-6).sqrt()
    w = w8[:, :600].double() * ws.double()[:, None]
    exact = t @ w.t()
    room = 0.501 * s.double()[:, None] * w.abs().sum(1)[None]
    assert bool(((y.double() - exact).abs() <= room).all())
    held, size = product64(v, s, w8, ws)
    assert bool(((y.double() - held).abs() <= 4 * 2.0 ** -24 * size).all())


def test_another_stream_and_replayed_graph(nncl):
    x = torch.randn(70, 1000, device="cuda")
    r = torch.randn(70, 1000, device="cuda")
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = nncl.NormInt8(x, residual=r)
    for i in range(3):
        x.copy_(torch.randn(70, 1000, generator=gen(i), device="cuda"))
        expect = nncl.NormInt8(x, residual=r)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, expect))


def test_refusals(nncl):
    x = torch.randn(4, 64, device="cuda")
    with pytest.raises(ShapeError, match="float32 or bfloat16"):
        nncl.NormInt8(x.half())
    with pytest.raises(ShapeError, match="residual must be"):
        nncl.NormInt8(x, residual=x.bfloat16())
    with pytest.raises(ShapeError, match="residual must be"):
        nncl.NormInt8(x, residual=x[:3])
    with pytest.raises(ShapeError, match="weight must"):
        nncl.NormInt8(x, x[0].bfloat16())
    with pytest.raises(ShapeError, match="weight must"):
        nncl.NormInt8(x, x[0, :63].contiguous())
    with pytest.raises(ShapeError, match="contiguous"):
        nncl.NormInt8(x.t())
    with pytest.raises(ShapeError, match="contiguous"):
        nncl.NormInt8(x[:, :4], residual=x.t()[:4, :4])
    for eps in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ShapeError, match="eps"):
            nncl.NormInt8(x, eps=eps)
    with pytest.raises(_native.MigemmArgumentError, match="eps"):
        nncl.NormInt8(x, eps=1e-60)
    with pytest.raises(ShapeError, match="at least one value"):
        nncl.NormInt8(x[:, :0])

"""GPU tests of NnClGlob.Sample against the definition in 64 bits.

The tokens have to be the same. The kernel's weights are off by 2^-39 of themselves and 2^-43 of the
largest, at most, so that their sums are off by less than 2^-30 of them for the vocabularies here
(2^17 2^-43 of the largest, which is part of the sum, and 2^-39); a token differs only where u times
the sum lies that near the border of two shares, on one row in 10^3 for the worst of them and far
fewer for others; inputs are fixed, and where all weights are equal they are exact. A probability
is a quotient of such numbers rounded to float32: within 2^-24 + 2^-30 of it, relatively."""
import numpy as np
import pytest
import torch

from my_pytchon_opencl_lib_amd import ShapeError, _native

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
INF = float("inf")


def say(*a):
    print(*a, flush=True)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def one(v, i):
    return float(v[i]) if isinstance(v, torch.Tensor) else float(np.float32(v))


def row64(x, u, t, k, p, least):
    """(token, probability) of one row of float64 logits."""
    if np.isnan(x).any() or not x.max() > -INF or not 0 <= t < INF or np.isnan(u + p + least):
        return -1, 0.0
    order = np.argsort(-x, kind="stable")
    if t == 0:
        return order[0], 1.0
    x = x[order]
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(x == x[0], 1.0, np.exp((x - x[0]) / t))
    w[w < min(least, 1.0)] = 0
    if k > 0:
        w[int(k):] = 0
    upto = np.cumsum(w)
    before = np.concatenate([[0.0], upto[:-1]])
    w[(before >= max(p, 0.0) * upto[-1]) & (np.arange(w.size) > 0)] = 0
    upto = np.cumsum(w)
    at = min(int((upto <= u * upto[-1]).sum()), int((w > 0).sum()) - 1)
    return order[at], w[at] / upto[-1]


def check(nncl, logits, uniforms, temperature=1.0, topK=0, topP=1.0, minP=0.0):
    tokens, chances = nncl.Sample(logits, uniforms, temperature, topK, topP, minP)
    assert tokens.dtype == torch.int32 and chances.dtype == torch.float32
    x, u = logits.double().cpu().numpy(), uniforms.double().cpu().numpy()
    want = [row64(x[i], u[i], one(temperature, i), one(topK, i), one(topP, i), one(minP, i))
            for i in range(x.shape[0])]
    assert tokens.tolist() == [int(w[0]) for w in want]
    got = chances.double().cpu().numpy()
    p = np.array([w[1] for w in want])
    assert (np.abs(got - p) <= (2.0 ** -24 + 2.0 ** -30) * p + 1e-45).all()
    return tokens


FILTERS = [(1.0, 0, 1.0, 0.0), (0.7, 50, 1.0, 0.0), (1.3, 0, 0.9, 0.0), (1.0, 0, 1.0, 0.1),
           (0.8, 40, 0.95, 0.05), (1.0, 5000, 0.5, 0.0), (0.0, 3, 0.5, 0.5), (2.0, 1, 1.0, 0.0),
           (5.0, 0, 0.999, 0.0), (0.05, 0, 0.3, 0.0), (1.0, 3, 0.01, 1.0), (30.0, 0, 0.6, 0.0)]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (5, 7), (4, 100), (17, 1000), (3, 4096),
                                        (9, 8193), (2, 32000), (5, 50001), (2, 131072),
                                        (1, 300007)])
def test_against_the_definition(nncl, rows, vocab, kind):
    say("sample", rows, vocab, kind)
    g = gen(rows + vocab)
    logits = (3 * torch.randn(rows, vocab, generator=g, device="cuda")).to(TYPES[kind])
    for f in FILTERS:
        check(nncl, logits, torch.rand(rows, generator=g, device="cuda"), *f)


@pytest.mark.parametrize("rows,vocab", [(96, 5003), (44, 50001), (30, 70003)])
@pytest.mark.parametrize("kind", TYPES)
def test_parameters_of_each_row(nncl, rows, vocab, kind):
    """Every filter on and off in one call, among rows whose parameters say nothing."""
    say("mixed", rows, vocab, kind)
    g = gen(5)
    logits = (2 * torch.randn(rows, vocab, generator=g, device="cuda")).to(TYPES[kind])
    logits[torch.rand(rows, vocab, generator=g, device="cuda") < 0.3] = -INF
    u = torch.rand(rows, generator=g, device="cuda")

    def pick(values, dtype=torch.float32):
        at = torch.randint(0, len(values), (rows,), generator=g, device="cuda")
        return torch.tensor(values, dtype=dtype, device="cuda")[at]
    t = pick([0.0, 0.5, 1.0, 1.7, 40.0])
    k = pick([0, 1, 2, 30, 3000, 10 ** 9, -4], torch.int32)
    p = pick([1.0, 0.9, 0.4, 1e-9, 0.0, -1.0, 7.0])
    m = pick([0.0, 0.01, 0.3, 1.0, 9.0, -2.0])
    check(nncl, logits, u, t, k, p, m)
    check(nncl, logits, u, t, 40, p, 0.1)
    t[3], t[4], t[5], p[6], m[7], u[8] = -1.0, INF, float("nan"), float("nan"), float("nan"), \
        float("nan")
    u[9], u[10], u[11] = 1.0, 3.0, -1.0  # outside [0, 1): the last and the first of the kept
    tokens, chances = nncl.Sample(logits, u, t, k, p, m)
    assert tokens[3:9].tolist() == [-1] * 6 and chances[3:9].tolist() == [0.0] * 6
    ok = torch.ones(rows, dtype=torch.bool, device="cuda")
    ok[3:12] = False
    same = nncl.Sample(logits[ok], u[ok], t[ok], k[ok], p[ok], m[ok])
    assert torch.equal(tokens[ok], same[0]) and torch.equal(chances[ok], same[1])
    t[9:12], k[9:12], p[9:12], m[9:12] = 1.0, 20, 1.0, 0.0
    tokens, _ = nncl.Sample(logits, u, t, k, p, m)
    best = torch.sort(logits[9:12].float(), dim=1, descending=True, stable=True).indices
    assert tokens[9:12].tolist() == [int(best[0, 19]), int(best[1, 19]), int(best[2, 0])]


@pytest.mark.parametrize("vocab", [700, 70001, 200003])
@pytest.mark.parametrize("values", [1, 2, 5])
def test_equal_logits_go_by_index(nncl, vocab, values):
    """Rows of one to five different logits: whole bins of equal tokens, cut by index."""
    say("ties", vocab, values)
    g = gen(vocab + values)
    rows = 6
    logits = torch.randint(0, values, (rows, vocab), generator=g, device="cuda").float()
    logits[1] -= 1e30
    logits[2] *= 1e-30
    logits[3] = torch.where(torch.rand(vocab, generator=g, device="cuda") < 0.5, -0.0, 0.0)
    for f in ((1.0, 0, 1.0, 0.0), (1.0, 0, 0.5, 0.0), (1.0, vocab // 2, 1.0, 0.0),
              (2.0, vocab - 3, 0.75, 0.0), (0.0, 0, 1.0, 0.0)):
        for u in (torch.rand(rows, generator=g, device="cuda"), torch.zeros(rows, device="cuda"),
                  torch.full((rows,), 1 - 2.0 ** -24, device="cuda")):
            check(nncl, logits, u, *f)
            check(nncl, logits.bfloat16(), u, *f)


def test_equal_logits_at_exact_borders(nncl):
    """Four equal tokens: u and top-p at the quarters fall on borders that are exact."""
    logits = torch.zeros(8, 4, device="cuda")
    u = torch.arange(8, device="cuda") / 8
    assert check(nncl, logits, u).tolist() == [0, 0, 1, 1, 2, 2, 3, 3]
    assert check(nncl, logits, u, topP=0.5).tolist() == [0, 0, 0, 0, 1, 1, 1, 1]
    assert check(nncl, logits, u, topK=3, topP=0.75).tolist() == [0, 0, 0, 1, 1, 1, 2, 2]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("vocab", [40, 9001, 60001])
def test_masks_infinities_and_nan(nncl, vocab, kind):
    say("masks", vocab, kind)
    dt = TYPES[kind]
    least = torch.finfo(dt).min
    g = gen(vocab)
    base = torch.randn(12, vocab, generator=g, device="cuda").to(dt)
    keep = torch.rand(12, vocab, generator=g, device="cuda") < 0.02
    x = base.clone()
    x[0] = -INF                       # nothing is left
    x[1, 1:] = -INF                   # one token is left
    x[2] = torch.where(keep[2], base[2], -INF)
    x[2, 5] = 1.0
    x[3] = torch.where(keep[3], base[3], least)
    x[4] = least                      # all equal
    x[5, vocab // 2] = float("nan")
    x[6, :] = -INF
    x[6, vocab - 1] = float("nan")
    x[7, 3] = x[7, vocab - 2] = INF   # two that outweigh the rest
    x[8] = INF
    x[9, 0], x[9, 1:] = torch.finfo(dt).max, least
    x[10, ::2] = -INF
    x[11, vocab - 1] = 1000.0
    for f in FILTERS:
        check(nncl, x, torch.rand(12, generator=g, device="cuda"), *f)
    tokens, chances = nncl.Sample(x, torch.rand(12, generator=g, device="cuda"))
    assert tokens[[0, 5, 6]].tolist() == [-1] * 3 and chances[[0, 5, 6]].tolist() == [0.0] * 3
    assert int(tokens[1]) == 0 and int(tokens[7]) in (3, vocab - 2) and float(chances[7]) == 0.5


def test_extreme_temperatures_and_spreads(nncl):
    g = gen(8)
    x = torch.randn(7, 30011, generator=g, device="cuda")
    x[1] *= 1e30
    x[2] *= 1e-30
    x[3] *= 3e38 / x[3].abs().max()
    x[4] = torch.linspace(0, -100, 30011)
    x[5] = torch.linspace(-1e-3, 1e-3, 30011)
    x[6, :] = 0
    x[6, 77] = 1e-40
    for t in (1e-40, 1e-20, 1e-3, 1.0, 1e3, 1e20, 3e38):
        for k, p, m in ((0, 1.0, 0.0), (0, 0.9, 0.0), (300, 0.9, 0.01), (9000, 1.0, 0.0)):
            check(nncl, x, torch.rand(7, generator=g, device="cuda"), t, k, p, m)


def test_the_largest_vocabulary(nncl):
    n = 1 << 20
    x = torch.randn(2, n, generator=gen(1), device="cuda")
    x[1] = 1.5
    for f in FILTERS[:6]:
        check(nncl, x, torch.tensor([0.3, 0.999], device="cuda"), *f)
    with pytest.raises(_native.MigemmArgumentError, match="2.20"):
        nncl.Sample(torch.zeros(1, n + 1, device="cuda"), torch.zeros(1, device="cuda"))


@pytest.mark.parametrize("kind", TYPES)
def test_rows_that_lie_apart(nncl, kind):
    """Slices of wider rows, beginning at odd elements, between values that would win."""
    big = torch.full((9, 6011), 50.0, device="cuda").to(TYPES[kind])
    big[:, 5:6006] = torch.randn(9, 6001, generator=gen(2), device="cuda").to(TYPES[kind])
    part = big[:, 5:6006]
    u = torch.rand(9, generator=gen(3), device="cuda")
    for f in FILTERS:
        check(nncl, part, u, *f)
        assert torch.equal(nncl.Sample(part, u, *f)[0], nncl.Sample(part.contiguous(), u, *f)[0])


def test_shares_of_many_draws(nncl):
    """Evenly spread random numbers give each token its share, to one draw."""
    x = torch.tensor([[0.3, -1.0, 2.0, -INF, 0.3, 1.2]], device="cuda")
    n = 20000
    u = (torch.arange(n, device="cuda") + 0.5) / n
    tokens, chances = nncl.Sample(x.expand(n, 6).contiguous(), u)
    p = torch.softmax(x[0].double(), 0)
    got = torch.bincount(tokens.long(), minlength=6).double()
    assert bool(((got - n * p).abs() <= 1.0).all())
    drawn = p[tokens.long()]
    assert bool(((chances.double() - drawn).abs() <= 2.0 ** -23 * drawn).all())


def test_another_stream_and_replayed_graph(nncl):
    x = torch.randn(20, 50001, generator=gen(4), device="cuda")
    u = torch.rand(20, generator=gen(5), device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = nncl.Sample(x, u, 0.9, 100, 0.9, 0.01)
    side.synchronize()
    assert torch.equal(other[0], nncl.Sample(x, u, 0.9, 100, 0.9, 0.01)[0])
    stream = torch.cuda.Stream()
    nncl.reserve_workspace(stream, 64 << 20)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = nncl.Sample(x, u, 0.9, 0, 0.9, 0.01)
    for i in range(4):
        x.copy_(2 * torch.randn(20, 50001, generator=gen(10 + i), device="cuda"))
        u.copy_(torch.rand(20, generator=gen(20 + i), device="cuda"))
        expect = nncl.Sample(x, u, 0.9, 0, 0.9, 0.01)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], expect[0]) and torch.equal(got[1], expect[1])


@pytest.mark.parametrize("kind", TYPES)
def test_whole_rows_and_rows_cut_over_work_groups_agree(nncl, kind):
    """49152 tokens: up to 48 rows are cut over work-groups, more are not. Both give the same bits,
    with filters of every kind (single numbers and one a row), and those of the definition."""
    g = gen(31)
    rows, vocab = 64, 49152
    x = (2.5 * torch.randn(rows, vocab, generator=g, device="cuda")).to(TYPES[kind])
    x[5] = 1.25
    x[6, 100:] = -INF
    x[7] = -INF
    x[8, 9] = float("nan")
    u = torch.rand(rows, generator=g, device="cuda")
    for f in FILTERS + [(1.0, 700, 0.8, 0.0), (1.5, 20000, 0.9, 0.0)]:
        say(f)
        whole = nncl.Sample(x, u, *f)
        for a, b in ((0, 1), (1, 9), (9, 40), (16, 64)):
            cut = nncl.Sample(x[a:b], u[a:b], *f)
            assert torch.equal(cut[0], whole[0][a:b]) and torch.equal(cut[1], whole[1][a:b])
        check(nncl, x[4:12], u[4:12], *f)


def test_two_streams_at_once(nncl):
    """Calls on two streams, each with its own workspace, give the bits of calls one by one."""
    xs = [torch.randn(3, 131072, generator=gen(i), device="cuda") for i in range(2)]
    us = [torch.rand(3, generator=gen(10 + i), device="cuda") for i in range(2)]
    want = [nncl.Sample(x, u, 0.8, 0, 0.9) for x, u in zip(xs, us)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(nncl.Sample(xs[i], us[i], 0.8, 0, 0.9))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(t, want[i][0]) and torch.equal(c, want[i][1]) for t, c in got[i])


@pytest.mark.parametrize("rows,vocab,uses", [(1, 40959, False), (41, 40960, False),
                                             (40, 40960, True), (1, 131072, True)])
def test_capture_needs_a_workspace_where_the_header_says(nncl, rows, vocab, uses):
    x = torch.randn(rows, vocab, generator=gen(vocab), device="cuda")
    u = torch.rand(rows, generator=gen(rows), device="cuda")
    stream = torch.cuda.Stream()
    _native.call("migemm_workspace_release", stream.cuda_stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    if uses:
        with pytest.raises(_native.MigemmRuntimeError, match="WORKSPACE"):
            with torch.cuda.graph(graph, stream=stream):
                nncl.Sample(x, u)
        torch.cuda.synchronize()
        nncl.reserve_workspace(stream, 8 << 20)
        graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = nncl.Sample(x, u)
    for i in range(3):
        u.copy_(torch.rand(rows, generator=gen(50 + i), device="cuda"))
        expect = nncl.Sample(x, u)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], expect[0]) and torch.equal(got[1], expect[1])


def test_the_same_call_gives_the_same_bits(nncl):
    x = torch.randn(3, 131072, generator=gen(6), device="cuda")
    u = torch.rand(3, generator=gen(7), device="cuda")
    first = nncl.Sample(x, u, topP=0.97)
    for _ in range(5):
        again = nncl.Sample(x, u, topP=0.97)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_refusals(nncl):
    x, u = torch.randn(4, 64, device="cuda"), torch.rand(4, device="cuda")
    with pytest.raises(ShapeError, match="float32 or bfloat16"):
        nncl.Sample(x.half(), u)
    with pytest.raises(ShapeError, match="axes"):
        nncl.Sample(x[0], u)
    with pytest.raises(ShapeError, match="uniforms must have the shape"):
        nncl.Sample(x, u[:3])
    with pytest.raises(ShapeError, match="uniforms must be"):
        nncl.Sample(x, u.double())
    with pytest.raises(ShapeError, match="contiguous"):
        nncl.Sample(x.t(), torch.rand(64, device="cuda"))
    for name, values in (("temperature", (-0.5, INF, float("nan"))), ("topK", (-1, 2 ** 31)),
                         ("topP", (-0.1, 1.5, float("nan"))), ("minP", (-0.1, 1.01, float("nan")))):
        for v in values:
            with pytest.raises(ShapeError, match=name):
                nncl.Sample(x, u, **{name: v})
        with pytest.raises(ShapeError, match=name):
            nncl.Sample(x, u, **{name: u[:3].to(torch.int32 if name == "topK" else torch.float32)})
        with pytest.raises(ShapeError, match=name + " must be"):
            nncl.Sample(x, u, **{name: u.double()})
    with pytest.raises(_native.MigemmArgumentError, match="top_p"):
        nncl.Sample(x, u, topP=0.0)
    with pytest.raises(TypeError):
        nncl.Sample(x, u, topK=2.5)
    with pytest.raises(ShapeError, match="at least one token"):
        nncl.Sample(x[:, :0], u)
    assert nncl.Sample(x[:0], u[:0])[0].shape == (0,)

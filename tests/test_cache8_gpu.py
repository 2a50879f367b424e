"""GPU tests of the 8-bit paged cache: NnClGlob.CacheTables, CacheSlots, CacheRelease,
CacheAppend, CacheRead and CacheAttention (cache.Int8Cache).

Tables and cache contents are compared with plain loops, bit for bit (every float32 step of the
rules is one correctly rounded operation). Attention is compared with the formula in 64 bits
over the cache's own contents. With A the largest scale * sum |q| |k| of a row and V the largest
|value|, a float32 score is off by at most (D + 8) 2^-24 A, a weight by twice that and 2^-21, and
the weighted mean by the weights' errors and (keys / 64 + 72) 2^-24 from the sums (64 keys a
step, then steps and ranges), all times V; a bfloat16 call adds 2^-8 V, which holds the rounding
of its result and of its weights (a weighted mean's, so they average), and 2^-9 of the result."""
import numpy as np
import pytest
import torch

from my_pytchon_opencl_lib_amd import ShapeError, _native
from my_pytchon_opencl_lib_amd.cache import Int8Cache

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
TINY = np.float32(2.0 ** -126)


def say(*a):
    print(*a, flush=True)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------------------ tables
def tables_by_loops(lengths, counts, table, free, count, tokens, page):
    table = [list(r) for r in table]
    slots, positions, starts, new = [-1] * tokens, [-1] * tokens, [0], []
    place, asked, left = 0, 0, count
    for i, (n, c) in enumerate(zip(lengths, counts)):
        n, c = max(n, 0), max(c, 0)
        first, place = place, place + c
        starts.append(min(place, tokens))
        fits = n + c <= len(table[i]) * page and place <= tokens
        need = -(-(n + c) // page) - -(-n // page) if fits else 0
        before, asked = asked, asked + need
        if not fits or (need and asked > count):
            new.append(n)
            continue
        for j in range(need):
            table[i][-(-n // page) + j] = free[count - 1 - before - j]
        left -= need
        new.append(n + c)
        for k in range(c):
            p = n + k
            if table[i][p // page] >= 0:
                slots[first + k] = table[i][p // page] * page + p % page
                positions[first + k] = p
    return table, slots, positions, starts, new, left


def check_tables(nncl, lengths, counts, columns, page, spare, tokens, seed):
    rng = np.random.default_rng(seed)
    had = [min(-(-max(n, 0) // page), columns) for n in lengths]
    order = rng.permutation(sum(had) + spare + 1).tolist()
    table, at = [], 0
    for h in had:
        table.append(order[at:at + h] + [-1] * (columns - h))
        at += h
    free = order[at:]
    expect = tables_by_loops(lengths, counts, table, free, spare, tokens, page)
    args = [ints(lengths), ints(counts), ints(table), ints(free), ints([spare])]
    before = [a.clone() for a in args]
    for _ in range(2):  # the same call again gives the same
        got = nncl.CacheTables(*args, tokens, page)
        assert args[2].tolist() == expect[0]
        for name, g, e in zip(("slots", "positions", "starts", "lengths"), got, expect[1:]):
            assert g.tolist() == e, name
        assert got[4].tolist() == [expect[5]]
    for k in (0, 1, 3, 4):
        assert torch.equal(args[k], before[k])
    # the slots of what is there now
    new = expect[4]
    total = sum(max(n, 0) for n in new)
    if total <= 200000 and all(n <= columns * page for n in new):
        zero = ints([0] * len(new))
        s2, p2, st2 = nncl.CacheSlots(zero, ints(new), args[2], total + 1, page)
        e2 = [expect[0][i][p // page] * page + p % page for i, n in enumerate(new)
              for p in range(n)]
        ok = [expect[0][i][p // page] >= 0 for i, n in enumerate(new) for p in range(n)]
        assert s2.tolist() == [e if o else -1 for e, o in zip(e2, ok)] + [-1]
        assert st2.tolist() == np.concatenate([[0], np.cumsum(new)]).tolist()


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("requests,most,new,spare", [(1, 0, 1, 1), (1, 100, 1, 0), (7, 200, 1, 3),
                                                     (33, 500, 40, 60), (64, 70, 1, 200),
                                                     (300, 90, 25, 300), (1500, 40, 3, 900),
                                                     (2, 5000, 3000, 400)])
def test_tables(nncl, requests, most, new, spare, page):
    say("tables", requests, most, new, spare, page)
    rng = np.random.default_rng(requests + page)
    lengths = rng.integers(0, most + 1, requests).tolist()
    counts = rng.integers(0, new + 1, requests).tolist()
    counts[0] = new
    columns = -(-(most + new) // page) + 1
    check_tables(nncl, lengths, counts, columns, page, spare, sum(counts) + 5, requests)
    # a step buffer that ends inside the requests, rows that are too short
    check_tables(nncl, lengths, counts, columns, page, spare, sum(counts) // 2, requests + 1)
    check_tables(nncl, lengths, counts, max(1, columns // 2), page, spare, sum(counts), 5)


def test_tables_pages_run_out_in_order(nncl):
    """Those before the one that does not fit get theirs, those after only if they need none."""
    check_tables(nncl, [16, 10, 32, 15, 0, 3], [1, 6, 33, 1, 16, 1], 8, 16, 3, 64, 0)
    check_tables(nncl, [0, 0, 0], [16, 17, 16], 8, 16, 2, 64, 0)
    check_tables(nncl, [0, 0, 0], [0, 0, 0], 1, 16, 0, 0, 0)
    check_tables(nncl, [-4, 5], [3, -7], 2, 16, 2, 4, 0)


def test_tables_with_numbers_out_of_range(nncl):
    """Lengths and counts near 2^31, page numbers outside: no position, and no fault."""
    big = 2 ** 31 - 1
    table = ints([[3, -1], [2, 4], [big, 0], [-5, 1]])
    slots, positions, starts, new, left = nncl.CacheTables(
        ints([big, 1, 3, 2]), ints([big, 2, 2, 1]), table, ints([7, 8, 9]), ints([100]), 40, 16)
    assert starts.tolist() == [0, 40, 40, 40, 40] and left.tolist() == [3]
    assert new.tolist() == [big, 1, 3, 2] and set(slots.tolist()) == {-1}
    slots, positions, starts, new, left = nncl.CacheTables(
        ints([1, 3, 2]), ints([2, 2, 1]), table[1:].contiguous(), ints([7, 8, 9]), ints([-4]), 6,
        16)
    assert starts.tolist() == [0, 2, 4, 5] and left.tolist() == [0]
    assert slots.tolist() == [33, 34, -1, -1, -1, -1]
    assert positions.tolist() == [1, 2, -1, -1, -1, -1]


@pytest.mark.parametrize("page", [16, 64])
def test_release_gives_pages_back(nncl, page):
    cache = Int8Cache(300, 1, 8, page)
    free, count = cache.freePages()
    table = cache.blockTable(9, 150)
    lengths = ints([0] * 9)
    counts = [page * 140, 1, 0, page, page + 1, 5 * page, 3, 9, page * 30 - 1]
    _, _, _, lengths, count = nncl.CacheTables(lengths, ints(counts), table, free, count,
                                               sum(counts), page)
    used = sum(-(-c // page) for c in counts)
    assert lengths.tolist() == counts and count.tolist() == [300 - used]
    held = table.clone()
    finished = [1, 0, 1, 0, 1, 0, 1, 0, 1]
    nncl.CacheRelease(ints(finished), lengths, table, free, count, page)
    assert lengths.tolist() == [0 if f else c for f, c in zip(finished, counts)]
    back = [p for i, f in enumerate(finished) if f for p in held[i].tolist() if p >= 0]
    assert count.tolist() == [300 - used + len(back)]
    assert free.tolist()[300 - used:300 - used + len(back)] == back
    for i, f in enumerate(finished):
        assert table[i].tolist() == ([-1] * 150 if f else held[i].tolist())
    # all pages are owned once: what is free and what the tables hold
    now = free.tolist()[:int(count)] + [p for p in table.view(-1).tolist() if p >= 0]
    assert sorted(now) == list(range(300))


# --------------------------------------------------------------------- append and read
class PlainCache:
    """The rules of append in numpy's float32, over [page, head, token, feature]."""

    def __init__(self, cache):
        d = cache.headDim
        self.page = cache.pageSize
        self.held = [cache.keys.cpu().numpy()[..., :d].astype(np.float32),
                     cache.values.cpu().numpy()[:, :, :d].transpose(0, 1, 3, 2)
                     .astype(np.float32)]
        self.scales = [cache.keyScales.cpu().numpy().copy(),
                       cache.valueScales.cpu().numpy().copy()]
        self.known = np.zeros((cache.pages, cache.pageSize), dtype=bool)

    def append(self, k, v, slots):
        pages = {}
        for i, s in enumerate(slots):
            if 0 <= s < self.known.size:
                pages.setdefault(s // self.page, []).append(i)
        f = np.float32
        for p, who in pages.items():
            off = [slots[i] % self.page for i in who]
            if 0 in off:
                self.known[p] = False
            self.known[p, off] = True
            for which, x in ((0, k), (1, v)):
                for h in range(x.shape[1]):
                    new = x[who, h].astype(f)
                    most = np.max(np.abs(new))
                    with np.errstate(all="ignore"):
                        s = f(most) / f(127)
                        s = f(np.nan) if not np.isfinite(most) else f(0) if s < TINY else s
                        old = f(0) if 0 in off else self.scales[which][p, h]
                        now = f(np.nan) if np.isnan(old) or np.isnan(s) else max(old, s)
                        ratio = f(old / now) if now > 0 else f(0)
                        inv = f(f(1) / now) if now > 0 else f(0)
                        a = self.held[which][p, h]
                        a[:] = np.rint((a * ratio).astype(f))
                        a[off] = np.rint((new * inv).astype(f))
                    self.scales[which][p, h] = now

    def values(self):
        with np.errstate(all="ignore"):
            return [h * s[:, :, None, None] for h, s in zip(self.held, self.scales)]


def same_cache(cache, plain, slots=None):
    """Scales of all pages, and the bytes of every token that was written."""
    assert np.array_equal(cache.keyScales.cpu().numpy(), plain.scales[0], equal_nan=True)
    assert np.array_equal(cache.valueScales.cpu().numpy(), plain.scales[1], equal_nan=True)
    now = PlainCache(cache)
    for which in (0, 1):
        ok = ~np.isnan(plain.scales[which])[:, :, None] & plain.known[:, None, :]
        assert np.array_equal(now.held[which][ok], plain.held[which][ok])


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("heads,dim,page", [(1, 8, 16), (3, 40, 16), (2, 64, 32), (2, 72, 64),
                                            (1, 128, 128), (2, 128, 64), (1, 192, 16),
                                            (1, 256, 128)])
def test_append_over_steps(nncl, heads, dim, page, kind):
    """Prompts that begin and end inside pages, then single tokens of growing and shrinking
    size, a request that rests, one without room; every byte and scale by the rule."""
    say("append", heads, dim, page, kind)
    cache = Int8Cache(40, heads, dim, page)
    cache.keys.random_(-127, 128)  # what pages held before must not matter
    cache.values.random_(-127, 128)
    cache.keyScales.fill_(5.0)
    cache.valueScales.fill_(5.0)
    plain = PlainCache(cache)
    free, count = cache.freePages()
    table = cache.blockTable(4, 40)
    lengths = ints([0, 0, 0, 0])
    rng = np.random.default_rng(dim)
    for step, counts in enumerate([[page + 3, 1, 2 * page, 0], [1, 1, 1, page - 1],
                                   [1, 0, 5, 2], [3, 1, 1, 30 * page], [page, page, 1, 1]]):
        tokens = sum(counts) + 2
        slots, _, _, lengths, count = nncl.CacheTables(lengths, ints(counts), table, free, count,
                                                       tokens, page)
        size = float(2.0 ** rng.integers(-3, 4))
        k = (size * torch.randn(tokens, heads, dim, generator=gen(step), device="cuda"))
        v = torch.randn(tokens, heads, dim, generator=gen(50 + step), device="cuda") / size
        if step == 2:
            k[0] = 0
        k, v = k.to(TYPES[kind]), v.to(TYPES[kind])
        nncl.CacheAppend(k, v, slots, cache)
        plain.append(k.float().cpu().numpy(), v.float().cpu().numpy(), slots.tolist())
        same_cache(cache, plain)
        # and again: the same tokens in the same slots change nothing
        nncl.CacheAppend(k, v, slots, cache)
        same_cache(cache, plain)
    # read back, with slots outside the pool
    total = int(lengths.sum())
    slots, _, _ = nncl.CacheSlots(ints([0] * 4), lengths, table, total, page)
    slots[3] = -1
    slots[4] = 40 * page
    for out in TYPES.values():
        rk, rv = nncl.CacheRead(cache, slots, out)
        for got, full in zip((rk, rv), plain.values()):
            s = np.array(slots.tolist())
            inside = (s >= 0) & (s < 40 * page)
            s = np.where(inside, s, 0)
            e = full[s // page, :, s % page]
            e = torch.from_numpy(np.where(inside[:, None, None], e, 0).astype(np.float32))
            assert torch.equal(got.cpu(), e.to(out))


def test_append_takes_slices_and_many_tokens(nncl):
    """k and v as slices of one projection; enough tokens that a work-group takes several
    pages."""
    heads, dim, page, tokens = 4, 64, 16, 5000
    cache = Int8Cache(400, heads, dim, page)
    plain = PlainCache(cache)
    qkv = torch.randn(tokens, 3 * heads * dim + 2, generator=gen(3), device="cuda")
    k = qkv[:, 1 + heads * dim:1 + 2 * heads * dim].unflatten(1, (heads, dim))
    v = qkv[:, 1 + 2 * heads * dim:1 + 3 * heads * dim].unflatten(1, (heads, dim))
    free, count = cache.freePages()
    table = cache.blockTable(3, 330)
    slots, _, _, lengths, _ = nncl.CacheTables(ints([0] * 3), ints([4000, 7, 993]), table, free,
                                               count, tokens, page)
    assert int((slots >= 0).sum()) == tokens
    nncl.CacheAppend(k, v, slots, cache)
    plain.append(k.cpu().numpy(), v.cpu().numpy(), slots.tolist())
    same_cache(cache, plain)


def test_append_of_values_that_are_not_finite(nncl):
    """They make their page's scale NaN for their head alone, until the page is begun again."""
    cache = Int8Cache(3, 2, 16, 16)
    plain = PlainCache(cache)
    for step, slots in enumerate([list(range(0, 20)), [20, 21], [22], list(range(0, 4))]):
        k = torch.randn(len(slots), 2, 16, generator=gen(step), device="cuda")
        v = torch.randn(len(slots), 2, 16, generator=gen(9 + step), device="cuda")
        if step == 0:
            k[2, 1, 3] = float("inf")
            v[5, 0, 0] = float("nan")
        if step == 1:
            k[1, 0, 15] = float("-inf")
        nncl.CacheAppend(k, v, ints(slots), cache)
        plain.append(k.cpu().numpy(), v.cpu().numpy(), slots)
        same_cache(cache, plain)
    assert cache.keyScales.isnan().tolist() == [[False, False], [True, False], [False, False]]


# ---------------------------------------------------------------------------- attention
def filled(heads, dim, page, pages, seed):
    """A cache with something in every slot."""
    cache = Int8Cache(pages, heads, dim, page)
    g = gen(seed)
    cache.keys.copy_(torch.randint(-127, 128, cache.keys.shape, generator=g, device="cuda"))
    cache.values.copy_(torch.randint(-127, 128, cache.values.shape, generator=g, device="cuda"))
    cache.keyScales.copy_(torch.rand(pages, heads, generator=g, device="cuda") * 0.02 + 0.005)
    cache.valueScales.copy_(torch.rand(pages, heads, generator=g, device="cuda") * 0.02 + 0.005)
    return cache


def attention64(q, cache, table, starts, positions, scale):
    """(result, A, V) in 64 bits over the cache's contents (module docstring)."""
    d, page = cache.headDim, cache.pageSize
    tokens, heads = q.shape[:2]
    group = heads // cache.kvHeads
    k = cache.keys[..., :d].double() * cache.keyScales.double()[:, :, None, None]
    v = cache.values[:, :, :d].transpose(2, 3).double() * \
        cache.valueScales.double()[:, :, None, None]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    room = torch.zeros(q.shape[:2] + (2,), dtype=torch.float64, device=q.device)
    st, pos = starts.tolist(), positions.tolist()
    for r in range(len(st) - 1):
        for t in range(st[r], st[r + 1]):
            n = pos[t] + 1
            at = [(table[r][p // page], p % page) for p in range(n)]
            at = [(a, b) for a, b in at if 0 <= a < cache.pages]
            if not at:
                continue
            a = torch.tensor([x[0] for x in at], device=q.device)
            b = torch.tensor([x[1] for x in at], device=q.device)
            for h in range(cache.kvHeads):
                kk, vv = k[a, h, b], v[a, h, b]
                x = q[t, h * group:(h + 1) * group].double()
                z = scale * (x @ kk.t())
                p = torch.softmax(z, 1)
                out[t, h * group:(h + 1) * group] = p @ vv
                room[t, h * group:(h + 1) * group, 0] = scale * (
                    x.abs() @ kk.abs().t()).amax(1)
                room[t, h * group:(h + 1) * group, 1] = vv.abs().max()
    return out, room[..., 0], room[..., 1]


def check_attention(got, want, keys):
    y, a, v = want
    d = y.shape[-1]
    bf = got.dtype == torch.bfloat16
    weight = 2 * (d + 8) * 2.0 ** -24 * a + 2.0 ** -21 + (2.0 ** -9 if bf else 0)
    tol = v * (2 * weight + (keys / 64 + 72) * 2.0 ** -24)
    tol = tol[..., None] + (2.0 ** -9 * y.abs() if bf else 0)
    off = (got.double() - y).abs()
    assert bool((off <= tol).all()), float((off - tol).max())
    # and on the whole: roundings that do not line up
    if float(y.norm()) > 0:
        far = float((got.double() - y).norm() / y.norm())
        assert far <= (3e-3 if bf else 2e-6), far


def step_of(nncl, cache, lengths, counts, extra, seed, columns=None):
    """A table of random pages, starts and positions of a step after which request i has
    lengths[i] tokens, the last counts[i] of them new."""
    page = cache.pageSize
    need = [-(-n // page) for n in lengths]
    columns = columns or max(max(need), 1) + 1
    order = np.random.default_rng(seed).permutation(cache.pages).tolist()
    table, at = [], 0
    for n in need:
        table.append(order[at:at + n] + [-1] * (columns - n))
        at += n
    assert at <= cache.pages
    tokens = sum(counts) + extra
    _, positions, starts = nncl.CacheSlots(ints([n - c for n, c in zip(lengths, counts)]),
                                           ints(counts), ints(table), tokens, page)
    return table, starts, positions, tokens


FEW = [  # heads, kv heads, head size, page, lengths after the step, new tokens
    (1, 1, 8, 16, [1], [1]),
    (2, 2, 32, 16, [1, 2, 15, 16, 17], [1, 1, 1, 1, 1]),
    (4, 1, 40, 32, [63, 64, 65, 31], [1, 1, 1, 1]),
    (8, 2, 64, 64, [300, 1, 257, 256], [1, 1, 1, 1]),
    (6, 2, 72, 16, [5, 0, 200], [2, 0, 5]),
    (8, 1, 96, 128, [129, 700], [1, 2]),
    (32, 8, 128, 64, [1000, 3, 65], [1, 1, 1]),
    (16, 1, 128, 16, [2000], [1]),
    (2, 1, 192, 32, [100, 40], [3, 1]),
    (3, 3, 256, 64, [130, 513], [1, 1]),
]
MANY = [
    (1, 1, 32, 16, [17], [17]),
    (2, 1, 40, 16, [200, 3, 64], [150, 3, 64]),
    (4, 4, 64, 32, [129, 40, 0, 300], [129, 1, 0, 20]),
    (8, 2, 64, 128, [260], [260]),
    (4, 2, 96, 64, [70, 200], [70, 33]),
    (4, 1, 128, 64, [190, 65], [190, 64]),
    (2, 2, 128, 16, [600, 5], [40, 5]),
    (2, 1, 192, 64, [100], [90]),
    (2, 1, 256, 16, [90, 600], [50, 60]),
]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("heads,kv,dim,page,lengths,counts", FEW + MANY)
def test_attention(nncl, heads, kv, dim, page, lengths, counts, kind):
    """Every head size and page size, groups, lengths around tiles and ranges, requests without
    tokens; hints right, absent and wrong; tokens past the step's end give 0."""
    say("attention", heads, kv, dim, page, lengths, counts, kind)
    cache = filled(kv, dim, page, sum(-(-n // page) for n in lengths) + 2, dim)
    table, starts, positions, tokens = step_of(nncl, cache, lengths, counts, 3, page)
    q = torch.randn(tokens, heads, dim, generator=gen(heads), device="cuda").to(TYPES[kind])
    want = attention64(q, cache, table, starts, positions, dim ** -0.5)
    for count, length in ((max(counts), max(lengths)), (0, 0), (1, 1), (10000, 70)):
        got = nncl.CacheAttention(q, cache, ints(table), starts, positions, maxCount=count,
                                  maxLength=length)
        assert got.dtype == q.dtype and got.shape == q.shape
        check_attention(got, want, max(lengths))
        assert not got[sum(counts):].any()
    again = nncl.CacheAttention(q, cache, ints(table), starts, positions, maxCount=10000,
                                maxLength=70)
    assert torch.equal(got, again)  # the same bits every time


@pytest.mark.parametrize("kind", TYPES)
def test_attention_scales_and_strided_queries(nncl, kind):
    cache = filled(2, 64, 16, 60, 1)
    table, starts, positions, tokens = step_of(nncl, cache, [300, 90], [30, 1], 0, 2)
    wide = torch.randn(tokens, 3 * 256 + 3, generator=gen(1), device="cuda").to(TYPES[kind])
    q = wide[:, 5:5 + 256].unflatten(1, (4, 64))
    for scale in (0.0, 1.0, 0.02):
        got = nncl.CacheAttention(q, cache, ints(table), starts, positions, scale=scale)
        check_attention(got, attention64(q, cache, table, starts, positions, scale), 300)


@pytest.mark.parametrize("counts", [[1, 1], [40, 30]])
def test_attention_rows_without_keys_and_lost_pages(nncl, counts):
    """Positions of -1 (and below) give 0, positions past the table's row end there, pages
    outside the pool are left out wherever they stand, starts are read as within the step."""
    cache = filled(2, 64, 16, 80, 4)
    lengths = [600, 500]
    table, starts, positions, tokens = step_of(nncl, cache, lengths, counts, 2, 7)
    for r, j, page in ((0, 0, -1), (0, 3, 80), (0, 20, 2 ** 31 - 1), (1, 5, -2 ** 31)):
        table[r][j] = page
    positions[0] = -1
    if counts[0] > 1:
        positions[3] = -2 ** 31
        positions[4] = 0   # only a lost page
        positions[5] = 15
        positions[6] = 16
    q = torch.randn(tokens, 4, 64, generator=gen(2), device="cuda")
    got = nncl.CacheAttention(q, cache, ints(table), starts, positions)
    want = attention64(q, cache, table, starts, positions.clamp(min=-1), 0.125)
    check_attention(got, want, 600)
    assert not got[0].any() and (counts[0] == 1 or not got[3:6].any())
    # a position past the row: as the row's last
    far = positions.clone()
    far[1] = 2 ** 31 - 1
    ends = positions.clone()
    ends[1] = len(table[0]) * 16 - 1
    for t in (far, ends):
        t = nncl.CacheAttention(q, cache, ints(table), starts, t)
        assert bool(t.isfinite().all())
        if counts[0] > 1:
            check_attention(t, attention64(q, cache, table, starts, ends.clamp(min=-1), 0.125),
                            700)
    # a request's first token beyond the step, a negative one
    odd = starts.clone()
    odd[2] = 10 ** 6
    assert bool(nncl.CacheAttention(q, cache, ints(table), odd, positions).isfinite().all())
    odd[0] = -7
    assert bool(nncl.CacheAttention(q, cache, ints(table), odd, positions).isfinite().all())


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("count", [1, 50])
def test_attention_and_what_is_not_finite(nncl, count, kind):
    """A page with a NaN scale reaches the rows that see a token of it, for its head, and no
    other row; a query that is not finite reaches its own rows."""
    cache = filled(2, 64, 16, 60, 4)
    table, starts, positions, tokens = step_of(nncl, cache, [400, 300], [count, count], 0, 3)
    q = torch.randn(tokens, 4, 64, generator=gen(5), device="cuda").to(TYPES[kind])
    want = attention64(q, cache, table, starts, positions, 0.125)
    clean = nncl.CacheAttention(q, cache, ints(table), starts, positions)
    cache.keyScales[table[0][23], 0] = float("nan")  # tokens 368..383
    cache.valueScales[table[0][24], 1] = float("nan")  # tokens 384..399
    q[-1, 0, 5] = float("inf")
    got = nncl.CacheAttention(q, cache, ints(table), starts, positions)
    bad = torch.zeros(tokens, 4, dtype=torch.bool, device="cuda")
    own = torch.arange(tokens, device="cuda") < count
    bad[:, :2] |= (own & (positions >= 368))[:, None]
    bad[:, 2:] |= (own & (positions >= 384))[:, None]
    bad[-1, 0] = True
    assert torch.equal(got.isnan(), bad[:, :, None].expand_as(got))
    if kind == "f32":
        assert torch.equal(got[~bad], clean[~bad])
    else:  # (a tile with such a scale rounds its weights another way)
        got[bad], clean[bad] = 0, 0
        check_attention(got, tuple(torch.where(bad if w.dim() == 2 else bad[..., None], 0, w)
                                   for w in want), 400)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("count", [1, 50])
def test_attention_over_scales_of_any_size(nncl, count, page, kind):
    """Pages whose values are all 0 (scale 0), tiny or huge among others: weights count in
    full, whatever their values' scale."""
    cache = filled(2, 64, page, 60, 4)
    table, starts, positions, tokens = step_of(nncl, cache, [400, 300], [count, count], 0, 3)
    for r, j, scale in ((0, 0, 0.0), (0, 1, 2.0 ** -126), (0, 2, 1e-30), (0, 4, 1e30),
                        (1, 0, 0.0), (1, 1, 3e-37), (1, 2, 0.0), (1, 3, 1e-12)):
        cache.valueScales[table[r][j]] = scale
    cache.keyScales[table[0][3]] = 0.0
    q = torch.randn(tokens, 4, 64, generator=gen(5), device="cuda").to(TYPES[kind])
    got = nncl.CacheAttention(q, cache, ints(table), starts, positions)
    want = attention64(q, cache, table, starts, positions, 0.125)
    assert bool(got.isfinite().all())
    for part in (slice(0, count), slice(count, 2 * count)):
        check_attention(got[part], tuple(w[part] for w in want), 400)


def test_attention_over_a_cache_past_32_bits(nncl):
    """Keys and values of more than 2^32 bytes each, a request in the last pages."""
    pages, heads, dim, page = 70000, 8, 128, 64
    say("cache of", pages * heads * dim * page, "bytes a side")
    cache = Int8Cache(pages, heads, dim, page)
    small = filled(heads, dim, page, 8, 3)
    cache.keys[-8:] = small.keys
    cache.values[-8:] = small.values
    cache.keyScales[-8:] = small.keyScales
    cache.valueScales[-8:] = small.valueScales
    for lengths, counts in (([200, 230], [1, 1]), ([200, 130], [60, 1])):
        table, starts, positions, tokens = step_of(nncl, small, lengths, counts, 0, 3)
        q = torch.randn(tokens, 16, dim, generator=gen(5), device="cuda")
        there = [[p + pages - 8 if p >= 0 else p for p in row] for row in table]
        a = nncl.CacheAttention(q, small, ints(table), starts, positions)
        b = nncl.CacheAttention(q, cache, ints(there), starts, positions)
        assert torch.equal(a, b)
    slots = ints([(pages - 1) * page + 5, (pages - 2) * page])
    k = torch.randn(2, heads, dim, device="cuda") * 9
    nncl.CacheAppend(k, k, slots, cache)
    nncl.CacheAppend(k, k, ints([7 * page + 5, 6 * page]), small)
    for a, b in zip(nncl.CacheRead(cache, slots), nncl.CacheRead(small, ints([7 * page + 5,
                                                                             6 * page]))):
        assert torch.equal(a, b)
    del cache
    torch.cuda.empty_cache()


def test_step_captured_in_a_graph(nncl):
    """Tables, append and attention of a decoding step, captured once and replayed: every
    replay gives the eager bits, with eager work between."""
    heads, kv, dim, page, requests = 8, 2, 64, 16, 5
    cache = filled(kv, dim, page, 400, 8)
    free, count = cache.freePages()
    table = cache.blockTable(requests, 60)
    lengths = ints([0] * requests)
    step = torch.randn(700, kv, dim, generator=gen(1), device="cuda")
    slots, _, _, lengths, count = nncl.CacheTables(lengths, ints([100, 300, 17, 1, 200]), table,
                                                   free, count, 700, page)
    nncl.CacheAppend(step, step, slots, cache)
    ones = ints([1] * requests)
    q = torch.zeros(requests, heads, dim, device="cuda")
    k, v = torch.zeros(requests, kv, dim, device="cuda"), torch.zeros(requests, kv, dim,
                                                                      device="cuda")
    stream = torch.cuda.Stream()
    nncl.reserve_workspace(stream, 64 << 20)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        slots, positions, starts, new, left = nncl.CacheTables(lengths, ones, table, free, count,
                                                               requests, page)
        nncl.CacheAppend(k, v, slots, cache)
        out = nncl.CacheAttention(q, cache, table, starts, positions, maxCount=1)
        lengths.copy_(new)
        count.copy_(left)
    for i in range(4):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=gen(10 * i + t.numel()), device="cuda"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert lengths.tolist() == [101 + i, 301 + i, 18 + i, 2 + i, 201 + i]
        again = nncl.CacheAttention(q, cache, table, starts, positions, maxCount=1)
        assert torch.equal(out, again)
        want = attention64(q, cache, table.tolist(), starts, positions, dim ** -0.5)
        check_attention(out, want, 400)


def test_refusals(nncl):
    with pytest.raises(ShapeError, match="headDim"):
        Int8Cache(4, 1, 12)
    with pytest.raises(ShapeError, match="headDim"):
        Int8Cache(4, 1, 264)
    with pytest.raises(ShapeError, match="pageSize"):
        Int8Cache(4, 1, 64, 48)
    cache = Int8Cache(4, 2, 64, 16)
    k = torch.zeros(3, 2, 64, device="cuda")
    slots = ints([0, 1, 2])
    with pytest.raises(ShapeError, match="k and v must be"):
        nncl.CacheAppend(k[:, :1], k[:, :1], slots, cache)
    with pytest.raises(ShapeError, match="one type"):
        nncl.CacheAppend(k, k.bfloat16(), slots, cache)
    with pytest.raises(ShapeError, match="rows of k"):
        nncl.CacheAppend(k.transpose(0, 1).contiguous().transpose(0, 1), k, slots, cache)
    with pytest.raises(ShapeError, match="slots"):
        nncl.CacheAppend(k, k, slots.long(), cache)
    with pytest.raises(ShapeError, match="slots"):
        nncl.CacheAppend(k, k, slots[:2], cache)
    table, starts, pos = cache.blockTable(2, 2), ints([0, 1, 3]), ints([0, 0, 1])
    q = torch.zeros(3, 4, 64, device="cuda")
    with pytest.raises(ShapeError, match="heads"):
        nncl.CacheAttention(q[:, :3], cache, table, starts, pos)
    with pytest.raises(ShapeError, match="starts"):
        nncl.CacheAttention(q, cache, table, starts[:2], pos)
    with pytest.raises(ShapeError, match="positions"):
        nncl.CacheAttention(q, cache, table, starts, pos[:2])
    with pytest.raises(_native.MigemmArgumentError, match="scale"):
        nncl.CacheAttention(q, cache, table, starts, pos, scale=float("nan"))
    with pytest.raises(_native.MigemmArgumentError, match="max_count"):
        nncl.CacheAttention(q, cache, table, starts, pos, maxCount=-1)
    with pytest.raises(ShapeError, match="float32 or bfloat16"):
        nncl.CacheAttention(q.double(), cache, table, starts, pos)
    with pytest.raises(_native.MigemmArgumentError, match="page_size"):
        nncl.CacheTables(pos, pos, cache.blockTable(3, 2), pos, ints([1]), 4, 48)
    with pytest.raises(ShapeError, match="counts"):
        nncl.CacheTables(pos, pos[:2], cache.blockTable(3, 2), pos, ints([1]), 4, 16)
    assert nncl.CacheAttention(q[:0], cache, table, starts, pos[:0]).shape == (0, 4, 64)
    assert nncl.CacheRead(cache, slots[:0])[0].shape == (0, 2, 64)
    nncl.CacheAppend(k[:0], k[:0], slots[:0], cache)

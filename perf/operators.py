"""Performance cases of the 8-bit serving operators, through their public entry points.

Each kind of case is one piece of work that a program that serves a model has it do:

  linear  NnClGlob.LinearInt8: a layer whose weight is held in 8 bits with a scale for each
          output channel; the rows of x are quantised on the fly, a scale for each
  tables  NnClGlob.CacheTables: the pages and the slots of the tokens that a step adds to a
          batch of requests, from the requests' lengths
  append  NnClGlob.CacheAppend: a step's keys and values into an 8-bit paged cache with a scale
          for each page and head; NnClGlob.CacheRead hands the touched pages back
  attend  NnClGlob.CacheAttention: causal attention of a step's queries over that cache

The cache of a case: keys int8 [pages, kv heads, page size, width], values int8 [pages, kv
heads, width, page size] (a head's values transposed within a page), width the head's size
rounded up to 32 (to 64 above 128), float32 scales [pages, kv heads] for each.

A scale is s = fl(a / 127) of the largest magnitude a it covers, 0 where that is subnormal and
NaN where a value is not finite; a value x is held as rint(fl(x * fl(1 / s))) (half to even).
"""
import math
import random

import torch

own = False

_TINY = 2.0 ** -126
_TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}
_glob = None


def glob():
    global _glob
    if _glob is None:
        from my_pytchon_opencl_lib_amd import NnClGlob
        _glob = NnClGlob("cuda:0")
    return _glob


def listed():
    return [
        # one token through a wide layer: bound by reading the weight
        {"name": "linear_token", "kind": "linear", "rows": 1, "fin": 4096, "fout": 11008,
         "type": "bfloat16"},
        # a small serving batch
        {"name": "linear_batch", "kind": "linear", "rows": 24, "fin": 2048, "fout": 4096,
         "type": "float32"},
        # no dimension a multiple of any tile, rows of odd length
        {"name": "linear_ragged", "kind": "linear", "rows": 1000, "fin": 777, "fout": 3000,
         "type": "float32"},
        # the prompts of a batch through the wide layer (the largest product)
        {"name": "linear_prompt", "kind": "linear", "rows": 8192, "fin": 4096, "fout": 11008,
         "type": "bfloat16"},
        # a decoding step of a small batch: one token a request (the smallest call)
        {"name": "tables_step", "kind": "tables", "requests": 32, "context": 4096, "new": 1,
         "page": 64, "pool": 1.0},
        # admitting many prompts at once in small pages, more than the pool holds
        {"name": "tables_admit", "kind": "tables", "requests": 512, "context": 1024, "new": 500,
         "page": 16, "pool": 0.8},
        # a decoding step: one token a request, old pages that are rescaled
        {"name": "append_step", "kind": "append", "requests": 64, "context": 2000, "new": 1,
         "kv": 8, "dim": 128, "page": 64, "type": "bfloat16"},
        # prompts that begin and end inside pages
        {"name": "append_prompt", "kind": "append", "requests": 5, "context": 100, "new": 2500,
         "kv": 8, "dim": 128, "page": 32, "type": "float32"},
        # a decoding step of a batch with grouped heads
        {"name": "attend_step", "kind": "attend", "requests": 32, "context": 4096, "new": 1,
         "mix": 1, "heads": 32, "kv": 8, "dim": 128, "page": 64, "type": "bfloat16"},
        # few requests with long contexts
        {"name": "attend_long", "kind": "attend", "requests": 2, "context": 131072, "new": 1,
         "mix": 1, "heads": 32, "kv": 8, "dim": 128, "page": 64, "type": "bfloat16"},
        # prompts, some of them continued from a cached part
        {"name": "attend_prompt", "kind": "attend", "requests": 4, "context": 1500, "new": 1500,
         "mix": 1, "heads": 32, "kv": 8, "dim": 128, "page": 64, "type": "bfloat16"},
        # short prompts among decoding requests, a head of keys for each head of queries
        {"name": "attend_mixed", "kind": "attend", "requests": 9, "context": 500, "new": 128,
         "mix": 2, "heads": 8, "kv": 8, "dim": 64, "page": 16, "type": "float32"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A size over [lo, hi], log-uniform; every second one rounded to a multiple of 32 (the
    widths of layers), the others as they fall, odd ones among them."""
    v = _log_int(rng, lo, hi)
    if rng.random() < 0.5 and v >= 32:
        v = v // 32 * 32
    return v


def draw(rng):
    kind = rng.choice(["linear", "tables", "append", "attend", "attend"])
    kind_type = rng.choice(["float32", "bfloat16"])
    if kind == "linear":
        return {"kind": kind, "rows": _log_int(rng, 1, 8192), "fin": _size(rng, 64, 4096),
                "fout": _size(rng, 64, 11008), "type": kind_type}
    page = rng.choice([16, 32, 64, 128])
    if kind == "tables":
        return {"kind": kind, "requests": _log_int(rng, 1, 512),
                "context": _log_int(rng, 1, 4096), "new": rng.choice([1, _log_int(rng, 2, 500)]),
                "page": page, "pool": rng.choice([1.0, 1.0, 0.5])}
    dim = rng.choice([32, 40, 64, 72, 80, 96, 128, 128, 192, 256])
    if kind == "append":
        new = rng.choice([1, _log_int(rng, 2, 2500)])
        return {"kind": kind, "requests": _log_int(rng, 1, 64 if new == 1 else 5),
                "context": _log_int(rng, 1, 2000), "new": new, "kv": _log_int(rng, 1, 16),
                "dim": dim, "page": page, "type": kind_type}
    kv = _log_int(rng, 1, 16)
    case = {"kind": kind, "requests": _log_int(rng, 1, 32), "context": _log_int(rng, 16, 32768),
            "new": 1, "mix": 1, "heads": kv * rng.choice([1, 2, 3, 4, 8]), "kv": kv, "dim": dim,
            "page": page, "type": kind_type}
    if rng.random() < 0.5:  # prompts
        case |= {"requests": _log_int(rng, 1, 8), "context": _log_int(rng, 16, 1500),
                 "new": _log_int(rng, 2, 1500), "mix": rng.choice([1, 1, 3])}
    while work(case)["bytes"] > 4e8:
        case["context"] = max(1, case["context"] // 2)
    while work(case)["flops"] > 1.5e11 or _scores(case) > 4e8:
        case["new"] = max(1, case["new"] // 2)
        case["requests"] = max(1, case["requests"] // 2)
    return case


# ---------------------------------------------------------------- lengths of a case's requests
def _lengths(case):
    """(tokens in the cache, new tokens) of each request: fixed by the case, so that its work
    is. Contexts are spread over [1/4, 1] of the longest, some prompts begin with none; where
    prompts are mixed in, every `mix`-th request brings one and the others one token; in a
    batch of eight and more one request rests."""
    rng = random.Random("%(requests)d %(context)d %(new)d" % case)
    olds, news = [], []
    for i in range(case["requests"]):
        old = max(1, int(case["context"] * rng.uniform(0.25, 1.0)))
        new = 1
        if case["new"] > 1 and i % case.get("mix", 1) == 0:
            new = max(1, int(case["new"] * rng.uniform(0.4, 1.0)))
            old = rng.choice([0, old])
        if i == 0:
            new = case["new"]
        if i == 5 and case["requests"] >= 8:
            new = 0
        olds.append(old)
        news.append(new)
    return olds, news


def _pages(n, page):
    return -(-n // page)


def _width(dim):
    return -(-dim // 32) * 32 if dim <= 128 else -(-dim // 64) * 64


def _scores(case):
    """Scores of the plain form: requests x heads x the longest step x the longest context."""
    olds, news = _lengths(case)
    return case["requests"] * case["heads"] * max(news) * max(a + b for a, b in zip(olds, news))


def work(case):
    kind = case["kind"]
    if kind == "linear":
        m, k, n = case["rows"], case["fin"], case["fout"]
        size = 4 if case["type"] == "float32" else 2
        return {"bytes": m * k * size + n * k + 8 * n + m * n * size, "flops": 2 * m * n * k}
    olds, news = _lengths(case)
    total = sum(news)
    if kind == "tables":
        page = case["page"]
        add = sum(_pages(a + b, page) - _pages(a, page) for a, b in zip(olds, news))
        # lengths, counts, starts, new lengths; free pages to table; slots and positions; the
        # entry of the page that each request goes on in
        return {"bytes": 16 * len(olds) + 8 * add + 8 * total + 4 * len(olds), "flops": 0}
    size = 4 if case["type"] == "float32" else 2
    one = case["kv"] * case["dim"]
    if kind == "append":
        back = sum(_pages(a + b, case["page"]) - a // case["page"] if b else 0
                   for a, b in zip(olds, news)) * case["page"]
        # new keys and values read and written in 8 bits, the touched pages handed back
        return {"bytes": 2 * one * (total * (size + 1) + back * (1 + size)), "flops": 0}
    pairs = sum(b * a + b * (b + 1) // 2 for a, b in zip(olds, news))
    keys = sum(a + b for a, b in zip(olds, news) if b)
    return {"bytes": 2 * keys * one + 2 * total * case["heads"] * case["dim"] * size,
            "flops": 4 * pairs * case["heads"] * case["dim"]}


# ------------------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _scale_of(a):
    s = a / torch.full_like(a, 127.0)
    s = torch.where(s < _TINY, torch.zeros_like(s), s)
    return torch.where(torch.isfinite(a), s, torch.full_like(s, math.nan))


def _held(x, s):
    return torch.round(x * torch.where(s > 0, torch.reciprocal(s), torch.zeros_like(s)))


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _cache(case, g, pages):
    """A cache whose every page is full: keys with a few large channels, plain values."""
    h, p, d = case["kv"], case["page"], case["dim"]
    w = _width(d)
    k = _randn(g, pages, h, p, d) * torch.exp(0.4 * _randn(g, 1, h, 1, d))
    ks = _scale_of(k.abs().amax((2, 3)))
    keys = torch.zeros(pages, h, p, w, dtype=torch.int8, device="cuda")
    keys[..., :d] = _held(k, ks[:, :, None, None])
    v = _randn(g, pages, h, d, p)
    vs = _scale_of(v.abs().amax((2, 3)))
    values = torch.zeros(pages, h, w, p, dtype=torch.int8, device="cuda")
    values[:, :, :d] = _held(v, vs[:, :, None, None])
    return {"keys": keys, "values": values, "key_scales": ks, "value_scales": vs}


def _handle(case, c):
    from my_pytchon_opencl_lib_amd.cache import Int8Cache
    cache = Int8Cache(c["keys"].shape[0], case["kv"], case["dim"], case["page"], device="cuda:0")
    cache.keys.copy_(c["keys"])
    cache.values.copy_(c["values"])
    cache.keyScales.copy_(c["key_scales"])
    cache.valueScales.copy_(c["value_scales"])
    return cache


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _table(g, counts, pages, columns):
    """A block table: counts[i] pages for request i, spread over the pool; -1 beyond."""
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    c = _ints(counts).long()
    first = torch.cumsum(c, 0) - c
    col = torch.arange(columns, device="cuda")
    at = (first[:, None] + col).clamp(max=max(pages - 1, 0))
    return torch.where(col < c[:, None], order[at], -1).to(torch.int32), order


def prepare(case, seed):
    g = _generator(seed)
    kind = case["kind"]
    s = {"case": case}
    if kind == "linear":
        dt = _TYPES[case["type"]]
        m, k, n = case["rows"], case["fin"], case["fout"]
        big = torch.where(torch.rand(k, generator=g, device="cuda") < 0.01, 8.0, 1.0)
        s["x"] = (_randn(g, m, k) * big).to(dt)
        weight = (torch.rand(n, k, generator=g, device="cuda") * 2 - 1) / math.sqrt(k)
        s["scales"] = _scale_of(weight.abs().amax(1))
        s["weight"] = torch.zeros(n, -(-k // 16) * 16, dtype=torch.int8, device="cuda")
        s["weight"][:, :k] = _held(weight, s["scales"][:, None])
        s["bias"] = _randn(g, n) * 0.1
        return s
    olds, news = _lengths(case)
    page = case["page"]
    had = [_pages(a, page) for a in olds]
    want = [_pages(a + b, page) for a, b in zip(olds, news)]
    if kind == "tables":
        spare = int(sum(w - h for w, h in zip(want, had)) * case["pool"])
        pages = sum(had) + spare
        s["table"], order = _table(g, had, pages, max(want) + 2)
        s["free"] = torch.cat([order[sum(had):], order[:0].new_zeros(1)])
        s["free_count"] = _ints([spare])
        s["lengths"], s["counts"] = _ints(olds), _ints(news)
        s["tokens"] = sum(news) + 3  # a step's buffers are a little larger than the step
        return s
    dt = _TYPES[case["type"]]
    pages = sum(want) + 3
    s["cache"] = _cache(case, g, pages)
    s["table"], _ = _table(g, want, pages, max(want) + 1)
    total = sum(news)
    owner = torch.repeat_interleave(torch.arange(len(news), device="cuda"), _ints(news))
    s["starts"] = torch.cat([_ints([0]), torch.cumsum(_ints(news), 0).to(torch.int32)])
    place = torch.arange(total, device="cuda") - s["starts"][owner]
    at = _ints(olds)[owner] + place
    s["positions"] = at.to(torch.int32)
    if kind == "append":
        s["slots"] = (s["table"][owner, at // page] * page + at % page).to(torch.int32)
        # growing values, as a step that outranges what its page holds
        s["k"] = (1.5 * _randn(g, total, case["kv"], case["dim"])).to(dt)
        s["v"] = (1.5 * _randn(g, total, case["kv"], case["dim"])).to(dt)
        back = [(i, a // page * page, a + b) for i, (a, b) in enumerate(zip(olds, news)) if b]
        who = torch.repeat_interleave(_ints([x[0] for x in back]),
                                      _ints([x[2] - x[1] for x in back])).long()
        pos = torch.cat([torch.arange(x[1], x[2], device="cuda") for x in back])
        s["back"] = (s["table"][who, pos // page] * page + pos % page).to(torch.int32)
    else:
        s["q"] = _randn(g, total, case["heads"], case["dim"]).to(dt)
        s["most"] = max(news)
        s["longest"] = max(a + b for a, b in zip(olds, news))
    if own:
        s["handle"] = _handle(case, s["cache"])
    return s


# ------------------------------------------------------------------------------ one pass
def run(s):
    kind = s["case"]["kind"]
    if not own:
        return {"linear": _linear, "tables": _tables, "append": _append,
                "attend": _attend}[kind](s)
    nncl = glob()
    if kind == "linear":
        return nncl.LinearInt8(s["x"], s["weight"], s["scales"], s["bias"])
    if kind == "tables":
        slots, positions, starts, lengths, free = nncl.CacheTables(
            s["lengths"], s["counts"], s["table"], s["free"], s["free_count"], s["tokens"],
            s["case"]["page"])
        return {"table": s["table"], "slots": slots, "positions": positions, "starts": starts,
                "lengths": lengths, "free": free}
    if kind == "append":
        nncl.CacheAppend(s["k"], s["v"], s["slots"], s["handle"])
        k, v = nncl.CacheRead(s["handle"], s["back"], s["k"].dtype)
        return {"k": k, "v": v}
    return nncl.CacheAttention(s["q"], s["handle"], s["table"], s["starts"], s["positions"],
                               maxCount=s["most"], maxLength=s["longest"])


def _linear(s):
    k = s["x"].shape[1]
    x = s["x"].float()
    scale = _scale_of(x.abs().amax(1))
    held = _held(x, scale[:, None])
    y = torch.matmul(held, s["weight"][:, :k].float().t())
    return (y * scale[:, None] * s["scales"] + s["bias"]).to(s["x"].dtype)


def _tables(s):
    page, tokens = s["case"]["page"], s["tokens"]
    n, c = s["lengths"].long().clamp(min=0), s["counts"].long().clamp(min=0)
    free, table = s["free"], s["table"]
    columns = table.shape[1]
    end = torch.cumsum(c, 0)
    start = end - c
    have = (n + page - 1) // page
    fits = (n + c <= columns * page) & (end <= tokens)
    asks = torch.where(fits, (n + c + page - 1) // page - have, 0)
    upto = torch.cumsum(asks, 0)
    held = s["free_count"].long()
    ok = fits & ((asks == 0) | (upto <= held))
    col = torch.arange(columns, device=n.device)
    rank = (upto - asks - have)[:, None] + col
    new = ok[:, None] & (col >= have[:, None]) & (col < (have + asks)[:, None])
    table = torch.where(new, free[(held - 1 - rank).clamp(0, free.numel() - 1)], table)
    t = torch.arange(tokens, device=n.device)
    r = torch.searchsorted(end, t, right=True)
    live = r < n.numel()
    r = r.clamp(max=n.numel() - 1)
    live = live & ok[r]
    at = torch.where(live, n[r] + t - start[r], 0)
    slots = torch.where(live, table[r, at // page].long() * page + at % page, -1)
    starts = torch.cat([end.new_zeros(1), end]).clamp(max=tokens)
    return {"table": table, "slots": slots.to(torch.int32),
            "positions": torch.where(live, at, -1).to(torch.int32),
            "starts": starts.to(torch.int32),
            "lengths": (n + torch.where(ok, c, 0)).to(torch.int32),
            "free": (held - torch.where(ok, asks, 0).sum()).to(torch.int32)}


def _appended(x, slots, page, held, scales):
    """held [pages, kv, page, dim] (float32) and its scales after x [T, kv, dim] at slots."""
    pages = held.shape[0]
    at, off = slots.long() // page, slots.long() % page
    x = x.float()
    most = torch.zeros_like(scales).index_reduce_(0, at, x.abs().amax(2), "amax")
    seen = torch.zeros(pages, device=x.device).index_fill_(0, at, 1.0) > 0
    fresh = torch.zeros(pages, device=x.device).index_reduce_(0, at, (off == 0).float(), "amax")
    old = torch.where(fresh[:, None] > 0, torch.zeros_like(scales), scales)
    now = torch.where(seen[:, None], torch.maximum(old, _scale_of(most)), scales)
    ratio = torch.where(now > 0, old / now, torch.zeros_like(now))
    again = torch.round(held * ratio[:, :, None, None])
    held = torch.where(seen[:, None, None, None], again, held)
    held[at, :, off] = _held(x, now[at][:, :, None])
    return held, now


def _append(s):
    page, d, c = s["case"]["page"], s["case"]["dim"], s["cache"]
    at, off = s["back"].long() // page, s["back"].long() % page
    out = {}
    for name, held, scales in (("k", c["keys"][..., :d], c["key_scales"]),
                               ("v", c["values"][:, :, :d].transpose(2, 3), c["value_scales"])):
        held, scales = _appended(s[name], s["slots"], page, held.float(), scales)
        out[name] = (held[at, :, off] * scales[at][:, :, None]).to(s[name].dtype)
    return out


def _attend(s):
    case, c = s["case"], s["cache"]
    page, d, kv = case["page"], case["dim"], case["kv"]
    group = case["heads"] // kv
    q, starts = s["q"], s["starts"].long()
    tokens, requests = q.shape[0], starts.numel() - 1
    pos = torch.arange(s["longest"], device=q.device)
    at = s["table"][:, pos // page].long().clamp(min=0)
    k = c["keys"][at, :, pos % page][..., :d].float() * c["key_scales"][at][..., None]
    v = c["values"].transpose(2, 3)[at, :, pos % page][..., :d].float()
    v = v * c["value_scales"][at][..., None]
    step = torch.arange(s["most"], device=q.device)
    t = starts[:-1, None] + step
    real = t < starts[1:, None]
    t = t.clamp(max=tokens - 1)
    sees = torch.where(real, s["positions"][t].long() + 1, 0)  # keys of each query
    rows = q[t].float().reshape(requests, -1, kv, group, d).permute(0, 2, 1, 3, 4)
    score = torch.matmul(rows.reshape(requests, kv, -1, d), k.permute(0, 2, 3, 1))
    score = score.reshape(requests, kv, -1, group, pos.numel()) * (1.0 / math.sqrt(d))
    mask = pos < sees[:, :, None]
    score = score.masked_fill_(~mask[:, None, :, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.reshape(requests, kv, -1, pos.numel()), v.permute(0, 2, 1, 3))
    o = o.reshape(requests, kv, -1, group, d)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    o = o.permute(0, 2, 1, 3, 4).reshape(requests, -1, case["heads"], d)
    n = torch.arange(tokens, device=q.device)
    r = torch.searchsorted(starts[1:].contiguous(), n, right=True).clamp(max=requests - 1)
    return o[r, n - starts[r]].to(q.dtype)


# ------------------------------------------------------------------- the definition, in 64 bits
def _exact_scale(a):
    """fl32(a / 127) as a 64-bit number; 0 where it is subnormal."""
    s = (a.double() / 127.0).float().double()
    return torch.where(s < _TINY, 0.0, s)


def _exact_held(x, s):
    """rint(fl32(x * fl32(1 / s))) as 64-bit numbers."""
    inv = torch.where(s > 0, (1.0 / s.clamp(min=_TINY)).float().double(), 0.0)
    return torch.round((x.double() * inv).float().double())


def exact(case, seed):
    global own
    kind = case["kind"]
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if kind == "tables":
        return None
    if kind == "linear":
        k = s["x"].shape[1]
        scale = _exact_scale(s["x"].double().abs().max(dim=1).values)
        x8 = _exact_held(s["x"], scale[:, None])
        y = x8 @ s["weight"][:, :k].double().t()
        return y * scale[:, None] * s["scales"].double()[None] + s["bias"].double()[None]
    page, d, c = case["page"], case["dim"], s["cache"]
    if kind == "append":
        out = {}
        slots = s["slots"].tolist()
        touched = {}
        for i, slot in enumerate(slots):
            touched.setdefault(slot // page, []).append(i)
        for name in ("k", "v"):
            if name == "k":
                held, scales = c["keys"][..., :d].double(), c["key_scales"].double()
            else:
                held = c["values"][:, :, :d].transpose(2, 3).double()
                scales = c["value_scales"].double()
            held, scales = held.contiguous(), scales.clone()
            for p, who in touched.items():
                off = torch.tensor([slots[i] % page for i in who], device="cuda")
                x = s[name][who[0]:who[-1] + 1].double()  # a page's tokens are neighbours
                before = torch.zeros_like(scales[p]) if slots[who[0]] % page == 0 else scales[p]
                after = torch.maximum(before, _exact_scale(x.abs().amax(dim=(0, 2))))
                ratio = (before / after).float().double()
                held[p] = torch.round((held[p] * ratio[:, None, None]).float().double())
                held[p][:, off] = _exact_held(x, after[None, :, None]).transpose(0, 1)
                scales[p] = after
            at, off = s["back"].long() // page, s["back"].long() % page
            out[name] = held[at, :, off] * scales[at].unsqueeze(2)
        return out
    starts, table = s["starts"].tolist(), s["table"]
    group = case["heads"] // case["kv"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for r in range(len(starts) - 1):
        a, b = starts[r], starts[r + 1]
        if a == b:
            continue
        last = s["positions"][a:b].long()
        length = int(last[-1]) + 1
        pages = table[r, :_pages(length, page)].long()
        for h in range(case["kv"]):
            k = c["keys"][pages, h].double() * c["key_scales"][pages, h].double()[:, None, None]
            v = c["values"][pages, h].double() * c["value_scales"][pages, h].double()[:, None, None]
            k = k.reshape(-1, k.shape[-1])[:length, :d]
            v = v.transpose(1, 2).reshape(-1, v.shape[1])[:length, :d]
            for e in range(h * group, (h + 1) * group):
                z = (s["q"][a:b, e].double() @ k.t()) / math.sqrt(d)
                z[torch.arange(length, device="cuda")[None] > last[:, None]] = -math.inf
                out[a:b, e] = torch.softmax(z, dim=1) @ v
    return out

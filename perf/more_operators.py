"""Performance cases of the rest of a decoder's step in 8 bits, through the public entry points.

Each kind of case is one piece of work that a program that serves a model has it do around the
layers and the attention of perf/operators.py:

  norm    NnClGlob.NormInt8: the residual's addition, the root-mean-square norm of the sum and
          its rows in 8 bits with a scale for each, as the next layer's product takes them
  layer   NnClGlob.MatmulInt8 and LinearInt8 with their epilogues: bias, activation, the
          product of a gate and its activation, and the residual, in the product's own launch
  sample  NnClGlob.Sample: a token for each row of logits, from temperature, min-p, top-k and
          top-p and one given random number a row, and the probability that it had

The 8-bit rule is that of the 8-bit operators: a scale is s = fl(a / 127) of the largest magnitude
a of a row, 0 where that is subnormal and NaN where a value is not finite; a value x is held as
rint(fl(x * fl(1 / s))) (half to even). The norm's sum of squares and its root are taken in 64
bits and rounded once: r = fl(1 / sqrt(mean(s^2) + eps)), y = fl(fl(s * r) * w).
"""
import math

import torch

own = False

_TINY = 2.0 ** -126
_EPS = 2.0 ** -20
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
        # one token between two layers: latency
        {"name": "norm_token", "kind": "norm", "rows": 1, "cols": 4096, "type": "bfloat16"},
        # no size a multiple of any tile, rows of odd length
        {"name": "norm_ragged", "kind": "norm", "rows": 1000, "cols": 777, "type": "float32"},
        # the prompts of a batch: bound by memory
        {"name": "norm_prompt", "kind": "norm", "rows": 8192, "cols": 4096, "type": "bfloat16"},
        # one token through a gated layer: bound by reading its two weights
        {"name": "gate_token", "kind": "layer", "rows": 1, "fin": 4096, "fout": 11008,
         "type": "bfloat16", "act": "silu", "gated": True, "residual": False, "held": False},
        # a small serving batch through the layer that closes a block
        {"name": "close_batch", "kind": "layer", "rows": 24, "fin": 4096, "fout": 2048,
         "type": "float32", "act": "none", "gated": False, "residual": True, "held": False},
        # no dimension a multiple of any tile
        {"name": "gelu_ragged", "kind": "layer", "rows": 1000, "fin": 777, "fout": 3000,
         "type": "float32", "act": "gelu", "gated": False, "residual": False, "held": True},
        # the prompts of a batch through the gated layer, rows as the norm leaves them (the
        # largest product)
        {"name": "gate_prompt", "kind": "layer", "rows": 4096, "fin": 4096, "fout": 11008,
         "type": "bfloat16", "act": "silu", "gated": True, "residual": False, "held": True},
        # one request's next token (the smallest sampling)
        {"name": "sample_token", "kind": "sample", "rows": 1, "vocab": 32000, "type": "float32",
         "temperature": 0.8, "topK": 50, "topP": 0.95, "minP": 0.0, "mixed": False,
         "masked": 0.0},
        # one request over a large vocabulary, the nucleus alone: every weight counts
        {"name": "sample_wide", "kind": "sample", "rows": 1, "vocab": 131072, "type": "bfloat16",
         "temperature": 1.0, "topK": 0, "topP": 0.9, "minP": 0.0, "mixed": False, "masked": 0.0},
        # a batch whose requests each ask for something else, greedy ones among them, under a
        # grammar that allows some of the tokens; an odd vocabulary
        {"name": "sample_mixed", "kind": "sample", "rows": 33, "vocab": 50001, "type": "bfloat16",
         "temperature": 1.0, "topK": 0, "topP": 1.0, "minP": 0.0, "mixed": True, "masked": 0.3},
        # a decoding step of a large batch
        {"name": "sample_batch", "kind": "sample", "rows": 64, "vocab": 131072, "type": "float32",
         "temperature": 0.7, "topK": 0, "topP": 0.95, "minP": 0.02, "mixed": False, "masked": 0.0},
        # samples for training by reinforcement: no filter, many rows (the most logits)
        {"name": "sample_many", "kind": "sample", "rows": 512, "vocab": 65536, "type": "float32",
         "temperature": 1.0, "topK": 0, "topP": 1.0, "minP": 0.0, "mixed": False, "masked": 0.0},
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
    kind = rng.choice(["norm", "layer", "layer", "sample", "sample"])
    kind_type = rng.choice(["float32", "bfloat16"])
    if kind == "norm":
        rows, cols = _log_int(rng, 1, 8192), _size(rng, 64, 12000)
        return {"kind": kind, "rows": max(1, min(rows, (8192 * 4096) // (2 * cols))),
                "cols": cols, "type": kind_type}
    if kind == "layer":
        act = rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh"])
        gated = rng.random() < 0.4
        return {"kind": kind, "rows": _log_int(rng, 1, 4096), "fin": _size(rng, 64, 4096),
                "fout": _size(rng, 64, 11008), "type": kind_type, "act": act, "gated": gated,
                "residual": rng.random() < 0.5 or (act == "none" and not gated),
                "held": rng.random() < 0.5}
    rows, vocab = _log_int(rng, 1, 512), _size(rng, 1000, 200000)
    return {"kind": kind, "rows": max(1, min(rows, (1 << 24) // vocab)), "vocab": vocab,
            "type": kind_type, "temperature": rng.choice([0.0] + [1.0] * 2 +
                                                   [round(rng.uniform(0.3, 1.6), 2)] * 5),
            "topK": rng.choice([0, 0, _log_int(rng, 1, 3000)]),
            "topP": rng.choice([1.0, round(rng.uniform(0.4, 0.99), 2)]),
            "minP": rng.choice([0.0, 0.0, round(rng.uniform(0.01, 0.2), 2)]),
            "mixed": rng.random() < 0.3, "masked": rng.choice([0.0, 0.0, 0.5, 0.999])}


def work(case):
    size = 4 if case["type"] == "float32" else 2
    if case["kind"] == "norm":
        r, k = case["rows"], case["cols"]
        # x and residual read, the sum and the row in 8 bits written; the values it stands for
        return {"bytes": r * k * (3 * size + 1) + 4 * r + 4 * k, "flops": 8 * r * k}
    if case["kind"] == "layer":
        m, k, n = case["rows"], case["fin"], case["fout"]
        wide = 2 * n if case["gated"] else n
        read = m * k * (1 if case["held"] else size) + wide * k + 8 * wide
        return {"bytes": read + m * n * size * (2 if case["residual"] else 1),
                "flops": 2 * m * wide * k}
    return {"bytes": case["rows"] * (case["vocab"] * size + 28),
            "flops": 4 * case["rows"] * case["vocab"]}


# ------------------------------------------------------------------------------ inputs
def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _rand(g, *shape):
    return torch.rand(*shape, generator=g, device="cuda")


def _scale_of(a):
    s = a / torch.full_like(a, 127.0)
    s = torch.where(s < _TINY, torch.zeros_like(s), s)
    return torch.where(torch.isfinite(a), s, torch.full_like(s, math.nan))


def _held(x, s):
    return torch.round(x * torch.where(s > 0, torch.reciprocal(s), torch.zeros_like(s)))


def _rows8(x):
    """(values int8 [rows, columns rounded up to 16], scales) of float32 rows."""
    s = _scale_of(x.abs().amax(1))
    v = torch.zeros(x.shape[0], -(-x.shape[1] // 16) * 16, dtype=torch.int8, device=x.device)
    v[:, :x.shape[1]] = _held(x, s[:, None])
    return v, s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = {"case": case}
    dt = _TYPES[case["type"]]
    if case["kind"] == "norm":
        r, k = case["rows"], case["cols"]
        # a residual stream with a few large channels, and what a block adds to it
        big = torch.where(_rand(g, k) < 0.01, 20.0, 1.0)
        s["residual"] = (_randn(g, r, k) * big).to(dt)
        s["x"] = _randn(g, r, k).to(dt)
        s["weight"] = 1 + 0.3 * _randn(g, k)
        return s
    if case["kind"] == "layer":
        m, k, n = case["rows"], case["fin"], case["fout"]
        wide = 2 * n if case["gated"] else n
        x = _randn(g, m, k) * torch.where(_rand(g, k) < 0.01, 8.0, 1.0)
        s["weight"], s["scales"] = _rows8((_rand(g, wide, k) * 2 - 1) * (2 / math.sqrt(k)))
        s["bias"] = _randn(g, wide) * 0.1
        s["residual"] = _randn(g, m, n).to(dt) if case["residual"] else None
        if case["held"]:
            s["rows"], s["rowScales"] = _rows8(x)
        else:
            s["x"] = x.to(dt)
        return s
    r, v = case["rows"], case["vocab"]
    logits = 2 * _randn(g, r, v)
    # the tokens that the context makes likely
    likely = torch.randint(0, v, (r, 24), generator=g, device="cuda")
    logits.scatter_add_(1, likely, 3 + 9 * _rand(g, r, 24))
    if case["masked"]:
        logits.masked_fill_(_rand(g, r, v) < case["masked"], -math.inf)
        logits[:, v // 2] = 1.0  # (a grammar allows something)
    s["logits"] = logits.to(dt)
    s["uniforms"] = _rand(g, r)
    s.update({name: case[name] for name in ("temperature", "topK", "topP", "minP")})
    if case["mixed"]:  # parameters of each request, on the GPU
        def pick(values):
            at = torch.randint(0, len(values), (r,), generator=g, device="cuda")
            return torch.tensor(values, device="cuda")[at]
        s["temperature"] = pick([0.0, 0.6, 0.9, 1.0, 1.3])
        s["topK"] = pick([0, 0, 1, 40, 500]).to(torch.int32)
        s["topP"] = pick([1.0, 1.0, 0.9, 0.5])
        s["minP"] = pick([0.0, 0.0, 0.05, 0.1])
    return s


# ------------------------------------------------------------------------------ one pass
def run(s):
    case = s["case"]
    if not own:
        return {"norm": _norm, "layer": _layer, "sample": _sample}[case["kind"]](s)
    nncl = glob()
    if case["kind"] == "norm":
        values, scales, total = nncl.NormInt8(s["x"], s["weight"], residual=s["residual"],
                                              eps=_EPS)
        return {"y": values[:, :case["cols"]] * scales[:, None], "sum": total}
    if case["kind"] == "layer":
        act = None if case["act"] == "none" else case["act"]
        if case["held"]:
            return nncl.MatmulInt8(s["rows"], s["rowScales"], s["weight"], s["scales"], s["bias"],
                                   dtype=_TYPES[case["type"]], activation=act,
                                   gated=case["gated"], residual=s["residual"])
        return nncl.LinearInt8(s["x"], s["weight"], s["scales"], s["bias"], activation=act,
                               gated=case["gated"], residual=s["residual"])
    tokens, probabilities = nncl.Sample(s["logits"], s["uniforms"], temperature=s["temperature"],
                                        topK=s["topK"], topP=s["topP"], minP=s["minP"])
    return {"tokens": tokens, "probabilities": probabilities}


def _norm(s):
    total = (s["x"].float() + s["residual"].float()).to(s["x"].dtype)
    x = total.float()
    mean = x.double().square().mean(1, keepdim=True)
    r = (1.0 / torch.sqrt(mean + _EPS)).float()
    y = x * r * s["weight"]
    scale = _scale_of(y.abs().amax(1))
    return {"y": _held(y, scale[:, None]) * scale[:, None], "sum": total}


def _activated(c, act):
    if act == "relu":
        return torch.where(c < 0, torch.zeros_like(c), c)
    if act == "silu":
        return c / (1 + torch.exp(-c))
    if act == "gelu":
        return 0.5 * c * (1 + torch.erf(c * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * c * (1 + torch.tanh(math.sqrt(2 / math.pi) * (c + 0.044715 * c * c * c)))
    return c


def _layer(s):
    case = s["case"]
    k, n = case["fin"], case["fout"]
    if case["held"]:
        held, scale = s["rows"][:, :k].float(), s["rowScales"]
    else:
        x = s["x"].float()
        scale = _scale_of(x.abs().amax(1))
        held = _held(x, scale[:, None])
    c = torch.matmul(held, s["weight"][:, :k].float().t())
    c = c * scale[:, None] * s["scales"] + s["bias"]
    y = _activated(c[:, :n], case["act"])
    if case["gated"]:
        y = y * c[:, n:]
    if case["residual"]:
        y = y + s["residual"].float()
    return y.to(_TYPES[case["type"]])


def _column(v, like):
    """A parameter of all rows, or of each, as a 64-bit column (numbers by way of 32 bits, as
    the rows' tensors hold them)."""
    if not isinstance(v, torch.Tensor):
        v = torch.full((like.shape[0],), v, dtype=torch.float32, device=like.device)
    return v.double()[:, None]


def _sample(s):
    logits, order = torch.sort(s["logits"].double(), dim=1, descending=True, stable=True)
    t, k, p, least = (_column(s[name], logits) for name in ("temperature", "topK", "topP", "minP"))
    w = torch.exp((logits - logits[:, :1]) / torch.where(t > 0, t, torch.ones_like(t)))
    w = torch.where(w >= least, w, torch.zeros_like(w))
    rank = torch.arange(w.shape[1], device=w.device)
    w = torch.where((k <= 0) | (rank < k), w, torch.zeros_like(w))
    upto = torch.cumsum(w, 1)
    before = torch.cat([torch.zeros_like(upto[:, :1]), upto[:, :-1]], 1)
    w = torch.where(before < p * upto[:, -1:], w, torch.zeros_like(w))
    upto = torch.cumsum(w, 1)
    at = (upto <= s["uniforms"].double()[:, None] * upto[:, -1:]).sum(1, keepdim=True)
    at = torch.minimum(at, (w > 0).sum(1, keepdim=True) - 1)
    at = torch.where(t > 0, at, torch.zeros_like(at))
    chance = torch.where(t > 0, w.gather(1, at) / upto[:, -1:], torch.ones_like(t))
    return {"tokens": order.gather(1, at)[:, 0].to(torch.int32),
            "probabilities": chance[:, 0].float()}


# ------------------------------------------------------------------- the definition, in 64 bits
def _exact_scale(a):
    """fl32(a / 127) as a 64-bit number; 0 where it is subnormal."""
    s = (a / 127.0).float().double()
    return torch.where(s < _TINY, 0.0, s)


def _exact_held(x, s):
    """rint(fl32(x * fl32(1 / s))) as 64-bit numbers."""
    inv = torch.where(s > 0, (1.0 / s.clamp(min=_TINY)).float().double(), 0.0)
    return torch.round((x * inv).float().double())


def _exact_chances(s):
    """The probability of each row's token, row by row: the tokens that a row may give, best first,
    are cut where the filters cut them, and the random number falls into one's share."""
    out = []
    for i, u in enumerate(s["uniforms"].tolist()):
        t, k, p, least = (float(v[i] if isinstance(v, torch.Tensor) else torch.tensor(v).float())
                          for v in (s[name] for name in ("temperature", "topK", "topP", "minP")))
        if t == 0:
            out.append(1.0)
            continue
        x = s["logits"][i].double()
        shares = ((x - x.max()) / t).exp()
        shares = shares[shares >= least].sort(descending=True).values
        if k > 0:
            shares = shares[:int(k)]
        enough = shares.cumsum(0) >= p * shares.sum()
        if bool(enough.any()):
            shares = shares[:int(enough.to(torch.uint8).argmax()) + 1]
        past = (shares.cumsum(0) > u * shares.sum()).to(torch.uint8)
        one = int(past.argmax()) if bool(past.any()) else int((shares > 0).sum()) - 1
        out.append(float(shares[one] / shares.sum()))
    return torch.tensor(out, dtype=torch.float64, device="cuda")


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "sample":
        return {"tokens": None, "probabilities": _exact_chances(s)}
    if case["kind"] == "norm":
        dt = s["x"].dtype
        total = (s["x"].double() + s["residual"].double())
        x = total.float().to(dt).double()
        root = (x.pow(2).sum(dim=1) / case["cols"] + _EPS).pow(-0.5).float().double()
        y = (x * root[:, None]).float().double() * s["weight"].double()
        y = y.float().double()
        scale = _exact_scale(y.abs().max(dim=1).values)
        return {"y": _exact_held(y, scale[:, None]) * scale[:, None], "sum": total}
    k, n = case["fin"], case["fout"]
    if case["held"]:
        held, scale = s["rows"][:, :k].double(), s["rowScales"].double()
    else:
        x = s["x"].double()
        scale = _exact_scale(x.abs().max(dim=1).values)
        held = _exact_held(x, scale[:, None])
    c = held @ s["weight"][:, :k].double().t()
    c = c * scale[:, None] * s["scales"].double()[None] + s["bias"].double()[None]
    g = c[:, :n]
    if case["act"] == "relu":
        g = g.clamp(min=0)
    elif case["act"] == "silu":
        g = g * torch.special.expit(g)
    elif case["act"] == "gelu":
        g = g * torch.special.ndtr(g)
    elif case["act"] == "gelu_tanh":
        g = g * torch.special.expit(2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g.pow(3)))
    if case["gated"]:
        g = g * c[:, n:]
    if case["residual"]:
        g = g + s["residual"].double()
    return g

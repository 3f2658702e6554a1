"""The attention block of a host that schedules a decoder itself, as cases that can be timed and compared.

Such a host has the products (`CudaBackend.had_q8`, `mv`, `mvq`) and calls three operators between them:

- `norm_rope`: q and k rows of a projection are normed per head, rotated to their positions, k and v go into the cache;
- `tree_attention`: the rows - one decoded token, a chain, or a tree of drafted tokens - attend to the cache and to their own ancestors,
  with the output gate of the 27B architecture where a case has it, and with the weight each slot received added up where it is asked for;
- `cache_evict`: a cache that has reached its budget keeps, per KV head, its latest slots and those with the largest weight.

Heads, head dimensions and rotated elements are the 27B architecture's (24 / 4 heads of 256, 64 rotated) or generic ones; activations are f32 over an f16
cache, as in the engine, or 16-bit throughout.  Values: N(0, 1) products in front of the norm; queries and keys behind it scaled so that scores spread
by a bit over two, which makes attention peaked without being one-hot; received weights with a heavy tail and slots that never received any (ties).
"""
import math

import torch

own = False

_ACT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_CACHE = {"f32": torch.float16, "f16": torch.float16, "bf16": torch.bfloat16}      # f32 activations go with an f16 cache


def listed():
    return [
        # ---- q / k norm, rotation, cache store -----------------------------------------------------------
        # a decoded token at the 27B shape: latency
        {"name": "place-1", "op": "place", "rows": 1, "heads": 24, "kv": 4, "dim": 256, "rot": 64, "layout": "half", "scaling": "none", "factor": 1.0, "at": 512, "norm": True, "type": "f32"},
        # a tree of drafts far into a stretched context, whole heads rotated in pairs of neighbours
        {"name": "place-29", "op": "place", "rows": 29, "heads": 32, "kv": 8, "dim": 128, "rot": 128, "layout": "interleaved", "scaling": "yarn", "factor": 4.0, "at": 120011, "norm": True, "type": "bf16"},
        # a long prompt at the 27B shape
        {"name": "place-4096", "op": "place", "rows": 4096, "heads": 24, "kv": 4, "dim": 256, "rot": 64, "layout": "half", "scaling": "none", "factor": 1.0, "at": 0, "norm": True, "type": "f32"},
        # ---- attention over the cache --------------------------------------------------------------------
        # a decoded token behind the benchmark's 512-token prompt
        {"name": "attend-1", "op": "attend", "rows": 1, "cached": 512, "heads": 24, "kv": 4, "dim": 256, "tree": False, "gate": True, "weights": False, "type": "f32"},
        # verification of a chain of three drafts, 16-bit, smaller heads
        {"name": "attend-4", "op": "attend", "rows": 4, "cached": 777, "heads": 32, "kv": 8, "dim": 128, "tree": False, "gate": False, "weights": False, "type": "f16"},
        # verification of a small tree at the reference's 2091-token prompt
        {"name": "attend-12", "op": "attend", "rows": 12, "cached": 2091, "heads": 24, "kv": 4, "dim": 256, "tree": True, "gate": True, "weights": False, "type": "f32"},
        # the same with the received weights added up, for a cache that will be cut
        {"name": "attend-9-weights", "op": "attend", "rows": 9, "cached": 8190, "heads": 24, "kv": 4, "dim": 256, "tree": True, "gate": True, "weights": True, "type": "f32"},
        # a decoded token over a very long context: the cache's bytes
        {"name": "attend-1-long", "op": "attend", "rows": 1, "cached": 131071, "heads": 24, "kv": 4, "dim": 256, "tree": False, "gate": False, "weights": False, "type": "bf16"},
        # a large tree over a long context: the largest product
        {"name": "attend-64", "op": "attend", "rows": 64, "cached": 30011, "heads": 24, "kv": 4, "dim": 256, "tree": True, "gate": True, "weights": False, "type": "f32"},
        # ---- eviction --------------------------------------------------------------------------------------
        # a small cache back to its budget
        {"name": "evict-1200", "op": "evict", "cached": 1200, "keep": 1024, "recent": 64, "kv": 8, "dim": 128, "type": "bf16"},
        # the engine's full context halved
        {"name": "evict-8192", "op": "evict", "cached": 8192, "keep": 4096, "recent": 257, "kv": 4, "dim": 256, "type": "f32"},
        # a very long context cut to a quarter
        {"name": "evict-131072", "op": "evict", "cached": 131072, "keep": 32768, "recent": 1024, "kv": 4, "dim": 256, "type": "f32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("place", "attend", "attend", "attend", "evict"))
    kind = rng.choice(("f32", "f32", "f16", "bf16"))
    kv = rng.choice((1, 2, 4, 8))
    dim = rng.choice((64, 80, 128, 256, 256))
    heads = kv * rng.choice((1, 2, 3, 4, 6, 8))
    if op == "place":
        scaling = rng.choice(("none", "linear", "ntk", "yarn"))
        return {"op": op, "rows": _log(rng, 1, min(4096, 4096 * 24 * 256 // ((heads + 2 * kv) * dim))), "heads": heads, "kv": kv, "dim": dim,
                "rot": rng.choice((dim, dim // 2, dim // 4)), "layout": rng.choice(("half", "interleaved")), "scaling": scaling,
                "factor": 1.0 if scaling == "none" else rng.choice((2.0, 4.0, 7.5)), "at": _log(rng, 1, 200000), "norm": rng.random() < 0.8, "type": kind}
    if op == "attend":
        rows = _log(rng, 1, 96)
        most = min(60000.0, 64 * 30011 * 24 * 256 / (rows * heads * dim))
        return {"op": op, "rows": rows, "cached": _log(rng, 1, max(2.0, most)), "heads": heads, "kv": kv, "dim": dim, "tree": rng.random() < 0.7, "gate": rng.random() < 0.5,
                "weights": rng.random() < 0.25, "type": kind}
    cached = _log(rng, 2, 131072)
    keep = max(1, min(int(cached * rng.uniform(0.1, 1.0)), 32768 * 4 * 256 // (kv * dim)))
    return {"op": op, "cached": cached, "keep": keep, "recent": int(keep * rng.uniform(0.0, 1.0)), "kv": kv, "dim": dim, "type": kind}


class _State:
    """What the caller keeps between calls."""


def _spare(n):
    return n + 37                                                # cache slots behind the last one used: they stay as they are


def _inputs(case, seed):
    """The tensors of a case, from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(1000003 * int(seed) + 17)
    rand = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    unit = lambda *shape: torch.rand(shape, generator=g, device="cuda")  # noqa: E731
    act, cache = _ACT[case["type"]], _CACHE[case["type"]]
    kv, dim = case["kv"], case["dim"]
    x = {}
    if case["op"] == "place":
        rows, heads, slots = case["rows"], case["heads"], _spare(case["rows"] + 5)
        x["q"], x["k"], x["v"] = rand(rows, heads, dim).to(act), rand(rows, kv, dim).to(act), rand(rows, kv, dim).to(act)
        x["q_norm"], x["k_norm"] = (0.5 + unit(dim), 0.5 + unit(dim)) if case["norm"] else (None, None)
        # a prompt's rows follow one another; a tree's rows share positions
        step = torch.arange(rows, device="cuda") if rows > 64 else (unit(rows) * (torch.arange(rows, device="cuda") + 1)).long()
        x["positions"] = (case["at"] + step).to(torch.int32)
        x["k_cache"], x["v_cache"] = rand(slots, kv, dim).to(cache), rand(slots, kv, dim).to(cache)
    elif case["op"] == "attend":
        rows, heads, slots = case["rows"], case["heads"], _spare(case["cached"] + case["rows"])
        x["q"] = (rand(rows, heads, dim) * (1.5 * math.sqrt(16 / math.sqrt(dim)))).to(act)
        x["k_cache"] = (rand(slots, kv, dim) * 1.5).to(cache)
        x["v_cache"] = rand(slots, kv, dim).to(cache)
        x["gate"] = rand(rows, heads, dim).to(act) if case["gate"] else None
        t = torch.arange(rows, device="cuda")
        x["parents"] = ((unit(rows) * (t + 1)).long() - 1).clamp(max=rows).minimum(t - 1).to(torch.int32) if case["tree"] else None
        x["weights"] = unit(kv, slots) if case["weights"] else None
    else:
        slots = _spare(case["cached"])
        w = torch.exp(2 * rand(kv, slots))
        x["weights"] = torch.where(unit(kv, slots) < 0.15, torch.zeros_like(w), w)
        x["k_cache"], x["v_cache"] = rand(slots, kv, dim).to(cache), rand(slots, kv, dim).to(cache)
    return x


def prepare(case, seed):
    s = _State()
    s.case = dict(case)
    s.__dict__.update(_inputs(case, seed))
    s.rope = None                                                # the table of frequencies, made once
    if case["op"] == "place":
        s.q_out = torch.zeros_like(s.q)
    elif case["op"] == "attend":
        s.out = torch.zeros_like(s.q)
    else:
        s.kept = torch.zeros(case["kv"], case["keep"], dtype=torch.int32, device="cuda")
    return s


_BASE, _ORIGINAL = 1e7, 32768                                    # rope base of the 27B architecture; context that a stretched one was trained with


def run(s):
    c = s.case
    if own:
        return _run_own(s, c)
    return {"place": _place, "attend": _attend, "evict": _evict}[c["op"]](s, c)


def _run_own(s, c):
    from irontimber_b200 import attention
    if c["op"] == "place":
        if s.rope is None:
            s.rope = attention.Rope(c["rot"], _BASE, c["layout"], c["scaling"], c["factor"], _ORIGINAL)
        attention.norm_rope(s.rope, s.q, s.k, s.v, s.q_out, s.k_cache, s.v_cache, 5, s.positions, q_norm=s.q_norm, k_norm=s.k_norm, eps=1e-6)
        return {"q": s.q_out, "k": s.k_cache, "v": s.v_cache}
    if c["op"] == "attend":
        attention.tree_attention(s.q, s.k_cache, s.v_cache, c["cached"], s.out, parents=s.parents, gate=s.gate, weights=s.weights)
        return {"out": s.out} if s.weights is None else {"out": s.out, "weights": s.weights}
    attention.cache_evict(s.k_cache, s.v_cache, s.weights, c["cached"], c["keep"], c["recent"], s.kept)
    return {"kept": s.kept, "k": s.k_cache, "v": s.v_cache, "weights": s.weights}


# ---- the plain forms ----------------------------------------------------------------------------------------------
def _frequencies(c):
    """Angle per position of every pair, in 64 bits, and the factor on sine and cosine."""
    n, f = c["rot"], c["factor"]
    i = torch.arange(n // 2, dtype=torch.float64, device="cuda")
    if c["scaling"] == "ntk":
        return torch.pow(_BASE * f ** (n / (n - 2)), -2 * i / n), 1.0
    w = torch.pow(torch.tensor(_BASE, dtype=torch.float64, device="cuda"), -2 * i / n)
    if c["scaling"] == "linear":
        return w / f, 1.0
    if c["scaling"] == "yarn":
        turn = [n * math.log(_ORIGINAL / (2 * math.pi * b)) / (2 * math.log(_BASE)) for b in (32.0, 1.0)]
        lo, hi = max(math.floor(turn[0]), 0), min(math.ceil(turn[1]), n - 1)
        r = ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return w * (1 - r) + w / f * r, 0.1 * math.log(f) + 1
    return w, 1.0


def _normed(x, w):
    x = x.float()
    return x if w is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w


def _rotated(x, c, cos, sin):
    n = c["rot"]
    a, b = (x[..., : n // 2], x[..., n // 2:n]) if c["layout"] == "half" else (x[..., 0:n:2], x[..., 1:n:2])
    y, z = a * cos - b * sin, a * sin + b * cos
    r = torch.cat((y, z), -1) if c["layout"] == "half" else torch.stack((y, z), -1).flatten(-2)
    return torch.cat((r, x[..., n:]), -1)


def _place(s, c):
    w, m = _frequencies(c)
    angle = s.positions.double()[:, None, None] * w
    cos, sin = (m * torch.cos(angle)).float(), (m * torch.sin(angle)).float()
    s.q_out.copy_(_rotated(_normed(s.q, s.q_norm), c, cos, sin))
    s.k_cache[5:5 + c["rows"]] = _rotated(_normed(s.k, s.k_norm), c, cos, sin).to(s.k_cache.dtype)
    s.v_cache[5:5 + c["rows"]] = s.v.to(s.v_cache.dtype)
    return {"q": s.q_out, "k": s.k_cache, "v": s.v_cache}


def _seen(parents, rows):
    """rows x rows: whether a row sees another, itself and its ancestors.  With A the matrix of parents, that is (1 - A)^-1."""
    t = torch.arange(rows, device="cuda")
    if parents is None:
        return t[:, None] >= t
    a = (parents[:, None] == t).double()
    one = torch.eye(rows, dtype=torch.float64, device="cuda")
    return torch.linalg.solve_triangular(one - a, one, upper=False, unitriangular=True) > 0.5


def _attend(s, c):
    rows, n, kv, dim = c["rows"], c["cached"], c["kv"], c["dim"]
    group = c["heads"] // kv
    k, v = (x[: n + rows].float().transpose(0, 1) for x in (s.k_cache, s.v_cache))            # kv, slots, dim
    q = s.q.float().view(rows, kv, group, dim).permute(1, 0, 2, 3).reshape(kv, rows * group, dim)
    score = torch.matmul(q, k.transpose(1, 2)) * dim ** -0.5
    seen = torch.cat((torch.ones(rows, n, dtype=torch.bool, device="cuda"), _seen(s.parents, rows)), 1)
    seen = seen.repeat_interleave(group, 0)
    score = score.masked_fill(~seen, -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = torch.matmul(p, v).view(kv, rows, group, dim).permute(1, 0, 2, 3).reshape(rows, c["heads"], dim)
    if s.gate is not None:
        o = o * torch.sigmoid(s.gate.float())
    s.out.copy_(o)
    if s.weights is None:
        return {"out": s.out}
    s.weights[:, : n + rows] += p.sum(1)
    return {"out": s.out, "weights": s.weights}


def _evict(s, c):
    n, keep, recent = c["cached"], c["keep"], c["recent"]
    order = torch.sort(s.weights[:, : n - recent], dim=1, descending=True, stable=True).indices[:, : keep - recent]
    last = torch.arange(n - recent, n, device="cuda").expand(c["kv"], recent)
    kept = torch.cat((torch.sort(order, dim=1).values, last), 1)                                # kv, keep
    s.kept.copy_(kept)
    s.weights[:, :keep] = torch.gather(s.weights, 1, kept)
    at = kept.t()[:, :, None].expand(keep, c["kv"], c["dim"])
    s.k_cache[:keep] = torch.gather(s.k_cache, 0, at)
    s.v_cache[:keep] = torch.gather(s.v_cache, 0, at)
    return {"kept": s.kept, "k": s.k_cache, "v": s.v_cache, "weights": s.weights}


# ---- what a pass cannot do without ---------------------------------------------------------------------------
def work(case):
    a, b = {"f32": 4, "f16": 2, "bf16": 2}[case["type"]], 2
    kv, dim = case["kv"], case["dim"]
    if case["op"] == "place":
        rows, heads = case["rows"], case["heads"]
        return {"bytes": rows * ((2 * heads + 2 * kv) * dim * a + 2 * kv * dim * b + 4), "flops": rows * (heads + kv) * (4 * dim * case["norm"] + 3 * case["rot"])}
    if case["op"] == "attend":
        rows, heads, n = case["rows"], case["heads"], case["cached"]
        return {"bytes": 2 * (n + rows) * kv * dim * b + rows * heads * dim * a * (3 if case["gate"] else 2) + (8 * kv * (n + rows) if case["weights"] else 0),
                "flops": 4 * rows * heads * dim * (n + (rows + 1) / 2)}
    n, keep = case["cached"], case["keep"]
    return {"bytes": 4 * kv * n + kv * keep * (4 * dim * b + 4 + 4), "flops": kv * n}


# ---- the definition in 64 bits --------------------------------------------------------------------------------
def exact(case, seed):
    x = _inputs(case, seed)
    return {"place": _place64, "attend": _attend64, "evict": _evict64}[case["op"]](x, case)


def _place64(x, c):
    rows, dim, rot, f = c["rows"], c["dim"], c["rot"], c["factor"]
    pairs = torch.zeros(rot // 2, 2, dtype=torch.long)
    freq = torch.zeros(rot // 2, dtype=torch.float64)
    m = 0.1 * math.log(f) + 1 if c["scaling"] == "yarn" else 1.0
    for i in range(rot // 2):
        pairs[i] = torch.tensor((i, i + rot // 2) if c["layout"] == "half" else (2 * i, 2 * i + 1))
        base = _BASE * f ** (rot / (rot - 2)) if c["scaling"] == "ntk" else _BASE
        freq[i] = base ** (-2.0 * i / rot)
        if c["scaling"] == "linear":
            freq[i] /= f
        if c["scaling"] == "yarn":
            # pairs that turn more than 32 times in the original context keep their frequency, those that turn less than once are stretched
            lo = max(math.floor(rot / 2 * math.log(_ORIGINAL / (32 * 2 * math.pi), _BASE)), 0)
            hi = min(math.ceil(rot / 2 * math.log(_ORIGINAL / (2 * math.pi), _BASE)), rot - 1)
            share = min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0)
            freq[i] = freq[i] * (1 - share) + freq[i] / f * share
    turn = torch.polar(torch.full((rows, rot // 2), m, dtype=torch.float64), x["positions"].cpu().double()[:, None] * freq).cuda()[:, None]
    pairs = pairs.cuda()

    def head(v, w):
        v = v.double()
        if w is not None:
            v = v / torch.sqrt((v * v).sum(-1, keepdim=True) / dim + 1e-6) * w.double()
        z = torch.complex(v[..., pairs[:, 0]], v[..., pairs[:, 1]]) * turn
        v = v.clone()
        v[..., pairs[:, 0]], v[..., pairs[:, 1]] = z.real, z.imag
        return v

    kc, vc = x["k_cache"].double(), x["v_cache"].double()
    kc[5:5 + rows], vc[5:5 + rows] = head(x["k"], x["k_norm"]), x["v"].double()
    return {"q": head(x["q"], x["q_norm"]), "k": kc, "v": vc}


def _attend64(x, c):
    rows, n, kv, dim, heads = c["rows"], c["cached"], c["kv"], c["dim"], c["heads"]
    parents = list(range(-1, rows - 1)) if x["parents"] is None else x["parents"].tolist()
    hidden = torch.ones(rows, n + rows, dtype=torch.bool)
    hidden[:, :n] = False
    for t in range(rows):
        j = t
        while j >= 0:
            hidden[t, n + j] = False
            j = parents[j]
    hidden = hidden.cuda()
    out = torch.zeros(rows, heads, dim, dtype=torch.float64, device="cuda")
    got = torch.zeros(kv, n + rows, dtype=torch.float64, device="cuda")
    for h in range(heads):
        g = h * kv // heads
        k, v = x["k_cache"][: n + rows, g].double(), x["v_cache"][: n + rows, g].double()
        z = x["q"][:, h].double() @ k.t() / math.sqrt(dim)
        z[hidden] = -math.inf
        p = torch.exp(z - torch.logsumexp(z, 1, keepdim=True))
        out[:, h] = p @ v
        got[g] += p.sum(0)
    if x["gate"] is not None:
        out = out / (1 + torch.exp(-x["gate"].double()))
    if x["weights"] is None:
        return {"out": out}
    weights = x["weights"].double()
    weights[:, : n + rows] += got
    return {"out": out, "weights": weights}


def _evict64(x, c):
    n, keep, recent = c["cached"], c["keep"], c["recent"]
    kc, vc, weights = (x[name].double() for name in ("k_cache", "v_cache", "weights"))
    kept = torch.zeros(c["kv"], keep, dtype=torch.int32, device="cuda")
    for g in range(c["kv"]):
        w = x["weights"][g, : n - recent].tolist()
        best = sorted(sorted(range(n - recent), key=lambda i: (-w[i], i))[: keep - recent])
        at = torch.tensor(best + list(range(n - recent, n)), dtype=torch.long, device="cuda")
        kept[g] = at
        for t, name in ((kc, "k_cache"), (vc, "v_cache")):
            t[:keep, g] = x[name][at, g].double()
        weights[g, :keep] = x["weights"][g, at].double()
    return {"kept": kept, "k": kc, "v": vc, "weights": weights}

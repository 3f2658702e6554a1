"""The attention block's operators against their definitions in 64 bits.

Tolerances, derived.  h = half a step relative to the value: f32 2^-24, f16 2^-11, bf16 2^-8 (h of the output's type; a cache's for the stored keys).
- norm_rope: the norm's factor is a sum of at most 256 squares (each lane 8 fused steps, 5 levels of a tree: 13 roundings, halved by the root), a division, a sum, a root, a
  division and two products: within 12 f32 half steps of x.  Angle: 2^-32 turns and a conversion to 24 bits of half a turn: pi 2^-24 + 2^-30 < 4 half steps, sine and cosine two more, times
  m one more, two products and a sum three more.  So 24 half steps of (|a| + |b|) of a pair cover both, and then the output type's own half step.
- tree_attention: a score is a sum of 256 products of f16 or bf16 values, exact one by one, added in f32 by at most 2 x 16 tensor-core steps of 16 (17 terms each, none below 2^-23 of the largest
  kept): |ds| <= 2^-17 sum |q||k| scale with room; splitting an f32 q leaves 2^-22 of its row's largest element.  exp2 adds 2^-22 relative, joining runs as much again.  p is then off by 2 |ds| (it and the
  sum), and the output by that times sum p|v|.  16-bit activations: p rounded: h sum p|v|.  The gate's sigmoid: 4 f32 half steps (__expf: 2 + |x| / 2^22 of them).  Then h of the output.
- weights: 2 |ds| + 2^-20 of what is received, and f32 half steps of the sum.
The worst case above grows with every term; all roundings being independent, the error's 2-norm for f32 stays below 1e-5 of the result's (the steps' 2^-23 times the square root of their number times
the scores' spread is below 2e-6).
- cache_evict: moves; equal.
"""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

ACT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CACHE = {"f32": torch.float16, "f16": torch.float16, "bf16": torch.bfloat16}
H32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


@pytest.fixture(scope="module")
def ops():
    from irontimber_b200 import attention, build
    build.build()
    torch.cuda.set_device(0)
    return attention


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def near(got, want, tol, what=""):
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}, worst {float((err / tol.clamp(min=1e-300)).max()):.3g} of the tolerance"


# ---- norm, rotation, store ---------------------------------------------------------------------------------------------
def norm_rope_64(x, w, pos, freq, m, layout, eps):
    """(result, what the error is measured by) in 64 bits."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()
    n = 2 * len(freq)
    if n == 0:
        return x, x.abs()
    f = torch.tensor(freq, dtype=torch.float64, device="cuda")
    ang = pos.double()[:, None, None] * f
    c, s = m * ang.cos(), m * ang.sin()
    ia, ib = (slice(0, n // 2), slice(n // 2, n)) if layout == "half" else (slice(0, n, 2), slice(1, n, 2))
    out, size = x.clone(), x.abs()
    a, b = x[..., ia], x[..., ib]
    out[..., ia], out[..., ib] = a * c - b * s, a * s + b * c
    size[..., ia] = size[..., ib] = (a.abs() + b.abs()) * m
    return out, size


@pytest.mark.parametrize("rows,heads,kv,dim,rot,layout,scaling,kind,norm", [
    (1, 24, 4, 256, 64, "half", "none", "f32", True), (29, 32, 8, 128, 128, "interleaved", "yarn", "bf16", True), (3, 5, 1, 64, 2, "half", "none", "f16", True), (257, 6, 2, 80, 20, "interleaved", "linear", "f32", False),
    (130, 1, 1, 8, 8, "half", "ntk", "f32", True), (2, 9, 3, 248, 246, "half", "yarn", "f16", False), (7, 16, 16, 256, 256, "interleaved", "none", "bf16", True), (5, 2, 2, 128, 0, "half", "none", "f32", True), (1, 1, 1, 16, 6, "interleaved", "linear", "f32", True)])
def test_norm_rope(ops, rows, heads, kv, dim, rot, layout, scaling, kind, norm):
    g = gen(rows * 1000 + dim)
    act, cache = ACT[kind], CACHE[kind]
    q, k, v = (3 * randn(g, rows, h, dim).to(act) for h in (heads, kv, kv))
    qn, kn = (randn(g, dim), randn(g, dim)) if norm else (None, None)
    kc, vc = randn(g, rows + 9, kv, dim).to(cache), randn(g, rows + 9, kv, dim).to(cache)
    kc0, vc0 = kc.clone(), vc.clone()
    rope = ops.Rope(rot, 1e7, layout, scaling, 1.0 if scaling == "none" else 4.0, 32768) if rot else None
    freq, m = rope.read() if rope else ([], 1.0)
    pos = torch.randint(0, 1 << 20, (rows,), generator=g, device="cuda", dtype=torch.int32)
    out = torch.empty_like(q)
    ops.norm_rope(rope, q, k, v, out, kc, vc, 4, pos, q_norm=qn, k_norm=kn, eps=1e-5)
    for got, x, w, h, what in ((out, q, qn, half_step(act), "q"), (kc[4:4 + rows], k, kn, half_step(cache), "k")):
        want, size = norm_rope_64(x, w, pos, freq, m, layout, 1e-5)
        near(got, want, 24 * H32 * size + h * want.abs() * 1.001 + (2.0 ** -25 if got.dtype == torch.float16 else 0), what)
    assert torch.equal(vc[4:4 + rows], v.to(cache))
    for now, was in ((kc, kc0), (vc, vc0)):
        assert torch.equal(now[:4], was[:4]) and torch.equal(now[4 + rows:], was[4 + rows:])


def test_norm_rope_positions(ops):
    """A number, a number plus a device value, far and negative positions; and the angle is exact however far."""
    g = gen(5)
    q = randn(g, 6, 2, 64)
    rope = ops.Rope(64, 1e4)
    freq, m = rope.read()
    out = torch.empty_like(q)
    base = torch.tensor([1000], dtype=torch.int32, device="cuda")
    for pos0, b in ((0, None), (7, None), (7, base), (-3, None), ((1 << 31) - 6, None), (-(1 << 31), None)):
        ops.norm_rope(rope, q, None, None, out, None, None, 0, pos0, base=b)
        pos = torch.arange(6, device="cuda", dtype=torch.float64) + pos0 + (1000 if b is not None else 0)
        # freq is read in 53 bits: at 2^31 its rounding alone is 2^-22 radians
        want, size = norm_rope_64(q, None, pos, freq, m, "half", 0.0)
        near(out, want, (24 * H32 + 2.0 ** -53 * abs(float(pos.abs().max()))) * size + H32 * want.abs(), f"pos0 {pos0}")


def test_norm_rope_in_place_strided_and_partial(ops):
    """A packed row of projections (q next to its gate, then k, then v), q in place; caches of [kv head][slot], both in one buffer; k and v alone."""
    g = gen(6)
    rows, heads, kv, dim = 11, 6, 2, 64
    row = randn(g, rows, heads * 2 * dim + 2 * kv * dim)
    row0 = row.clone()
    q = row[:, :heads * 2 * dim].view(rows, heads, 2 * dim)[..., :dim]
    k, v = (row[:, heads * 2 * dim + i * kv * dim:][:, :kv * dim].view(rows, kv, dim) for i in (0, 1))
    both = torch.zeros(kv, 20, 2 * dim, dtype=torch.float16, device="cuda")
    kc, vc = both[..., :dim].transpose(0, 1), both[..., dim:].transpose(0, 1)
    rope = ops.Rope(32, 1e4, "interleaved")
    w = randn(g, dim)
    ref_out, ref_k, ref_v = torch.empty(rows, heads, dim, device="cuda"), torch.zeros(20, kv, dim, dtype=torch.float16, device="cuda"), torch.zeros(20, kv, dim, dtype=torch.float16, device="cuda")
    ops.norm_rope(rope, q.contiguous(), k.contiguous(), v.contiguous(), ref_out, ref_k, ref_v, 9, 3, q_norm=w, k_norm=w)
    ops.norm_rope(rope, None, k, v, None, kc, vc, 9, 3, k_norm=w)
    assert torch.equal(kc, ref_k) and torch.equal(vc, ref_v)
    both.zero_()
    ops.norm_rope(rope, q, k, v, q, kc, vc, 9, 3, q_norm=w, k_norm=w)
    assert torch.equal(q, ref_out) and torch.equal(kc, ref_k) and torch.equal(vc, ref_v)
    gates = row[:, :heads * 2 * dim].view(rows, heads, 2 * dim)[..., dim:]
    assert torch.equal(gates, row0[:, :heads * 2 * dim].view(rows, heads, 2 * dim)[..., dim:]) and torch.equal(row[:, heads * 2 * dim:], row0[:, heads * 2 * dim:])


def test_norm_rope_rows_outside_the_cache_are_not_stored(ops):
    g = gen(7)
    k = randn(g, 5, 1, 8)
    for add in (-3, 0, 4, 100, -100):
        kc, vc = torch.zeros(6, 1, 8, dtype=torch.float16, device="cuda"), torch.zeros(6, 1, 8, dtype=torch.float16, device="cuda")
        ops.norm_rope(None, None, k, k, None, kc, vc, 1, 0, base=torch.tensor([add], dtype=torch.int32, device="cuda"))
        want = torch.zeros_like(kc)
        for t in range(5):
            if 0 <= 1 + add + t < 6:
                want[1 + add + t] = k[t].half()
        assert torch.equal(kc, want) and torch.equal(vc, want)


def test_norm_rope_of_nothing_zeros_and_infinities(ops):
    out = torch.full((2, 1, 64), 7.0, device="cuda")
    ops.norm_rope(None, torch.zeros(0, 1, 64, device="cuda"), None, None, out[:0], None, None, 0, 0)
    q = torch.zeros(2, 1, 64, device="cuda"); q[1, 0, 5] = math.inf
    w = torch.ones(64, device="cuda")
    ops.norm_rope(ops.Rope(64), q, None, None, out, None, None, 0, 3, q_norm=w, eps=1e-6)
    assert torch.equal(out[0], torch.zeros_like(out[0])) and out[1].isnan().any()


# ---- attention -----------------------------------------------------------------------------------------------------------
def seen_rows(parents, rows):
    """rows x rows, by walking up."""
    see = torch.zeros(rows, rows, dtype=torch.bool)
    for t in range(rows):
        j = t
        while j >= 0:
            see[t, j] = True
            nxt = j - 1 if parents is None else parents[j]
            j = nxt if 0 <= nxt < j else -1
    return see.cuda()


def tree_64(q, kc, vc, cached, parents, gate, scale, dtype):
    """(out, its tolerance, received, its tolerance) in 64 bits; kc, vc as the caller holds them.  Masked slots are left out of every sum."""
    rows, heads, dim = q.shape
    kv, n = kc.shape[1], cached + rows
    see = torch.cat((torch.ones(rows, cached, dtype=torch.bool, device="cuda"), seen_rows(parents, rows)), 1)
    scale = scale or dim ** -0.5
    out, tol = torch.zeros(rows, heads, dim, dtype=torch.float64, device="cuda"), torch.zeros(rows, heads, dim, dtype=torch.float64, device="cuda")
    got, gtol = torch.zeros(kv, n, dtype=torch.float64, device="cuda"), torch.zeros(kv, n, dtype=torch.float64, device="cuda")
    kc, vc = kc[:n].double(), vc[:n].double()
    rounding = 0.0 if dtype == torch.float32 else half_step(dtype)
    for h in range(heads):
        k, v = kc[:, h * kv // heads], vc[:, h * kv // heads]
        for t0 in range(0, rows, 16):
            rs = slice(t0, min(rows, t0 + 16))
            m = see[rs]
            s = torch.where(m, q[rs, h].double() @ torch.nan_to_num(k, 0, 0, 0).t() * scale if not torch.isfinite(k).all() else q[rs, h].double() @ k.t() * scale, -math.inf)
            ds = 2.0 ** -17 * abs(scale) * (q[rs, h].double().abs() @ torch.nan_to_num(k, 0, 0, 0).abs().t()).masked_fill(~m, 0).amax(-1, keepdim=True) + 2.0 ** -21
            p = torch.softmax(s, -1)
            vv = torch.nan_to_num(v, 0, 0, 0) if not torch.isfinite(v).all() else v
            out[rs, h] = p @ vv
            tol[rs, h] = (2 * ds + rounding) * (p @ vv.abs())
            got[h * kv // heads] += p.sum(0)
            gtol[h * kv // heads] += ((2 * ds + 2.0 ** -20) * p).sum(0)
    if gate is not None:
        z = 1 / (1 + torch.exp(-gate.double()))
        out, tol = out * z, tol * z + (out * z).abs() * H32 * (8 + gate.double().abs())
    return out, tol + out.abs() * (half_step(dtype) * 1.001 + 2 * H32) + (2.0 ** -25 if dtype == torch.float16 else 1e-38), got, gtol


def random_parents(rows, seed):
    r = torch.Generator().manual_seed(seed)
    return [int(torch.randint(-1, t, (1,), generator=r)) if t else -1 for t in range(rows)]


def make(kind, rows, cached, heads, kv, dim, seed, spare=13):
    g = gen(seed)
    act, cache = ACT[kind], CACHE[kind]
    q = (1.5 * (16 / math.sqrt(dim)) ** 0.5 * randn(g, rows, heads, dim)).to(act)
    kc, vc = (1.5 * randn(g, cached + rows + spare, kv, dim)).to(cache), randn(g, cached + rows + spare, kv, dim).to(cache)
    return q, kc, vc, g


CASES = [
    # rows, cached, heads, kv, dim, tree, gate, kind: tokens, chains and trees; product rows on either side of 16, 32, 64; slots on either side of a tile
    (1, 0, 1, 1, 64, False, False, "f32"), (1, 0, 6, 1, 256, False, True, "f16"), (1, 63, 24, 4, 256, False, True, "f32"), (1, 64, 24, 4, 256, False, False, "bf16"), (1, 512, 24, 4, 256, False, True, "f32"),
    (1, 5000, 16, 16, 128, False, False, "f16"), (2, 62, 8, 1, 64, False, False, "f32"), (2, 63, 16, 2, 128, True, True, "bf16"), (3, 777, 6, 1, 80, True, False, "f32"), (4, 777, 32, 8, 128, False, False, "f16"),
    (5, 1000, 12, 2, 8, True, True, "f32"), (6, 129, 6, 1, 248, True, False, "bf16"), (11, 200, 6, 1, 256, True, True, "f32"), (12, 2091, 24, 4, 256, True, True, "f32"), (16, 0, 4, 4, 128, True, False, "f16"),
    (33, 31, 3, 3, 64, True, False, "f32"), (64, 640, 24, 4, 256, True, True, "f32"), (65, 700, 8, 2, 128, False, True, "bf16"), (64, 2000, 16, 4, 256, True, False, "f16"), (100, 28, 40, 1, 64, True, False, "f32"),
    (256, 300, 4, 2, 128, True, False, "bf16"), (256, 0, 2, 1, 256, False, True, "f32"), (128, 5, 200, 200, 16, True, False, "f16"), (1, 40000, 8, 1, 256, False, False, "bf16")]


@pytest.mark.parametrize("rows,cached,heads,kv,dim,tree,gate,kind", CASES)
def test_tree_attention(ops, rows, cached, heads, kv, dim, tree, gate, kind):
    q, kc, vc, g = make(kind, rows, cached, heads, kv, dim, rows * 7 + cached)
    parents = random_parents(rows, cached + rows) if tree else None
    par = torch.tensor(parents, dtype=torch.int32, device="cuda") if tree else None
    z = randn(g, rows, heads, dim).to(ACT[kind]) if gate else None
    out, got = torch.empty_like(q), torch.rand(kv, cached + rows + 5, generator=g, device="cuda")
    was = got.clone()
    ops.tree_attention(q, kc, vc, cached, out, parents=par, gate=z)
    want, tol, rec, rtol = tree_64(q, kc, vc, cached, parents, z, 0, ACT[kind])
    near(out, want, tol, "out")
    if kind == "f32":
        assert float((out.double() - want).norm() / want.norm()) < 1e-5
    again = torch.empty_like(q)
    ops.tree_attention(q, kc, vc, cached, again, parents=par, gate=z, weights=got)
    assert torch.equal(again, out), "the weights change nothing"
    n = cached + rows
    near(got[:, :n], was[:, :n].double() + rec, rtol + 2 * H32 * (was[:, :n] + rec), "weights")
    assert torch.equal(got[:, n:], was[:, n:])


@pytest.mark.parametrize("rows,kind", [(1, "f32"), (20, "f16"), (12, "bf16"), (64, "f32")])
def test_what_masked_slots_hold_does_not_matter(ops, rows, kind):
    """NaN, infinities and the type's lowest value behind the last slot and in rows that others do not see; the row that does see one gets it."""
    heads, kv, dim, cached = 6, 2, 128, 100
    q, kc, vc, g = make(kind, rows, cached, heads, kv, dim, 3)
    parents = [-1] * rows                      # siblings: every row sees itself alone
    par = torch.tensor(parents, dtype=torch.int32, device="cuda")
    clean, dirty, got = torch.empty_like(q), torch.empty_like(q), torch.zeros(kv, cached + rows, device="cuda")
    ops.tree_attention(q, kc, vc, cached, clean, parents=par)
    for bad in (math.nan, math.inf, -math.inf, torch.finfo(kc.dtype).min):
        k2, v2 = kc.clone(), vc.clone()
        k2[cached + rows:], v2[cached + rows:] = bad, bad
        ops.tree_attention(q, k2, v2, cached, dirty, parents=par)
        assert torch.equal(dirty, clean), bad
        if rows == 1:
            continue
        k2[cached + 1], v2[cached + 1] = bad, bad
        k2[cached + 1, 0, 5:], v2[cached + rows - 1, 1, 7] = 0.5, bad
        ops.tree_attention(q, k2, v2, cached, dirty, parents=par, weights=got)
        others = [t for t in range(rows) if t not in (1, rows - 1)]
        assert torch.equal(dirty[others], clean[others]), bad
        if rows - 1 != 1:
            # the last row: only element 7 of kv head 1 is touched
            last, was = dirty[rows - 1].clone(), clean[rows - 1].clone()
            if not math.isfinite(bad):
                assert not torch.isfinite(last[heads // kv:, 7]).any()
            last[heads // kv:, 7] = was[heads // kv:, 7] = 0
            assert torch.equal(last, was)
        if math.isnan(bad):
            assert dirty[1].isnan().any()


def test_device_length(ops):
    """`length` stands in for the number of cached slots; what lies behind is not seen, be it NaN."""
    rows, heads, kv, dim, most = 5, 12, 2, 128, 900
    for kind in ("f32", "bf16"):
        q, kc, vc, g = make(kind, rows, most, heads, kv, dim, 4)
        parents = random_parents(rows, 2)
        par = torch.tensor(parents, dtype=torch.int32, device="cuda")
        for n in (0, 1, 63, 64, 500, 900, 5000, -7):
            k2, v2 = kc.clone(), vc.clone()
            real = min(max(n, 0), most)
            k2[real + rows:], v2[real + rows:] = math.nan, math.nan
            out, got = torch.empty_like(q), torch.zeros(kv, most + rows, device="cuda")
            ops.tree_attention(q, k2, v2, most, out, parents=par, length=torch.tensor([n], dtype=torch.int32, device="cuda"), weights=got)
            want, tol, rec, rtol = tree_64(q, k2, v2, real, parents, None, 0, ACT[kind])
            near(out, want, tol, f"{kind} {n}")
            near(got[:, :real + rows], rec, rtol + 2 * H32 * rec, f"weights {n}")
            assert not got[:, real + rows:].any()


@pytest.mark.parametrize("rows,heads,kv,dim", [(1, 8, 1, 128), (4, 4, 2, 64), (3, 9, 3, 128), (9, 6, 6, 40), (8, 16, 2, 256), (13, 5, 1, 64), (13, 5, 1, 72), (16, 16, 2, 128), (43, 3, 1, 128), (64, 8, 2, 256), (37, 7, 1, 256)])
@pytest.mark.parametrize("cached,most", [(0, 0), (120, 120), (129, 700), (2300, 2300), (9000, 9000), (700, 41000)])
def test_received_weights_of_few_and_many_rows(ops, rows, heads, kv, dim, cached, most):
    """Product rows and lengths on both sides of every choice; `length` below `cached`; NaN and infinities where nobody looks; what lies behind the last slot stays."""
    q, kc, vc, g = make("f32", rows, most, heads, kv, dim, rows + cached)
    kc[cached + rows:], vc[cached + rows:] = math.nan, math.inf
    parents = random_parents(rows, dim)
    par = torch.tensor(parents, dtype=torch.int32, device="cuda")
    was = torch.rand(kv, most + rows + 5, generator=g, device="cuda")
    out, got = torch.empty_like(q), was.clone()
    length = torch.tensor([cached], dtype=torch.int32, device="cuda") if cached != most else None
    ops.tree_attention(q, kc, vc, most, out, parents=par, length=length, weights=got)
    want, tol, rec, rtol = tree_64(q, kc, vc, cached, parents, None, 0, torch.float32)
    n = cached + rows
    near(out, want, tol, "out")
    near(got[:, :n], was[:, :n].double() + rec, rtol + 2 * H32 * (was[:, :n] + rec), "weights")
    assert torch.equal(got[:, n:], was[:, n:])
    more = was.clone()                      # a workspace for a longer cache, with what the last call left in it
    ws = torch.full((ops.tree_attention_workspace(rows, heads, kv, dim, 2 * most + 1, weights=True),), 255, dtype=torch.uint8, device="cuda")
    ops.tree_attention(q, kc, vc, most, out, parents=par, length=length, weights=more, workspace=ws)
    assert torch.equal(more, got)


@pytest.mark.parametrize("kind,rows,heads,kv,dim,cached", [("f32", 130, 64, 2, 16, 8200), ("f32", 66, 66, 1, 72, 15600), ("bf16", 256, 40, 2, 136, 6800), ("f16", 256, 32, 4, 64, 8300)])
def test_received_weights_whose_scores_are_not_kept(ops, kind, rows, heads, kv, dim, cached):
    """More than 256 MB of scores: K is read again."""
    assert 4 * rows * heads * cached > 1 << 28 and rows * heads // kv > max(64, dim)
    q, kc, vc, g = make(kind, rows, cached, heads, kv, dim, rows)
    parents = random_parents(rows, dim)
    par = torch.tensor(parents, dtype=torch.int32, device="cuda")
    was = torch.rand(kv, cached + rows + 5, generator=g, device="cuda")
    for real in (cached, 700):
        k2, v2 = kc.clone(), vc.clone()
        k2[real + rows:], v2[real + rows:] = math.nan, math.inf
        out, got = torch.empty_like(q), was.clone()
        ops.tree_attention(q, k2, v2, cached, out, parents=par, length=torch.tensor([real], dtype=torch.int32, device="cuda"), weights=got)
        want, tol, rec, rtol = tree_64(q, k2, v2, real, parents, None, 0, ACT[kind])
        near(out, want, tol, "out")
        near(got[:, :real + rows], was[:, :real + rows].double() + rec, rtol + 2 * H32 * (was[:, :real + rows] + rec), "weights")
        assert torch.equal(got[:, real + rows:], was[:, real + rows:])


def test_parents_that_are_not_smaller_rows_count_as_none(ops):
    q, kc, vc, g = make("f16", 6, 70, 4, 2, 64, 8)
    bad = [3, 1, 0, 2, 1 << 30, -9]           # forward, itself, fine, fine, far away, negative
    out, want = torch.empty_like(q), torch.empty_like(q)
    ops.tree_attention(q, kc, vc, 70, out, parents=torch.tensor(bad, dtype=torch.int32, device="cuda"))
    ops.tree_attention(q, kc, vc, 70, want, parents=torch.tensor([-1, -1, 0, 2, -1, -1], dtype=torch.int32, device="cuda"))
    assert torch.equal(out, want)


def test_a_chain_is_the_tree_of_its_parents_and_rows_are_those_of_single_calls(ops):
    rows, cached = 9, 200
    q, kc, vc, g = make("f32", rows, cached, 8, 2, 128, 9)
    chain, tree = torch.empty_like(q), torch.empty_like(q)
    ops.tree_attention(q, kc, vc, cached, chain)
    ops.tree_attention(q, kc, vc, cached, tree, parents=torch.arange(-1, rows - 1, dtype=torch.int32, device="cuda"))
    assert torch.equal(chain, tree)
    for t in range(rows):
        one = torch.empty_like(q[:1])
        ops.tree_attention(q[t:t + 1], kc, vc, cached + t, one)
        want, tol, _, _ = tree_64(q[t:t + 1], kc, vc, cached + t, None, None, 0, torch.float32)
        near(one, want, tol); near(chain[t:t + 1], want, tol)


def test_layouts_and_alignments(ops):
    """q next to its gate in one row, out in place, caches of [kv head][slot], k and v interleaved in one buffer, scales, offsets of 4 elements."""
    rows, cached, heads, kv, dim = 7, 333, 6, 2, 64
    for kind in ("f32", "f16"):
        q, kc, vc, g = make(kind, rows, cached, heads, kv, dim, 10)
        z = randn(g, rows, heads, dim).to(ACT[kind])
        want = torch.empty_like(q)
        ops.tree_attention(q, kc, vc, cached, want, gate=z, scale=0.21)
        row = torch.cat((torch.zeros(rows, 4, dtype=q.dtype, device="cuda"), torch.stack((q, z), 2).reshape(rows, -1)), 1)
        qs, zs = (row[:, 4:].view(rows, heads, 2, dim)[:, :, i] for i in (0, 1))
        both = torch.empty(kv, kc.shape[0], 2, dim + 8, dtype=kc.dtype, device="cuda").fill_(math.nan)
        k2, v2 = (both[:, :, i, :dim].transpose(0, 1) for i in (0, 1))
        k2.copy_(kc); v2.copy_(vc)
        out = torch.zeros(rows, heads, dim + 4, dtype=q.dtype, device="cuda")
        ops.tree_attention(qs, k2, v2, cached, out[..., 4:], gate=zs, scale=0.21)
        assert torch.equal(out[..., 4:], want) and not out[..., :4].any()
        ops.tree_attention(q, kc, vc, cached, q, gate=z, scale=0.21)              # out is q itself
        assert torch.equal(q, want)
    q, kc, vc, g = make("f32", 3, 100, 4, 2, 64, 11)
    for scale in (-0.3, 1e-30, 40.0):
        out = torch.empty_like(q)
        ops.tree_attention(q, kc, vc, 100, out, scale=scale)
        s, tol, _, _ = tree_64(q, kc, vc, 100, None, None, scale, torch.float32)
        near(out, s, tol.clamp(max=50), f"scale {scale}")


def test_values_of_any_size(ops):
    """Rows of q far above and below f16's range, scores that leave one slot, probabilities below f16's smallest step; a row of zeros."""
    q, kc, vc, g = make("f32", 4, 300, 4, 2, 128, 12)
    for size in (1e-20, 1e6, 1e30, 0.0):
        x = q * size
        x[1, :, 3] *= 1e-9
        for scale in (0.1 / max(size, 1e-20), 20 / max(size, 1e-20)):
            if scale > 3e38:
                continue
            out = torch.empty_like(q)
            ops.tree_attention(x, kc, vc, 300, out, scale=scale)
            want, tol, _, _ = tree_64(x, kc, vc, 300, None, None, scale, torch.float32)
            near(out, want, tol, f"{size} {scale}")


def test_offsets_beyond_32_bits(ops):
    """The last slots of a cache whose byte and element offsets pass 2^32."""
    free = torch.cuda.mem_get_info()[0]
    if free < 40 << 30:
        pytest.skip("needs 30 GB")
    kv, dim, slots = 2, 256, (1 << 23) + 300
    kc = torch.zeros(kv, slots, dim, dtype=torch.float16, device="cuda")
    vc = torch.zeros(kv, slots, dim, dtype=torch.float16, device="cuda")
    g = gen(13)
    n, rows = slots - 20, 3
    tail = 1000
    kc[:, n - tail:] = randn(g, kv, tail + 20, dim).half(); vc[:, n - tail:] = randn(g, kv, tail + 20, dim).half()
    q = 3 * randn(g, rows, 8, dim)
    out, got = torch.empty_like(q), torch.zeros(kv, n + rows, device="cuda")
    ops.tree_attention(q, kc.transpose(0, 1), vc.transpose(0, 1), n, out, weights=got)
    # the slots of zeros: score 0, value 0; they only add exp(0) each to the sum
    k, v = (x[:, n - tail:n + rows].double().repeat_interleave(4, 0) for x in (kc, vc))
    s = torch.einsum("thd,hjd->htj", q.double(), k) / 16
    hide = torch.arange(tail + rows, device="cuda")[None] > tail + torch.arange(rows, device="cuda")[:, None]
    s = s.masked_fill(hide, -math.inf)
    e = torch.exp(s)
    total = e.sum(-1) + (n - tail)
    want = torch.einsum("htj,hjd->thd", e, v) / total.t()[..., None]
    # a sum of 2^23 equal terms per run of some 113,000: f32 sums of a thread's 28,000 steps are within 28,000 half steps in the worst case, and all round alike
    size = torch.einsum("htj,hjd->thd", e, v.abs()) / total.t()[..., None]
    near(out, want, (2 * 2.0 ** -17 * 150 + 28000 * H32) * size + 1e-30)
    p = (e / total[..., None]).view(kv, 4, rows, -1).sum((1, 2))
    near(got[:, n - tail:], p, (2 * 2.0 ** -17 * 150 + 28000 * H32) * p)
    rope = ops.Rope(64)
    base = torch.tensor([slots - 3], dtype=torch.int32, device="cuda")
    x = randn(g, 3, kv, dim)
    ops.norm_rope(rope, None, x, x, None, kc.transpose(0, 1), vc.transpose(0, 1), 0, 0, base=base)
    assert torch.equal(vc[:, -3:].transpose(0, 1), x.half())


def test_the_same_call_gives_the_same_bits_on_any_stream_and_beside_others(ops):
    q, kc, vc, g = make("f32", 12, 3000, 24, 4, 256, 14)
    par = torch.tensor(random_parents(12, 5), dtype=torch.int32, device="cuda")
    want, w0 = torch.empty_like(q), torch.zeros(4, 3100, device="cuda")
    ops.tree_attention(q, kc, vc, 3000, want, parents=par, weights=w0)
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs, ws = [torch.empty_like(q) for _ in range(12)], [torch.zeros(4, 3100, device="cuda") for _ in range(12)]
    torch.cuda.synchronize()
    for i, (o, w) in enumerate(zip(outs, ws)):
        if i % 2:
            with torch.cuda.stream(streams[i % 3]):
                ops.tree_attention(q, kc, vc, 3000, o, parents=par, weights=w)
        else:
            ops.tree_attention(q, kc, vc, 3000, o, parents=par, weights=w, stream=streams[i % 3])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs) and all(torch.equal(w, w0) for w in ws)


def test_recorded_graphs(ops):
    """The whole block recorded once, replayed at growing lengths; two recorded graphs have workspaces of their own."""
    kind, rows, heads, kv, dim, most = "f32", 3, 12, 2, 128, 400
    g = gen(15)
    x = randn(g, rows, heads + 2 * kv, dim)
    kc, vc = torch.zeros(most + rows, kv, dim, dtype=torch.float16, device="cuda"), torch.zeros(most + rows, kv, dim, dtype=torch.float16, device="cuda")
    n = torch.tensor([0], dtype=torch.int32, device="cuda")
    rope = ops.Rope(64, 1e6, "half", "yarn", 2.0, 128)
    w = randn(g, dim)
    q, out = torch.empty(rows, heads, dim, device="cuda"), torch.empty(rows, heads, dim, device="cuda")

    def step(o):
        ops.norm_rope(rope, x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:], q, kc, vc, 0, 0, q_norm=w, k_norm=w, base=n)
        ops.tree_attention(q, kc, vc, most, o, length=n)

    step(out)
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], [torch.empty_like(out) for _ in range(2)]
    for gr, o in zip(graphs, outs):
        with torch.cuda.graph(gr):
            step(o)
    for i in range(20):
        x.copy_(randn(g, rows, heads + 2 * kv, dim))
        n.fill_(20 * i)
        step(out)
        kept = kc.clone()
        for gr in graphs:
            gr.replay()
        for gr in graphs:
            gr.replay()
        assert torch.equal(outs[0], out) and torch.equal(outs[1], out) and torch.equal(kc, kept)
        want, tol, _, _ = tree_64(q, kc, vc, 20 * i, None, None, 0, torch.float32)
        near(out, want, tol, f"at {20 * i}")


# ---- eviction --------------------------------------------------------------------------------------------------------------
def evict_plain(w, n, keep, recent):
    """Kept slots of a head: by weight, ties to the lower slot, NaN lowest."""
    w = [(-math.inf, 1) if x != x else (x + 0.0, 0) for x in w[:n - recent].tolist()]
    best = sorted(range(n - recent), key=lambda i: (-w[i][0], w[i][1], i))[:keep - recent]
    return sorted(best) + list(range(n - recent, n))


def fill(g, kv, n, what):
    w = torch.rand(kv, n, generator=g, device="cuda")
    if what == "ties":
        w = (w * 4).floor()
    elif what == "same":
        w = torch.full_like(w, 0.25)
    elif what == "close":
        w = 1 + (w * 50).floor() * 2.0 ** -23
    elif what == "odd":
        w = torch.randn(kv, n, generator=g, device="cuda")
        for i, x in enumerate((math.nan, math.inf, -math.inf, -0.0, 0.0, 1e-45, -math.nan)):
            w[:, i::17] = x
    elif what == "rising":
        w = torch.arange(n, device="cuda").float().repeat(kv, 1)
    elif what == "falling":
        w = -torch.arange(n, device="cuda").float().repeat(kv, 1)
    return w


@pytest.mark.parametrize("n,keep,recent,kv,dim,what", [
    (1, 1, 0, 1, 8, "rand"), (1, 0, 0, 2, 64, "rand"), (2, 1, 0, 2, 64, "ties"), (2, 1, 1, 2, 64, "rand"), (33, 32, 0, 1, 64, "odd"), (100, 100, 10, 2, 128, "rand"), (1200, 1024, 64, 8, 128, "rand"), (1200, 600, 600, 1, 80, "rand"),
    (2049, 2048, 7, 3, 256, "same"), (5000, 17, 3, 4, 256, "ties"), (8192, 4096, 0, 4, 256, "close"), (8193, 4096, 0, 4, 64, "odd"), (9000, 8999, 1, 2, 128, "falling"), (9000, 4500, 100, 2, 256, "rising"),
    (30000, 10000, 129, 4, 256, "rand"), (70001, 35000, 1000, 1, 64, "ties"), (70000, 69999, 0, 2, 128, "odd"),
    (4096, 2000, 5, 2, 64, "ties"), (4097, 2000, 5, 2, 64, "ties"), (200000, 150000, 77, 1, 64, "rising"), (262144, 200001, 3, 1, 16, "rand"), (300001, 100000, 64, 2, 64, "rand"), (524288, 524287, 1, 1, 8, "same")])
def test_cache_evict(ops, n, keep, recent, kv, dim, what):
    g = gen(n + keep)
    spare = 11
    kc, vc = randn(g, n + spare, kv, dim).half(), randn(g, n + spare, kv, dim).half()
    w = torch.cat((fill(g, kv, n, what), torch.rand(kv, spare, generator=g, device="cuda")), 1)
    k0, v0, w0 = kc.clone(), vc.clone(), w.clone()
    kept = torch.full((kv, keep + 3), -5, dtype=torch.int32, device="cuda")
    ops.cache_evict(kc, vc, w, n, keep, recent, kept[:, :keep])
    assert (kept[:, keep:] == -5).all()
    for h in range(kv):
        at = torch.tensor(evict_plain(w0[h].cpu(), n, keep, recent), dtype=torch.long, device="cuda")
        assert torch.equal(kept[h, :keep].long(), at), h
        for now, was in ((kc[:, h], k0[:, h]), (vc[:, h], v0[:, h])):
            assert torch.equal(now[:keep], was[at]) and torch.equal(now[keep:], was[keep:])
        assert torch.equal(w[h, :keep].view(torch.int32), w0[h, at].view(torch.int32)) and torch.equal(w[h, keep:].view(torch.int32), w0[h, keep:].view(torch.int32))


@pytest.mark.parametrize("n", [1100, 2500, 7000, 90000])
@pytest.mark.parametrize("together,equal", [(1, False), (127, False), (128, False), (129, False), (129, True), (600, False), (1024, False), (1024, True), (1025, False), (1025, True)])
def test_cache_evict_weights_close_together(ops, n, together, equal):
    """The smallest kept weight is one of `together` that agree in sign, exponent and six bits, at either end of them and in their middle; the others lie far on both sides."""
    g = gen(n + together)
    w = torch.cat((1.0 + torch.arange(together, device="cuda").float() * 2.0 ** -23 * (0 if equal else 117), torch.rand(n - together, generator=g, device="cuda") * 0.5))
    w[together:][torch.rand(n - together, generator=g, device="cuda") < 0.4] += 3.0
    w = w[torch.randperm(n, generator=g, device="cuda")]
    above = int((w >= 3.0).sum())
    for keep in {above + 1, above + (together + 1) // 2, above + together}:
        kc, now = torch.arange(n, device="cuda").half()[:, None, None].expand(n, 1, 8).contiguous(), w[None].clone()
        was, kept = kc.clone(), torch.empty(1, keep, dtype=torch.int32, device="cuda")
        ops.cache_evict(kc, kc.clone(), now, n, keep, 0, kept)
        at = torch.tensor(evict_plain(w.cpu(), n, keep, 0), dtype=torch.long, device="cuda")
        assert torch.equal(kept[0].long(), at), keep
        assert torch.equal(kc[:keep], was[at]) and torch.equal(now[0, :keep], w[at])


@pytest.mark.parametrize("n", [900, 6000, 90000])
@pytest.mark.parametrize("scale,shift", [(2.0 ** -40, 0.0), (2.0 ** 30, 0.0), (-1.0, 0.0), (2.0 ** -21, -2.0 ** -22), (2.0 ** 11, 0.0), (2.0 ** -149 * 900, 0.0)])
def test_cache_evict_weights_of_any_size(ops, n, scale, shift):
    """Weights far below one, far above, negative, around the ends of the range that the first histogram spreads over, and below the normal numbers."""
    g = gen(n)
    w = torch.rand(2, n, generator=g, device="cuda") * scale + shift
    for keep, recent in ((1, 0), (n // 3, 5), (n - 1, 0)):
        kc, now = randn(g, n, 2, 8).half(), w.clone()
        was, kept = kc.clone(), torch.empty(2, keep, dtype=torch.int32, device="cuda")
        ops.cache_evict(kc, kc.clone(), now, n, keep, recent, kept)
        for h in range(2):
            at = torch.tensor(evict_plain(w[h].cpu(), n, keep, recent), dtype=torch.long, device="cuda")
            assert torch.equal(kept[h].long(), at), (keep, h)
            assert torch.equal(kc[:keep, h], was[at, h]) and torch.equal(now[h, :keep].view(torch.int32), w[h, at].view(torch.int32))


def test_cache_evict_layouts(ops):
    """[kv head][slot] caches, k and v in one buffer, weights and kept with strides, without kept (its own workspace), bf16."""
    g = gen(1)
    n, keep, recent, kv, dim = 700, 300, 20, 3, 64
    both = randn(g, kv, n, 2, dim).bfloat16()
    kc, vc = (both[:, :, i].transpose(0, 1) for i in (0, 1))
    w = torch.rand(kv, n + 9, generator=g, device="cuda")
    k1, v1, w1 = kc.contiguous(), vc.contiguous(), w[:, :n].contiguous()
    kept = torch.empty(kv, keep, dtype=torch.int32, device="cuda")
    ops.cache_evict(k1, v1, w1, n, keep, recent, kept)
    ops.cache_evict(kc, vc, w, n, keep, recent)
    assert torch.equal(kc, k1) and torch.equal(vc, v1) and torch.equal(w[:, :n], w1)


# ---- together ----------------------------------------------------------------------------------------------------------------
def test_a_request_that_drafts_trees_and_cuts_its_cache(ops):
    """As a host uses the operators on a backend's stream, between the library's own products: projections from the arena, norm and rotation into the cache, a
    tree of drafts, the accepted path kept, the cache cut when it is full, the output projection.  Every step against 64 bits from the state before it."""
    import numpy as np
    from irontimber_b200.backend import CudaBackend
    e, heads, kv, dim, rows, budget = 1024, 4, 2, 64, 5, 48
    width = (heads * 2 + 2 * kv) * dim
    be = CudaBackend(0, arena_floats=1 << 17)
    try:
        rng = np.random.default_rng(3)
        w_in, w_out = be.mat_synth(1, width, e), be.mat_synth(2, e, 1024)
        q8, q8o = be.q8_rows(e, rows), be.q8_rows(1024, rows)
        be.set_signs(np.where(rng.integers(0, 2, e) == 1, 1.0, -1.0).astype(np.float32))
        X, P, O, Y = 0, 8192, 8192 + 8 * width, 8192 + 8 * width + 8 * 1024
        proj, o, y = be.view(P, rows, width), be.view(O, rows, 1024), be.view(Y, rows, e)
        with torch.cuda.stream(be.torch_stream):
            o.zero_()
            q = proj[:, :heads * 2 * dim].view(rows, heads, 2 * dim)[..., :dim]
            gate = proj[:, :heads * 2 * dim].view(rows, heads, 2 * dim)[..., dim:]
            k, v = (proj[:, (heads * 2 + i * kv) * dim:][:, :kv * dim].view(rows, kv, dim) for i in (0, 1))
            kc, vc = (torch.zeros(80, kv, dim, dtype=torch.float16, device="cuda") for _ in range(2))
            got = torch.zeros(kv, 80, device="cuda")
            norm = torch.rand(dim, device="cuda") + 0.5
            rope = ops.Rope(32, 1e6, "half", "yarn", 4.0, 64)
            freq, m = rope.read()
            parents = [-1, 0, 0, 1, 2]
            par = torch.tensor(parents, dtype=torch.int32, device="cuda")
            depth = torch.tensor([0, 1, 1, 2, 2], dtype=torch.int32, device="cuda")
            n, pos, cuts = 0, 0, 0
            attn = o[:, :heads * dim].view(rows, heads, dim)
            for turn in range(30):
                be.upload(X, rng.standard_normal((rows, e)).astype(np.float32))
                be.had_q8(e, rows, X, e, q8)
                be.mv(w_in, rows, q8, P, width)
                raw = proj.clone()
                positions = depth + pos
                be.norm_rope(rope, q, k, v, q, kc, vc, n, positions, q_norm=norm, k_norm=norm)
                rq = raw[:, :heads * 2 * dim].view(rows, heads, 2 * dim)
                want, size = norm_rope_64(rq[..., :dim], norm, positions, freq, m, "half", 1e-6)
                near(q, want, 24 * H32 * size + H32 * want.abs(), "q")
                before = got.clone()
                be.tree_attention(q, kc, vc, n, attn, parents=par, gate=gate, weights=got)
                want, tol, rec, rtol = tree_64(q, kc, vc, n, parents, rq[..., dim:], 0, torch.float32)
                near(attn, want, tol, "attention")
                near(got[:, :n + rows], before[:, :n + rows] + rec, rtol + 2 * H32 * (before[:, :n + rows] + rec), "weights")
                be.had_q8(1024, rows, O, 1024, q8o, signs=False)
                be.mv(w_out, rows, q8o, Y, e)
                assert torch.isfinite(y).all()
                path = [0, 2, 4] if turn % 2 else [0]                  # the accepted rows move next to one another
                for c in (kc, vc):
                    c[n:n + len(path)] = c[[n + j for j in path]]
                got[:, n:n + len(path)] = got[:, [n + j for j in path]]
                got[:, n + len(path):] = 0
                n += len(path); pos += len(path)
                if n > budget:
                    k0, w0 = kc.clone(), got.clone()
                    kept = torch.empty(kv, 32, dtype=torch.int32, device="cuda")
                    be.cache_evict(kc, vc, got, n, 32, 8, kept)
                    for h in range(kv):
                        at = evict_plain(w0[h].cpu(), n, 32, 8)
                        assert kept[h].tolist() == at and torch.equal(kc[:32, h], k0[at, h])
                    n, cuts = 32, cuts + 1
            assert cuts >= 1
            # the block recorded and replayed by the backend
            length = torch.tensor([n], dtype=torch.int32, device="cuda")
            be.tree_attention(q, kc, vc, n, attn, parents=par, length=length)
            want = attn.clone()
            be.capture_begin()
            be.tree_attention(q, kc, vc, n, attn, parents=par, length=length)
            gr = be.capture_end()
            attn.zero_()
            be.tree_attention(q[:1], kc, vc, n, attn[:1])               # another use of the same workspace in between
            be.graph_launch(gr)
            assert torch.equal(attn, want)
            be.graph_destroy(gr)
            torch.cuda.synchronize()
    finally:
        be.close()


def test_inputs_of_a_kernel_that_lets_others_begin_early(ops):
    """The library's products let the next kernel begin while they run; q, gate and parents that such a kernel (and one behind it) writes have to be complete when they are read."""
    import numpy as np
    from irontimber_b200.backend import CudaBackend
    e, heads, dim, cached = 5120, 2, 64, 128 * 40
    width = 2 * heads * dim
    be = CudaBackend(0, arena_floats=1 << 20)
    try:
        rng = np.random.default_rng(4)
        w_big, w = be.mat_synth(1, 60000, e), be.mat_synth(2, width, e)
        q8 = be.q8_rows(e, 4)
        be.set_signs(np.ones(e, np.float32))
        Y = 4 * e
        x, y = be.view(0, 4, e), be.view(Y, 4, width)
        q, z = y[:, :heads * dim].view(4, heads, dim), y[:, heads * dim:].view(4, heads, dim)
        with torch.cuda.stream(be.torch_stream):
            kc, vc = (torch.randn(cached + 4, 1, dim, device="cuda").half() for _ in range(2))
            out, want, got = torch.empty(4, heads, dim, device="cuda"), torch.empty(4, heads, dim, device="cuda"), torch.zeros(1, cached + 4, device="cuda")
            ref = torch.zeros(1, cached + 4, device="cuda")
            par = torch.tensor([-1, 0, 0, 1], dtype=torch.int32, device="cuda")
            for turn in range(40):
                y.fill_(float("nan"))
                be.upload(0, rng.standard_normal((4, e)).astype(np.float32))
                be.had_q8(e, 4, 0, e, q8)
                be.mv(w_big, 4, q8, Y + 4 * width, 60000)
                be.mv(w, 4, q8, Y, width)                            # q and gate, right in front of the call that reads them
                be.tree_attention(q, kc, vc, cached, out, parents=par, gate=z, scale=1e-3, weights=got)
                be.sync()
                be.tree_attention(q, kc, vc, cached, want, parents=par, gate=z, scale=1e-3, weights=ref)
                be.sync()
                assert torch.equal(out, want) and torch.equal(got, ref) and torch.isfinite(out).all()
    finally:
        be.close()


def test_first_refusals_on_a_device(ops):
    from irontimber_b200._lib import IronTimberError
    q, kc, vc, g = make("f32", 2, 100, 4, 2, 64, 1)
    out = torch.full_like(q, 3.0)
    with pytest.raises(IronTimberError, match="workspace"):
        ops.tree_attention(q, kc, vc, 100, out, workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    with pytest.raises(IronTimberError, match="cached slots"):
        ops.tree_attention(q, kc[:101], vc[:101], 100, out)
    assert (out == 3.0).all()
    ops.tree_attention(q[:0], kc, vc, 100, out[:0])                 # no rows

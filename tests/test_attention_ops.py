"""The attention block's operators without a GPU: frequencies of a rotation, workspaces, and every refusal (arguments are checked before the device is touched, so
a call that passes all checks fails here for want of one, and only then)."""
import ctypes as C
import math

import pytest

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def lib():
    from irontimber_b200 import _lib, build
    build.build()
    return _lib.load()


def freqs(n, base, scaling, factor, original, fast=32.0, slow=1.0):
    """The definitions, pair by pair, in Python's floats."""
    if scaling == "ntk":
        base = base * factor ** (n / (n - 2))
    out = []
    for i in range(n // 2):
        f = base ** (-2 * i / n)
        if scaling == "linear":
            f /= factor
        if scaling == "yarn":
            lo = max(math.floor(n * math.log(original / (fast * 2 * math.pi)) / (2 * math.log(base))), 0)
            hi = min(math.ceil(n * math.log(original / (slow * 2 * math.pi)) / (2 * math.log(base))), n - 1)
            r = min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0)
            f = f * (1 - r) + f / factor * r
        out.append(f)
    return out, 0.1 * math.log(factor) + 1 if scaling == "yarn" else 1.0


@pytest.mark.parametrize("n,base,scaling,factor,original", [
    (64, 1e7, "none", 1.0, 0), (2, 1e4, "none", 1.0, 0), (128, 1e4, "linear", 4.0, 0), (6, 5e5, "ntk", 2.5, 0), (256, 1e4, "yarn", 8.0, 4096), (64, 1e7, "yarn", 4.0, 32768),
    (20, 1e6, "yarn", 1.0, 1), (64, 1e4, "yarn", 40.0, 1 << 20)])
def test_frequencies_are_the_definitions(lib, n, base, scaling, factor, original):
    from irontimber_b200.attention import Rope
    for layout in ("half", "interleaved"):
        rope = Rope(n, base, layout, scaling, factor, original)
        got, m = rope.read()
        want, wm = freqs(n, base, scaling, factor, original)
        assert len(got) == n // 2 and all(abs(g - w) <= 8 * 2.0 ** -52 * w * (1 + math.log(base)) for g, w in zip(got, want))   # pow: the exponent's rounding times ln base
        assert abs(m - wm) < 1e-14
        rope.close(); rope.close()


@pytest.mark.parametrize("change", [dict(n_rot=0), dict(n_rot=63), dict(n_rot=258), dict(base=1.0), dict(base=math.inf), dict(base=math.nan), dict(scaling="linear", factor=0.5),
                                    dict(scaling="yarn", factor=math.nan, original=4096), dict(scaling="yarn", factor=2.0, original=0), dict(scaling="ntk", n_rot=2, factor=2.0),
                                    dict(scaling="yarn", factor=2.0, original=4096, beta_fast=1.0, beta_slow=2.0)])
def test_rope_refusals(lib, change):
    from irontimber_b200._lib import IronTimberError
    from irontimber_b200.attention import Rope
    with pytest.raises(IronTimberError) as e:
        Rope(**{"n_rot": 64, "base": 1e4, **change})
    assert e.value.code == -1
    for bad in (dict(layout="quarter"), dict(scaling="cubic")):
        with pytest.raises(ValueError):
            Rope(64, **bad)
    assert lib.it_rope_create(None, None) == -1 and lib.it_rope_read(None, None, None) == -1
    lib.it_rope_destroy(None)


A = 1 << 20          # stand-ins for device addresses, far enough apart; nothing here may be read


def norm_rope_args(**change):
    from irontimber_b200.attention import NormRopeArgs
    a = dict(type=0, cache_type=1, rows=5, heads=6, kv_heads=2, head_dim=64, q=A, q_row=384, q_head=64, k=2 * A, k_row=128, k_head=64, v=3 * A, v_row=128, v_head=64,
             q_out=4 * A, qo_row=384, qo_head=64, k_cache=5 * A, kc_slot=128, kc_head=64, v_cache=6 * A, vc_slot=128, vc_head=64, slots=64, slot0=3,
             pos0=7, eps=1e-6)
    a.update(change)
    return NormRopeArgs(**a)


def tree_args(**change):
    from irontimber_b200.attention import TreeAttentionArgs
    a = dict(type=0, cache_type=1, rows=5, heads=6, kv_heads=2, head_dim=64, q=A, q_row=384, q_head=64, out=4 * A, o_row=384, o_head=64, k_cache=5 * A, kc_slot=128, kc_head=64,
             v_cache=6 * A, vc_slot=128, vc_head=64, slots=300, cached=200, workspace=16 * A, workspace_bytes=1 << 28)
    a.update(change)
    return TreeAttentionArgs(**a)


def evict_args(**change):
    from irontimber_b200.attention import CacheEvictArgs
    a = dict(kv_heads=2, head_dim=64, k_cache=5 * A, kc_slot=128, kc_head=64, v_cache=6 * A, vc_slot=128, vc_head=64, weights=7 * A, w_head=300, kept=8 * A, kept_head=100,
             slots=300, n=200, keep=100, recent=10, workspace=16 * A, workspace_bytes=1 << 20)
    a.update(change)
    return CacheEvictArgs(**a)


def refused(lib, call, args, part):
    assert call(None, C.byref(args)) == -1, part
    assert part in lib.it_last_error().decode()


def test_calls_without_a_fault_get_as_far_as_the_device(lib):
    if torch.cuda.is_available():
        pytest.skip("addresses here are stand-ins")
    for call, args in ((lib.it_norm_rope, norm_rope_args()), (lib.it_tree_attention, tree_args()), (lib.it_cache_evict, evict_args())):
        assert call(None, C.byref(args)) == -2       # IT_ECUDA: no device
    assert lib.it_norm_rope(None, C.byref(norm_rope_args(q=None, q_out=None, heads=2))) == -2
    assert lib.it_norm_rope(None, C.byref(norm_rope_args(k=None, v=None, k_cache=None, v_cache=None))) == -2
    assert lib.it_norm_rope(None, C.byref(norm_rope_args(q_out=A))) == -2                                        # in place
    assert lib.it_tree_attention(None, C.byref(tree_args(out=A))) == -2
    assert lib.it_tree_attention(None, C.byref(tree_args(kc_slot=64, kc_head=300 * 64, vc_slot=64, vc_head=300 * 64))) == -2      # [kv head][slot][element]
    assert lib.it_tree_attention(None, C.byref(tree_args(kv_heads=1, kc_head=0, vc_head=0))) == -2                # an axis of one: its stride does not matter
    assert lib.it_cache_evict(None, C.byref(evict_args(k_cache=None))) == -2
    # a whole packed row of projections, q in place
    assert lib.it_norm_rope(None, C.byref(norm_rope_args(q_row=640, qo_row=640, q_out=A, k=A + 384 * 4, k_row=640, v=A + 512 * 4, v_row=640))) == -2


@pytest.mark.parametrize("change,part", [
    (dict(type=3), "types"), (dict(cache_type=2), "types"), (dict(type=2), "types"), (dict(type=1, cache_type=0), "types"), (dict(rows=-1), "rows"), (dict(head_dim=68), "head dimension"),
    (dict(head_dim=264), "head dimension"), (dict(head_dim=0), "head dimension"), (dict(kv_heads=4), "kv heads"), (dict(kv_heads=0), "kv heads"), (dict(q=None, k=None, v=None), "neither"), (dict(v=None), "come together"),
    (dict(q_out=None), "q_out"), (dict(q=A + 4), "multiples of 4"), (dict(q_head=62), "multiples of 4"), (dict(q_head=32), "multiples of 4"), (dict(q_row=320), "multiples of 4"), (dict(q_out=A, qo_head=128, qo_row=768), "overlaps q"),
    (dict(q_out=A + 64), "overlaps q"), (dict(q_out=2 * A), "overlaps k or v"), (dict(k_cache=None), "without caches"), (dict(k_cache=5 * A + 8), "16-byte"), (dict(kc_slot=132), "multiples of 8"), (dict(vc_head=60), "multiples of 8"),
    (dict(slot0=60), "rows at slots"), (dict(slot0=-1), "rows at slots"), (dict(slots=0), "16-byte"), (dict(eps=-1.0), "eps"), (dict(eps=math.nan), "eps"), (dict(positions=A + 2), "aligned to its type")])
def test_norm_rope_refusals(lib, change, part):
    refused(lib, lib.it_norm_rope, norm_rope_args(**change), part)


def test_norm_rope_refuses_more_rotated_elements_than_a_head_has(lib):
    from irontimber_b200.attention import Rope
    rope = Rope(128)
    refused(lib, lib.it_norm_rope, norm_rope_args(rope=rope.handle), "rotated")


@pytest.mark.parametrize("change,part", [
    (dict(type=3), "types"), (dict(type=1, cache_type=2), "types"), (dict(rows=257), "rows"), (dict(rows=-1), "rows"), (dict(head_dim=20), "head dimension"), (dict(heads=5), "kv heads"), (dict(cached=-1), "cached"), (dict(cached=1 << 30), "cached"),
    (dict(cached=296), "cached slots"), (dict(q=None), "null"), (dict(out=None), "null"), (dict(v_cache=None), "null"), (dict(q=A + 8), "multiples of 4"), (dict(gate=9 * A, g_row=384, g_head=30), "multiples of 4"),
    (dict(k_cache=5 * A + 4), "16-byte"), (dict(kc_slot=0), "16-byte"), (dict(kc_head=-64), "16-byte"), (dict(vc_slot=100), "16-byte"), (dict(weights=9 * A, w_head=204), "overlap"), (dict(scale=math.nan), "scale"), (dict(scale=math.inf), "scale"),
    (dict(out=A + 16), "overlaps q"), (dict(out=A, weights=9 * A, w_head=300), "overlaps q"), (dict(gate=4 * A, g_row=768, g_head=128), "overlaps gate"), (dict(parents=A + 1), "aligned to its type"), (dict(length=A + 2), "aligned to its type")])
def test_tree_attention_refusals(lib, change, part):
    refused(lib, lib.it_tree_attention, tree_args(**change), part)


@pytest.mark.parametrize("change,part", [
    (dict(kv_heads=0), "kv heads"), (dict(head_dim=12), "head dimension"), (dict(recent=101), "keep"), (dict(keep=201), "keep"), (dict(n=301), "keep"), (dict(recent=-1), "keep"), (dict(slots=1 << 21, n=(1 << 19) + 1), "keep"),
    (dict(weights=None), "weights"), (dict(w_head=199), "weights"), (dict(k_cache=5 * A + 8), "16-byte"), (dict(vc_slot=60), "16-byte"), (dict(kept_head=99), "kept"), (dict(workspace=None), "workspace"),
    (dict(workspace_bytes=800), "workspace"), (dict(workspace=A + 128), "workspace")])
def test_cache_evict_refusals(lib, change, part):
    refused(lib, lib.it_cache_evict, evict_args(**change), part)


def test_null_arguments(lib):
    n = C.c_size_t()
    for call in (lib.it_norm_rope, lib.it_tree_attention, lib.it_cache_evict):
        assert call(None, None) == -1
    for call in (lib.it_tree_attention_workspace, lib.it_cache_evict_workspace):
        assert call(None, C.byref(n)) == -1
    assert lib.it_tree_attention_workspace(C.byref(tree_args()), None) == -1


def test_workspace_goes_by_sizes_alone(lib):
    from irontimber_b200.attention import tree_attention_workspace
    n = C.c_size_t()
    assert lib.it_tree_attention_workspace(C.byref(tree_args(q=None, out=None, k_cache=None, v_cache=None, workspace=None)), C.byref(n)) == 0 and n.value > 0
    assert tree_attention_workspace(5, 6, 2, 64, 200) == n.value
    assert lib.it_tree_attention_workspace(C.byref(tree_args(rows=0)), C.byref(n)) == 0 and n.value == 0
    # runs of a cache are at most one wave of CTAs: never more than this, however long it is
    assert tree_attention_workspace(256, 24, 4, 256, (1 << 30) - 1) < 64 << 20 and tree_attention_workspace(1, 1, 1, 256, (1 << 30) - 1) < 4 << 20
    # scores for the received weights: 4 bytes a product row and slot, in whole tiles, up to 256 MB or while the product rows are at most 64 or the head dimension
    for rows, heads, kv, dim, cached, kept in ((1, 6, 1, 64, 1000, True), (65, 1, 1, 64, 1000, True), (64, 64, 64, 64, 100000, True), (65, 64, 64, 64, 100000, False), (128, 32, 32, 128, 50000, True), (129, 32, 32, 128, 50000, False),
                                                (65, 64, 64, 64, 16064, False), (65, 64, 64, 64, 16000, True), (256, 4, 4, 256, 100000, True)):
        plain, more = tree_attention_workspace(rows, heads, kv, dim, cached), tree_attention_workspace(rows, heads, kv, dim, cached, weights=True)
        assert more - plain == (4 * rows * heads * ((cached + rows + 127) // 128 * 128) if kept else 256 << 20)
        assert tree_attention_workspace(rows, heads, kv, dim, cached // 3, weights=True) <= more
    assert lib.it_cache_evict_workspace(C.byref(evict_args(workspace=None, weights=None)), C.byref(n)) == 0 and n.value >= 800
    assert lib.it_cache_evict_workspace(C.byref(evict_args(keep=0, recent=0)), C.byref(n)) == 0 and n.value == 0


def test_tensors_are_checked_before_the_library_sees_them(lib):
    from irontimber_b200 import attention
    q, kc = torch.zeros(3, 4, 64), torch.zeros(50, 2, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="not on a CUDA device"):
        attention.tree_attention(q, kc, kc.clone(), 10, torch.zeros_like(q), workspace=torch.zeros(1 << 22, dtype=torch.uint8))
    with pytest.raises(ValueError, match="out has the shape"):
        attention.tree_attention(q, kc, kc.clone(), 10, torch.zeros(3, 4, 32))
    with pytest.raises(TypeError, match="out is torch.float16"):
        attention.tree_attention(q, kc, kc.clone(), 10, torch.zeros(3, 4, 64, dtype=torch.float16))
    with pytest.raises(ValueError, match="not contiguous"):
        attention.tree_attention(torch.zeros(3, 4, 128)[..., ::2], kc, kc.clone(), 10, torch.zeros_like(q))
    with pytest.raises(TypeError, match="a cache is"):
        attention.tree_attention(q, kc.float(), kc.float(), 10, torch.zeros_like(q))
    with pytest.raises(ValueError, match="weights are"):
        attention.tree_attention(q, kc, kc.clone(), 10, torch.zeros_like(q), weights=torch.zeros(2, 12))
    with pytest.raises(ValueError, match="parents is"):
        attention.tree_attention(q, kc, kc.clone(), 10, torch.zeros_like(q), parents=torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError, match="kept is"):
        attention.cache_evict(kc, kc.clone(), torch.zeros(2, 50), 40, 20, 3, torch.zeros(2, 19, dtype=torch.int32))
    with pytest.raises(ValueError, match="k has the shape"):
        attention.norm_rope(None, q, torch.zeros(3, 1, 64), torch.zeros(3, 1, 64), torch.zeros_like(q), kc, kc.clone(), 0, 0)
    # another device than the CUDA ones is refused by the types of the pair first, when those do not fit
    from irontimber_b200._lib import IronTimberError
    with pytest.raises(IronTimberError, match="types"):
        attention.tree_attention(q.bfloat16(), kc, kc.clone(), 10, torch.zeros_like(q, dtype=torch.bfloat16))

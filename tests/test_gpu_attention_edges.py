"""The attention block's operators where a result could lose bits or pass on what it must not; tolerances as in test_gpu_attention_ops.py."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from tests.test_gpu_attention_ops import ACT, CACHE, H32, gen, half_step, make, near, ops, random_parents, randn, tree_64  # noqa: E402,F401


@pytest.mark.parametrize("kind,rows,cached,heads,kv,dim,spread", [
    ("bf16", 1, 5000, 24, 4, 256, 0.1), ("f16", 1, 5000, 24, 4, 256, 0.1), ("bf16", 1, 400, 8, 2, 128, 0.1), ("f16", 4, 777, 32, 8, 128, 0.3), ("bf16", 5, 3000, 12, 2, 64, 0.1), ("f16", 9, 2500, 16, 4, 256, 0.1),
    ("bf16", 16, 6000, 8, 2, 72, 0.1), ("f16", 64, 2000, 16, 4, 256, 0.1), ("bf16", 64, 2000, 16, 4, 256, 0.1), ("bf16", 64, 1900, 32, 8, 128, 0.1), ("f16", 256, 700, 4, 2, 128, 1.0), ("bf16", 40, 60, 6, 1, 256, 0.5)])
def test_results_of_16_bit_activations_are_rounded_once(ops, kind, rows, cached, heads, kv, dim, spread):
    """Scores near one another, so that thousands of slots make up a result.  An element x before its last rounding, d off the exact value w, rounds as w does or both lie within d of the border between
    the two: |out - w| <= |round(w) - w| + 2 d.  In the 2-norm d is 1e-5 of w (as for f32 activations) and what two halves leave of a p: h^2, and for f16 2^-25 of the 2^6 that p is at its row's largest,
    which over n slots of one size is below sqrt(n) 2^-31."""
    q, kc, vc, g = make(kind, rows, cached, heads, kv, dim, rows + dim)
    q = (q.float() * spread).to(q.dtype)
    parents = random_parents(rows, cached)
    out = torch.empty_like(q)
    ops.tree_attention(q, kc, vc, cached, out, parents=torch.tensor(parents, dtype=torch.int32, device="cuda"))
    want = tree_64(q, kc, vc, cached, parents, None, 0, ACT[kind])[0]
    once = float((want.to(q.dtype).double() - want).norm())
    left = 1e-5 + half_step(q.dtype) ** 2 + (math.sqrt(cached + rows) * 2.0 ** -31 if kind == "f16" else 0)
    assert float((out.double() - want).norm()) <= once + 2 * left * float(want.norm())


def test_workspaces_of_other_streams_are_not_used(ops):
    """Calls that allocate, on the current stream and on others in turn, behind work that keeps the current stream busy while its blocks are freed."""
    q, kc, vc, g = make("f32", 12, 3000, 24, 4, 256, 20)
    par = torch.tensor(random_parents(12, 5), dtype=torch.int32, device="cuda")
    want, w0 = torch.empty_like(q), torch.zeros(4, 3100, device="cuda")
    ops.tree_attention(q, kc, vc, 3000, want, parents=par, weights=w0)
    other = torch.cuda.Stream()
    a, b = torch.randn(4096, 4096, device="cuda"), torch.empty(4096, 4096, device="cuda")
    nbytes = ops.tree_attention_workspace(12, 24, 4, 256, 4095, weights=True)
    outs, ws = [torch.empty_like(q) for _ in range(24)], [torch.zeros(4, 3100, device="cuda") for _ in range(24)]
    torch.cuda.synchronize()
    for i, (o, w) in enumerate(zip(outs, ws)):
        for _ in range(3):
            torch.mm(a, a, out=b)
        torch.empty(nbytes, dtype=torch.uint8, device="cuda").fill_(255)                # freed with its write still queued
        for s in (other, other.cuda_stream) if i % 2 else (None,):
            ops.tree_attention(q, kc, vc, 3000, o, parents=par, weights=w, stream=s)
        if i % 2:
            with torch.cuda.stream(other):
                w.mul_(0.5)                                                            # two equal calls have added to it
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    assert all(torch.equal(w, w0) for w in ws)


@pytest.mark.parametrize("rows,heads,kv,dim,cached,real", [
    (4, 2, 2, 64, 100, 100), (20, 6, 2, 128, 100, 100), (64, 8, 2, 256, 2000, 2000), (7, 1, 1, 64, 30000, 30000), (12, 24, 4, 256, 2091, 1900), (130, 64, 2, 16, 8200, 8200), (130, 64, 2, 16, 8200, 700)])
def test_a_row_that_is_not_a_number_weighs_only_what_it_sees(ops, rows, heads, kv, dim, cached, real):
    """A NaN or infinite key of a tree row makes that row's weights NaN, for the slots that it sees.  Those of its siblings, which nobody but they see, are what they were: with the weights formed
    by their own launch, beside the joining, and in a second walk over the keys."""
    q, kc, vc, g = make("f32", rows, cached, heads, kv, dim, rows + real)
    parents = [-1] * rows
    par = torch.tensor(parents, dtype=torch.int32, device="cuda")
    length = None if real == cached else torch.tensor([real], dtype=torch.int32, device="cuda")
    out, clean = torch.empty_like(q), torch.zeros(kv, cached + rows, device="cuda")
    ops.tree_attention(q, kc, vc, cached, out, parents=par, weights=clean, length=length)
    others = [real + t for t in range(rows) if t != 1]
    for bad in (math.nan, math.inf):
        k2 = kc.clone()
        k2[real + 1] = bad
        got = torch.zeros_like(clean)
        ops.tree_attention(q, k2, vc, cached, out, parents=par, weights=got, length=length)
        assert torch.equal(got[:, others], clean[:, others])
        if math.isnan(bad):
            assert got[:, real + 1].isnan().all() and got[:, :real].isnan().all()
        assert not got[:, real + rows:].any()


@pytest.mark.parametrize("cached,rows", [(6900, 255), (2000, 9)])
def test_a_key_of_minus_infinity_gets_no_weight(ops, cached, rows):
    """Every row scores it -inf, in a whole tile and in one that reaches behind the cached slots; the product tile's rows behind the last are zeros, and 0 * inf is not a number."""
    heads, kv, dim = 40, 2, 136
    assert rows * heads // kv % 64 and (4 * rows * heads * cached > 1 << 28) == (rows == 255)
    q, kc, vc, g = make("bf16", rows, cached, heads, kv, dim, rows)
    q[..., 0] = q[..., 0].abs() + 0.5
    par = torch.tensor(random_parents(rows, dim), dtype=torch.int32, device="cuda")
    out, got = torch.empty_like(q), torch.zeros(kv, cached + rows, device="cuda")
    for at in (5, cached - 1):
        kc[at, :, 0] = -math.inf
    ops.tree_attention(q, kc, vc, cached, out, parents=par, weights=got)
    assert torch.isfinite(out).all() and torch.isfinite(got).all()
    assert not got[:, 5].any() and not got[:, cached - 1].any() and (got[:, 6:cached - 1] > 0).any(1).all()


@pytest.mark.parametrize("rows,cached,heads,kv,dim,kind", [
    (5, 100, 6, 2, 128, "f32"), (5, 100, 6, 2, 128, "f16"), (1, 0, 2, 1, 64, "bf16"), (9, 128, 4, 2, 256, "f32"), (40, 120, 2, 1, 256, "bf16"), (64, 0, 8, 2, 128, "f32"), (64, 1000, 4, 1, 256, "f16"), (200, 300, 2, 2, 64, "f32"),
    (3, 128 * 300 - 1, 4, 4, 64, "f32")])
def test_an_infinite_value_of_a_row_reaches_those_that_see_it_as_it_is(ops, rows, cached, heads, kv, dim, kind):
    """In the first tile that a run has and in later ones, and for rows that have seen nothing before; the sign is the value's.  Elements beside it are what they were."""
    q, kc, vc, g = make(kind, rows, cached, heads, kv, dim, rows + cached)
    parents = random_parents(rows, 3)
    par = torch.tensor(parents, dtype=torch.int32, device="cuda")
    clean, out = torch.empty_like(q), torch.empty_like(q)
    ops.tree_attention(q, kc, vc, cached, clean, parents=par)
    for at in {0, rows // 2, rows - 1}:
        sees = []
        for t in range(rows):
            j = t
            while j > at:
                j = parents[j]
            sees.append(j == at)
        for bad in (math.inf, -math.inf):
            v2 = vc.clone()
            v2[cached + at, :, 3] = bad
            ops.tree_attention(q, kc, v2, cached, out, parents=par)
            seen = torch.tensor(sees, device="cuda")
            assert (out[seen][..., 3] == bad).all()
            assert torch.equal(out[~seen], clean[~seen])
            assert torch.equal(out[..., :3], clean[..., :3]) and torch.equal(out[..., 4:], clean[..., 4:])


def test_a_backend_records_with_its_own_workspace_only(ops):
    """Refused while recording: a call that would need a larger workspace, and one that would take it from torch's allocator.  The recording goes on, and what it holds is launched beside larger calls."""
    from irontimber_b200.backend import CudaBackend
    be = CudaBackend(0, arena_floats=1 << 12)
    try:
        with torch.cuda.stream(be.torch_stream):
            q, kc, vc, g = make("f32", 3, 5000, 8, 2, 128, 21)
            big = torch.randn(200, 8, 128, device="cuda")
            want, out, more = torch.empty_like(q), torch.zeros_like(q), torch.empty_like(big)
            w = torch.zeros(2, 5003, device="cuda")
            be.tree_attention(q, kc, vc, 5000, want)
            be.capture_begin()
            be.tree_attention(q, kc, vc, 5000, out)
            with pytest.raises(ValueError, match="before it is recorded"):
                be.tree_attention(big, kc, vc, 4800, more)
            with pytest.raises(ValueError, match="needs workspace="):
                ops.tree_attention(q, kc, vc, 5000, want)
            gr = be.capture_end()
            be.tree_attention(big, kc, vc, 4800, more)
            be.tree_attention(q, kc, vc, 5000, want.clone(), weights=w)
            be.graph_launch(gr)
            be.tree_attention(big, kc, vc, 4800, more)
            be.sync()
            assert torch.equal(out, want) and be.L.it_graph_kernel_nodes(gr) == 2
            be.graph_destroy(gr)
    finally:
        be.close()


def test_a_backend_is_closed_in_a_recording(ops):
    """As a `finally` does after a refusal: the recording is given up, nothing is raised, and the next backend works."""
    from irontimber_b200.backend import CudaBackend
    for _ in range(2):
        be = CudaBackend(0, arena_floats=1 << 12)
        q, kc, vc, g = make("f32", 3, 500, 8, 2, 128, 22)
        torch.cuda.synchronize()
        be.tree_attention(q, kc, vc, 500, torch.empty_like(q))
        be.capture_begin()
        be.tree_attention(q, kc, vc, 500, torch.empty_like(q))
        be.close()


def test_evictions_are_recorded_and_run_beside_one_another(ops):
    """One recorded eviction replayed on other contents, and evictions of two caches on two streams at once, each with a workspace of its own."""
    from tests.test_gpu_attention_ops import evict_plain
    g = gen(23)
    n, keep, recent, kv, dim = 9000, 5000, 70, 2, 64
    state = [[randn(g, n, kv, dim).half(), randn(g, n, kv, dim).half(), torch.rand(kv, n, generator=g, device="cuda")] for _ in range(2)]
    kept = [torch.empty(kv, keep, dtype=torch.int32, device="cuda") for _ in range(2)]
    first = [[x.clone() for x in s] for s in state]
    ops.cache_evict(*state[0], n, keep, recent, kept[0])                # outside of recording

    def check(i, was):
        for h in range(kv):
            at = torch.tensor(evict_plain(was[2][h].cpu(), n, keep, recent), dtype=torch.long, device="cuda")
            assert torch.equal(kept[i][h].long(), at)
            assert all(torch.equal(state[i][k][:keep, h], was[k][at, h]) and torch.equal(state[i][k][keep:], was[k][keep:]) for k in (0, 1))
            assert torch.equal(state[i][2][h, :keep], was[2][h, at])

    check(0, first[0])
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        ops.cache_evict(*state[0], n, keep, recent, kept[0])
    for turn in range(4):
        was = [randn(g, n, kv, dim).half(), randn(g, n, kv, dim).half(), torch.rand(kv, n, generator=g, device="cuda")]
        for x, y in zip(state[0], was):
            x.copy_(y)
        gr.replay()
        check(0, was)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for turn in range(8):
        for i in (0, 1):
            for x, y in zip(state[i], first[i]):
                x.copy_(y)
        torch.cuda.synchronize()
        for i in (0, 1):
            ops.cache_evict(*state[i], n, keep, recent, kept[i], stream=streams[i])
        torch.cuda.synchronize()
        for i in (0, 1):
            check(i, first[i])


def test_a_recorded_call_with_weights_adds_them_at_every_replay(ops):
    """Kept scores (by their own launch and beside the joining) and the second walk, at a length that moves between replays."""
    for kind, rows, heads, kv, dim, most in (("f32", 1, 6, 1, 64, 3000), ("f32", 20, 24, 4, 256, 2091), ("bf16", 256, 40, 2, 136, 6800)):
        q, kc, vc, g = make(kind, rows, most, heads, kv, dim, 24)
        par = torch.tensor(random_parents(rows, 1), dtype=torch.int32, device="cuda")
        n = torch.tensor([most], dtype=torch.int32, device="cuda")
        out, got, want, ref = torch.empty_like(q), torch.zeros(kv, most + rows, device="cuda"), torch.empty_like(q), torch.zeros(kv, most + rows, device="cuda")
        ops.tree_attention(q, kc, vc, most, want, parents=par, length=n, weights=ref)
        ref.zero_()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            ops.tree_attention(q, kc, vc, most, out, parents=par, length=n, weights=got)
        for real in (most, 0, 127, most - 1, 128):
            n.fill_(real)
            gr.replay()
            ops.tree_attention(q, kc, vc, most, want, parents=par, length=n, weights=ref)
            assert torch.equal(out, want) and torch.equal(got, ref)

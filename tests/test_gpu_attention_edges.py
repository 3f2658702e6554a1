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

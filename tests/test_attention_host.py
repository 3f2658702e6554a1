"""What attention.py and CudaBackend do on the host around a launch, without a GPU: whose memory a workspace is, how much is kept, and what is refused."""
import contextlib
import types

import pytest

torch = pytest.importorskip("torch")


class Streams:
    """Torch's streams and allocator as far as a workspace needs them: blocks belong to the stream that is current when they are asked for."""

    def __init__(self, monkeypatch):
        self.now, self.blocks = "current", []
        monkeypatch.setattr(torch.cuda, "stream", self.stream)
        monkeypatch.setattr(torch.cuda, "ExternalStream", lambda ptr, device=None: f"stream {ptr} of {device}")
        monkeypatch.setattr(torch.cuda, "default_stream", lambda device=None: f"default of {device}")
        monkeypatch.setattr(torch, "empty", self.empty)

    @contextlib.contextmanager
    def stream(self, s):
        was, self.now = self.now, s
        yield
        self.now = was

    def empty(self, n, dtype=None, device=None):
        assert dtype is torch.uint8
        block = types.SimpleNamespace(owner=self.now, numel=lambda: n, device=device, record_stream=lambda s: None)
        self.blocks.append(block)
        return block


@pytest.mark.parametrize("stream,owner", [(None, "current"), ("another", "another"), (77, "stream 77 of 3"), (0, "default of 3")])
def test_a_workspace_comes_from_the_pool_of_the_stream_that_uses_it(monkeypatch, stream, owner):
    """Memory of another stream's pool may be a block that was just freed there and that queued kernels still write."""
    from irontimber_b200 import attention
    s = Streams(monkeypatch)
    assert attention._workspace(1000, 3, stream).owner == owner and s.now == "current"


def backend():
    """A CudaBackend without a device."""
    from irontimber_b200.backend import CudaBackend
    be = CudaBackend.__new__(CudaBackend)
    be.device, be.ctx, be._torch_stream, be._workspaces, be.arena_floats = 0, None, "the backend's", [], 1 << 20
    return be


def test_a_backends_workspace_comes_from_its_streams_pool(monkeypatch):
    s = Streams(monkeypatch)
    assert backend()._workspace(1000).owner == "the backend's" and s.now == "current"


def test_what_a_backend_keeps_is_bounded_by_the_largest_request(monkeypatch):
    """A cache that grows by views, or calls of more and more rows, ask for a little more each time; earlier workspaces stay, since recorded graphs may know them."""
    from irontimber_b200 import attention
    for requests in ([attention.tree_attention_workspace(64, 24, 4, 256, n, weights=True) for n in range(1000, 131072, 128)],
                     [attention.tree_attention_workspace(r, 24, 4, 256, 131072, weights=True) for r in range(1, 257)], range(1, 200000, 999), [10, 10, 5, 10]):
        s, be = Streams(monkeypatch), backend()
        for n in requests:
            assert be._workspace(n).numel() >= n
        assert sum(w.numel() for w in be._workspaces) <= 4 * max(max(requests), 256)
        assert len(be._workspaces) <= 30 and len(s.blocks) == len(be._workspaces)


class Recorder:
    """The library's recording calls."""

    @staticmethod
    def it_capture_begin(ctx):
        return 0

    it_capture_end = staticmethod(lambda ctx, out: 0)
    it_ctx_stream = staticmethod(lambda ctx: 4711)
    it_ctx_destroy = it_sync = it_graph_destroy = staticmethod(lambda ctx: 0)


def test_a_recorded_call_does_not_allocate(monkeypatch):
    """The backend's own workspace has to be there; one from torch's allocator would be freed, and handed on, with the graph still writing to it."""
    from irontimber_b200 import _lib, attention
    s, be = Streams(monkeypatch), backend()
    be.L, be.ctx = Recorder, 1
    be._workspace(5000)
    mine = types.SimpleNamespace(cuda_stream=4711)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda index: mine)
    be.capture_begin()
    assert be._workspace(5000) is s.blocks[0] and be._workspace(10) is s.blocks[0]
    with pytest.raises(ValueError, match="before it is recorded"):
        be._workspace(5001)
    for stream in (mine, 4711, None):
        with pytest.raises(ValueError, match="needs workspace="):
            attention._workspace(100, 0, stream)
    attention._workspace(100, 0, 4712)
    be.capture_end()
    assert be._workspace(5001) is s.blocks[-1] and attention._workspace(100, 0, 4711) is s.blocks[-1]
    be.capture_begin()
    be.close()
    assert not _lib.RECORDING


def test_what_a_wait_that_ran_out_leaves_behind(tmp_path):
    """An attention's outputs are NaN.  An eviction's caches are not: the next call's message must not say so, nor that they are as they were."""
    import ctypes
    import os
    import re
    import subprocess
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "irontimber_b200", "csrc")
    sites = [int(n) for n in re.findall(r"atomicExch\(p?\.?\w*status, (\d+)\)|abort_flag, p\.status, (\d+)\)", open(os.path.join(csrc, "it_tree_attention_tc.cu")).read()) for n in n if n]
    src = open(os.path.join(csrc, "it_cache_evict.cu")).read()
    assert "atomicExch(p.status, IT_SITE_EVICT_MOVE)" in src and src.count("p.status,") == 1 and len(sites) >= 8
    (tmp_path / "t.cpp").write_text('#include "it_ops_sites.h"\nextern "C" const char* text(int site) { return it_ops_after_timeout(site); }\nextern "C" int evict() { return IT_SITE_EVICT_MOVE; }\n')
    subprocess.run(["g++", "-Wall", "-Werror", "-shared", "-fPIC", "-I", csrc, str(tmp_path / "t.cpp"), "-o", str(tmp_path / "t.so")], check=True)
    lib = ctypes.CDLL(str(tmp_path / "t.so"))
    lib.text.restype = ctypes.c_char_p
    assert all(s != lib.evict() and b"NaN" in lib.text(s) for s in sites)
    assert b"NaN" not in lib.text(lib.evict()) and b"moved in part" in lib.text(lib.evict())


from tests.test_attention_ops import A, evict_args, lib, norm_rope_args, refused, tree_args  # noqa: E402,F401


@pytest.mark.parametrize("change,part", [
    (dict(q_out=5 * A), "q_out overlaps k_cache"), (dict(q_out=6 * A + 512), "q_out overlaps v_cache"), (dict(q_out=5 * A - 64), "q_out overlaps k_cache")])
def test_norm_rope_does_not_write_what_it_writes_elsewhere(lib, change, part):
    refused(lib, lib.it_norm_rope, norm_rope_args(**change), part)


W = dict(weights=9 * A, w_head=300)


@pytest.mark.parametrize("change,part", [
    (dict(out=5 * A), "out overlaps k_cache"), (dict(out=6 * A + 204 * 128 * 2 + 192), "out overlaps v_cache"), (dict(out=9 * A + 4 * 300 + 16, **W), "out overlaps weights"), (dict(out=16 * A), "out overlaps the workspace"), (dict(out=16 * A + 512, **W), "out overlaps the workspace"),
    (dict(W, weights=16 * A), "weights overlaps the workspace"), (dict(W, weights=5 * A + 4), "weights overlaps k_cache"), (dict(W, weights=A), "weights overlaps q"),
    (dict(gate=11 * A, g_row=384, g_head=64, weights=11 * A + 4, w_head=300), "weights overlaps gate"), (dict(workspace=A + 256), "the workspace overlaps q"), (dict(workspace=5 * A), "the workspace overlaps k_cache"),
    (dict(workspace=6 * A), "the workspace overlaps v_cache"), (dict(gate=16 * A, g_row=384, g_head=64), "the workspace overlaps gate")])
def test_tree_attention_does_not_write_what_it_reads(lib, change, part):
    refused(lib, lib.it_tree_attention, tree_args(**change), part)


@pytest.mark.parametrize("change,part", [
    (dict(workspace=7 * A), "the workspace overlaps weights"), (dict(workspace=8 * A), "the workspace overlaps kept"), (dict(workspace=5 * A), "the workspace overlaps k_cache"), (dict(kept=7 * A + 4 * 300), "weights overlaps kept"),
    (dict(weights=6 * A), "weights overlaps v_cache"), (dict(kept=5 * A + 256), "kept overlaps k_cache")])
def test_cache_evict_does_not_write_what_it_reads(lib, change, part):
    refused(lib, lib.it_cache_evict, evict_args(**change), part)


def test_memory_next_to_one_another_is_not_refused(lib):
    if torch.cuda.is_available():
        pytest.skip("addresses here are stand-ins")
    import ctypes as C
    n = C.c_size_t()
    assert lib.it_tree_attention_workspace(C.byref(tree_args(**W)), C.byref(n)) == 0
    for args in (tree_args(out=5 * A - 5 * 384 * 4), tree_args(out=5 * A + 205 * 128 * 2), tree_args(out=9 * A + 4 * (300 + 208), **W), tree_args(out=16 * A - 5 * 384 * 4, **W),
                 tree_args(v_cache=5 * A + 128, kc_slot=256, vc_slot=256),                              # k and v of a slot side by side
                 tree_args(gate=4 * A, g_row=384, g_head=64, **W)):                                     # out in gate's place
        assert lib.it_tree_attention(None, C.byref(args)) == -2, lib.it_last_error()                    # as far as the device
    assert lib.it_norm_rope(None, C.byref(norm_rope_args(q_out=5 * A - 5 * 384 * 4))) == -2
    assert lib.it_cache_evict(None, C.byref(evict_args(kept=7 * A + 4 * (300 + 200)))) == -2


def test_missing_tensors_and_closed_ropes_are_refused(lib):
    from irontimber_b200 import attention
    q, kc = torch.zeros(3, 2, 64), torch.zeros(50, 2, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="q or k is missing"):
        attention.norm_rope(None, None, None, None, None, None, None, 0, 0)
    with pytest.raises(ValueError, match="q_out is missing"):
        attention.norm_rope(None, q, None, None, None, None, None, 0, 0)
    with pytest.raises(ValueError, match="v is missing"):
        attention.norm_rope(None, None, q, None, None, kc, kc.clone(), 0, 0)
    with pytest.raises(ValueError, match="v_cache is missing"):
        attention.norm_rope(None, None, q, q, None, kc, None, 0, 0)
    rope = attention.Rope(64)
    rope.close()
    with pytest.raises(ValueError, match="rope is closed"):
        attention.norm_rope(rope, q, None, None, q.clone(), None, None, 0, 0)
    for args, part in (((None, kc, kc, 10, q), "q is missing"), ((q, None, kc, 10, q), "k_cache is missing"), ((q, kc, None, 10, q), "v_cache is missing"), ((q, kc, kc.clone(), 10, None), "out is missing")):
        with pytest.raises(ValueError, match=part):
            attention.tree_attention(*args)
    with pytest.raises(ValueError, match="weights is missing"):
        attention.cache_evict(kc, kc.clone(), None, 40, 20, 3)


@pytest.mark.parametrize("off,shape", [(-4, (4,)), (-8, (2, 2)), (2, (4,)), (0, ((1 << 20) + 1,)), ((1 << 20) - 4, (5,)), (0, (-1, 8)), (0, (-2, -2)), (0, (1 << 32, 1 << 32)), (0, (1 << 62, 4))])
def test_a_view_stays_in_the_arena(off, shape):
    """In front of it, behind it, sizes below zero and sizes whose product does not fit 64 bits."""
    with pytest.raises(ValueError, match="in an arena of"):
        backend().view(off, *shape)

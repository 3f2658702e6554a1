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

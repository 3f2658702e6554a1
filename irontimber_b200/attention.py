"""The attention block of a host with its own schedule: norm and rotation of q and k with the cache store, attention of a token, a
chain or a tree of drafted tokens, eviction from the cache (it_norm_rope, it_tree_attention, it_cache_evict of include/irontimber_cuda.h).

Tensors are torch CUDA tensors of one device; work is launched on `stream` (torch's current stream of that device unless one is given) and nothing waits.
Activations are f32 over an f16 cache, or f16 / bf16 for both.  Heads are contiguous, everything else may have strides: a cache tensor is
[slot, kv head, element] whatever its memory order (`cache.transpose(0, 1)` of a [kv head, slot, element] one).  `CudaBackend` has the same calls on its own
stream.  All arithmetic runs in libirontimber_cuda.so; this file only marshals arguments.

In a graph: torch.cuda.graph gives a call that allocates its workspace memory of the graph's own; any other way of recording needs workspace=, memory that lives as long as the graph and that nothing
uses while it runs.
"""
import ctypes as C
import functools
import struct

import torch

from . import _lib

TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
LAYOUTS = {"half": 0, "interleaved": 1}
SCALINGS = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3}
_P, _I32, _I64 = C.c_void_p, C.c_int32, C.c_int64


class RopeConfig(C.Structure):
    """it_rope_config"""
    _fields_ = [("n_rot", _I32), ("layout", _I32), ("scaling", _I32),
                ("base", C.c_double), ("factor", C.c_double), ("original_ctx", C.c_double), ("beta_fast", C.c_double), ("beta_slow", C.c_double)]


class NormRopeArgs(C.Structure):
    """it_norm_rope_args"""
    _fields_ = [("type", _I32), ("cache_type", _I32), ("rows", _I32), ("heads", _I32), ("kv_heads", _I32), ("head_dim", _I32), ("rope", _P),
                ("q", _P), ("q_row", _I64), ("q_head", _I64), ("k", _P), ("k_row", _I64), ("k_head", _I64), ("v", _P), ("v_row", _I64), ("v_head", _I64),
                ("q_out", _P), ("qo_row", _I64), ("qo_head", _I64), ("k_cache", _P), ("kc_slot", _I64), ("kc_head", _I64),
                ("v_cache", _P), ("vc_slot", _I64), ("vc_head", _I64), ("slots", _I64), ("slot0", _I64), ("positions", _P), ("base", _P),
                ("q_norm", _P), ("k_norm", _P), ("pos0", _I32), ("eps", C.c_float)]


class TreeAttentionArgs(C.Structure):
    """it_tree_attention_args"""
    _fields_ = [("type", _I32), ("cache_type", _I32), ("rows", _I32), ("heads", _I32), ("kv_heads", _I32), ("head_dim", _I32),
                ("q", _P), ("q_row", _I64), ("q_head", _I64), ("gate", _P), ("g_row", _I64), ("g_head", _I64), ("out", _P), ("o_row", _I64), ("o_head", _I64),
                ("k_cache", _P), ("kc_slot", _I64), ("kc_head", _I64), ("v_cache", _P), ("vc_slot", _I64), ("vc_head", _I64),
                ("slots", _I64), ("cached", _I64), ("parents", _P), ("length", _P), ("weights", _P), ("w_head", _I64),
                ("workspace", _P), ("workspace_bytes", C.c_size_t), ("scale", C.c_float)]


class CacheEvictArgs(C.Structure):
    """it_cache_evict_args"""
    _fields_ = [("kv_heads", _I32), ("head_dim", _I32), ("k_cache", _P), ("kc_slot", _I64), ("kc_head", _I64), ("v_cache", _P), ("vc_slot", _I64), ("vc_head", _I64),
                ("weights", _P), ("w_head", _I64), ("kept", _P), ("kept_head", _I64), ("slots", _I64), ("n", _I64), ("keep", _I64), ("recent", _I64),
                ("workspace", _P), ("workspace_bytes", C.c_size_t)]


class Rope:
    """Frequencies of a rotation of the first n_rot elements of a head (it_rope_create); made once and used on any device."""

    def __init__(self, n_rot, base=10000.0, layout="half", scaling="none", factor=1.0, original=0, beta_fast=32.0, beta_slow=1.0):
        self.handle = None
        cfg = RopeConfig(n_rot, _word(LAYOUTS, layout, "layout"), _word(SCALINGS, scaling, "scaling"), base, factor, original, beta_fast, beta_slow)
        h = _P()
        self._destroy = _lib.load().it_rope_destroy
        _lib.check(_lib.load().it_rope_create(C.byref(cfg), C.byref(h)))
        self.handle, self.n_rot = h, n_rot

    def read(self):
        """(angle per position of every pair, factor on sine and cosine)"""
        freq, m = (C.c_double * (self.n_rot // 2))(), C.c_double()
        _lib.check(_lib.load().it_rope_read(self.handle, freq, C.byref(m)))
        return list(freq), m.value

    def close(self):
        if self.handle:
            self._destroy(self.handle)
            self.handle = None

    def __del__(self):
        self.close()


def _word(table, word, what):
    if word not in table:
        raise ValueError(f"{what} is one of {', '.join(table)}: got {word!r}")
    return table[word]


# A call of a few microseconds is half arguments: tensors are asked for each fact once, the argument structure is packed in one go, and the device and stream
# are looked up without building objects.
_NORM_ROPE, _TREE, _EVICT = struct.Struct("@6iP" + "Pqq" * 6 + "qqPPPPif"), struct.Struct("@6i" + "Pqq" * 5 + "qqPPPqPNf0q"), struct.Struct("@2i" + "Pqq" * 2 + "PqPqqqqqPN")
assert (_NORM_ROPE.size, _TREE.size, _EVICT.size) == (C.sizeof(NormRopeArgs), C.sizeof(TreeAttentionArgs), C.sizeof(CacheEvictArgs))
_current_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else None
_current_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else None
_NONE3 = (0, 0, 0)
_MOST_CACHED = (1 << 30) - 1
_F16, _BF16, _F32, _I32T = torch.float16, torch.bfloat16, torch.float32, torch.int32


def _three(x, name, shape, dtype, index):
    """Address and outer strides of a [a, b, element] tensor of this shape with contiguous elements."""
    try:
        st = x.stride()
    except AttributeError:
        raise ValueError(f"{name} is missing") from None
    if x.shape != shape or x.dtype is not dtype or x.get_device() != index or st[2] != 1:
        _refuse_three(x, name, shape, dtype, index)
    return x.data_ptr(), st[0], st[1]


def _refuse_three(x, name, shape, dtype, index):
    if x.shape != shape:
        raise ValueError(f"{name} has the shape {tuple(x.shape)}, not {tuple(shape)}")
    if x.dtype is not dtype:
        raise TypeError(f"{name} is {x.dtype}, not {dtype}")
    if x.get_device() != index:
        raise ValueError(f"{name} is on {x.device}, not on the device of the others")
    if shape[2] > 1:
        raise ValueError(f"the elements of a head of {name} are not contiguous")


def _flat(x, name, n, dtype, index):
    """Address of a contiguous vector of at least n elements; 0 for None."""
    if x is None:
        return 0
    st = x.stride()
    if len(st) != 1 or x.numel() < n or x.dtype is not dtype or x.get_device() != index or (st[0] != 1 and n > 1):
        raise ValueError(f"{name} is {tuple(x.shape)} {x.dtype} on {x.device}: a contiguous vector of {n} {dtype} on the device of the others is wanted")
    return x.data_ptr()


def _caches(k, v, index):
    """Shape, type and the addresses and strides of a pair of caches."""
    try:
        shape, dtype = k.shape, k.dtype
    except AttributeError:
        raise ValueError("k_cache is missing") from None
    if dtype is not _F16 and dtype is not _BF16:
        raise TypeError(f"a cache is float16 or bfloat16, not {dtype}")
    st = k.stride()
    if len(st) != 3 or st[2] != 1 or k.get_device() != index:
        if len(st) != 3:
            raise ValueError(f"k_cache has the shape {tuple(shape)}, not three dimensions")
        _refuse_three(k, "k_cache", shape, dtype, index)
    return shape, TYPES[dtype], (k.data_ptr(), st[0], st[1]), _three(v, "v_cache", shape, dtype, index)


def _rows(x, name):
    try:
        shape = x.shape
    except AttributeError:
        raise ValueError(f"{name} is missing") from None
    if len(shape) != 3:
        raise ValueError(f"{name} has the shape {tuple(shape)}, not three dimensions")
    return shape


def _launch(call, args, index, stream):
    if index < 0:
        raise ValueError("tensors are not on a CUDA device")
    if index != (_current_device() if _current_device else torch.cuda.current_device()):
        with torch.cuda.device(index):
            return _launch(call, args, index, stream)
    if stream is None:
        stream = _current_stream(index) if _current_stream else torch.cuda.current_stream(index).cuda_stream
    elif not isinstance(stream, int):
        stream = stream.cuda_stream
    code = call(stream, args)
    if code:
        _lib.check(code)


def norm_rope(rope, q, k, v, q_out, k_cache, v_cache, slot0, positions, q_norm=None, k_norm=None, eps=1e-6, base=None, stream=None):
    """q_out = rotate(norm(q)); k_cache[slot0 + t] = rotate(norm(k[t])); v_cache[slot0 + t] = v[t].

    q, q_out: [row, head, element] (q_out may be q); k, v: [row, kv head, element]; q_norm, k_norm: f32 weights of a head, or None for no norm; rope None: no
    rotation.  positions: int32 tensor [row], or the position of row 0.  base: int32 tensor whose value is added to slots (and to positions that
    are a number), read on the device.  q and q_out, or k, v and the caches, may be None."""
    some, name = (q, "q") if q is not None else (k, "k") if k is not None else (None, "q or k")
    if rope is not None and rope.handle is None:
        raise ValueError("rope is closed")
    shape = rows, heads, dim = _rows(some, name)
    act, index = some.dtype, some.get_device()
    t = ct = TYPES.get(act, -1)
    kv, slots, qp, qo, kp, vp, kc, vc = 1, 0, _NONE3, _NONE3, _NONE3, _NONE3, _NONE3, _NONE3
    if t == 0:
        ct = 1
    if q is not None:
        qp, qo = _three(q, "q", shape, act, index), _three(q_out, "q_out", shape, act, index)
    if k is not None:
        (slots, kv, d), ct, kc, vc = _caches(k_cache, v_cache, index)
        want = (rows, kv, dim)
        if d != dim:
            raise ValueError(f"caches of {kv} heads of {d} for heads of {dim}")
        kp, vp = _three(k, "k", want, act, index), _three(v, "v", want, act, index)
    pos0 = 0
    if isinstance(positions, torch.Tensor):
        positions = _flat(positions, "positions", rows, _I32T, index)
    else:
        pos0, positions = positions, 0
    args = _NORM_ROPE.pack(t, ct, rows, heads, kv, dim, rope.handle.value if rope is not None else 0, *qp, *kp, *vp, *qo, *kc, *vc, slots, slot0, positions, _flat(base, "base", 1, _I32T, index),
                           _flat(q_norm, "q_norm", dim, _F32, index), _flat(k_norm, "k_norm", dim, _F32, index), pos0, eps)
    _launch(_load().it_norm_rope, args, index, stream)


def tree_attention(q, k_cache, v_cache, cached, out, parents=None, gate=None, scale=0.0, length=None, weights=None, workspace=None, stream=None):
    """out = softmax(scale q.k) v (* sigmoid(gate)): rows q [row, head, element] whose keys and values are in slots cached .. cached + rows - 1.

    parents: int32 [row], the row that a row continues or -1 for the cache; None: a chain.  scale 0: head_dim^-1/2.  length: int32 tensor, the number of cached
    slots (at most `cached`), read on the device.  weights: f32 [kv head, slot], to which the softmax weight that every slot received is added.
    workspace: a uint8 tensor of tree_attention_workspace() bytes (asked with weights=True when weights are given); None: one from torch's allocator."""
    shape = rows, heads, dim = _rows(q, "q")
    act, index = q.dtype, q.get_device()
    (slots, kv, d), ct, kc, vc = _caches(k_cache, v_cache, index)
    if d != dim:
        raise ValueError(f"caches of heads of {d} for heads of {dim}")
    t = TYPES.get(act, -1)
    qp, op = _three(q, "q", shape, act, index), _three(out, "out", shape, act, index)
    gp = _three(gate, "gate", shape, act, index) if gate is not None else _NONE3
    wp, wh = _weights(weights, kv, cached + rows, index) if weights is not None else (0, 0)
    parents, length = _flat(parents, "parents", rows, _I32T, index), _flat(length, "length", 1, _I32T, index)
    if workspace is None:
        workspace = _workspace(_tree_bytes(t, ct, rows, heads, kv, dim) if not wp else _tree_bytes(t, ct, rows, heads, kv, dim, min((cached | 4095) + 1, _MOST_CACHED), True), index, stream)
    else:
        _check_workspace(workspace, index)
    args = _TREE.pack(t, ct, rows, heads, kv, dim, *qp, *gp, *op, *kc, *vc, slots, cached, parents, length, wp, wh, workspace.data_ptr(), workspace.numel(), scale)
    _launch(_load().it_tree_attention, args, index, stream)


def cache_evict(k_cache, v_cache, weights, n, keep, recent, kept=None, workspace=None, stream=None):
    """Cuts a cache of n slots to `keep` a KV head: the last `recent`, and of the others those with the largest weight (f32 [kv head, slot]; ties: the
    lower slot).  They move to the front in their order, in place, in both caches and the weights; kept (int32 [kv head, keep]) gets the slots they had.
    workspace: a uint8 tensor of cache_evict_workspace() bytes; None: one from torch's allocator."""
    if weights is None:
        raise ValueError("weights is missing")
    index = weights.get_device()
    (slots, kv, dim), _, kc, vc = _caches(k_cache, v_cache, index)
    wp, wh = _weights(weights, kv, n, index)
    kp = kh = 0
    if kept is not None:
        if kept.shape != (kv, keep) or kept.dtype is not torch.int32 or kept.get_device() != index or (keep > 1 and kept.stride(1) != 1):
            raise ValueError(f"kept is {tuple(kept.shape)} {kept.dtype}: int32 {(kv, keep)} with contiguous rows is wanted")
        kp, kh = kept.data_ptr(), kept.stride(0)
    if workspace is None:
        workspace = _workspace(cache_evict_workspace(kv, n, keep), index, stream)
    else:
        _check_workspace(workspace, index)
    args = _EVICT.pack(kv, dim, *kc, *vc, wp, wh, kp, kh, slots, n, keep, recent, workspace.data_ptr(), workspace.numel())
    _launch(_load().it_cache_evict, args, index, stream)


_load = _lib.load


def _weights(w, kv, n, index):
    st, shape = w.stride(), w.shape
    if len(st) != 2 or shape[0] != kv or shape[1] < n or w.dtype is not _F32 or w.get_device() != index or (st[1] != 1 and n > 1):
        raise ValueError(f"weights are {tuple(w.shape)} {w.dtype} on {w.device}: f32 [{kv}, {n} or more] with contiguous rows on the device of the others are wanted")
    return w.data_ptr(), st[0]


def _workspace(nbytes, index, stream):
    if index < 0:
        raise ValueError("tensors are not on a CUDA device")
    if _lib.RECORDING and (stream if isinstance(stream, int) else stream.cuda_stream if stream is not None else torch.cuda.current_stream(index).cuda_stream) in _lib.RECORDING:
        raise ValueError("a call that a CudaBackend records needs workspace=: one from torch's allocator would be handed on while the graph still uses it")
    if stream is None:
        return torch.empty(nbytes, dtype=torch.uint8, device=index)
    # Torch hands memory out, and takes it back, in the order of the stream that is current: a block that was just freed on another one may still be written by what is queued there.
    if isinstance(stream, int):
        stream = torch.cuda.ExternalStream(stream, device=index) if stream else torch.cuda.default_stream(index)
    with torch.cuda.stream(stream):
        return torch.empty(nbytes, dtype=torch.uint8, device=index)


def _check_workspace(w, index):
    if w.dtype is not torch.uint8 or w.get_device() != index or not w.is_contiguous():
        raise ValueError("a workspace is a contiguous uint8 tensor on the tensors' device")
    return w


@functools.lru_cache(maxsize=256)
def _tree_bytes(t, ct, rows, heads, kv, dim, cached=_MOST_CACHED, weights=False):
    """Bytes of workspace.  A call that allocates asks for any number of cached slots if it has no weights (they then matter only while they are few), else for the next 4096."""
    need = C.c_size_t()
    _lib.check(_lib.load().it_tree_attention_workspace(C.byref(TreeAttentionArgs(t, ct, rows, heads, kv, dim, cached=cached, weights=256 if weights else None)), C.byref(need)))
    return need.value


@functools.lru_cache(maxsize=256)
def cache_evict_workspace(kv_heads, n, keep):
    """Bytes of workspace for an eviction of these sizes."""
    need = C.c_size_t()
    _lib.check(_lib.load().it_cache_evict_workspace(C.byref(CacheEvictArgs(kv_heads, 8, n=n, slots=n, keep=keep)), C.byref(need)))
    return need.value


def tree_attention_workspace(rows, heads, kv_heads, head_dim, cached, dtype=torch.float32, weights=False):
    """Bytes of workspace for a call of these sizes, with weights or without; enough for fewer cached slots too."""
    t = TYPES.get(dtype, -1)
    return _tree_bytes(t, 1 if t == 0 else t, rows, heads, kv_heads, head_dim, cached, bool(weights))

"""The attention block of a host with its own schedule: norm and rotation of q and k with the cache store, attention of a token, a
chain or a tree of drafted tokens, eviction from the cache (it_norm_rope, it_tree_attention, it_cache_evict of include/irontimber_cuda.h).

Tensors are torch CUDA tensors of one device; work is launched on `stream` (torch's current stream of that device unless one is given) and nothing waits.
Activations are f32 over an f16 cache, or f16 / bf16 for both.  Heads are contiguous, everything else may have strides: a cache tensor is
[slot, kv head, element] whatever its memory order (`cache.transpose(0, 1)` of a [kv head, slot, element] one).  `CudaBackend` has the same calls on its own
stream.  All arithmetic runs in libirontimber_cuda.so; this file only marshals arguments.
"""
import ctypes as C

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


def _three(x, name, shape, dtype, device):
    """A [a, b, element] tensor of this shape with contiguous elements."""
    if x.dim() != 3 or (shape is not None and tuple(x.shape) != shape):
        raise ValueError(f"{name} has the shape {tuple(x.shape)}" + (f", not {shape}" if shape else ", not three dimensions"))
    if x.dtype != dtype:
        raise TypeError(f"{name} is {x.dtype}, not {dtype}")
    if x.device != device:
        raise ValueError(f"{name} is on {x.device}, not {device}")
    if x.shape[2] > 1 and x.stride(2) != 1:
        raise ValueError(f"the elements of a head of {name} are not contiguous")
    return x.data_ptr()


def _flat(x, name, n, dtype, device):
    if x.dim() != 1 or x.shape[0] < n or x.dtype != dtype or x.device != device or (n > 1 and x.stride(0) != 1):
        raise ValueError(f"{name} is {tuple(x.shape)} {x.dtype} on {x.device}: a contiguous vector of {n} {dtype} on {device} is wanted")
    return x.data_ptr()


def _caches(k, v, device):
    """Pointers and shape of a pair of caches."""
    _three(k, "k_cache", None, k.dtype, device)
    _three(v, "v_cache", tuple(k.shape), k.dtype, device)
    if k.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"a cache is float16 or bfloat16, not {k.dtype}")
    return k.shape


def _launch(call, args, device, stream):
    if not device.type == "cuda":
        raise ValueError(f"tensors are on {device}, not on a CUDA device")
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return _launch(call, args, device, stream)
    if stream is None:
        stream = torch.cuda.current_stream(device)
    _lib.check(call(getattr(stream, "cuda_stream", stream), C.byref(args)))


def norm_rope(rope, q, k, v, q_out, k_cache, v_cache, slot0, positions, q_norm=None, k_norm=None, eps=1e-6, base=None, stream=None):
    """q_out = rotate(norm(q)); k_cache[slot0 + t] = rotate(norm(k[t])); v_cache[slot0 + t] = v[t].

    q, q_out: [row, head, element] (q_out may be q); k, v: [row, kv head, element]; q_norm, k_norm: f32 weights of a head, or None for no norm; rope None: no
    rotation.  positions: int32 tensor [row], or the position of row 0.  base: int32 tensor whose value is added to slots (and to positions that
    are a number), read on the device.  q and q_out, or k, v and the caches, may be None."""
    some = q if q is not None else k
    device, act, rows, dim = some.device, some.dtype, some.shape[0], some.shape[2]
    a = NormRopeArgs(type=TYPES.get(act, -1), rows=rows, head_dim=dim, rope=rope.handle if rope is not None else None, slot0=slot0, eps=eps)
    a.heads = a.kv_heads = 1
    a.cache_type = 1 if act == torch.float32 else a.type
    if q is not None:
        a.q, a.q_out = _three(q, "q", None, act, device), _three(q_out, "q_out", tuple(q.shape), act, device)
        (a.q_row, a.q_head, _), (a.qo_row, a.qo_head, _) = q.stride(), q_out.stride()
        a.heads = q.shape[1]
    if k is not None:
        a.k, a.v = _three(k, "k", (rows, k.shape[1], dim), act, device), _three(v, "v", tuple(k.shape), act, device)
        slots, kv, d = _caches(k_cache, v_cache, device)
        if kv != k.shape[1] or d != dim:
            raise ValueError(f"caches of {kv} heads of {d} for {k.shape[1]} heads of {dim}")
        (a.k_row, a.k_head, _), (a.v_row, a.v_head, _) = k.stride(), v.stride()
        a.k_cache, a.v_cache, a.slots, a.cache_type = k_cache.data_ptr(), v_cache.data_ptr(), slots, TYPES[k_cache.dtype]
        (a.kc_slot, a.kc_head, _), (a.vc_slot, a.vc_head, _) = k_cache.stride(), v_cache.stride()
        a.kv_heads = kv
        if q is None:
            a.heads = kv
    if isinstance(positions, torch.Tensor):
        a.positions = _flat(positions, "positions", rows, torch.int32, device)
    else:
        a.pos0 = positions
    if base is not None:
        a.base = _flat(base, "base", 1, torch.int32, device)
    if q_norm is not None:
        a.q_norm = _flat(q_norm, "q_norm", dim, torch.float32, device)
    if k_norm is not None:
        a.k_norm = _flat(k_norm, "k_norm", dim, torch.float32, device)
    _launch(_lib.load().it_norm_rope, a, device, stream)


def tree_attention(q, k_cache, v_cache, cached, out, parents=None, gate=None, scale=0.0, length=None, weights=None, workspace=None, stream=None):
    """out = softmax(scale q.k) v (* sigmoid(gate)): rows q [row, head, element] whose keys and values are in slots cached .. cached + rows - 1.

    parents: int32 [row], the row that a row continues or -1 for the cache; None: a chain.  scale 0: head_dim^-1/2.  length: int32 tensor, the number of cached
    slots (at most `cached`), read on the device.  weights: f32 [kv head, slot], to which the softmax weight that every slot received is added.
    workspace: a uint8 tensor of tree_attention_workspace() bytes; None: one from torch's allocator."""
    device, act = q.device, q.dtype
    rows, heads, dim = q.shape
    slots, kv, d = _caches(k_cache, v_cache, device)
    if d != dim:
        raise ValueError(f"caches of heads of {d} for heads of {dim}")
    a = TreeAttentionArgs(TYPES.get(act, -1), TYPES[k_cache.dtype], rows, heads, kv, dim)
    a.q, a.out = _three(q, "q", None, act, device), _three(out, "out", (rows, heads, dim), act, device)
    (a.q_row, a.q_head, _), (a.o_row, a.o_head, _) = q.stride(), out.stride()
    if gate is not None:
        a.gate = _three(gate, "gate", (rows, heads, dim), act, device)
        a.g_row, a.g_head, _ = gate.stride()
    a.k_cache, a.v_cache, a.slots, a.cached, a.scale = k_cache.data_ptr(), v_cache.data_ptr(), slots, cached, scale
    (a.kc_slot, a.kc_head, _), (a.vc_slot, a.vc_head, _) = k_cache.stride(), v_cache.stride()
    if parents is not None:
        a.parents = _flat(parents, "parents", rows, torch.int32, device)
    if length is not None:
        a.length = _flat(length, "length", 1, torch.int32, device)
    if weights is not None:
        a.weights, a.w_head = _weights(weights, kv, cached + rows, device)
    L = _lib.load()
    need = C.c_size_t()
    _lib.check(L.it_tree_attention_workspace(C.byref(a), C.byref(need)))
    _workspace(a, workspace, need.value, device, stream)
    _launch(L.it_tree_attention, a, device, stream)


def cache_evict(k_cache, v_cache, weights, n, keep, recent, kept=None, workspace=None, stream=None):
    """Cuts a cache of n slots to `keep` a KV head: the last `recent`, and of the others those with the largest weight (f32 [kv head, slot]; ties: the
    lower slot).  They move to the front in their order, in place, in both caches and the weights; kept (int32 [kv head, keep]) gets the slots they had."""
    device = weights.device
    slots, kv, dim = _caches(k_cache, v_cache, device)
    a = CacheEvictArgs(kv, dim, k_cache.data_ptr(), k_cache.stride(0), k_cache.stride(1), v_cache.data_ptr(), v_cache.stride(0), v_cache.stride(1))
    a.slots, a.n, a.keep, a.recent = slots, n, keep, recent
    a.weights, a.w_head = _weights(weights, kv, n, device)
    if kept is not None:
        if tuple(kept.shape) != (kv, keep) or kept.dtype != torch.int32 or kept.device != device or (keep > 1 and kept.stride(1) != 1):
            raise ValueError(f"kept is {tuple(kept.shape)} {kept.dtype}: int32 {(kv, keep)} with contiguous rows is wanted")
        a.kept, a.kept_head = kept.data_ptr(), kept.stride(0)
    L = _lib.load()
    if kept is None or workspace is not None:
        need = C.c_size_t()
        _lib.check(L.it_cache_evict_workspace(C.byref(a), C.byref(need)))
        _workspace(a, workspace, need.value, device, stream)
    _launch(L.it_cache_evict, a, device, stream)


def _weights(w, kv, n, device):
    if w.dim() != 2 or w.shape[0] != kv or w.shape[1] < n or w.dtype != torch.float32 or w.device != device or (n > 1 and w.stride(1) != 1):
        raise ValueError(f"weights are {tuple(w.shape)} {w.dtype} on {w.device}: f32 [{kv}, {n} or more] with contiguous rows on {device} are wanted")
    return w.data_ptr(), w.stride(0)


def _workspace(a, workspace, need, device, stream):
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=device)
        if stream is not None:               # torch hands the memory out again in the order of the current stream
            workspace.record_stream(stream if isinstance(stream, torch.cuda.Stream) else torch.cuda.ExternalStream(stream, device=device))
    elif workspace.dtype != torch.uint8 or workspace.device != device or not workspace.is_contiguous():
        raise ValueError("a workspace is a contiguous uint8 tensor on the tensors' device")
    a.workspace, a.workspace_bytes = workspace.data_ptr(), workspace.numel()


def tree_attention_workspace(rows, heads, kv_heads, head_dim, cached, dtype=torch.float32):
    """Bytes of workspace for a call of these sizes."""
    t = TYPES.get(dtype, -1)
    a = TreeAttentionArgs(t, 1 if t == 0 else t, rows, heads, kv_heads, head_dim)
    a.cached = cached
    need = C.c_size_t()
    _lib.check(_lib.load().it_tree_attention_workspace(C.byref(a), C.byref(need)))
    return need.value

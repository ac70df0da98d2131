"""Rows of tokens over the caches: the plan of a step's drafts, the head norms
with the rotary position, and attention of several rows a sequence (a prompt,
one token of each sequence of a batch, a tree of drafted tokens).

The order in a step: draft_plan once; in each layer linear_i8_multi (q, k, v),
qk_norm_rope, tree_attention, linear_i8 (o); token_logprobs over the logits.
After a tree is judged, the caller moves the accepted rows' keys and values to
the positions they now have (their slots are those of their rows) and adds
their number to cache_len.

KVCache, QKNorm and Rope hold one layer's caches, norm weights and the rotary
tables with their C descriptions; a program builds them once. The tensors stay
the caller's and must not be freed or resized while the description is in use.
Every tensor of a call has to be on the current device.
"""
from __future__ import annotations

import ctypes

from . import FP16, FP32, _check, _need, _ptr, _torch, lib

_sz = ctypes.c_size_t
_vp = ctypes.c_void_p
_i = ctypes.c_int


class _CacheC(ctypes.Structure):
    _fields_ = [("k", _vp), ("v", _vp), ("batch", _i), ("kv_heads", _i), ("max_seq", _i), ("head_dim", _i),
                ("seq_stride", _sz), ("head_stride", _sz), ("row_stride", _sz)]


class _NormC(ctypes.Structure):
    _fields_ = [("q_w", _vp), ("q_s", _vp), ("k_w", _vp), ("k_s", _vp), ("group_size", _i), ("eps", ctypes.c_float)]


class _RopeC(ctypes.Structure):
    _fields_ = [("cos", _vp), ("sin", _vp), ("rows", _i), ("axes", _i), ("sections", _i * 3), ("interleaved", _i)]


_lib = _plan_fn = _rope_fn = _attn_fn = None


def _L():
    global _lib, _plan_fn, _rope_fn, _attn_fn
    if _lib is None:
        L = lib()
        sigs = {
            "q3vl_draft_plan": (_i, [_vp, _vp, _vp, _vp, _i, _sz, _i, _i, _vp, _i, _vp, _vp, _vp]),
            "q3vl_qk_norm_rope": (_i, [_vp, _sz, _vp, _sz, _vp, _sz, _vp, _sz, _i, _sz, _i, _vp, _vp, _vp, _vp, _vp, _vp]),
            "q3vl_tree_attention_workspace_bytes": (_sz, [_sz, _i, _i, _i, _vp]),
            "q3vl_tree_attention": (_i, [_vp, _sz, _vp, _sz, _i, _sz, _i, _vp, _vp, _vp, _vp, _i, _i, _i, ctypes.c_float,
                                         _vp, _sz, _vp]),
        }
        for name, (res, args) in sigs.items():
            fn = getattr(L, name)
            fn.restype, fn.argtypes = res, args
        _plan_fn, _rope_fn, _attn_fn = L.q3vl_draft_plan, L.q3vl_qk_norm_rope, L.q3vl_tree_attention
        _lib = L
    return _lib


# A call costs 3 to 6 us in the library (its launches), so the checks around it
# are kept short, as the linears' are: the usual tensor passes in one
# expression and only another one is looked at again for its error.
def _device():
    """(torch, the current device's index)"""
    torch = _torch()
    try:
        return torch, torch._C._cuda_getDevice()
    except RuntimeError:  # no device at all
        return torch, -2


def _raw_stream(stream, torch, dev):
    return torch._C._cuda_getCurrentRawStream(dev) if stream is None else stream.cuda_stream


def _here(t, name, dev):
    if t.get_device() != dev:
        raise ValueError(f"{name} must be on the current device")


def _rows(t, dtypes, name, dev):
    """Row stride of a 2-d device tensor whose rows are contiguous (views of
    wider rows too)."""
    torch = _torch()
    if isinstance(t, torch.Tensor) and t.get_device() == dev and t.dtype in dtypes and t.dim() == 2:
        n, m = t.shape
        s, u = t.stride()
        if s >= m and u == 1:
            return s
        if (u == 1 or m <= 1) and (s >= m or n <= 1):
            return max(s, m)
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a device tensor")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(map(str, dtypes))}, got {t.dtype}")
    _here(t, name, dev)
    raise ValueError(f"{name} must be 2-d with contiguous rows")


def _is_vec(t, dtype, dev):
    return isinstance(t, _torch().Tensor) and t.get_device() == dev and t.dtype is dtype and t.is_contiguous()


def _vec(t, dtype, n, name, dev):
    """Refuses what is not a contiguous device tensor of n values (None: any
    number). Callers ask _is_vec first."""
    if _is_vec(t, dtype, dev) and (n is None or t.numel() == n):
        return
    _need(t, dtype, name)
    _here(t, name, dev)
    raise ValueError(f"{name} must hold {n} values, got {t.numel()}")


def _mask_words(mask, rows, dev):
    torch = _torch()
    if not (isinstance(mask, torch.Tensor) and mask.get_device() == dev and mask.dtype is torch.int64 and mask.is_contiguous()
            and mask.dim() == 2):
        _need(mask, torch.int64, "mask", 2)
        _here(mask, "mask", dev)
    n, words = mask.shape
    if n != rows:
        raise ValueError("mask must have a line for each row")
    return words


def _workspace(t, dev):
    """(address, bytes) of a call's workspace; none: the library's own."""
    if t is None:
        return None, 0
    if not (isinstance(t, _torch().Tensor) and t.get_device() == dev and t.is_contiguous()):
        raise ValueError("workspace must be a contiguous tensor on the current device")
    return t.data_ptr(), t.numel() * t.element_size()


def _empty(like, stream, *shape, dtype=None):
    """An output of a call on `stream`: memory of that stream's own."""
    if stream is None:
        return like.new_empty(*shape) if dtype is None else like.new_empty(*shape, dtype=dtype)
    with _torch().cuda.stream(stream):
        return like.new_empty(*shape, dtype=dtype or like.dtype)


class KVCache:
    """One layer's caches of a batch: k, v fp16 [batch, kv_heads, max_seq,
    head_dim] (head_dim 64 or 128; any strides that keep a row contiguous and
    16-byte aligned, the same for both). The decode step's caches
    [layers, kv_heads, max_seq, head_dim] are KVCache(k[l][None], v[l][None])."""

    def __init__(self, k, v):
        torch = _torch()
        for t, n in ((k, "k"), (v, "v")):
            if not isinstance(t, torch.Tensor):
                raise TypeError(f"{n} must be a torch.Tensor")
            if not t.is_cuda:
                raise ValueError(f"{n} must be a device tensor")
            if t.dtype != torch.float16:
                raise TypeError(f"{n} must be torch.float16, got {t.dtype}")
            if t.dim() != 4 or t.stride(3) != 1:
                raise ValueError(f"{n} must be [batch, kv_heads, max_seq, head_dim] with contiguous rows")
        if k.shape != v.shape or k.stride() != v.stride() or k.device != v.device:
            raise ValueError("k and v must have the same shape, strides and device")
        B, H, S, D = k.shape
        st = [k.stride(0) if B > 1 else 0, k.stride(1) if H > 1 else 0, k.stride(2) if S > 1 else D]
        if any(x % 8 for x in st) or k.data_ptr() % 16 or v.data_ptr() % 16:
            raise ValueError("cache rows must be 16-byte aligned")
        self.k, self.v = k, v
        self.c = _CacheC(k.data_ptr(), v.data_ptr(), B, H, S, D, *st)
        self.ref = ctypes.byref(self.c)
        self.device, self.dev = k.device, k.get_device()


class QKNorm:
    """One layer's head norms: int8 weights [head_dim], fp32 scales
    [head_dim / gs]."""

    def __init__(self, q_w, q_s, k_w, k_s, gs, eps):
        torch = _torch()
        for w, s, n in ((q_w, q_s, "q"), (k_w, k_s, "k")):
            _need(w, torch.int8, n + "_w")
            _need(s, torch.float32, n + "_s")
            if gs <= 0 or w.numel() % gs or s.numel() != w.numel() // gs:
                raise ValueError(f"{n}_w and {n}_s do not match in groups of {gs}")
        if q_w.numel() != k_w.numel():
            raise ValueError("q_w and k_w must have the same size")
        self.t = (q_w, q_s, k_w, k_s)
        self.head_dim, self.dev = q_w.numel(), q_w.get_device()
        if any(t.get_device() != self.dev for t in self.t):
            raise ValueError("the norm's tensors must be on one device")
        self.c = _NormC(q_w.data_ptr(), q_s.data_ptr(), k_w.data_ptr(), k_s.data_ptr(), gs, eps)
        self.ref = ctypes.byref(self.c)


class Rope:
    """Rotary tables cos, sin fp32 [rows, head_dim/2]. sections None: a row has
    one position. sections (time, height, width): three positions a row, that
    many frequencies each, in that order or interleaved (frequency 3 n + a by
    axis a = 1, 2, the rest by time)."""

    def __init__(self, cos, sin, sections=None, interleaved=False):
        torch = _torch()
        for t, n in ((cos, "cos"), (sin, "sin")):
            _need(t, torch.float32, n, 2)
        if cos.shape != sin.shape:
            raise ValueError("cos and sin must have the same shape")
        if cos.device != sin.device:
            raise ValueError("cos and sin must be on one device")
        self.t, self.dev = (cos, sin), cos.get_device()
        self.head_dim, self.axes = 2 * cos.shape[1], 1 if sections is None else 3
        sec = (0, 0, 0) if sections is None else tuple(sections)
        if len(sec) != 3:
            raise ValueError("sections must be (time, height, width)")
        self.c = _RopeC(cos.data_ptr(), sin.data_ptr(), cos.shape[0], self.axes, (_i * 3)(*sec), int(bool(interleaved)))
        self.ref = ctypes.byref(self.c)


def draft_plan(parents, row_start, cache_len, max_seq, max_rows, pos_delta=None, mask=None, pos=None, slots=None, stream=None):
    """Plans a step over drafts: parents int32 [rows] (-1: follows the last
    cached token), row_start int32 [batch + 1], cache_len int32 [batch],
    pos_delta int32 [batch] added to the positions. Returns mask int64
    [rows, words] (64 ancestor bits a word, the row's own among them), pos
    int32 [rows] and slots int64 [rows]. Rows behind the last sequence get
    position and slot -1, rows that cannot be planned (a bad parent, no room in
    the cache, past max_rows) position -2 and slot -1."""
    torch, dev = _device()
    i32, T = torch.int32, torch.Tensor
    if not (isinstance(parents, T) and parents.dtype is i32 and parents.get_device() == dev and parents.is_contiguous()):
        _vec(parents, i32, None, "parents", dev)
    if not (isinstance(cache_len, T) and cache_len.dtype is i32 and cache_len.get_device() == dev and cache_len.is_contiguous()):
        _vec(cache_len, i32, None, "cache_len", dev)
    rows, batch = parents.numel(), cache_len.numel()
    if not (isinstance(row_start, T) and row_start.dtype is i32 and row_start.get_device() == dev and row_start.is_contiguous()
            and row_start.numel() == batch + 1):
        _vec(row_start, i32, batch + 1, "row_start", dev)
    if pos_delta is not None:
        _vec(pos_delta, i32, batch, "pos_delta", dev)
    if mask is None:
        words = max(1, -(-max_rows // 64))
        mask = _empty(parents, stream, rows, words, dtype=torch.int64)
    else:
        words = _mask_words(mask, rows, dev)
    if pos is None:
        pos = _empty(parents, stream, rows)
    else:
        _vec(pos, i32, rows, "pos", dev)
    if slots is None:
        slots = _empty(parents, stream, rows, dtype=torch.int64)
    else:
        _vec(slots, torch.int64, rows, "slots", dev)
    rc = (_plan_fn or _L().q3vl_draft_plan)(
        parents.data_ptr(), row_start.data_ptr(), cache_len.data_ptr(), _ptr(pos_delta), batch, rows, max_rows, max_seq,
        mask.data_ptr(), words, pos.data_ptr(), slots.data_ptr(), _raw_stream(stream, torch, dev))
    if rc:
        _check(rc)
    return mask, pos, slots


def qk_norm_rope(q, k, v, cache, slots, pos, norm, rope, out=None, out_dtype=None, stream=None):
    """Head norms and rotation of q [rows, heads * head_dim], k and v
    [rows, kv_heads * head_dim] (fp32; views of wider rows are fine). Returns
    the queries (out, or a new tensor of out_dtype: torch.float32, the default,
    or torch.float16); k and v go to the cache's rows that slots int64 [rows]
    names (batch index * max_seq + row; another value: not stored). pos int32
    [rows], or [rows, 3] under a Rope with sections. Rows at position -1 hold
    no token and are left alone; out may be q."""
    torch, dev = _device()
    f32 = (torch.float32,)
    ldq, ldk, ldv = _rows(q, f32, "q", dev), _rows(k, f32, "k", dev), _rows(v, f32, "v", dev)
    c = cache.c
    D = c.head_dim
    rows, qn = q.shape
    if qn % D or k.shape != (rows, c.kv_heads * D) or v.shape != k.shape:
        raise ValueError("shape mismatch between q, k, v and the cache")
    if norm.head_dim != D or rope.head_dim != D:
        raise ValueError("norm and rope must have the cache's head_dim")
    if not cache.dev == norm.dev == rope.dev == dev:
        raise ValueError("cache, norm and rope must be on the current device")
    if out is None:
        out = _empty(q, stream, rows, qn, dtype=out_dtype)
    elif out_dtype is not None and out.dtype != out_dtype:
        raise TypeError("out has another dtype than out_dtype")
    ldo = _rows(out, (torch.float32, torch.float16), "out", dev)
    if out.shape != q.shape:
        raise ValueError("out must have q's shape")
    _vec(slots, torch.int64, rows, "slots", dev)
    _vec(pos, torch.int32, rows * rope.axes, "pos", dev)
    rc = (_rope_fn or _L().q3vl_qk_norm_rope)(
        q.data_ptr(), ldq, k.data_ptr(), ldk, v.data_ptr(), ldv, out.data_ptr(), ldo,
        FP16 if out.dtype is torch.float16 else FP32, rows, qn // D, cache.ref, slots.data_ptr(), pos.data_ptr(), norm.ref,
        rope.ref, _raw_stream(stream, torch, dev))
    if rc:
        _check(rc)
    return out


def tree_attention_workspace_bytes(cache, rows, heads, max_rows, max_len=None) -> int:
    return _L().q3vl_tree_attention_workspace_bytes(rows, heads, max_rows, max_len or 0, cache.ref)


def alloc_tree_attention_workspace(cache, rows, heads, max_rows, max_len=None):
    """Device workspace for tree_attention at these sizes."""
    torch = _torch()
    n = tree_attention_workspace_bytes(cache, rows, heads, max_rows, max_len)
    return torch.empty(max(n, 256), dtype=torch.uint8, device=cache.device)


def tree_attention(q, cache, row_start, cache_len, max_rows, mask=None, max_len=None, scale=None, out=None, workspace=None,
                   stream=None):
    """Attention of q [rows, heads * head_dim] (fp32 or fp16) over the cache:
    row t of sequence b (rows row_start[b] .. row_start[b + 1] - 1) sees the
    cache_len[b] cached positions and, of the step's own rows, those set in its
    mask line (int64 [rows, words], draft_plan's) or, with mask None, rows 0 ..
    t. Their keys and values are in the cache already (qk_norm_rope). max_rows:
    the most rows of one sequence; max_len: the most positions, cached and new,
    of one (a hint for splitting the work, default the whole cache). scale:
    default 1 / sqrt(head_dim). out may be q. A row that sees nothing gives 0.
    workspace: alloc_tree_attention_workspace with the same max_rows and
    max_len."""
    torch, dev = _device()
    ldq = _rows(q, (torch.float32, torch.float16), "q", dev)
    c = cache.c
    D, batch = c.head_dim, c.batch
    rows, qn = q.shape
    if qn % D:
        raise ValueError("q's rows must be whole heads of the cache's head_dim")
    if cache.dev != dev:
        raise ValueError("cache must be on the current device")
    if out is None:
        out = _empty(q, stream, rows, qn)
        ldo = qn
    else:
        ldo = _rows(out, (q.dtype,), "out", dev)
        if out.shape != q.shape:
            raise ValueError("out must have q's shape")
    _vec(row_start, torch.int32, batch + 1, "row_start", dev)
    _vec(cache_len, torch.int32, batch, "cache_len", dev)
    words = 0 if mask is None else _mask_words(mask, rows, dev)
    wp, wb = _workspace(workspace, dev)
    rc = (_attn_fn or _L().q3vl_tree_attention)(
        q.data_ptr(), ldq, out.data_ptr(), ldo, FP16 if q.dtype is torch.float16 else FP32, rows, qn // D, cache.ref,
        row_start.data_ptr(), cache_len.data_ptr(), _ptr(mask), words, max_rows, max_len or 0,
        D ** -0.5 if scale is None else scale, wp, wb, _raw_stream(stream, torch, dev))
    if rc:
        _check(rc)
    return out

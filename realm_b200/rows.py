"""Row plans: the operators of a step's rows over the paged cache.

    with pool.plan(tenants, n_heads) as plan:          # a step's rows, once
        for layer in ...:
            plan.append(layer, k, v, q=q, q_out=q2, q_norm=..., k_norm=..., rope=rope_table(...))
            plan.attention(layer, q2, scale, softcap=50.0, out=o)
    sample_filtered(ctx, logits, [SamplingFilter(0.8, top_k=40, top_p=0.9, min_p=0.02)], uniforms)

Arrays are numpy (host; the call copies and waits) or CUDA torch tensors (the
call enqueues and returns). CUDA calls are ordered with torch's current stream:
without events where the context runs on that stream (Context(stream=...)), by
events in both directions where it has a stream of its own. Rows may lie apart
(slices of one projection's output); heads and elements are contiguous.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass
from typing import Optional, Sequence

import numpy as np

from . import F16, F32, PTR_DEVICE, PTR_HOST, _check, _lib, _sig  # noqa: E402
from .sampling import _prev_arrays

_vp, _u32, _u64, _i32, _f = C.c_void_p, C.c_uint32, C.c_uint64, C.c_int32, C.c_float
ASYNC = 2
BAD_HANDLE = -20  # RB_ERR_BAD_HANDLE
MAX_VOCAB = 262144


class _PlanDesc(C.Structure):
    _fields_ = [("n_heads", _u32), ("n_rows", _u32), ("tenants", _vp), ("positions", _vp), ("begin", _vp),
                ("end", _vp), ("window", _u32)]


class _AppendDesc(C.Structure):
    _fields_ = [("dtype", _i32), ("rope_style", _i32), ("q", _vp), ("k", _vp), ("v", _vp), ("q_out", _vp),
                ("ldq", _u64), ("ldk", _u64), ("ldv", _u64), ("ldo", _u64), ("q_norm", _vp), ("k_norm", _vp),
                ("eps", _f), ("rotary", _u32), ("rope", _vp), ("rope_len", _u32)]


class _AttentionDesc(C.Structure):
    _fields_ = [("dtype", _i32), ("scale", _f), ("softcap", _f), ("q", _vp), ("out", _vp), ("ldq", _u64),
                ("ldo", _u64), ("slopes", _vp)]


class _Filter(C.Structure):
    _fields_ = [("temperature", _f), ("top_k", _u32), ("top_p", _f), ("min_p", _f), ("repetition_penalty", _f)]


_sig("rb_plan_create", [_vp, _i32, C.POINTER(_PlanDesc), C.POINTER(_i32)])
_sig("rb_plan_destroy", [_vp, _i32])
_sig("rb_plan_append", [_vp, _i32, _u32, C.POINTER(_AppendDesc), _u32])
_sig("rb_plan_attention", [_vp, _i32, _u32, C.POINTER(_AttentionDesc), _u32])
_sig("rb_plan_partition", [_u32, _vp, _u32, _u32, _u32, _i32, _vp, _u32])
_sig("rb_sample_filtered", [_vp, _i32, _vp, _u64, _u32, _u32, _vp, _vp, _vp, _vp, _vp, _vp, _u32])


def _is_tensor(a) -> bool:
    return hasattr(a, "data_ptr")


_TORCH = {}  # torch's dtypes by name


def _torch_dtype(name):
    import torch
    _TORCH[name] = getattr(torch, name)
    return _TORCH[name]


def _vec(a, dtype, n, name):
    """Pointer of a contiguous vector of n elements, or None."""
    if a is None:
        return None
    if _is_tensor(a):
        if a.dtype is (_TORCH.get(dtype) or _torch_dtype(dtype)) and a.numel() == n and a.is_contiguous():
            return a.data_ptr()
    elif a.dtype == dtype and a.size == n and a.flags.c_contiguous:
        return a.ctypes.data
    raise ValueError(f"{name}: {n} contiguous {dtype} values wanted")


def _writable(a, name):
    """a, an output: not a numpy array that is read-only."""
    if a is not None and not _is_tensor(a) and not a.flags.writeable:
        raise ValueError(f"{name}: read-only")
    return a


def _rows3(a, n, heads, hd, name):
    """(pointer, elements between rows) of a [n][heads][hd] (or [n][heads * hd]) array."""
    if _is_tensor(a):
        shape, stride, ptr = a.shape, a.stride(), a.data_ptr()
    else:
        shape, ptr = a.shape, a.ctypes.data
        if any(s % a.itemsize for s in a.strides):
            raise ValueError(f"{name}: rows lie whole elements apart, got strides of {a.strides} bytes")
        stride = [s // a.itemsize for s in a.strides]
    if len(shape) == 3:
        ok = shape[0] == n and shape[1] == heads and shape[2] == hd and stride[2] == 1 and \
            (stride[1] == hd or heads == 1)
    else:
        ok = len(shape) == 2 and shape[0] == n and shape[1] == heads * hd and stride[1] == 1
    if n == 1:
        ld = heads * hd
    else:
        ld = stride[0]
        ok = ok and ld >= heads * hd
    if not ok:
        raise ValueError(f"{name}: [{n}][{heads}][{hd}] with contiguous heads wanted, got {tuple(shape)} / {tuple(stride)}")
    return ptr, ld


def _mat(a, n, width, dtype, device, name):
    """(pointer, elements between rows) of a tensor [n][width] of `dtype` on `device` (its index)."""
    st = a.stride()
    if a.shape == (n, width) and (st[1] == 1 or width == 1) and a.dtype is dtype and a.get_device() == device:
        if n == 1:
            return a.data_ptr(), width
        if st[0] >= width:
            return a.data_ptr(), st[0]
    raise ValueError(f"{name}: [{n}][{width}] of {dtype} on the context's device wanted, rows contiguous, got "
                     f"{tuple(a.shape)} / {tuple(st)} of {a.dtype} on {a.device}")


_DTYPES = {"torch.float32": F32, "torch.float16": F16, "float32": F32, "float16": F16}
_SEEN = {}  # dtype objects met so far


def _dtype(arrays, ctx):
    """(dtype id, flags) of arrays that share a type and a memory space."""
    dtype = arrays[0].dtype
    for a in arrays:
        if a.dtype != dtype:
            raise ValueError(f"mixed types {dtype} and {a.dtype}")
    dt = _SEEN.get(dtype)
    if dt is None:
        dt = _DTYPES.get(str(dtype))
        if dt is None:
            raise ValueError(f"unsupported type {dtype}")
        _SEEN[dtype] = dt
    return dt, _space(arrays, ctx)


def _space(arrays, ctx):
    """Flags of arrays that are all host arrays, or all tensors on the context's device."""
    dev = _is_tensor(arrays[0])
    for a in arrays:
        if a is not None and (_is_tensor(a) != dev or (dev and a.get_device() != ctx.device)):
            raise ValueError("host arrays, or tensors on the context's device, wanted: not a mix")
    return PTR_DEVICE | ASYNC if dev else PTR_HOST


_raw_stream = None


def _current_stream(device: int) -> int:
    """The cudaStream_t of torch's current stream."""
    global _raw_stream
    if _raw_stream is None:
        import torch
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
            (lambda d: torch.cuda.current_stream(d).cuda_stream)
    return _raw_stream(device)


class _Order:
    """Orders a device call on a context's own stream after torch's current one, and what follows there after it."""

    def __init__(self, ctx):
        import torch
        self.cur = torch.cuda.current_stream(ctx.device)
        self.ext = ctx.torch_stream()
        self.ext.wait_stream(self.cur)

    def done(self):
        self.cur.wait_stream(self.ext)


def _call(ctx, flags, fn, *args):
    if not flags & PTR_DEVICE or _current_stream(ctx.device) == ctx._stream_id:
        rc = fn(*args, flags)
    else:
        order = _Order(ctx)
        rc = fn(*args, flags)
        order.done()
    if rc < 0:
        _check(rc)


def _indices(a, name):
    """One 32-bit unsigned value per row, or None; anything that would not keep its value is refused."""
    if a is None:
        return None
    a = np.asarray(a)
    if a.size == 0:
        return np.empty(0, np.uint32)
    kind, size = a.dtype.kind, a.itemsize
    # (a negative value of 8 bytes is a large one without its sign)
    ok = kind == "u" and size <= 4 or \
        (kind in "iu" and (a.view(np.uint64).max() <= 0xffffffff if size == 8 else a.min() >= 0))
    if a.ndim != 1 or not ok:
        raise ValueError(f"{name}: integers of at least 0, one per row, wanted")
    return np.ascontiguousarray(a, np.uint32)


class RowPlan:
    """The rows of one step over a KV pool (rb_plan_create); see KVPool.plan. Ends with close(), with its pool, or
    when nothing refers to it."""

    handle = -1

    def __init__(self, pool, tenants, n_heads: int, positions=None, begin=None, end=None, window: int = 0):
        self.pool, self.ctx, self.n_heads = pool, pool.ctx, int(n_heads)
        arr = [_indices(tenants, "tenants"), _indices(positions, "positions"), _indices(begin, "begin"),
               _indices(end, "end")]
        if int(window) != window or not 0 <= window <= 0xffffffff:
            raise ValueError("window: a length of at least 0, or 0 for none, wanted")
        self.n_rows = len(arr[0])
        for a in arr[1:]:
            if a is not None and len(a) != self.n_rows:
                raise ValueError("tenants, positions, begin and end have one entry per row")
        d = _PlanDesc(self.n_heads, self.n_rows, *[None if a is None else a.ctypes.data for a in arr], int(window))
        h = _i32()
        _check(_lib.rb_plan_create(self.ctx.handle, pool.handle, C.byref(d), C.byref(h)))
        self.handle = h.value
        self._append, self._attention = _AppendDesc(), _AttentionDesc()
        self._append_ref, self._attention_ref = C.byref(self._append), C.byref(self._attention)

    def append(self, layer: int, k, v, q=None, q_out=None, q_norm=None, k_norm=None, eps: float = 1e-6, rope=None,
               adjacent: bool = False):
        """Norms, rotation and append of the rows (rb_plan_append); returns q_out (made when q is
        given and it is not). rope: [positions][rotary] float32, cosines then sines (rope_table)."""
        n, H, kv, hd = self.n_rows, self.n_heads, self.pool.n_kv, self.pool.hd
        if q is not None and q_out is None:
            if _is_tensor(q):
                import torch
                q_out = torch.empty((n, H, hd), dtype=q.dtype, device=q.device)
            else:
                q_out = np.empty((n, H, hd), q.dtype)
        dt, flags = _dtype((k, v) if q is None else (k, v, q, q_out), self.ctx)
        if q_norm is not None or k_norm is not None or rope is not None:
            _space((k, q_norm, k_norm, rope), self.ctx)
        d = self._append
        d.dtype, d.rope_style, d.eps = dt, int(bool(adjacent)), eps
        d.k, d.ldk = _rows3(k, n, kv, hd, "k")
        d.v, d.ldv = _rows3(v, n, kv, hd, "v")
        d.q, d.ldq = (None, 0) if q is None else _rows3(q, n, H, hd, "q")
        d.q_out, d.ldo = (None, 0) if q is None else _rows3(_writable(q_out, "q_out"), n, H, hd, "q_out")
        d.q_norm, d.k_norm = _vec(q_norm, "float32", hd, "q_norm"), _vec(k_norm, "float32", hd, "k_norm")
        if rope is None:
            d.rope, d.rope_len, d.rotary = None, 0, 0
        else:
            d.rope_len, d.rotary = rope.shape
            d.rope = _vec(rope, "float32", d.rope_len * d.rotary, "rope")
        _call(self.ctx, flags, _lib.rb_plan_append, self.ctx._h, self.handle, layer, self._append_ref)
        return q_out

    def attention(self, layer: int, q, scale: float, softcap: float = 0.0, slopes=None, out=None):
        """Masked attention of the rows over the cache (rb_plan_attention); returns out."""
        n, H, hd = self.n_rows, self.n_heads, self.pool.hd
        if out is None:
            if _is_tensor(q):
                import torch
                out = torch.empty((n, H, hd), dtype=q.dtype, device=q.device)
            else:
                out = np.empty((n, H, hd), q.dtype)
        dt, flags = _dtype((q, out), self.ctx)
        if slopes is not None:
            _space((q, slopes), self.ctx)
        d = self._attention
        d.dtype, d.scale, d.softcap = dt, scale, softcap
        d.q, d.ldq = _rows3(q, n, H, hd, "q")
        d.out, d.ldo = _rows3(_writable(out, "out"), n, H, hd, "out")
        d.slopes = _vec(slopes, "float32", H, "slopes")
        _call(self.ctx, flags, _lib.rb_plan_attention, self.ctx._h, self.handle, layer, self._attention_ref)
        return out

    def close(self):
        """Frees the plan; its pool's tokens stay."""
        h, self.handle = self.handle, -1
        if h >= 0 and self.ctx.handle:
            rc = _lib.rb_plan_destroy(self.ctx.handle, h)
            if rc != BAD_HANDLE:  # gone with its pool
                _check(rc)

    def __del__(self):
        if self.handle >= 0 and _lib is not None:
            self.close()

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()


def rope_table(n_positions: int, rotary: int, theta: float = 10000.0, scaling: float = 1.0, device=None):
    """[n_positions][rotary] float32: cosines, then sines, of position / scaling * theta^(-2i / rotary),
    computed in 64 bits. numpy, or a tensor on `device`."""
    f = theta ** (-np.arange(0, rotary, 2, dtype=np.float64) / max(1, rotary)) / scaling
    a = np.arange(n_positions, dtype=np.float64)[:, None] * f
    t = np.concatenate([np.cos(a), np.sin(a)], 1).astype(np.float32)
    if device is None:
        return t
    import torch
    return torch.from_numpy(t).to(device)


@dataclass
class SamplingFilter:
    """rb_sampling_filter: how a row's token is drawn."""
    temperature: float = 1.0
    top_k: int = 0
    top_p: float = 1.0
    min_p: float = 0.0
    repetition_penalty: float = 1.0

    def c(self) -> _Filter:
        return _Filter(float(self.temperature), int(self.top_k), float(self.top_p), float(self.min_p),
                       float(self.repetition_penalty))


def pack_filters(filters: Sequence[SamplingFilter], device):
    """The filters as a tensor on `device` ([n][20] bytes), for sample_filtered on CUDA tensors."""
    import torch
    if not filters:
        return torch.empty((0, C.sizeof(_Filter)), dtype=torch.uint8, device=device)
    arr = (_Filter * len(filters))(*[f.c() for f in filters])
    return torch.frombuffer(bytearray(arr), dtype=torch.uint8).view(len(filters), C.sizeof(_Filter)).to(device)


def sample_filtered(ctx, logits, filters, uniforms, prev=None, out=None, probs=None):
    """One token per row of logits [n][vocab] (rb_sample_filtered); returns the tokens.

    Host: numpy logits (float32 or float16), a list of SamplingFilter, uniforms, prev as per-row token
    lists; out: a uint32 or int32 array; probs: a float32 array that receives the tokens' probabilities.
    CUDA: tensors; filters from pack_filters, prev a pair (tokens, offsets) of int32 tensors; the call
    does not wait, and a row without a token left holds -1."""
    if not _is_tensor(logits):
        x = np.ascontiguousarray(logits)
        x = x[None] if x.ndim == 1 else x
        n, v = x.shape
        dt, _ = _dtype([x], ctx)
        _space([x, out, probs], ctx)
        if len(filters) != n:
            raise ValueError("one filter per row wanted")
        arr = (_Filter * n)(*[f.c() for f in filters])
        u = np.ascontiguousarray(uniforms, np.float32).reshape(n)
        pf, po = _prev_arrays(prev, n)
        tok = np.empty(n, np.uint32) if out is None else _writable(out, "out")
        at = _vec(tok, "int32" if getattr(tok, "dtype", None) == np.int32 else "uint32", n, "out")
        pp = _vec(_writable(probs, "probs"), "float32", n, "probs")
        _check(_lib.rb_sample_filtered(ctx.handle, dt, x.ctypes.data, v, n, v, arr,
                                       None if pf is None else pf.ctypes.data, None if po is None else po.ctypes.data,
                                       u.ctypes.data, at, pp, PTR_HOST))
        return tok
    import torch
    n, v = logits.shape
    if logits.stride(1) != 1 and v > 1:
        raise ValueError("logits rows have to be contiguous")
    dt, flags = _dtype([logits], ctx)
    if out is None:
        out = torch.empty(n, dtype=torch.int32, device=logits.device)
    prev = prev or (None, None)
    _space([logits, filters, uniforms, out, probs, *prev], ctx)
    if prev[0] is not None and prev[0].numel() == 0 and prev[1] is not None:  # no row has a history; no memory either
        _vec(prev[1], "int32", n + 1, "prev offsets")
        prev = (None, None)
    _call(
        ctx, flags, _lib.rb_sample_filtered, ctx._h, dt, logits.data_ptr(), logits.stride(0) if n > 1 else v, n, v,
        _vec(filters, "uint8", n * C.sizeof(_Filter), "filters"),
        None if prev[0] is None else _vec(prev[0], "int32", prev[0].numel(), "prev tokens"),
        None if prev[1] is None else _vec(prev[1], "int32", n + 1, "prev offsets"),
        _vec(uniforms, "float32", n, "uniforms"), _vec(out, "int32", n, "out"),
        _vec(probs, "float32", n, "probs"))
    return out


def partition(rows, n_heads: int, n_kv: int, num_sms: int, f16_cache: bool) -> np.ndarray:
    """Test hook: the work lists of rows [n][4] (position, first key, one past the last, tenant)."""
    r = np.ascontiguousarray(rows, np.int32)
    n = _check(_lib.rb_plan_partition(len(r), r.ctypes.data, n_heads, n_kv, num_sms, int(f16_cache), None, 0))
    out = np.empty((n, 10), np.int32)
    _check(_lib.rb_plan_partition(len(r), r.ctypes.data, n_heads, n_kv, num_sms, int(f16_cache), out.ctypes.data, n))
    return out

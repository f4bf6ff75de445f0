"""Low-rank adapters of many tenants beside one shared projection.

    adapters = ctx.adapters(n, k, n_slots=64, max_rank=64)       # of a projection [n][k]
    adapters.set(3, down, up, scale=alpha / rank)                # tenant 3's: down [rank][k], up [n][rank]
    y = weight.matmul(x, rows, out=y)
    adapters.add(x, slots, y)                                    # y[r] += scale up (down x[r]) of slots[r]

The reference gives every tenant dequantised weights with the product of its factors added
(crates/realm-runtime/src/lora.rs); here the quantised weight stays shared, and one call
serves rows of any mix of adapters.
"""
from __future__ import annotations

import ctypes as C
import sys

import numpy as np

from . import PTR_DEVICE, _check, _lib, _sig
from .rows import (ASYNC, BAD_HANDLE, _SEEN, _Order, _call, _current_stream, _dtype, _is_tensor, _mat, _rows3, _vec,
                   _writable)

_vp, _u32, _u64, _i32, _f = C.c_void_p, C.c_uint32, C.c_uint64, C.c_int32, C.c_float


class _AdaptersDesc(C.Structure):
    _fields_ = [("dtype", _i32), ("n_rows", _u32), ("slots", _vp), ("x", _vp), ("y", _vp), ("out", _vp),
                ("ldx", _u64), ("ldy", _u64), ("ldo", _u64)]


_sig("rb_adapters_create", [_vp, _u32, _u32, _u32, _u32, C.POINTER(_i32)])
_sig("rb_adapters_destroy", [_vp, _i32])
_sig("rb_adapters_set", [_vp, _i32, _u32, _i32, _u32, _vp, _vp, _f, _u32])
_sig("rb_adapters_clear", [_vp, _i32, _u32])
_sig("rb_adapters_add", [_vp, _i32, C.POINTER(_AdaptersDesc), _u32])
_sig("rb_test_adapters_portable", [_vp, _i32])
_sig("rb_adapters_check", [_vp, _i32, C.POINTER(_AdaptersDesc), _u32])


def _size(v, name, most=0xffffffff):
    if int(v) != v or not 0 <= v <= most:
        raise ValueError(f"{name}: an integer of at least 0 wanted")
    return int(v)


def _change(ctx, flags, fn, *args):
    """_call, for what changes a slot: ordered with torch's current stream also without tensors, since captured calls
    that read the slot are replayed there."""
    torch = sys.modules.get("torch")
    if flags & PTR_DEVICE or torch is None or not torch.cuda.is_initialized() or \
            _current_stream(ctx.device) == ctx._stream_id:
        return _call(ctx, flags, fn, *args)
    order = _Order(ctx)
    rc = fn(*args, flags)
    order.done()
    _check(rc)


class AdapterSet:
    """Adapters of a projection [n][k] in `n_slots` slots of up to `max_rank` (rb_adapters_create), held in fp16.
    Ends with close(), with its context, or when nothing refers to it."""

    handle = -1

    def __init__(self, ctx, n: int, k: int, n_slots: int, max_rank: int):
        self.ctx, self.n, self.k = ctx, _size(n, "n"), _size(k, "k")
        self.n_slots, self.max_rank = _size(n_slots, "n_slots"), _size(max_rank, "max_rank")
        h = _i32()
        _check(_lib.rb_adapters_create(ctx.handle, self.n, self.k, self.n_slots, self.max_rank, C.byref(h)))
        self.handle = h.value
        self._desc = _AdaptersDesc()
        self._ref = C.byref(self._desc)

    def set(self, slot: int, down, up, scale: float = 1.0):
        """Puts an adapter in `slot`: down [rank][k], up [n][rank], contiguous, float16 or float32 (rounded to
        float16 behind a power of two), numpy arrays or CUDA tensors. Calls made before it keep the old one."""
        dt, flags = _dtype((down, up), self.ctx)
        rank = down.shape[0] if len(down.shape) == 2 else -1
        name = str(down.dtype).replace("torch.", "")
        if tuple(down.shape) != (rank, self.k) or tuple(up.shape) != (self.n, rank):
            raise ValueError(f"down [rank][{self.k}] and up [{self.n}][rank] wanted, got {tuple(down.shape)} and "
                             f"{tuple(up.shape)}")
        _change(self.ctx, flags, _lib.rb_adapters_set, self.ctx.handle, self.handle, _size(slot, "slot"), dt, rank,
              _vec(down, name, rank * self.k, "down"), _vec(up, name, rank * self.n, "up"), scale)

    def clear(self, slot: int):
        """Empties a slot; ordered like set()."""
        _change(self.ctx, 0, lambda *a: _lib.rb_adapters_clear(*a[:3]), self.ctx.handle, self.handle, _size(slot, "slot"))

    def add(self, x, slots, y, out=None, _product=None):
        """y with scale up (down x) of every row's adapter added (rb_adapters_add), in place, or in `out`; returns it.

        x [rows][k], y and out [rows][n]: float32 or float16, numpy arrays or CUDA tensors; rows may lie apart.
        slots: int32, -1 for rows without an adapter."""
        if out is None:
            out = y
        n_rows = x.shape[0]
        d = self._desc
        d.n_rows = n_rows
        if _is_tensor(x):
            if not (_is_tensor(y) and _is_tensor(slots) and _is_tensor(out)):
                raise ValueError("host arrays, or tensors on the context's device, wanted: not a mix")
            t, dev, flags = x.dtype, self.ctx.device, PTR_DEVICE | ASYNC
            d.dtype = _SEEN[t] if t in _SEEN else _dtype((x,), self.ctx)[0]
            if slots.get_device() != dev:
                raise ValueError("slots: a tensor on the context's device wanted")
            d.slots = _vec(slots, "int32", n_rows, "slots")
            d.x, d.ldx = _mat(x, n_rows, self.k, t, dev, "x")
            d.y, d.ldy = _mat(y, n_rows, self.n, t, dev, "y")
            d.out, d.ldo = (d.y, d.ldy) if out is y else _mat(out, n_rows, self.n, t, dev, "out")
        else:
            d.dtype, flags = _dtype((x, y, out), self.ctx)
            if _is_tensor(slots):
                raise ValueError("host arrays, or tensors on the context's device, wanted: not a mix")
            given = np.asarray(slots)
            if given.size and (given.dtype.kind not in "iu" or given.min() < -2 ** 31 or given.max() >= 2 ** 31):
                raise ValueError("slots: 32-bit integers wanted")
            slots = np.ascontiguousarray(given, np.int32)
            d.slots = _vec(slots, "int32", n_rows, "slots")
            if n_rows:
                d.x, d.ldx = _rows3(x, n_rows, 1, self.k, "x")
                d.y, d.ldy = _rows3(y, n_rows, 1, self.n, "y")
                d.out, d.ldo = (d.y, d.ldy) if out is y else _rows3(out, n_rows, 1, self.n, "out")
                _writable(out, "out")
        if _product is not None:  # Weight.matmul: writes y once nothing is refused
            _check(_lib.rb_adapters_check(self.ctx.handle, self.handle, self._ref, flags))
            _product()
        _call(self.ctx, flags, _lib.rb_adapters_add, self.ctx.handle, self.handle, self._ref)
        return out

    def close(self):
        h, self.handle = self.handle, -1
        if h >= 0 and self.ctx.handle:
            rc = _lib.rb_adapters_destroy(self.ctx.handle, h)
            if rc != BAD_HANDLE:
                _check(rc)

    def __del__(self):
        if self.handle >= 0 and _lib is not None:
            self.close()

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

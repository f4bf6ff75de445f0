"""The norms around a block with its gate and residual, in one pass.

    x, h = residual_norm(ctx, y, x, post_norm=w1, gate=g, scale=s, pre_norm=w2)

y: the block's output, x: the residual stream; the new stream is x + s g norm(y) w1, and h
its norm by w2, what the next block reads.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import PTR_DEVICE, PTR_HOST, _lib, _sig
from .rows import ASYNC, _DTYPES, _SEEN, _call, _dtype, _is_tensor, _mat, _rows3, _space, _vec, _writable

_vp, _u32, _u64, _i32, _f = C.c_void_p, C.c_uint32, C.c_uint64, C.c_int32, C.c_float


class _ResidualDesc(C.Structure):
    _fields_ = [("dtype", _i32), ("x_dtype", _i32), ("n_rows", _u32), ("dim", _u32), ("y", _vp), ("x", _vp),
                ("gate", _vp), ("x_out", _vp), ("out", _vp), ("ldy", _u64), ("ldx", _u64), ("ldg", _u64),
                ("ldxo", _u64), ("ldo", _u64), ("post_norm", _vp), ("pre_norm", _vp), ("scale", _f), ("eps", _f)]


_sig("rb_residual_norm", [_vp, C.POINTER(_ResidualDesc), _u32])


def _empty(like):
    if _is_tensor(like):
        import torch
        return torch.empty(tuple(like.shape), dtype=like.dtype, device=like.device)
    return np.empty(like.shape, like.dtype)


def residual_norm(ctx, y, x, post_norm=None, gate=None, scale: float = 1.0, pre_norm=None, eps: float = 1e-6,
                  x_out=None, out=None):
    """x_out = x + scale * gate * norm(y) * post_norm and out = norm(x_out) * pre_norm (rb_residual_norm);
    returns (x_out, out), out None without pre_norm.

    y, x [rows][dim], float32 or float16 each, numpy arrays or CUDA tensors; rows may lie apart. post_norm None: y
    as it is. gate: [dim] or [rows][dim] in y's type. x_out has x's type and may be x, out y's type and may be y."""
    if len(y.shape) != 2:
        raise ValueError(f"y: [rows][dim] wanted, got {tuple(y.shape)}")
    n, dim = y.shape
    if x_out is None:
        x_out = _empty(x)
    if pre_norm is None:
        if out is not None:
            raise ValueError("out goes with pre_norm")
    elif out is None:
        out = _empty(y)
    d = _ResidualDesc(n_rows=n, dim=dim, scale=scale, eps=eps)
    if _is_tensor(y):
        _tensors(ctx, d, n, dim, y, x, post_norm, gate, pre_norm, x_out, out)
        flags = PTR_DEVICE | ASYNC
    else:
        _arrays(ctx, d, n, dim, y, x, post_norm, gate, pre_norm, x_out, out)
        flags = PTR_HOST
    _call(ctx, flags, _lib.rb_residual_norm, ctx._h, C.byref(d))
    return x_out, out


def _tensors(ctx, d, n, dim, y, x, post_norm, gate, pre_norm, x_out, out):
    dev, ty, tx = ctx.device, y.dtype, x.dtype
    for a in (x, post_norm, gate, pre_norm, x_out, out):
        if a is not None and not _is_tensor(a):
            raise ValueError("host arrays, or tensors on the context's device, wanted: not a mix")
    d.dtype, d.x_dtype = _type(ty), _type(tx)
    d.y, d.ldy = _mat(y, n, dim, ty, dev, "y")
    d.x, d.ldx = _mat(x, n, dim, tx, dev, "x")
    d.x_out, d.ldxo = _mat(x_out, n, dim, tx, dev, "x_out")
    if out is not None:
        d.out, d.ldo = _mat(out, n, dim, ty, dev, "out")
        d.pre_norm = _weight(pre_norm, dim, dev, "pre_norm")
    if post_norm is not None:
        d.post_norm = _weight(post_norm, dim, dev, "post_norm")
    if gate is not None:
        if gate.dim() == 1:
            d.gate, d.ldg = _mat(gate[None], 1, dim, ty, dev, "gate")[0], 0
        else:
            d.gate, d.ldg = _mat(gate, n, dim, ty, dev, "gate")


def _weight(w, dim, dev, name):
    if w.get_device() != dev:
        raise ValueError(f"{name}: on the context's device wanted")
    return _vec(w, "float32", dim, name)


def _type(t):
    dt = _SEEN.get(t)
    if dt is None:
        dt = _DTYPES.get(str(t))
        if dt is None:
            raise ValueError(f"unsupported type {t}")
        _SEEN[t] = dt
    return dt


def _arrays(ctx, d, n, dim, y, x, post_norm, gate, pre_norm, x_out, out):
    _space((y, x, post_norm, gate, pre_norm, x_out, out), ctx)
    d.dtype, _ = _dtype([a for a in (y, gate, out) if a is not None], ctx)
    d.x_dtype, _ = _dtype((x, x_out), ctx)
    d.post_norm, d.pre_norm = _vec(post_norm, "float32", dim, "post_norm"), _vec(pre_norm, "float32", dim, "pre_norm")
    if not n:
        return
    d.y, d.ldy = _rows3(y, n, 1, dim, "y")
    d.x, d.ldx = _rows3(x, n, 1, dim, "x")
    d.x_out, d.ldxo = _rows3(_writable(x_out, "x_out"), n, 1, dim, "x_out")
    if out is not None:
        d.out, d.ldo = _rows3(_writable(out, "out"), n, 1, dim, "out")
    if gate is not None:
        if len(gate.shape) == 1:
            d.gate, d.ldg = _vec(gate, str(gate.dtype), dim, "gate"), 0
        else:
            d.gate, d.ldg = _rows3(gate, n, 1, dim, "gate")

"""Drafted decoding: a small model (or a lookup in the request's own history) proposes
tokens, the target runs over all of them in one step, and the accepted ones are
distributed as the target's own (crates/realm-runtime/src/speculative.rs has the loop).

    q[:, i] = filter_probs(ctx, draft_logits, filters)        # what draft i was drawn from
    p = filter_probs(ctx, target_logits, filters)             # a row more than drafts, per request
    tokens, accepted = verify_drafts(ctx, p, drafts, uniforms, offsets, draft_probs=q)

The rows of a request that were not accepted stay in the cache; a plan whose positions start
below the cache's length overwrites them.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import PTR_DEVICE, _lib, _sig
from .rows import ASYNC, _Filter, _call, _dtype, _is_tensor, _mat, _rows3, _space, _vec, _writable
from .sampling import _prev_arrays

_vp, _u32, _u64, _i32 = C.c_void_p, C.c_uint32, C.c_uint64, C.c_int32


class _VerifyDesc(C.Structure):
    _fields_ = [("n_requests", _u32), ("n_rows", _u32), ("vocab", _u32), ("offsets", _vp), ("probs", _vp),
                ("draft_probs", _vp), ("ldp", _u64), ("ldq", _u64), ("drafts", _vp), ("uniforms", _vp),
                ("tokens", _vp), ("accepted", _vp)]


_sig("rb_filter_probs", [_vp, _i32, _vp, _u64, _u32, _u32, _vp, _vp, _vp, _vp, _u64, _u32])
_sig("rb_verify_drafts", [_vp, C.POINTER(_VerifyDesc), _u32])


def _matrix(a, name):
    if len(a.shape) != 2:
        raise ValueError(f"{name}: [rows][vocab] wanted, got {tuple(a.shape)}")
    return a.shape


def filter_probs(ctx, logits, filters, prev=None, out=None):
    """The distribution that sample_filtered draws from, for every row of logits [n][vocab] (rb_filter_probs):
    float32 [n][vocab], 0 for tokens that are not kept. Arguments as sample_filtered; rows may lie apart."""
    n, v = _matrix(logits, "logits")
    dt, flags = _dtype([logits], ctx)
    if _is_tensor(logits):
        if out is None:
            import torch
            out = torch.empty((n, v), dtype=torch.float32, device=logits.device)
        prev = prev or (None, None)
        _space([logits, filters, out, *prev], ctx)
        if prev[0] is not None and prev[0].numel() == 0 and prev[1] is not None:  # no row has a history; no memory either
            _vec(prev[1], "int32", n + 1, "prev offsets")
            prev = (None, None)
        fp = _vec(filters, "uint8", n * C.sizeof(_Filter), "filters")
        pt = None if prev[0] is None else _vec(prev[0], "int32", prev[0].numel(), "prev tokens")
        po = None if prev[1] is None else _vec(prev[1], "int32", n + 1, "prev offsets")
    else:
        if out is None:
            out = np.empty((n, v), np.float32)
        _space([logits, out], ctx)
        if len(filters) != n:
            raise ValueError("one filter per row wanted")
        arr = (_Filter * n)(*[f.c() for f in filters])
        tok, off = _prev_arrays(prev, n)
        fp, pt, po = C.addressof(arr), None if tok is None else tok.ctypes.data, None if off is None else off.ctypes.data
    if _dtype([out], ctx)[0] != 0:
        raise ValueError(f"out: float32 wanted, got {out.dtype}")
    if n:
        xp, ldx = _rows3(logits, n, 1, v, "logits")
        op, ldo = _rows3(_writable(out, "out"), n, 1, v, "out")
        _call(ctx, flags, _lib.rb_filter_probs, ctx.handle, dt, xp, ldx, n, v, fp, pt, po, op, ldo)
    return out


def verify_drafts(ctx, probs, drafts, uniforms, offsets, draft_probs=None, tokens=None, accepted=None):
    """Verifies drafted tokens against the target's probabilities (rb_verify_drafts); returns (tokens, accepted).

    Request r has the rows offsets[r] .. offsets[r + 1] of probs [rows][vocab] (float32), one more than drafts.
    drafts, uniforms [rows]: of row i the token drafted there and the random number that tests it; a request's
    last row has no draft, and its uniform draws the request's token. draft_probs [rows][vocab]: what the drafts were drawn
    from, or None. tokens [rows]: the accepted drafts, the drawn token, then -1; accepted [requests]: how many drafts.
    CUDA tensors (drafts, offsets, tokens, accepted int32; the call does not wait), or numpy arrays."""
    n, v = _matrix(probs, "probs")
    m = len(offsets) - 1
    if m < 0:
        raise ValueError("offsets: one more than requests wanted")
    d = _VerifyDesc(n_requests=m, n_rows=n, vocab=v)
    if _is_tensor(probs):
        import torch
        dev, flags, f32 = ctx.device, PTR_DEVICE | ASYNC, torch.float32
        if tokens is None:
            tokens = torch.full((n,), -1, dtype=torch.int32, device=probs.device)
        if accepted is None:
            accepted = torch.empty(m, dtype=torch.int32, device=probs.device)
        _space([probs, drafts, uniforms, offsets, draft_probs, tokens, accepted], ctx)
        d.probs, d.ldp = _mat(probs, n, v, f32, dev, "probs")
        if draft_probs is not None:
            d.draft_probs, d.ldq = _mat(draft_probs, n, v, f32, dev, "draft_probs")
    else:
        drafts, offsets = (np.ascontiguousarray(a, np.int32) if not _is_tensor(a) else a for a in (drafts, offsets))
        uniforms = uniforms if _is_tensor(uniforms) else np.ascontiguousarray(uniforms, np.float32)
        tokens = np.full(n, -1, np.int32) if tokens is None else tokens
        accepted = np.empty(m, np.int32) if accepted is None else accepted
        flags = _space([probs, drafts, uniforms, offsets, draft_probs, tokens, accepted], ctx)
        if _dtype([probs] if draft_probs is None else [probs, draft_probs], ctx)[0] != 0:
            raise ValueError(f"probs: float32 wanted, got {probs.dtype}")
        if draft_probs is not None and _matrix(draft_probs, "draft_probs") != (n, v):
            raise ValueError(f"draft_probs: [{n}][{v}] wanted, got {tuple(draft_probs.shape)}")
        if n:
            d.probs, d.ldp = _rows3(probs, n, 1, v, "probs")
            if draft_probs is not None:
                d.draft_probs, d.ldq = _rows3(draft_probs, n, 1, v, "draft_probs")
    d.offsets = _vec(offsets, "int32", m + 1, "offsets")
    d.drafts = _vec(drafts, "int32", n, "drafts")
    d.uniforms = _vec(uniforms, "float32", n, "uniforms")
    d.tokens = _vec(_writable(tokens, "tokens"), "int32", n, "tokens")
    d.accepted = _vec(_writable(accepted, "accepted"), "int32", m, "accepted")
    _call(ctx, flags, _lib.rb_verify_drafts, ctx.handle, C.byref(d))
    return tokens, accepted

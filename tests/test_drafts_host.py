"""What the operators of a step with adapters and drafts check on the host, without a GPU."""
import ctypes as C

import numpy as np
import pytest


class _Ctx:
    """Stands in for a context where a call has to be refused before it reaches the library, or by it."""
    handle, _h, device, _stream_id = None, None, 0, 0


def _refused(fn, *a, **kw):
    """The library's own refusal: there is no context."""
    import realm_b200 as rb
    with pytest.raises(rb.RealmError) as e:
        fn(*a, **kw)
    assert e.value.code == -20


def test_residual_norm_arguments():
    import realm_b200 as rb
    y, x, w = np.ones((4, 64), np.float32), np.ones((4, 64), np.float16), np.ones(64, np.float32)
    _refused(rb.residual_norm, _Ctx, y, x, post_norm=w, gate=w, pre_norm=w)
    _refused(rb.residual_norm, _Ctx, y, x, gate=y)
    for kw in (dict(pre_norm=w[1:]), dict(post_norm=w.astype(np.float64)), dict(gate=w.astype(np.float16)), dict(out=y.copy()),
               dict(x_out=y.copy()), dict(gate=np.ones((3, 64), np.float32)), dict(pre_norm=w, out=x.copy())):
        with pytest.raises(ValueError):
            rb.residual_norm(_Ctx, y, x, **kw)
    for a, b in ((y[0], x[0]), (y[:3], x), (y.astype(np.int32), x), (y.T.copy().T, x), (y, x[:, :32])):
        with pytest.raises(ValueError):
            rb.residual_norm(_Ctx, a, b)


def test_verify_drafts_arguments():
    import realm_b200 as rb
    p, d, u, o = np.ones((5, 9), np.float32), np.zeros(5, int), np.zeros(5), [0, 3, 5]
    _refused(rb.verify_drafts, _Ctx, p, d, u, o)
    _refused(rb.verify_drafts, _Ctx, p, d, u, o, draft_probs=p.copy())
    for kw in (dict(draft_probs=p[:4]), dict(draft_probs=p.astype(np.float16)), dict(tokens=np.zeros(4, np.int32)),
               dict(tokens=np.zeros(5, np.int64)), dict(accepted=np.zeros(3, np.int32))):
        with pytest.raises(ValueError):
            rb.verify_drafts(_Ctx, p, d, u, o, **kw)
    for a in ((p[0], d, u, o), (p.astype(np.float64), d, u, o), (p, d[1:], u, o), (p, d, u[1:], o), (p, d, u, []), (p[:, ::2], d, u, o)):
        with pytest.raises(ValueError):
            rb.verify_drafts(_Ctx, *a)


def test_filter_probs_arguments():
    import realm_b200 as rb
    x, f = np.ones((2, 9), np.float16), [rb.SamplingFilter()] * 2
    _refused(rb.filter_probs, _Ctx, x, f)
    _refused(rb.filter_probs, _Ctx, x, f, prev=[[1], []])
    for a, kw in (((x, f[:1]), {}), ((x[0], f), {}), ((x.astype(np.int32), f), {}), ((x, f), dict(out=np.ones((2, 9), np.float16))),
                  ((x, f), dict(out=np.ones((2, 8), np.float32)))):
        with pytest.raises(ValueError):
            rb.filter_probs(_Ctx, *a, **kw)


def test_adapters_arguments():
    import realm_b200 as rb
    _refused(rb.AdapterSet, _Ctx, 64, 128, 4, 8)
    for a in ((-1, 128, 4, 8), (64, 128, 4.5, 8), (64, 2 ** 33, 4, 8)):
        with pytest.raises(ValueError):
            rb.AdapterSet(_Ctx, *a)
    s = rb.AdapterSet.__new__(rb.AdapterSet)  # as one whose library object is gone
    s.ctx, s.n, s.k, s.n_slots, s.max_rank = _Ctx, 64, 128, 4, 8
    from realm_b200.adapters import _AdaptersDesc
    s._desc = _AdaptersDesc()
    s._ref = C.byref(s._desc)
    x, y = np.ones((3, 128), np.float32), np.ones((3, 64), np.float32)
    _refused(s.add, x, [0, -1, 3], y)
    _refused(s.set, 0, np.ones((8, 128), np.float16), np.ones((64, 8), np.float16))
    _refused(s.clear, 1)
    for a in ((x, [0, 1], y), (x, np.array([2**40, 0, 0]), y), (x, [0.5, 0, 0], y), (x, [2 ** 40, 0, 0], y), (x[:, :64], [0, 0, 0], y), (x, [0, 0, 0], y[:2]),
              (x.astype(np.float16), [0, 0, 0], y)):
        with pytest.raises(ValueError):
            s.add(*a)
    for a in ((np.ones((8, 127), np.float32), np.ones((64, 8), np.float32)), (np.ones((8, 128), np.float32), np.ones((64, 7), np.float32)),
              (np.ones((8, 128), np.float32), np.ones((64, 8), np.float16)), (np.ones(128, np.float32), np.ones((64, 1), np.float32))):
        with pytest.raises(ValueError):
            s.set(0, *a)
    with pytest.raises(ValueError, match="slot"):
        s.clear(-1)


def test_null_pointers_and_descriptors():
    """The C entries refuse what a binding might pass; none of these reach a device."""
    from realm_b200 import _lib
    n = C.c_int32()
    assert _lib.rb_adapters_create(None, 1, 1, 1, 1, C.byref(n)) == -20
    assert _lib.rb_adapters_destroy(None, 0) == -20
    assert _lib.rb_adapters_set(None, 0, 0, 0, 1, None, None, 1.0, 0) == -20
    assert _lib.rb_adapters_clear(None, 0, 0) == -20
    assert _lib.rb_adapters_add(None, 0, None, 0) == -20
    assert _lib.rb_verify_drafts(None, None, 0) == -20
    assert _lib.rb_residual_norm(None, None, 0) == -20
    assert _lib.rb_filter_probs(None, 0, None, 0, 0, 0, None, None, None, None, 0, 0) == -20

"""What a projection with adapters refuses on the host, without a GPU: before the product is asked for."""
import ctypes as C

import numpy as np
import pytest


class _Ctx:
    """Stands in for a context: the library refuses what reaches it."""
    handle, _h, device, _stream_id = None, None, 0, 0


def _pair():
    import realm_b200 as rb
    from realm_b200.adapters import _AdaptersDesc
    w, s = rb.Weight.__new__(rb.Weight), rb.AdapterSet.__new__(rb.AdapterSet)
    w.ctx, w.n, w.k, w.handle = _Ctx, 64, 128, 0
    s.ctx, s.n, s.k, s.n_slots, s.max_rank = _Ctx, 64, 128, 4, 8
    s._desc = _AdaptersDesc()
    s._ref = C.byref(s._desc)
    return w, s


def test_arguments():
    import realm_b200 as rb
    w, s = _pair()
    w._product = lambda *a: pytest.fail("the product was asked for")
    x, out = np.ones((3, 128), np.float32), np.ones((3, 64), np.float32)
    with pytest.raises(rb.RealmError) as e:  # all is well but for the context
        w.matmul(x, 3, out=out, adapters=s, slots=[0, -1, 1])
    assert e.value.code == -20
    for a, o, slots in ((x[:2], out, [0, 0, 0]), (x, out[:2], [0, 0, 0]), (x, out, [0, 0]), (x, out, [0.5, 0, 0]),
                        (x, out.astype(np.float16), [0, 0, 0]), (x, out.astype(np.float64), [0, 0, 0]), (x, out, None)):
        with pytest.raises(ValueError):
            w.matmul(a, 3, out=o, adapters=s, slots=slots)
    with pytest.raises(ValueError, match="together"):
        w.matmul(x, 3, out=out, slots=[0, 0, 0])


def test_the_check_alone():
    from realm_b200 import _lib
    assert _lib.rb_adapters_check(None, 0, None, 0) == -20

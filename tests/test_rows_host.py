"""What row plans and the operators' bindings check on the host, without a GPU."""
import os
import subprocess
import sys

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class _Pool:
    """Stands in for a pool where a call has to be refused before it reaches the library."""
    n_kv, hd, handle = 2, 64, 0

    class ctx:
        handle, _h, device = None, None, 0


@pytest.mark.parametrize("name", ["tenants", "positions", "begin", "end"])
@pytest.mark.parametrize("bad", [np.array([3, -1]), np.array([0, 2 ** 32]), np.array([-5, 0], np.int8), [1, -2], [0.5, 1.0],
                                 np.array([1.0, 2.0]), [[0, 1]], np.array([True, False])])
def test_rows_that_are_not_indices_are_refused(name, bad):
    """Before, a begin of -1 wrapped around to a key past all others, and the row saw none."""
    from realm_b200 import RowPlan
    rows = dict(tenants=[0, 1], positions=[4, 5], begin=[0, 0], end=[5, 6])
    with pytest.raises(ValueError, match=name):
        RowPlan(_Pool, n_heads=4, **dict(rows, **{name: bad}))


@pytest.mark.parametrize("bad", [-1, 2 ** 32, 1.5])
def test_windows_that_are_not_lengths_are_refused(bad):
    from realm_b200 import RowPlan
    with pytest.raises(ValueError, match="window"):
        RowPlan(_Pool, [0, 1], 4, window=bad)


def test_integer_rows_of_any_type_reach_the_library():
    import realm_b200 as rb
    for t in (np.int8, np.int64, np.uint64, np.uint32, list, tuple):
        a = t([0, 1]) if t in (list, tuple) else np.array([0, 1], t)
        with pytest.raises(rb.RealmError) as e:  # there is no context
            rb.RowPlan(_Pool, a, 4, positions=a, end=a, window=np.int64(7))
        assert e.value.code == -20


def test_no_memory_is_an_error_not_an_abort():
    """The work lists of many short runs do not fit the address space that the process may use."""
    code = """
import resource, sys
sys.path.insert(0, %r)
import numpy as np, realm_b200 as rb
from realm_b200 import rows as R
n = 1 << 19
rows = np.zeros((n, 4), np.int32)
rows[:, 2], rows[:, 3] = 1, np.arange(n) %% 2
have = int(open("/proc/self/statm").read().split()[0]) * resource.getpagesize()
resource.setrlimit(resource.RLIMIT_AS, (have + (64 << 20),) * 2)
try:
    R.partition(rows, 64, 8, 148, False)
except rb.RealmError as e:
    print("refused", e.code)
""" % ROOT
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "refused -26", (r.returncode, r.stdout, r.stderr[-500:])


def _plan(n_rows, n_heads=2):
    """A plan without a library behind it: its calls get past the binding's checks and then fail (-20)."""
    from realm_b200 import RowPlan, rows as R
    p = RowPlan.__new__(RowPlan)
    p.pool, p.ctx, p.n_heads, p.n_rows = _Pool, _Pool.ctx, n_heads, n_rows
    p._append, p._attention = R._AppendDesc(), R._AttentionDesc()
    p._append_ref, p._attention_ref = R.C.byref(p._append), R.C.byref(p._attention)
    return p


def _code(f):
    import realm_b200 as rb
    with pytest.raises(rb.RealmError) as e:
        f()
    return e.value.code


def test_rows_that_lie_parts_of_an_element_apart_are_refused():
    """A field of packed records: 515 bytes from row to row. Before, the 3 were dropped and other memory was read."""
    x = np.zeros(3, [("q", "f4", (2, 64)), ("tail", "u1", 3)])["q"]
    k = np.zeros((3, 2, 64), np.float32)
    for f in (lambda p: p.append(0, x, k), lambda p: p.append(0, k, x), lambda p: p.append(0, k, k, q=x),
              lambda p: p.attention(0, x, 1.0), lambda p: p.attention(0, k, 1.0, out=x)):
        with pytest.raises(ValueError, match="515"):
            f(_plan(3))
    wide = np.zeros((3, 2, 64 + 64), np.float32)
    assert _code(lambda: _plan(3).append(0, k, k, q=k)) == -20 and wide[:, 0, :64].strides == (1024, 4)
    assert _code(lambda: _plan(3).append(0, wide.reshape(3, 256)[:, :128].reshape(3, 2, 64), k)) == -20


def test_read_only_outputs_are_refused():
    """Before, the library wrote into them (a mapped file's pages, or memory that others share)."""
    import realm_b200 as rb
    k = np.zeros((3, 2, 64), np.float32)
    ro = np.frombuffer(bytes(k.nbytes), np.float32).reshape(k.shape)
    assert not ro.flags.writeable
    for f in (lambda: _plan(3).append(0, k, k, q=k, q_out=ro), lambda: _plan(3).attention(0, k, 1.0, out=ro),
              lambda: rb.sample_filtered(_Pool.ctx, np.zeros((2, 5), np.float32), [rb.SamplingFilter()] * 2, [0.1, 0.2],
                                         probs=np.frombuffer(bytes(8), np.float32))):
        with pytest.raises(ValueError, match="read-only"):
            f()
    assert _code(lambda: _plan(3).append(0, ro, ro, q=ro, q_out=k.copy())) == -20  # inputs may be


@pytest.mark.parametrize("heads,kv,rows", [(32, 8, 2000), (8, 1, 512), (4, 4, 3000)])
def test_units_of_long_contexts_are_bounded(heads, kv, rows):
    """Many rows over 131072 keys and more: no unit of the tile kernel takes more than 32768 keys, so that its sums on the
    tensor core stay short; each key is in one unit."""
    from realm_b200 import rows as R
    end = 140001
    pos = np.arange(end - rows, end)
    r = np.stack([pos, np.zeros(rows, int), pos + 1, np.zeros(rows, int)], 1)
    units = R.partition(r, heads, kv, 148, True)
    assert (units[:, 0] == 1).all()
    k0, k1 = units[:, 7], units[:, 8]
    assert (k1 - k0).max() <= 256 * 128
    items = {}
    for u in units:
        items.setdefault((u[2], u[3], u[5]), []).append((u[7], u[8]))
    for spans in items.values():
        spans.sort()
        assert spans[0][0] == 0 and all(a[1] == b[0] for a, b in zip(spans, spans[1:])) and len(spans) >= 5

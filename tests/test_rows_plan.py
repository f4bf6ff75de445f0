"""Work lists of row plans (rb_plan_partition, host code): every row sees each of
its keys in exactly one unit, no unit leaves its item's keys, and partial results
get slots of their own."""
import numpy as np
import pytest


def _rows(spec):
    """spec: (tenant, positions, lo, hi) per row."""
    return np.array([[p, lo, hi, t] for t, p, lo, hi in spec], np.int32)


def _causal(tenant, first, n, window=0):
    return [(tenant, p, max(0, p - window + 1) if window else 0, p + 1) for p in range(first, first + n)]


CASES = {
    "one token": _causal(0, 0, 1),
    "one long": _causal(3, 5000, 1),
    "mixed decode": sum([_causal(t, 100 * t + 7, 1) for t in range(13)], []),
    "no keys": [(0, 4, 0, 0)],
    "no keys in a run": [(0, 4, 0, 5), (0, 5, 0, 0), (0, 6, 0, 7)],
    "prompt": _causal(0, 0, 300),
    "chunk after context": _causal(1, 4000, 77),
    "window": _causal(0, 1000, 64, window=33),
    "documents": [(0, p, p // 50 * 50, p + 1) for p in range(260)],
    "prefix": [(0, p, 0, max(p + 1, 40)) for p in range(90)],
    "decode and prompt": _causal(0, 900, 1) + _causal(1, 0, 200) + _causal(2, 17, 3),
    "same tenant twice": _causal(0, 10, 2) + _causal(1, 5, 1) + _causal(0, 40, 2),
}


@pytest.mark.parametrize("name", CASES)
@pytest.mark.parametrize("heads,kv", [(1, 1), (8, 8), (32, 8), (12, 2), (40, 1)])
@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("sms", [1, 148])
def test_units_cover_every_key_once(name, heads, kv, f16, sms):
    from realm_b200 import rows as R
    rows = _rows(CASES[name])
    rep = heads // kv
    units = R.partition(rows, heads, kv, sms, f16)
    seen = [[np.zeros(max(1, hi), np.int64) for _ in range(heads)] for _, _, hi, _ in rows]
    touched = np.zeros((len(rows), heads), np.int64)
    slots = set()
    direct = np.zeros((len(rows), heads), np.int64)
    for kind, cta, row0, v0, nv, kvh, tenant, k0, k1, slot in units:
        assert k0 % 16 == 0 and 0 <= k0 <= k1 and 0 <= kvh < kv and 0 < nv <= (256 if kind else 8) and 0 <= v0 < rep
        assert f16 or kind == 0
        if slot >= 0:
            mine = set(range(slot, slot + nv))
            assert not mine & slots
            slots |= mine
        for i in range(nv):
            row, head = row0 + (v0 + i) // rep, kvh * rep + (v0 + i) % rep
            assert rows[row][3] == tenant
            lo, hi = max(k0, rows[row][1]), min(k1, rows[row][2])
            if hi > lo:
                seen[row][head][lo:hi] += 1
            touched[row, head] += 1
            direct[row, head] += slot < 0
    for r, (pos, lo, hi, t) in enumerate(rows):
        for h in range(heads):
            if hi > lo:
                assert (seen[r][h][lo:hi] == 1).all() and not seen[r][h][:lo].any()
            assert touched[r, h] >= 1
            assert direct[r, h] == (touched[r, h] == 1)  # one unit writes the output, several leave parts
    assert slots == set(range(len(slots)))


def test_warps_share_pages_evenly():
    from realm_b200 import rows as R
    rows = _rows(sum([_causal(t, 511 + 480 * t, 1) for t in range(16)], []))
    units = R.partition(rows, 32, 8, 148, True)
    load = np.zeros(units[:, 1].max() + 1, np.int64)
    np.add.at(load, units[:, 1], (units[:, 8] - units[:, 7] + 15) // 16)
    # warps in groups of eight, one a kv head, on the same keys
    assert (units[:, 5] == units[:, 1] % 8).all()
    assert len(load) == 2 * 4 * 148 and load.max() - load.min() <= 1


def test_refusals():
    import realm_b200 as rb
    from realm_b200 import rows as R
    with pytest.raises(rb.RealmError):
        R.partition(_rows(_causal(0, 0, 1)), 3, 2, 148, True)
    with pytest.raises(rb.RealmError):
        R.partition(_rows(_causal(0, 0, 1)), 0, 1, 148, True)


def test_rope_table_is_correct_at_long_positions():
    import realm_b200 as rb
    t = rb.rope_table(70001, 64, theta=1e6)
    i = 70000 * (1e6 ** (-2.0 * 3 / 64))
    assert abs(t[70000, 3] - np.cos(i)) < 1e-7 and abs(t[70000, 35] - np.sin(i)) < 1e-7

"""GPU tests of the row plans' operators against plain forms in 64 bits.

Bounds, with u = 2^-24 (fp32) and h = 2^-11 (half an ulp of fp16, relative):
- append: the sum of squares, the inverse root and the rotation are a few dozen
  fp32 roundings, bounded by 64 u of the largest value; fp16 results add h.
- attention, fp32 rows: a score of hd products is off by at most
  e = (hd u + 2^-21) scale sum |q||k| (sums in fp32, operands split into two
  halves of 11 bits) plus 2^-20 of its own size for cap and bias; a weight by twice
  that, so an output by (2 e + 2^-19) max |v|. fp16 rows: the probabilities and
  the result are rounded to fp16 as well: + h max |v| each.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U, HALF = 2.0 ** -24, 2.0 ** -11


def _np(x):
    return x.detach().cpu().double().numpy() if hasattr(x, "detach") else np.asarray(x, np.float64)


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------
def _append_ref(x, w, rope, pos, adjacent):
    x = x.astype(np.float64)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-5) * w.astype(np.float64)
    if rope is not None and rope.shape[1]:
        half = rope.shape[1] // 2
        c, s = rope[pos, :half].astype(np.float64)[:, None], rope[pos, half:].astype(np.float64)[:, None]
        i = np.arange(half)
        i, j = (2 * i, 2 * i + 1) if adjacent else (i, i + half)
        a, b = x[..., i].copy(), x[..., j].copy()
        x[..., i], x[..., j] = a * c - b * s, b * c + a * s
    return x


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("typ,cache", [("float16", "F16"), ("float32", "F16"), ("float32", "F32"), ("float16", "F32")])
@pytest.mark.parametrize("norm,rotary,adjacent", [(True, 1.0, False), (False, 0.5, True), (True, 8, False), (True, 8, True),
                                                  (False, 0, False), (True, 1.0, True), (False, 24, False)])
def test_append(ctx, hd, typ, cache, norm, rotary, adjacent):
    import torch
    import realm_b200 as rb
    rng = np.random.default_rng(hd + len(typ) + int(8 * rotary))
    H, kv, lens = 6, 3, [1, 16, 37]
    rot = int(rotary * hd) if isinstance(rotary, float) else rotary
    pool = ctx.kv_pool(2, kv, hd, getattr(rb, cache), n_pages=32, max_tenants=4, max_seq=128)
    try:
        pool.shuffle(5)
        rope = rb.rope_table(128, rot) if rot else None
        wq, wk = (rng.normal(1, 0.3, hd).astype(np.float32) for _ in range(2)) if norm else (None, None)
        seen = {t: ([], []) for t in range(3)}
        for t in range(3):
            pool.create(t)
        for step in range(2):  # the second step continues the first
            tenant = np.concatenate([np.full(n, t) for t, n in enumerate(lens)])
            pos = np.concatenate([np.arange(n) + step * n for n in lens])
            n = len(tenant)
            x = (rng.normal(0, 2, (n, H + 2 * kv, hd))).astype(typ)
            dev = torch.from_numpy(x).cuda()
            d = lambda a: None if a is None else torch.from_numpy(a).cuda()  # noqa: E731
            with pool.plan(tenant, H, positions=pos if step else None) as plan:
                got = plan.append(1, dev[:, H:H + kv], dev[:, H + kv:], q=dev[:, :H], q_norm=d(wq), k_norm=d(wk),
                                  eps=1e-5, rope=d(rope), adjacent=adjacent)
            got = _np(got)
            ref = _append_ref(x[:, :H], wq, rope, pos, adjacent)
            top = np.abs(ref).max()
            tol = 64 * U * top + (HALF * np.abs(ref) if typ == "float16" else 0) + 2.0 ** -24
            assert (np.abs(got - ref) <= tol).all(), np.abs(got - ref).max()
            kref = _append_ref(x[:, H:H + kv], wk, rope, pos, adjacent)
            for t in range(3):
                seen[t][0].append(kref[tenant == t])
                seen[t][1].append(x[tenant == t, H + kv:].astype(np.float64))
        for t in range(3):
            assert pool.len(t, 1) == 2 * lens[t] and pool.len(t, 0) == 0
            k, v = (a.reshape(-1, kv, hd).astype(np.float64) for a in pool.gather(t, 1))
            kr, vr = np.concatenate(seen[t][0]), np.concatenate(seen[t][1])
            tol = 64 * U * np.abs(kr).max() + (HALF * np.abs(kr) if cache == "F16" else 0) + 2.0 ** -24
            assert (np.abs(k - kr) <= tol).all()
            assert (v == (vr.astype(np.float16) if cache == "F16" else vr)).all()
    finally:
        pool.close()


def test_append_host_arrays_in_place_and_overwrite(ctx):
    import torch
    import realm_b200 as rb
    rng = np.random.default_rng(3)
    pool = ctx.kv_pool(1, 2, 64, rb.F32, n_pages=8, max_tenants=1, max_seq=64)
    try:
        pool.create(0)
        x = rng.normal(0, 1, (20, 4, 64)).astype(np.float32)
        rope = rb.rope_table(64, 64)
        with pool.plan([0] * 20, 2) as plan:
            q = plan.append(0, x[:, 2:3].repeat(2, 1), x[:, 3:4].repeat(2, 1), q=x[:, :2], rope=rope)
        ref = _append_ref(x[:, :2], None, rope, np.arange(20), False)
        assert np.abs(q - ref).max() <= 64 * U * np.abs(ref).max()
        # positions below the length are overwritten, the length stays
        y = torch.randn(3, 2, 64, device="cuda")
        z = y.clone()
        with pool.plan([0] * 3, 2, positions=[10, 11, 12]) as plan:
            plan.append(0, y, y, q=z, q_out=z)
        assert torch.equal(y, z)
        k, v = (a.reshape(20, 2, 64) for a in pool.gather(0, 0))
        assert pool.len(0) == 20 and (k[10:13] == y.cpu().numpy()).all() and (v[:10] == x[:10, 3:4]).all()
    finally:
        pool.close()


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def _attn_ref(q, k, v, pos, lo, hi, scale, cap, slopes):
    """q [n][H][hd], k, v [L][kv][hd] of one tenant; 64 bits. Returns out and the largest sum |q||k| scale."""
    n, H, hd = q.shape
    rep = H // k.shape[1]
    out = np.zeros((n, H, hd))
    amp = 0.0
    for r in range(n):
        if hi[r] <= lo[r]:
            continue
        for h in range(H):
            kk, vv = k[lo[r]:hi[r], h // rep], v[lo[r]:hi[r], h // rep]
            x = kk @ q[r, h] * scale
            amp = max(amp, (np.abs(kk) @ np.abs(q[r, h])).max() * abs(scale))
            if cap:
                x = cap * np.tanh(x / cap)
            if slopes is not None:
                x = x - slopes[h] * np.abs(pos[r] - np.arange(lo[r], hi[r]))
            p = np.exp(x - x.max())
            out[r, h] = p @ vv / p.sum()
    return out, amp


def _check_attention(ctx, hd, H, kv, typ, cache, tenants, cap=0.0, bias=False, window=0, q_scale=1.0, strided=False,
                     dirty=None, seed=0, scale=None):
    """tenants: (cached length, rows' positions, begin, end) each; begin/end None: the defaults."""
    import torch
    import realm_b200 as rb
    rng = np.random.default_rng(seed + hd + H)
    L = [t[0] for t in tenants]
    pool = ctx.kv_pool(1, kv, hd, rb.F16 if cache == "F16" else rb.F32, n_pages=sum((n + 15) // 16 for n in L) + 2,
                       max_tenants=len(L), max_seq=max(L) + 16)
    try:
        pool.shuffle(seed + 1)
        if dirty is not None:
            pool.pages().fill_(dirty)
        ct = np.float16 if cache == "F16" else np.float32
        K = [rng.normal(0, 1, (n, kv, hd)).astype(ct) for n in L]
        V = [rng.normal(0, 1, (n, kv, hd)).astype(ct) for n in L]
        for t, n in enumerate(L):
            pool.create(t)
            with pool.plan([t] * n, H) as p:
                p.append(0, torch.from_numpy(K[t]).cuda(), torch.from_numpy(V[t]).cuda())
        ten = np.concatenate([np.full(len(t[1]), i) for i, t in enumerate(tenants)])
        pos = np.concatenate([np.asarray(t[1]) for t in tenants])
        beg = np.concatenate([np.zeros(len(t[1]), int) if t[2] is None else np.asarray(t[2]) for t in tenants])
        end = np.concatenate([np.asarray(t[1]) + 1 if t[3] is None else np.asarray(t[3]) for t in tenants])
        n = len(ten)
        q = (rng.normal(0, q_scale, (n, H, hd))).astype(typ)
        slopes = (2.0 ** -np.arange(1, H + 1)).astype(np.float32) if bias else None
        scale = 1 / np.sqrt(hd) if scale is None else scale
        dq = torch.from_numpy(q).cuda()
        out = None
        if strided:
            wide = torch.full((n, H * hd + 24), 7.0, dtype=dq.dtype, device="cuda")
            wide[:, 8:8 + H * hd] = dq.reshape(n, -1)
            dq = wide[:, 8:8 + H * hd]
            outw = torch.full((n, H * hd + 9), 7.0, dtype=dq.dtype, device="cuda")
            out = outw[:, 3:3 + H * hd]
        with pool.plan(ten, H, positions=pos, begin=beg, end=end, window=window) as plan:
            got = plan.attention(0, dq, scale, softcap=cap, slopes=None if slopes is None else torch.from_numpy(slopes).cuda(),
                                 out=out)
            again = plan.attention(0, dq, scale, softcap=cap,
                                   slopes=None if slopes is None else torch.from_numpy(slopes).cuda()).clone()
        if strided:
            assert (outw[:, :3] == 7).all() and (outw[:, 3 + H * hd:] == 7).all()
        got = got.reshape(n, H, hd)
        assert torch.equal(got, again.reshape(n, H, hd))  # no order of atomics in the result
        got = _np(got)
        ref, amp, vmax = np.zeros((n, H, hd)), 0.0, 0.0
        for t in range(len(L)):
            m = ten == t
            lo = np.maximum(beg[m], pos[m] - window + 1) if window else beg[m]
            ref[m], a = _attn_ref(q[m].astype(np.float64), K[t].astype(np.float64), V[t].astype(np.float64), pos[m],
                                  np.minimum(lo, end[m]), end[m], scale, cap, slopes)
            amp, vmax = max(amp, a), max(vmax, float(np.abs(V[t]).max()) if L[t] else 0.0)
        far = max(L) * (0.5 if bias else 0.0)
        e = (hd * U + 2.0 ** -21) * amp + 2.0 ** -20 * (amp + far)
        tol = (2 * e + 2.0 ** -19) * vmax + (2 * HALF * vmax if typ == "float16" else 0)
        assert np.isfinite(got).all()
        assert np.abs(got - ref).max() <= tol, (np.abs(got - ref).max(), tol)
        norm = np.linalg.norm(ref)
        if norm:
            rel = np.linalg.norm(got - ref) / norm
            # 1e-5: fp32 sums; a score is known to 2^-22 of its parts, a weight to twice that; fp16:
            # two roundings of independent sign, each at most h, 0.6 h in the mean square
            assert rel <= 1e-5 + 2.0 ** -21 * (amp + cap + far) + (0 if typ == "float32" else 1.2 * HALF), rel
    finally:
        pool.close()


TYPES = [("float16", "F16"), ("float32", "F16"), ("float32", "F32"), ("float16", "F32")]


@pytest.mark.parametrize("typ,cache", TYPES)
@pytest.mark.parametrize("hd,H,kv", [(64, 4, 4), (128, 8, 2), (128, 5, 1), (64, 24, 2), (128, 48, 1)])
@pytest.mark.parametrize("cap,bias,window", [(0.0, False, 0), (30.0, False, 0), (0.0, True, 0), (5.0, True, 50)])
def test_single_tokens(ctx, typ, cache, hd, H, kv, cap, bias, window):
    lens = [1, 15, 16, 17, 63, 200, 777]
    _check_attention(ctx, hd, H, kv, typ, cache, [(n, [n - 1], None, None) for n in lens], cap, bias, window, q_scale=2.0)


@pytest.mark.parametrize("typ,cache", TYPES)
@pytest.mark.parametrize("hd,H,kv", [(64, 2, 2), (128, 4, 1), (128, 6, 2), (64, 16, 1)])
@pytest.mark.parametrize("cap,bias", [(0.0, False), (20.0, False), (0.0, True)])
def test_prompts(ctx, typ, cache, hd, H, kv, cap, bias):
    """Whole prompts, a chunk after cached tokens, a single row: lengths around tile and page edges."""
    t = [(n, np.arange(n), None, None) for n in (1, 2, 33, 127, 130, 260)]
    t += [(300, np.arange(211, 300), None, None), (140, [139], None, None)]
    _check_attention(ctx, hd, H, kv, typ, cache, t, cap, bias, q_scale=2.0, strided=True)


@pytest.mark.parametrize("typ,cache", TYPES)
@pytest.mark.parametrize("hd,H,kv", [(64, 4, 4), (128, 8, 2)])
@pytest.mark.parametrize("kind", ["document", "prefix", "window", "empty", "reversed", "sparse"])
def test_masks(ctx, typ, cache, hd, H, kv, kind):
    n = 290
    pos = np.arange(n)
    beg = end = None
    window = 0
    if kind == "document":
        beg = pos // 37 * 37
    elif kind == "prefix":
        end = np.maximum(pos + 1, 150)
    elif kind == "window":
        window = 20
    elif kind == "empty":  # every third row sees nothing
        end = np.where(pos % 3 == 1, 0, pos + 1)
    elif kind == "reversed":  # rows in no order, one of them twice
        pos = np.concatenate([pos[::-1], [100, 100]])
    else:
        pos = np.array([3, 250, 17, 289, 0])
        beg, end = np.array([2, 200, 17, 0, 0]), np.array([3, 290, 18, 290, 1])
    _check_attention(ctx, hd, H, kv, typ, cache, [(n, pos, beg, end), (40, [39], [40], [40]), (40, [39], [0], [0])],
                     cap=10.0 if kind == "prefix" else 0.0, bias=kind == "prefix", window=window)


@pytest.mark.parametrize("typ,cache", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("cap", [3.0, 10.0, 22.0, 60.0])
def test_caps(ctx, typ, cache, hd, cap):
    """Scores from far below the cap to far above it, in rows that see different keys, over several blocks."""
    _check_attention(ctx, hd, 4, 1, typ, cache, [(700, np.arange(600, 700), None, None), (300, [299], None, None)], cap=cap,
                     q_scale=3.0)


@pytest.mark.parametrize("typ,cache", TYPES)
@pytest.mark.parametrize("scale", [-0.125, 0.0, 1e-25])
@pytest.mark.parametrize("cap", [0.0, 20.0])
def test_scales(ctx, typ, cache, scale, cap):
    _check_attention(ctx, 128, 8, 2, typ, cache, [(300, np.arange(230, 300), None, None), (40, [39], None, None)], cap=cap,
                     scale=scale)


@pytest.mark.parametrize("typ,cache", TYPES)
def test_large_scores(ctx, typ, cache):
    """Scores far apart (one weight is nearly 1) and large capped ones."""
    for cap in (0.0, 50.0):
        _check_attention(ctx, 128, 8, 2, typ, cache, [(400, np.arange(250, 400), None, None), (900, [899], None, None)],
                         cap=cap, q_scale=20.0)


@pytest.mark.parametrize("typ,cache", TYPES)
@pytest.mark.parametrize("dirt", [float("nan"), float("inf")])
def test_what_is_not_seen_does_not_matter(ctx, typ, cache, dirt):
    """Not-a-number and infinities in the rest of the pages never reach an output."""
    _check_attention(ctx, 128, 8, 2, typ, cache, [(37, [36], None, None), (5, [4], None, None), (1, [0], None, None),
                                                  (200, np.arange(100, 200), None, None)], dirty=dirt)


@pytest.mark.parametrize("typ,cache", TYPES)
@pytest.mark.parametrize("dirt", [float("nan"), float("inf")])
def test_masked_keys_of_the_same_tenant_do_not_matter(ctx, typ, cache, dirt):
    """A document whose keys and values are not finite leaves the tenant's other documents alone."""
    import torch
    import realm_b200 as rb
    H, kv, hd, n = 8, 2, 128, 260
    rng = np.random.default_rng(2)
    bad = slice(70, 141)
    pos = np.arange(n)
    beg = np.where(pos < 70, 0, np.where(pos < 141, 70, 141))
    pool = ctx.kv_pool(1, kv, hd, rb.F16 if cache == "F16" else rb.F32, n_pages=40, max_tenants=1, max_seq=n)
    try:
        pool.create(0)
        ct = np.float16 if cache == "F16" else np.float32
        q = rng.normal(0, 1, (n, H, hd)).astype(typ)
        outs = []
        for fill in (0.0, dirt):
            k, v = (rng2.normal(0, 1, (n, kv, hd)).astype(ct) for rng2 in (np.random.default_rng(7), np.random.default_rng(8)))
            k[bad], v[bad] = fill, fill
            with pool.plan([0] * n, H, positions=pos, begin=beg) as p:
                p.append(0, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda())
                outs.append(p.attention(0, torch.from_numpy(q).cuda(), 0.1).clone())
            # one token at a time
            for r in (69, 141, 200):
                with pool.plan([0], H, positions=[r], begin=[beg[r]]) as p:
                    one = p.attention(0, torch.from_numpy(q[r:r + 1]).cuda(), 0.1)
                assert torch.isfinite(one).all()
        good = np.r_[0:70, 141:n]
        assert torch.isfinite(outs[0]).all()
        assert torch.equal(outs[0][good], outs[1][good])
        assert not torch.isfinite(outs[1][bad]).any()
    finally:
        pool.close()


def test_host_arrays_and_layers(ctx):
    import realm_b200 as rb
    rng = np.random.default_rng(9)
    pool = ctx.kv_pool(3, 2, 64, rb.F16, n_pages=12, max_tenants=2, max_seq=64)
    try:
        pool.create(1)
        ks = [rng.normal(0, 1, (30, 2, 64)).astype(np.float32) for _ in range(3)]
        q = rng.normal(0, 1, (1, 4, 64)).astype(np.float32)
        with pool.plan([1] * 30, 4) as p:
            for layer in range(3):
                p.append(layer, ks[layer], ks[layer])
        with pool.plan([1], 4, positions=[29]) as p:
            for layer in range(3):
                got = p.attention(layer, q, 0.125)
                k = ks[layer].astype(np.float16).astype(np.float64)
                ref, _ = _attn_ref(q.astype(np.float64), k, k, [29], [0], [30], 0.125, 0, None)
                assert np.abs(got - ref).max() < 1e-4
    finally:
        pool.close()


def test_agrees_with_attention_forward(ctx):
    """Plain causal rows: the same result as the framework's decode attention."""
    import torch
    import realm_b200 as rb
    pool = ctx.kv_pool(1, 4, 128, rb.F16, n_pages=64, max_tenants=3, max_seq=400)
    try:
        lens = [390, 17, 64]
        for t, n in enumerate(lens):
            pool.create(t)
            pool.append(t, 0, torch.randn(n, 4, 128, device="cuda"), torch.randn(n, 4, 128, device="cuda"))
        q = torch.randn(3, 16, 128, device="cuda")
        old = torch.empty(3, 16, 128, device="cuda")
        pool.attention_forward(0, [0, 1, 2], q, 16, 0.088, positions=[n - 1 for n in lens], out=old)
        with pool.plan([0, 1, 2], 16, positions=[n - 1 for n in lens]) as p:
            new = p.attention(0, q, 0.088)
        assert (old - new).abs().max() < 2e-5
    finally:
        pool.close()


def test_other_streams(ctx):
    """Calls are ordered with torch's current stream, whichever it is."""
    import torch
    import realm_b200 as rb
    pool = ctx.kv_pool(1, 4, 64, rb.F16, n_pages=160, max_tenants=1, max_seq=2100)
    try:
        pool.create(0)
        side = torch.cuda.Stream()
        big = torch.randn(4096, 4096, device="cuda")
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            for _ in range(8):
                big = (big @ big).clamp(-1, 1)  # keeps the stream busy, so that a missing wait shows
            k = torch.full((2000, 4, 64), 3.0, device="cuda") * (big[0, 0] * 0 + 1)
            with pool.plan([0] * 2000, 8) as p:
                p.append(0, k, k)
                o = p.attention(0, torch.ones(2000, 8, 64, device="cuda"), 0.1)
            o = o + 1
        side.synchronize()
        # every value is 3, so o is 4 within the bound above (a missing wait reads other memory)
        e = (64 * U + 2.0 ** -21 + 2.0 ** -20) * 0.1 * 64 * 3
        assert (o - 4).abs().max() <= (2 * e + 2.0 ** -19) * 3
    finally:
        pool.close()


def test_pages_outlive_a_closed_pool(ctx):
    """A tensor of pages() keeps the pool's memory; the pool itself cannot be used any more."""
    import torch
    import realm_b200 as rb
    free = torch.cuda.mem_get_info()[0]
    pool = ctx.kv_pool(1, 2, 64, rb.F32, n_pages=4096, max_tenants=1, max_seq=64)  # 64 MB
    pool.create(0)
    k = torch.randn(20, 2, 64, device="cuda")
    with pool.plan([0] * 20, 2) as p:
        p.append(0, k, k)
    view = pool.pages()
    assert view.shape == (4096, 1, 2, 2, 16, 64)
    pool.close()
    ctx.sync()
    assert torch.equal(view[0, 0, 1].permute(1, 0, 2), k[:16])
    with pytest.raises(rb.RealmError):
        pool.create(0)
    assert free - torch.cuda.mem_get_info()[0] >= 64 << 20
    del view
    assert free - torch.cuda.mem_get_info()[0] < 64 << 20


def test_context_on_a_stream_of_the_caller():
    import torch
    import realm_b200 as rb
    s = torch.cuda.Stream()
    for handle in (0, s.cuda_stream):
        with rb.Context(0, stream=handle) as c:
            assert (c.stream or 0) == handle
            pool = c.kv_pool(1, 1, 64, rb.F16, n_pages=4, max_tenants=1, max_seq=32)
            pool.create(0)
            k = np.ones((5, 1, 64), np.float32)
            with pool.plan([0] * 5, 1) as p:
                p.append(0, k, k)
                assert (p.attention(0, k, 1.0) == 1).all()
            pool.close()
    torch.cuda.synchronize()


def test_plan_refusals(ctx):
    import torch
    import realm_b200 as rb
    pool = ctx.kv_pool(2, 2, 64, rb.F16, n_pages=6, max_tenants=3, max_seq=200)

    def code(f):
        with pytest.raises(rb.RealmError) as e:
            f()
        return e.value.code

    try:
        pool.create(0)
        pool.create(1)
        assert code(lambda: pool.plan([2], 2)) == -2                       # no such tenant
        assert code(lambda: pool.plan([7], 2)) == -2
        assert code(lambda: pool.plan([0], 3)) == -23                      # heads
        assert code(lambda: pool.plan([0], 0)) == -23
        assert code(lambda: pool.plan([0], 130)) == -23
        assert code(lambda: pool.plan([], 2)) == -3
        assert code(lambda: pool.plan([0], 2, positions=[200])) == -22
        assert code(lambda: pool.plan([0], 2, end=[201])) == -22
        free = pool.free_pages()
        assert code(lambda: pool.plan([0] * 50 + [1] * 60, 2)) == -21      # 4 + 4 pages of 6
        assert pool.free_pages() == free
        with pytest.raises(ValueError):
            pool.plan([0, 0], 2, end=[1])
        x = torch.zeros(4, 2, 64, device="cuda")
        p = pool.plan([0] * 4, 2)
        assert code(lambda: p.attention(0, x, 1.0)) == -7                  # nothing cached yet
        assert code(lambda: p.append(2, x, x)) == -2                       # layer
        p.append(0, x, x)
        assert code(lambda: p.attention(1, x, 1.0)) == -7
        assert code(lambda: p.attention(0, x, 1.0, softcap=-1.0)) == -3
        assert code(lambda: p.attention(0, x, float("nan"))) == -3
        with pytest.raises(ValueError):
            p.attention(0, x[:3], 1.0)
        with pytest.raises(ValueError):
            p.attention(0, x.double(), 1.0)
        with pytest.raises(ValueError):
            p.attention(0, x.transpose(0, 1), 1.0)
        with pytest.raises(ValueError):
            p.attention(0, x, 1.0, out=np.zeros((4, 2, 64), np.float32))
        with pytest.raises(ValueError):
            p.append(0, x, x.half())
        rope = torch.zeros(3, 64, device="cuda")
        assert code(lambda: p.append(0, x, x, rope=rope)) == -3            # table too short
        assert code(lambda: p.append(0, x, x, rope=torch.zeros(9, 12, device="cuda"))) == -23
        assert code(lambda: p.append(0, x, x, rope=torch.zeros(9, 72, device="cuda"))) == -23
        gap = pool.plan([0], 2, positions=[6])
        assert code(lambda: gap.append(0, x[:1], x[:1])) == -3             # position 4 is missing
        mixed = pool.plan([0, 0], 2, positions=[3, 2])
        assert code(lambda: mixed.append(0, x[:2], x[:2])) == -3           # not ascending
        pool.clear(0)
        assert code(lambda: p.attention(0, x, 1.0)) == -7
        assert code(lambda: p.append(0, x, x)) == -7
        pool.destroy(0)
        assert code(lambda: p.append(0, x, x)) == -2
        p.close()
        assert code(lambda: p.append(0, x, x)) == -20
    finally:
        pool.close()
    with pytest.raises(rb.RealmError):
        pool.plan([0], 2)


# ---------------------------------------------------------------------------
# sampling
# ---------------------------------------------------------------------------
def _sample_ref(x, f, u, prev=()):
    """The definition, with the weights in fp32 and everything after them exact."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float32))
    for t in prev:
        if t < len(x):
            x[t] = x[t] / np.float32(f.repetition_penalty) if x[t] > 0 else x[t] * np.float32(f.repetition_penalty)
    if f.temperature < 1e-7:
        return int(np.argmax(x)), 1.0
    y = (x / np.float32(f.temperature)).astype(np.float32)
    m = y.max()
    import torch
    with np.errstate(invalid="ignore"):
        w = torch.exp(torch.from_numpy((y - m).astype(np.float32)).cuda()).cpu().numpy()
    w[y == m] = 1
    w[~(w >= np.float32(min(f.min_p, 1.0)))] = 0
    W = np.floor(w.astype(np.float64) * 2.0 ** 40).astype(np.uint64).astype(object)
    order = np.lexsort((np.arange(len(w)), -w.astype(np.float64)))
    ranked = W[order]
    if 0 < f.top_k < len(w):
        ranked[f.top_k:] = 0
    if 0 < f.top_p < 1:
        before = np.cumsum(ranked) - ranked
        want = max(1, int(float(sum(ranked)) * float(np.float32(f.top_p))))
        ranked = np.where(before < want, ranked, 0)
    kept = np.zeros(len(w), object)
    kept[order] = ranked
    total = int(sum(kept))
    run = np.cumsum(kept)
    tok = int(np.argmax(run > int(float(np.float32(u)) * float(total))))
    return tok, float(kept[tok]) / total


FILTERS = [(0.0, 0, 1.0, 0.0), (1.0, 0, 1.0, 0.0), (0.7, 40, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (1.3, 50, 0.95, 0.02),
           (1.0, 0, 1.0, 0.1), (1.0, 1, 1.0, 0.0), (0.9, 10 ** 6, 0.5, 0.0), (2.0, 7, 1e-9, 0.0), (1.0, 0, 0.8, 5.0)]


@pytest.mark.parametrize("V", [1, 2, 7, 1000, 8193, 21000, 32000, 100000, 151937, 262144])
@pytest.mark.parametrize("typ", ["float32", "float16"])
def test_sample_filtered(ctx, V, typ):
    import torch
    import realm_b200 as rb
    rng = np.random.default_rng(V)
    n = 2 * len(FILTERS)
    fs = [rb.SamplingFilter(*FILTERS[i % len(FILTERS)], repetition_penalty=1.2 if i >= len(FILTERS) else 1.0)
          for i in range(n)]
    x = (rng.normal(0, 3, (n, V))).astype(typ)
    x[::3] = np.round(x[::3])          # many ties
    x[1::4, ::5] = -np.inf             # masked tokens
    x[2::5, V // 2:] = np.nan
    x[:, 0] = 1.0
    prev = [list(rng.integers(0, V, 6)) + [0, 0] if i >= len(FILTERS) else [] for i in range(n)]
    u = (rng.integers(0, 2 ** 23, n) / 2 ** 23).astype(np.float32)
    u[0], u[3] = 0.0, 1 - 2.0 ** -24
    probs = np.zeros(n, np.float32)
    got = rb.sample_filtered(ctx, x, fs, u, prev=prev, probs=probs)
    ref = [_sample_ref(x[i], fs[i], u[i], prev[i]) for i in range(n)]
    assert [int(t) for t in got] == [t for t, _ in ref]
    assert np.allclose(probs, [p for _, p in ref], rtol=2.0 ** -22, atol=0)
    # the same on device tensors, with rows apart
    wide = torch.full((n, V + 5), 99.0, dtype=torch.from_numpy(x).dtype, device="cuda")
    wide[:, :V] = torch.from_numpy(x).cuda()
    flat = torch.tensor([t for p in prev for t in p], dtype=torch.int32, device="cuda")
    off = torch.tensor(np.concatenate([[0], np.cumsum([len(p) for p in prev])]), dtype=torch.int32, device="cuda")
    dp = torch.empty(n, device="cuda")
    dev = rb.sample_filtered(ctx, wide[:, :V], rb.pack_filters(fs, "cuda"), torch.from_numpy(u).cuda(),
                             prev=(flat, off), probs=dp)
    assert (dev.cpu().numpy() == got.astype(np.int32)).all() and (dp.cpu().numpy() == probs).all()


def test_sample_infinities_and_refusals(ctx):
    import torch
    import realm_b200 as rb
    F = rb.SamplingFilter
    x = np.zeros((1, 9), np.float32)
    x[0, [2, 5]] = np.inf
    assert rb.sample_filtered(ctx, x, [F()], [0.1])[0] == 2
    assert rb.sample_filtered(ctx, x, [F()], [0.9])[0] == 5
    assert rb.sample_filtered(ctx, x, [F(0.0)], [0.9])[0] == 2   # ties: the lowest index
    x[:] = -np.inf
    for f in (F(), F(0.0)):
        with pytest.raises(rb.RealmError) as e:
            rb.sample_filtered(ctx, x, [f], [0.5])
        assert e.value.code == -3 and "weighted index" in str(e.value)
    dev = rb.sample_filtered(ctx, torch.from_numpy(x).cuda(), rb.pack_filters([F()], "cuda"), torch.zeros(1, device="cuda"))
    assert dev.item() == -1
    with pytest.raises(rb.RealmError) as e:
        rb.sample_filtered(ctx, np.zeros((1, 262145), np.float32), [F()], [0.5])
    assert e.value.code == -23
    with pytest.raises(ValueError):
        rb.sample_filtered(ctx, np.zeros((2, 5), np.float32), [F()], [0.5, 0.5])
    with pytest.raises(ValueError):
        rb.sample_filtered(ctx, np.zeros((1, 5), np.float64), [F()], [0.5])
    with pytest.raises(ValueError):
        rb.sample_filtered(ctx, torch.zeros(1, 5, device="cuda"), [F()], torch.zeros(1, device="cuda"))
    assert len(rb.sample_filtered(ctx, np.zeros((0, 5), np.float32), [], [])) == 0


def test_sample_frequencies(ctx):
    """Draws over a small vocabulary follow the filtered distribution."""
    import realm_b200 as rb
    rng = np.random.default_rng(4)
    V, n = 12, 4000
    x = np.tile(rng.normal(0, 1.5, V).astype(np.float32), (n, 1))
    f = rb.SamplingFilter(0.9, top_k=8, top_p=0.95, min_p=0.01)
    got = rb.sample_filtered(ctx, x, [f] * n, ((np.arange(n) + 0.5) / n).astype(np.float32))
    p = np.array([_sample_ref(x[0], f, (i + 0.5) / n)[0] for i in range(n)])
    assert (np.bincount(got, minlength=V) == np.bincount(p, minlength=V)).all()


@pytest.mark.parametrize("typ", ["float32", "float16"])
@pytest.mark.parametrize("V", [3000, 9001, 23001, 40003, 90001])
def test_sample_many_rows(ctx, V, typ):
    """Many rows take fewer CTAs each: the same tokens as one row at a time, for every vocabulary range."""
    import torch
    import realm_b200 as rb
    n = 300
    g = torch.Generator("cuda").manual_seed(V)
    x = (torch.randn(n, V, device="cuda", generator=g) * 3).to(getattr(torch, typ))
    u = torch.rand(n, device="cuda", generator=g)
    fs = [rb.SamplingFilter(0.9, 60 if i % 2 else 0, 0.9 if i % 3 else 1.0, 0.001) for i in range(n)]
    probs = torch.empty(n, device="cuda")
    got = rb.sample_filtered(ctx, x, rb.pack_filters(fs, "cuda"), u, probs=probs)
    for i in range(0, n, 23):
        tok, p = _sample_ref(x[i].cpu().numpy(), fs[i], float(u[i]))
        assert got[i].item() == tok and abs(probs[i].item() - p) <= 2.0 ** -22 * p
        one = rb.sample_filtered(ctx, x[i:i + 1], rb.pack_filters(fs[i:i + 1], "cuda"), u[i:i + 1])
        assert one.item() == tok


@pytest.mark.parametrize("typ", ["float32", "float16"])
@pytest.mark.parametrize("V", [6007, 50000, 140001])
def test_sample_few_and_many_candidates(ctx, V, typ):
    """Rows of which few or most tokens weigh enough, together, at one end, equal or all over the vocabulary."""
    import torch
    import realm_b200 as rb
    rng = np.random.default_rng(V)
    i = np.arange(V)
    kinds = [np.zeros(V),                                   # all equal
             np.where(i < 5000, 1.0, -30.0),                # 5000 equal ones at the front
             np.where(i >= V - 300, 2.0 + i % 7, -40.0),    # all at the end
             np.where(i % 97 == 5, 3.0, -50.0 + i % 3),     # spread, with ties
             np.where(i == V // 2, 40.0, -5.0 * (i % 11)),  # one token
             -np.sqrt(i) / 4.0,                             # sorted
             rng.normal(0, 4, V), rng.normal(0, 0.5, V), rng.normal(0, 12, V),
             np.where(i % 1999 == 7, np.inf, 1.0)]          # infinities
    filters = [(1.0, 0, 0.9, 0.01), (0.7, 40, 0.95, 0.0), (1.0, 3000, 1.0, 0.0), (1.3, 7000, 0.5, 1e-3), (0.0, 0, 1.0, 0.0),
               (2.0, 1, 1.0, 0.5), (1.0, 0, 1.0, 0.2), (1e4, 50, 0.3, 0.0), (3e38, 0, 0.4, 0.5)]
    fs, x = [], []
    for k in kinds:
        for f in filters:
            fs.append(rb.SamplingFilter(*f))
            x.append(k)
    x = np.stack(x).astype(typ)
    n = len(fs) * 3
    u = (rng.integers(0, 2 ** 23, n) / 2 ** 23).astype(np.float32)
    dx = torch.from_numpy(x).cuda().repeat(3, 1)
    probs = torch.empty(n, device="cuda")
    got = rb.sample_filtered(ctx, dx, rb.pack_filters(fs * 3, "cuda"), torch.from_numpy(u).cuda(), probs=probs)
    for r in range(n):
        tok, p = _sample_ref(x[r % len(fs)], fs[r % len(fs)], float(u[r]))
        assert got[r].item() == tok and abs(probs[r].item() - p) <= 2.0 ** -22 * p, (r, got[r].item(), tok)

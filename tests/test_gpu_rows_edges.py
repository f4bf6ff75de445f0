"""Edges of the row plans' operators: what calls refuse, lifetimes, streams, and inputs
on which a kernel's rounding shows. References are plain forms in 64 bits; each
tolerance is derived where it stands, with U = 2^-24 (fp32) and HALF = 2^-11 (fp16)."""
import os
import subprocess
import sys

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
U, HALF = 2.0 ** -24, 2.0 ** -11


def _np(x):
    return x.detach().cpu().double().numpy()


def _cuda(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _code(f):
    import realm_b200 as rb
    with pytest.raises(rb.RealmError) as e:
        f()
    return e.value.code


# ---------------------------------------------------------------------------
# sampling
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("typ", ["float32", "float16"])
@pytest.mark.parametrize("rows,V", [(1, 9), (3, 5000), (200, 33000), (40, 151937)])
@pytest.mark.parametrize("top_k,min_p", [(0, 0.0), (5, 0.0), (0, 0.3), (2000, 0.0)])
def test_a_uniform_of_one_draws_the_last_kept_token(ctx, typ, rows, V, top_k, min_p):
    """Float64 draws just below 1 round to 1.0f: every row still writes a token, the last of those kept."""
    import torch
    import realm_b200 as rb
    rng = np.random.default_rng(V + top_k)
    x = np.round(rng.normal(0, 1.5, (rows, V)) * 4).astype(typ) / 4  # exact in both types: ties by the index
    want = []
    for r in range(rows):
        order = np.lexsort((np.arange(V), -x[r].astype(np.float64)))
        kept = order[:top_k] if 0 < top_k < V else order
        if min_p:  # exp(-1.25) = 0.2865 < 0.3 < exp(-1) = 0.3679
            kept = kept[x[r][kept].astype(np.float64) >= float(x[r].max()) - 1.0]
        want.append(kept.max())
    f = rb.SamplingFilter(1.0, top_k=top_k, min_p=min_p)
    one = np.full(rows, np.nextafter(1.0, 0.0))
    probs = np.full(rows, -7, np.float32)
    assert (rb.sample_filtered(ctx, x, [f] * rows, one, probs=probs) == want).all()
    assert (probs > 0).all()
    for u in (1.0, 1.5, float("inf")):
        out = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
        probs = torch.full((rows,), -7.0, device="cuda")
        rb.sample_filtered(ctx, _cuda(x), rb.pack_filters([f] * rows, "cuda"), torch.full((rows,), u, device="cuda"),
                           out=out, probs=probs)
        assert (out.cpu().numpy() == want).all() and (probs > 0).all()
    # below 0 and not a number: the first kept token
    for u in (-1.0, float("nan")):
        out = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
        rb.sample_filtered(ctx, _cuda(x), rb.pack_filters([f] * rows, "cuda"), torch.full((rows,), u, device="cuda"), out=out)
        got = out.cpu().numpy()
        for r in range(rows):
            order = np.lexsort((np.arange(V), -x[r].astype(np.float64)))
            kept = order[:top_k] if 0 < top_k < V else order
            if min_p:
                kept = kept[x[r][kept].astype(np.float64) >= float(x[r].max()) - 1.0]
            assert got[r] == kept.min()


# ---------------------------------------------------------------------------
# lifetimes
# ---------------------------------------------------------------------------
def _small_model(ctx, rb):
    return rb.Model(ctx, dict(n_layers=2, hidden=256, n_heads=4, n_kv_heads=2, head_dim=64, ffn=256, vocab=256, max_seq=64,
                              rms_eps=1e-5, layer_eps=1e-5, rope_theta=1e4, kv_dtype=rb.F32, max_tenants=2, kv_pages=8192))


@pytest.mark.parametrize("owner", ["pool", "model"])
def test_a_tensor_of_pages_outlives_the_context(owner):
    import torch
    import realm_b200 as rb
    free = torch.cuda.mem_get_info()[0]
    k = torch.randn(20, 2, 64, device="cuda")
    with rb.Context(0) as c:
        if owner == "pool":
            pool = c.kv_pool(2, 2, 64, rb.F32, n_pages=8192, max_tenants=1, max_seq=64)  # 256 MB
            pool.create(0)
        else:
            model = _small_model(c, rb)
            model.tenant_create(0)
            pool = model.kv
        with pool.plan([0] * 20, 2) as p:
            p.append(1, k, k)
        view = pool.pages()[:, 1]
    assert torch.equal(view[0, 1].permute(1, 0, 2), k[:16])
    view.fill_(3.0)  # the whole of it
    assert (view == 3.0).all()
    assert free - torch.cuda.mem_get_info()[0] >= 256 << 20
    del view
    assert free - torch.cuda.mem_get_info()[0] < 256 << 20


def test_a_tensor_of_pages_outlives_its_model(ctx):
    import torch
    import realm_b200 as rb
    model = _small_model(ctx, rb)
    model.tenant_create(0)
    k = torch.randn(20, 2, 64, device="cuda")
    with model.kv.plan([0] * 20, 2) as p:
        p.append(0, k, k)
    view = model.kv.pages()
    kv = model.kv
    model.close()
    assert torch.equal(view[0, 0, 0].permute(1, 0, 2), k[:16])
    assert _code(kv.pages) == -20 and _code(lambda: kv.create(1)) == -20


def test_a_plan_ends_with_its_pool(ctx):
    """A plan of a closed pool stays refused when other pools and plans have come, and leaves them alone."""
    import torch
    import realm_b200 as rb
    a = ctx.kv_pool(1, 4, 128, rb.F32, n_pages=8, max_tenants=1, max_seq=64)
    a.create(0)
    old = a.plan([0] * 2, 8)
    x, y = torch.zeros(2, 4, 128, device="cuda"), torch.zeros(2, 8, 128, device="cuda")
    a.close()
    b = ctx.kv_pool(1, 4, 128, rb.F32, n_pages=8, max_tenants=1, max_seq=64)
    try:
        b.create(0)
        for plan in (b.plan([0] * 60, 8), b.plan([0] * 60, 8)):
            assert _code(lambda: old.append(0, x, x)) == -20
            assert _code(lambda: old.attention(0, y, 1.0)) == -20
            assert b.len(0) == 0
            plan.close()
            plan.close()
        old.close()
        assert b.plan([0], 8).handle > old.handle
    finally:
        b.close()


def test_a_plan_ends_with_its_model(ctx):
    import torch
    import realm_b200 as rb
    model = _small_model(ctx, rb)
    model.tenant_create(0)
    k = torch.randn(20, 2, 64, device="cuda")
    plan = model.kv.plan([0] * 20, 4)
    plan.append(0, k, k)
    model.close()
    other = ctx.kv_pool(1, 2, 64, rb.F16, n_pages=8, max_tenants=1, max_seq=64)
    try:
        assert _code(lambda: plan.append(0, k, k)) == -20
        assert _code(lambda: plan.attention(0, torch.zeros(20, 4, 64, device="cuda"), 1.0)) == -20
        plan.close()
    finally:
        other.close()


def test_a_plan_that_nothing_refers_to_is_freed(ctx):
    import torch
    import realm_b200 as rb
    pool = ctx.kv_pool(1, 1, 128, rb.F16, n_pages=16, max_tenants=16, max_seq=64)
    try:
        pool.create(0)
        rows = np.zeros(1 << 20, np.uint32)
        free = torch.cuda.mem_get_info()[0]
        for _ in range(4):  # 2^20 rows of 64 heads are 16 MB and more of lists
            pool.plan(rows, 64, positions=rows)
        assert free - torch.cuda.mem_get_info()[0] < 16 << 20
    finally:
        pool.close()


# ---------------------------------------------------------------------------
# streams
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("which", ["default", "side"])
@pytest.mark.parametrize("current", ["default", "side"])
def test_every_call_takes_cuda_tensors_on_a_context_of_the_callers_stream(which, current):
    """The calls that were there before row plans, and row plans, whatever torch's current stream is."""
    import torch
    import realm_b200 as rb
    side = torch.cuda.Stream()
    own = torch.cuda.default_stream() if which == "default" else side
    rng = np.random.default_rng(0)
    with rb.Context(0, stream=own.cuda_stream) as c:
        assert c.stream == own.cuda_stream
        blocks = c.quantize(rb.Q4_K, rng.normal(0, 0.1, (256, 256)).astype(np.float32))
        w = c.upload_weight(rb.Q4_K, 256, 256, blocks)
        pool = c.kv_pool(1, 2, 64, rb.F16, n_pages=8, max_tenants=2, max_seq=64)
        pool.create(0)
        pool.create(1)
        with torch.cuda.stream(torch.cuda.default_stream() if current == "default" else torch.cuda.Stream()):
            x = _cuda(rng.normal(0, 1, (3, 256)).astype(np.float32))
            got = w.matmul(x, 3, out=torch.empty(3, 256, device="cuda"))
            host = w.matmul(x.cpu().numpy(), 3)
            assert np.array_equal(got.cpu().numpy(), host)
            k = torch.ones(5, 2, 64, device="cuda")
            pool.append(0, 0, k, k * 3)
            o = pool.attention_forward(0, [0], k[:1], 2, 0.1, positions=[4], out=torch.empty(1, 2, 64, device="cuda"))
            # five equal keys: 3 within the rounding of five weights and their sum
            assert (o - 3).abs().max() <= 3 * 16 * U
            with pool.plan([1] * 5, 2) as p:
                p.append(0, k, k * 3)
                o = p.attention(0, k, 0.1)
            assert (o - 3).abs().max() <= 3 * 2.0 ** -20  # probabilities in two fp16 parts: 22 bits
            t = rb.sample_filtered(c, torch.zeros(2, 4, device="cuda"), rb.pack_filters([rb.SamplingFilter()] * 2, "cuda"),
                                   torch.tensor([0.1, 0.9], device="cuda"))
            assert t.tolist() == [0, 3]
        pool.close()
        w.free()


def test_the_example_runs():
    r = subprocess.run([sys.executable, os.path.join(ROOT, "examples", "local_global_decode.py")], capture_output=True,
                       text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    assert r.stdout.count("prompt of") == 3


def test_calls_wait_on_their_own_contexts_stream(ctx):
    """Another context that came and went changes nothing."""
    import torch
    import realm_b200 as rb
    rng = np.random.default_rng(1)
    w = ctx.upload_weight(rb.Q4_K, 256, 256, ctx.quantize(rb.Q4_K, rng.normal(0, 0.1, (256, 256)).astype(np.float32)))
    value = rng.normal(0, 1, (3, 256)).astype(np.float32)
    want = w.matmul(value, 3)
    value, x, out = _cuda(value), torch.zeros(3, 256, device="cuda"), torch.empty(3, 256, device="cuda")
    big = torch.randn(4096, 4096, device="cuda")
    with rb.Context(0), rb.Context(0):
        pass
    torch.cuda.synchronize()
    for _ in range(20):
        big = (big @ big).clamp(-1, 1)  # keeps torch's stream busy, so that a missing wait shows
    x.copy_(value + big[:3, :256] * 0)
    w.matmul(x, 3, out=out)
    assert np.array_equal(out.cpu().numpy(), want)
    w.free()


def test_empty_histories_on_cuda_tensors(ctx):
    """The first token of a batch: no row has a history, and the tensor of all of them is empty."""
    import torch
    import realm_b200 as rb
    x = torch.randn(3, 1000, device="cuda", generator=torch.Generator("cuda").manual_seed(0))
    u = torch.tensor([0.2, 0.5, 0.8], device="cuda")
    f = rb.pack_filters([rb.SamplingFilter(0.7, top_k=20, repetition_penalty=1.3)] * 3, "cuda")
    none = (torch.empty(0, dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda"))
    assert torch.equal(rb.sample_filtered(ctx, x, f, u, prev=none), rb.sample_filtered(ctx, x, f, u))


def test_empty_batches_on_cuda_tensors(ctx):
    import torch
    import realm_b200 as rb
    for typ in (torch.float32, torch.float16):
        t = rb.sample_filtered(ctx, torch.empty(0, 1000, dtype=typ, device="cuda"), rb.pack_filters([], "cuda"),
                               torch.empty(0, device="cuda"), probs=torch.empty(0, device="cuda"))
        assert t.shape == (0,) and t.dtype == torch.int32


# ---------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------
def test_memory_off_its_alignment_is_refused(ctx):
    """Device memory that a kernel could not read by words: an error from the call, nothing launched."""
    import ctypes as C
    import torch
    import realm_b200 as rb
    from realm_b200 import rows as R
    x = torch.zeros(2, 8, device="cuda")
    u = torch.zeros(2, device="cuda")
    packed = rb.pack_filters([rb.SamplingFilter()] * 2, "cuda")
    odd = torch.zeros(41, dtype=torch.uint8, device="cuda")[1:]
    odd.copy_(packed.reshape(-1))
    assert _code(lambda: rb.sample_filtered(ctx, x, odd, u)) == -3
    ok = dict(params=packed.data_ptr(), prev=u.data_ptr(), prev_off=u.data_ptr(), uniforms=u.data_ptr(),
              out=torch.zeros(2, device="cuda").data_ptr(), probs=u.data_ptr())
    for name in ok:
        a = dict(ok, **{name: ok[name] + 2})
        rc = rb.lib().rb_sample_filtered(ctx.handle, rb.F32, x.data_ptr(), 8, 2, 8, a["params"], a["prev"], a["prev_off"],
                                         a["uniforms"], a["out"], a["probs"], rb.PTR_DEVICE)
        assert rc == -3, name
    pool = ctx.kv_pool(1, 2, 64, rb.F16, n_pages=2, max_tenants=1, max_seq=32)
    try:
        pool.create(0)
        with pool.plan([0], 4) as p:
            k = torch.zeros(1, 4, 64, device="cuda")
            at = k.data_ptr()
            good = dict(q=at, k=at, v=at, q_out=at, q_norm=at, k_norm=at, rope=at)
            for name in good:
                d = R._AppendDesc(dtype=rb.F32, ldq=256, ldk=128, ldv=128, ldo=256, eps=1e-6, rotary=64, rope_len=1,
                                  **dict(good, **{name: at + 2}))
                assert rb.lib().rb_plan_append(ctx.handle, p.handle, 0, C.byref(d), rb.PTR_DEVICE) == -3, name
            assert pool.len(0) == 0
            p.append(0, k[:, :2], k[:, :2])
            good = dict(q=at, out=at, slopes=at)
            for name in good:
                d = R._AttentionDesc(dtype=rb.F32, scale=1.0, ldq=256, ldo=256, **dict(good, **{name: at + 2}))
                assert rb.lib().rb_plan_attention(ctx.handle, p.handle, 0, C.byref(d), rb.PTR_DEVICE) == -3, name
    finally:
        pool.close()


def test_rows_too_far_apart_are_refused(ctx):
    """Distances whose bytes would not fit 64 bits."""
    import ctypes as C
    import realm_b200 as rb
    from realm_b200 import rows as R
    x = np.zeros(1024, np.float32)
    at = x.ctypes.data
    pool = ctx.kv_pool(1, 1, 64, rb.F16, n_pages=2, max_tenants=1, max_seq=32)
    try:
        pool.create(0)
        with pool.plan([0, 0], 1) as p:
            for ld in ((1 << 62) + 64, 1 << 61, (1 << 36) + 1):
                d = R._AppendDesc(dtype=rb.F32, k=at, v=at, ldk=64, ldv=ld)
                assert rb.lib().rb_plan_append(ctx.handle, p.handle, 0, C.byref(d), rb.PTR_HOST) == -3
                d = R._AppendDesc(dtype=rb.F32, k=at, v=at, ldk=ld, ldv=64)
                assert rb.lib().rb_plan_append(ctx.handle, p.handle, 0, C.byref(d), rb.PTR_HOST) == -3
                assert pool.len(0) == 0
                f = rb.SamplingFilter().c()
                rc = rb.lib().rb_sample_filtered(ctx.handle, rb.F32, at, ld, 2, 8, (R._Filter * 2)(f, f), None, None, at, at,
                                                 None, rb.PTR_HOST)
                assert rc == -3
            p.append(0, x[:128].reshape(2, 1, 64), x[:128].reshape(2, 1, 64))
            for ld in ((1 << 62) + 64, 1 << 61, (1 << 36) + 1):
                for ldq, ldo in ((ld, 64), (64, ld)):
                    d = R._AttentionDesc(dtype=rb.F32, scale=1.0, q=at, out=at, ldq=ldq, ldo=ldo)
                    assert rb.lib().rb_plan_attention(ctx.handle, p.handle, 0, C.byref(d), rb.PTR_HOST) == -3
    finally:
        pool.close()


def test_histories_out_of_order_are_refused(ctx):
    """Host offsets that fall, or pass the last one: the kernel would read past the tokens."""
    import realm_b200 as rb
    from realm_b200 import rows as R
    x, u = np.zeros((2, 8), np.float32), np.zeros(2, np.float32)
    f = rb.SamplingFilter(repetition_penalty=1.2).c()
    tokens, out = np.zeros(4, np.uint32), np.zeros(2, np.uint32)
    for off, rc in (([0, 9, 4], -3), ([5, 2, 4], -3), ([0, 3, 2], -3), ([0, 1, 4], 2), ([2, 2, 4], 2)):
        off = np.array(off, np.uint32)
        assert rb.lib().rb_sample_filtered(ctx.handle, rb.F32, x.ctypes.data, 8, 2, 8, (R._Filter * 2)(f, f),
                                           tokens.ctypes.data, off.ctypes.data, u.ctypes.data, out.ctypes.data, None,
                                           rb.PTR_HOST) == rc, off


def test_sampled_tokens_go_to_the_callers_array(ctx):
    """numpy: `out` as uint32 or int32, filled and returned, as on CUDA tensors."""
    import torch
    import realm_b200 as rb
    x = np.random.default_rng(0).normal(0, 3, (6, 700)).astype(np.float32)
    f, u = [rb.SamplingFilter(0.8, top_k=30)] * 6, np.linspace(0.05, 0.95, 6)
    want = rb.sample_filtered(ctx, x, f, u)
    for t in (np.uint32, np.int32):
        out, probs = np.full(6, 12345, t), np.zeros(6, np.float32)
        assert rb.sample_filtered(ctx, x, f, u, out=out, probs=probs) is out
        assert (out == want).all() and (probs > 0).all()
    for out in (np.zeros(5, np.uint32), np.zeros(6, np.int64), np.zeros(12, np.int32)[::2], torch.zeros(6, dtype=torch.int32),
                torch.zeros(6, dtype=torch.int32, device="cuda")):
        with pytest.raises(ValueError):
            rb.sample_filtered(ctx, x, f, u, out=out)
    with pytest.raises(ValueError):
        rb.sample_filtered(ctx, x, f, u, probs=torch.zeros(6, device="cuda"))


# ---------------------------------------------------------------------------
# rounding
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("typ", ["float32", "float16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("shape", ["row of 32 heads", "run of 40 rows"])
def test_light_keys_beside_a_heavy_one_whose_value_is_zero(ctx, typ, hd, shape):
    """One key has nearly all the weight and a value of 0, and thousands of equal ones 2^-u of it each: the
    output is theirs alone, and shows what their weights are rounded to. Another u for every query vector.

    A weight of fp32 rows is off by 2^-22 of itself (two fp16 parts) and by what its score is off, and by
    2^-37 of the heaviest one (p counts from 2^12 and more, in steps of 2^-24). The score has a magnitude
    of u ln 2, made of q in 22 bits and a few fp32 roundings: 2^-22 (u + 4) with some room. fp16 rows: q is
    an exact input; probabilities and output are rounded to fp16, h / 2 each, with room 2 h together."""
    import realm_b200 as rb
    n, H, L = (1, 32, 5000) if shape[0:3] == "row" else (40, 1, 5000)
    u = np.linspace(9.3, 30.7, n * H).reshape(n, H)
    q = np.zeros((n, H, hd), typ)
    k = np.zeros((L, 1, hd), np.float16)
    k[0, 0, 5], k[1:, 0, 5] = 8.0, -8.0
    q[:, :, 5] = u * np.log(2) / 16  # scale 1: the scores differ by u ln 2
    v = np.ones((L, 1, hd), np.float16)
    v[0] = 0
    pool = ctx.kv_pool(1, 1, hd, rb.F16, n_pages=L // 16 + 1, max_tenants=1, max_seq=L)
    try:
        pool.create(0)
        with pool.plan([0] * L, H) as p:
            p.append(0, _cuda(k), _cuda(v))
        with pool.plan([0] * n, H, positions=[L - 1] * n) as p:
            got = _np(p.attention(0, _cuda(q), 1.0))
    finally:
        pool.close()
    w = (L - 1) * np.exp(-16.0 * q[:, :, 5].astype(np.float64))
    ref = (w / (1 + w))[:, :, None]
    rel = 2.0 ** -21 * (u + 4) if typ == "float32" else 2 * HALF + 2.0 ** -21 * (u + 4)
    tol = rel[:, :, None] * ref + (L - 1) * 2.0 ** -37 + (2.0 ** -25 if typ == "float16" else 0)
    assert (np.abs(got - ref) <= tol).all(), (np.abs(got - ref) / tol).max()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("bias", [False, True])
def test_small_capped_scores_beside_rows_with_large_ones(ctx, hd, bias):
    """Rows of one warp: every other one has scores of several caps, the rest scores of up to 1.5, where two
    kinds of keys with values 1 and -1 show the ratio of their weights. fp32 rows.

    A small score x is off by 2^-22 |x| (q in 22 bits) and a few fp32 roundings of its size, so a weight by
    2^-20 with |x| <= 1.5, and by 2^-22 for its own two parts; the output, a difference of two such shares,
    by no more than 2^-19."""
    import realm_b200 as rb
    n, L, cap = 64, 256, 50.0
    q = np.zeros((n, 1, hd), np.float32)
    a = np.linspace(0.02, 1.5, n)
    q[:, 0, 3] = np.where(np.arange(n) % 2, 100.0 * (1 + a), a)
    k = np.zeros((L, 1, hd), np.float16)
    k[0::2, 0, 3], k[1::2, 0, 3] = 1.0, -0.75
    v = np.ones((L, 1, hd), np.float16)
    v[1::2] = -1
    slopes = np.zeros(1, np.float32) if bias else None
    pool = ctx.kv_pool(1, 1, hd, rb.F16, n_pages=L // 16, max_tenants=1, max_seq=L)
    try:
        pool.create(0)
        with pool.plan([0] * L, 1) as p:
            p.append(0, _cuda(k), _cuda(v))
        with pool.plan([0] * n, 1, positions=[L - 1] * n) as p:
            got = _np(p.attention(0, _cuda(q), 1.0, softcap=cap, slopes=None if slopes is None else _cuda(slopes)))
    finally:
        pool.close()
    x = cap * np.tanh(q[:, 0, 3].astype(np.float64)[:, None] * np.array([1.0, -0.75]) / cap)
    ref = np.tanh((x[:, 0] - x[:, 1]) / 2)
    err = np.abs(got[:, 0] - ref[:, None]).max(1)
    assert (err[0::2] <= 2.0 ** -19).all(), err[0::2].max()
    assert (err[1::2] <= 2.0 ** -18).all()  # one kind of key has the whole weight


@pytest.mark.parametrize("typ,cache", [("float16", "F16"), ("float32", "F16"), ("float32", "F32"), ("float16", "F32")])
@pytest.mark.parametrize("shape", ["row", "run"])
@pytest.mark.parametrize("bias", [False, True])
def test_caps_far_from_the_scores(ctx, typ, cache, shape, bias):
    """A cap so large that it changes nothing gives what no cap gives, and one so small that all scores are equal the mean
    of the values; one score is exactly 0. Bounds: twice the error of one of them, scores of up to 8."""
    import torch
    import realm_b200 as rb
    L, H, hd = 300, 4, 64
    n = 1 if shape == "row" else 40
    g = torch.Generator("cuda").manual_seed(5)
    k = torch.randn(L, 1, hd, device="cuda", generator=g)
    k[17] = 0
    v = torch.randn(L, 1, hd, device="cuda", generator=g)
    q = (torch.randn(n, H, hd, device="cuda", generator=g) * 2).to(getattr(torch, typ))
    slopes = torch.full((H,), 2.0 ** -6, device="cuda") if bias else None
    pool = ctx.kv_pool(1, 1, hd, rb.F16 if cache == "F16" else rb.F32, n_pages=L // 16 + 1, max_tenants=1, max_seq=L)
    try:
        pool.create(0)
        with pool.plan([0] * L, H) as p:
            p.append(0, k, v)
        with pool.plan([0] * n, H, positions=[L - 1] * n) as p:
            run = lambda cap: p.attention(0, q, 0.125, softcap=cap, slopes=slopes).double()  # noqa: E731
            none = run(0.0)
            top = v.abs().max().item()
            tol = top * (4 * HALF if typ == "float16" else 2.0 ** -18)
            for cap in (1e9, 1e20, 1e30, 3e38):
                assert ((run(cap) - none).abs() <= tol).all(), cap
            d = torch.arange(L - 1, -1, -1, device="cuda", dtype=torch.float64)
            w = torch.softmax(-d * 2.0 ** -6 if bias else d * 0, 0)
            c = v.to(torch.float16 if cache == "F16" else torch.float32).double()[:, 0]
            for cap in (1e-9, 1e-30, 1e-38, 1e-40, 1e-45):
                assert ((run(cap) - w @ c).abs() <= tol).all(), cap
    finally:
        pool.close()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("shape", ["prompt of documents", "row of 64 heads"])
def test_fp32_rows_lose_little_to_the_order_of_their_sums(ctx, hd, shape):
    """fp32 rows over up to 300 keys, against plain fp32 products of the same inputs: the error against 64 bits stays
    within 1.5 times theirs, or 1e-6. (Parts of 22 bits alone cost about what fp32's own roundings do.)"""
    import torch
    import realm_b200 as rb
    H, kv = (8, 2) if shape[0] == "p" else (64, 1)
    L = 1200 if shape[0] == "p" else 300
    g = torch.Generator("cuda").manual_seed(hd)
    k = torch.randn(L, kv, hd, device="cuda", generator=g).half()
    v = torch.randn(L, kv, hd, device="cuda", generator=g).half()
    pos = np.arange(L) if shape[0] == "p" else np.array([L - 1])
    beg = pos // 300 * 300
    q = torch.randn(len(pos), H, hd, device="cuda", generator=g) * 2.5
    pool = ctx.kv_pool(1, kv, hd, rb.F16, n_pages=L // 16 + 1, max_tenants=1, max_seq=L)
    try:
        pool.create(0)
        with pool.plan([0] * L, H) as p:
            p.append(0, k, v)
        with pool.plan([0] * len(pos), H, positions=pos, begin=beg) as p:
            got = {cap: p.attention(0, q, hd ** -0.5, softcap=cap) for cap in (0.0, 30.0)}
    finally:
        pool.close()
    at, lo, hi = torch.arange(L, device="cuda"), _cuda(beg)[:, None], _cuda(pos)[:, None]
    seen = ((at >= lo) & (at <= hi))[:, None]
    before = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    try:
        for cap, o in got.items():
            outs = []
            for t in (torch.float64, torch.float32):
                kk, vv = (a.to(t).repeat_interleave(H // kv, 1) for a in (k, v))
                x = torch.einsum("nhd,lhd->nhl", q.to(t), kk) * hd ** -0.5
                x = cap * torch.tanh(x / cap) if cap else x
                w = torch.softmax(x.masked_fill(~seen, -torch.inf), -1)
                outs.append(torch.einsum("nhl,lhd->nhd", w, vv).double())
            ref, plain = outs
            e, f = ((a.double() - ref).norm() / ref.norm() for a in (o, plain))
            assert e <= max(1e-6, 1.5 * f), (cap, e.item(), f.item())
    finally:
        torch.backends.cuda.matmul.allow_tf32 = before


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows", [1, 5])
def test_long_sums_of_positive_values(ctx, hd, rows):
    """fp32 rows over thousands of positive values: whatever is cut off a running sum adds up instead of cancelling.
    The sums of a page cut off at most 2 x 2^-23 of themselves (two products of 16 keys each), the rest is rounded:
    a page's share, some hundreds of shares and the parts' join 2^-24 each with any sign, and weights in 22 bits:
    2^-21 in all, with room for the scores' 2^-22 S (S: the weighted mean of |x|, below 2 here)."""
    import torch
    import realm_b200 as rb
    H, kv, T, L = 8, 2, 24, 8000
    g = torch.Generator("cuda").manual_seed(hd)
    pool = ctx.kv_pool(1, kv, hd, rb.F16, n_pages=T * L // 16, max_tenants=T, max_seq=L)
    try:
        K, V = [], []
        for t in range(T):
            pool.create(t)
            K.append(torch.randn(L, kv, hd, device="cuda", generator=g).half())
            V.append((torch.rand(L, kv, hd, device="cuda", generator=g) + 0.5).half())
            with pool.plan([t] * L, H) as p:
                p.append(0, K[t], V[t])
        ten, pos = np.repeat(np.arange(T), rows), np.tile(np.arange(L - rows, L), T)
        q = torch.randn(len(ten), H, hd, device="cuda", generator=g)
        with pool.plan(ten, H, positions=pos) as p:
            got = p.attention(0, q, hd ** -0.5)
    finally:
        pool.close()
    num = den = 0.0
    for r in range(len(ten)):
        k = K[ten[r]][:pos[r] + 1].double().repeat_interleave(H // kv, 1)
        v = V[ten[r]][:pos[r] + 1].double().repeat_interleave(H // kv, 1)
        w = torch.softmax(torch.einsum("hd,khd->hk", q[r].double(), k) * hd ** -0.5, -1)
        ref = torch.einsum("hk,khd->hd", w, v)
        num, den = num + (got[r].double() - ref).square().sum().item(), den + ref.square().sum().item()
    assert (num / den) ** 0.5 <= 2.0 ** -21 + 2.0 ** -21, (num / den) ** 0.5


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("values", ["positive", "random"])
def test_chunks_over_long_contexts(ctx, hd, cap, values):
    """fp32 rows, chunks of 512 rows over 2500 tokens, more of them than SMs. Random values: the error against 64 bits stays
    within 1.5 times that of plain fp32 products, or 1e-6. Positive values: what the tensor core cuts off has one sign;
    at most 2^-23 of the running sum after each 16 keys of each part, 32 times before it is added to the rest: 2^-18."""
    import torch
    import realm_b200 as rb
    H, kv, T, L, rows = 8, 2, 12, 2500, 512
    g = torch.Generator("cuda").manual_seed(hd)
    pool = ctx.kv_pool(1, kv, hd, rb.F16, n_pages=T * (L // 16 + 1), max_tenants=T, max_seq=L)
    K, V = [], []
    try:
        for t in range(T):
            pool.create(t)
            K.append(torch.randn(L, kv, hd, device="cuda", generator=g).half())
            v = torch.randn(L, kv, hd, device="cuda", generator=g)
            V.append((v.abs() + 0.25 if values == "positive" else v).half())
            with pool.plan([t] * L, H) as p:
                p.append(0, K[t], V[t])
        ten, pos = np.repeat(np.arange(T), rows), np.tile(np.arange(L - rows, L), T)
        q = torch.randn(T, rows, H, hd, device="cuda", generator=g)
        with pool.plan(ten, H, positions=pos) as p:
            got = p.attention(0, q.view(-1, H, hd), hd ** -0.5, softcap=cap).view(q.shape)
    finally:
        pool.close()
    seen = (torch.arange(L, device="cuda") <= torch.arange(L - rows, L, device="cuda")[:, None])[:, None]
    before = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    e = f = n = 0.0
    try:
        for t in range(T):
            outs = []
            for typ in (torch.float64, torch.float32):
                k, v = (a[t].to(typ).repeat_interleave(H // kv, 1) for a in (K, V))
                x = torch.einsum("nhd,lhd->nhl", q[t].to(typ), k) * hd ** -0.5
                x = cap * torch.tanh(x / cap) if cap else x
                outs.append(torch.einsum("nhl,lhd->nhd", torch.softmax(x.masked_fill(~seen, -torch.inf), -1), v).double())
            e, f, n = (a + b.square().sum().item() for a, b in ((e, got[t].double() - outs[0]), (f, outs[1] - outs[0]),
                                                                (n, outs[0])))
    finally:
        torch.backends.cuda.matmul.allow_tf32 = before
    e, f = (e / n) ** 0.5, (f / n) ** 0.5
    assert e <= (2.0 ** -18 if values == "positive" else max(1e-6, 1.5 * f)), (e, f)


@pytest.mark.parametrize("hd", [64, 128])
def test_scores_that_rise_by_far(ctx, hd):
    """fp32 rows whose scores climb block by block, by hundreds in all, so that what the earlier keys gave fades out,
    and rows whose first keys come late. A weight is off by 2^-22 and by its score's rounding, 2^-23 of up to 400, twice:
    2^-13 with room; values are up to 1."""
    import torch
    import realm_b200 as rb
    H, L, n = 4, 2048, 300
    g = torch.Generator("cuda").manual_seed(hd)
    k = torch.zeros(L, 1, hd, dtype=torch.float16, device="cuda")
    k[:, 0, 0] = torch.arange(L, device="cuda") / 64.0 + torch.rand(L, device="cuda", generator=g)
    v = (torch.rand(L, 1, hd, device="cuda", generator=g) * 2 - 1).half()
    q = torch.randn(n, H, hd, device="cuda", generator=g)
    q[:, :, 0] = torch.linspace(-12, 12, n * H, device="cuda").view(n, H)
    beg = np.where(np.arange(n) % 7 == 3, 1400, 0)
    pool = ctx.kv_pool(1, 1, hd, rb.F16, n_pages=L // 16, max_tenants=1, max_seq=L)
    try:
        pool.create(0)
        with pool.plan([0] * L, H) as p:
            p.append(0, k, v)
        rep = 40  # more items than SMs: none is cut
        with pool.plan([0] * (n * rep), H, positions=[L - 1] * (n * rep), begin=np.tile(beg, rep)) as p:
            got = p.attention(0, q.repeat(rep, 1, 1), 1.0).view(rep, n, H, hd)
    finally:
        pool.close()
    assert (got - got[:1]).abs().max() <= 2.0 ** -13  # the same rows at other places of their tiles
    seen = torch.arange(L, device="cuda") >= _cuda(beg)[:, None, None]
    x = torch.einsum("nhd,ld->nhl", q.double(), k[:, 0].double()).masked_fill(~seen, -torch.inf)
    ref = torch.einsum("nhl,ld->nhd", torch.softmax(x, -1), v[:, 0].double())
    assert (got[0].double() - ref).abs().max() <= 2.0 ** -13


def test_fp16_chunks_over_very_long_contexts(ctx):
    """fp16 rows over 200000 positive values, more items than SMs: the error stays that of the rows' own rounding, 2^-11
    of the output in the mean square (probabilities' errors average out over the keys)."""
    import torch
    import realm_b200 as rb
    H, hd, L, n = 1, 64, 200000, 64
    g = torch.Generator("cuda").manual_seed(1)
    k = torch.randn(L, 1, hd, device="cuda", generator=g).half()
    v = (torch.rand(L, 1, hd, device="cuda", generator=g) + 0.5).half()
    q = torch.randn(n, H, hd, device="cuda", generator=g).half()
    pool = ctx.kv_pool(1, 1, hd, rb.F16, n_pages=L // 16, max_tenants=1, max_seq=L)
    try:
        pool.create(0)
        with pool.plan([0] * L, H) as p:
            p.append(0, k, v)
        rep = 600
        with pool.plan([0] * (n * rep), H, positions=[L - 1] * (n * rep)) as p:
            got = p.attention(0, q.repeat(rep, 1, 1), hd ** -0.5)[:n].double()
    finally:
        pool.close()
    w = torch.softmax(torch.einsum("nhd,ld->nhl", q.double(), k[:, 0].double()) * hd ** -0.5, -1)
    ref = torch.einsum("nhl,ld->nhd", w, v[:, 0].double())
    assert ((got - ref).norm() / ref.norm()).item() <= HALF


def test_prompts_over_a_models_pool(ctx):
    """Row plans on the pool of a model: a chunk of fp32 rows over several blocks of keys, as over a pool of the caller's."""
    import torch
    import realm_b200 as rb
    cfg = dict(n_layers=1, hidden=256, n_heads=4, n_kv_heads=2, head_dim=64, ffn=256, vocab=256, max_seq=1024, rms_eps=1e-5,
               layer_eps=1e-5, rope_theta=1e4, kv_dtype=rb.F16, max_tenants=1)
    g = torch.Generator("cuda").manual_seed(0)
    k, v = (torch.randn(1000, 2, 64, device="cuda", generator=g) for _ in range(2))
    q = torch.randn(700, 8, 64, device="cuda", generator=g)
    outs = []
    with rb.Context(0) as c:
        model = rb.Model(c, cfg)
        model.tenant_create(0)
        pool = c.kv_pool(1, 2, 64, rb.F16, n_pages=64, max_tenants=1, max_seq=1024)
        pool.create(0)
        for kv in (model.kv, pool):
            with kv.plan([0] * 1000, 8) as p:
                p.append(0, k, v)
            with kv.plan([0] * 700, 8, positions=range(300, 1000)) as p:
                outs.append(p.attention(0, q, 0.125))
    assert torch.equal(*outs) and torch.isfinite(outs[0]).all()


# ---------------------------------------------------------------------------
# steps as a batcher makes them
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("typ,cache", [("float16", "F16"), ("float32", "F16"), ("float32", "F32"), ("float16", "F32")])
@pytest.mark.parametrize("hd,H", [(64, 16), (128, 16), (128, 8), (64, 64)])
@pytest.mark.parametrize("cap,bias,window", [(0.0, False, 0), (30.0, False, 0), (0.0, True, 0), (20.0, True, 3001)])
def test_warps_with_several_units(ctx, typ, cache, hd, H, cap, bias, window):
    """Twenty tenants of 500 to 8000 tokens on 8 kv heads: decode rows, runs of three rows, rows without keys between
    them, and a chunk of 40 rows. Warps take shares of several items, so their loads run over the ends of units.

    A score is known to 2^-22 of its parts (q in 22 bits, a few fp32 roundings) and a weight to twice that and the
    2^-22 of its own two parts; the errors of different keys are independent, so the norm of the output's error is
    at most 2^-21 (2 + S) of its norm, with S the largest weighted mean of |x| + |bias|. fp16 rows: probabilities
    and outputs are rounded, each by 0.41 h in the mean square; 0.7 h together."""
    import torch
    import realm_b200 as rb
    from realm_b200 import rows as R
    kv = 8
    rng = np.random.default_rng(hd + H)
    g = torch.Generator("cuda").manual_seed(hd + H)
    L = [int(n) for n in np.linspace(500, 8000, 20) + np.arange(20) % 16]
    dt = torch.float16 if cache == "F16" else torch.float32
    pool = ctx.kv_pool(1, kv, hd, rb.F16 if cache == "F16" else rb.F32, n_pages=sum((n + 15) // 16 for n in L),
                       max_tenants=len(L), max_seq=max(L))
    try:
        pool.shuffle(3)
        pool.pages().fill_(float("nan"))
        K, V = [], []
        for t, n in enumerate(L):
            pool.create(t)
            K.append(torch.randn(n, kv, hd, device="cuda", generator=g).to(dt))
            V.append(torch.randn(n, kv, hd, device="cuda", generator=g).to(dt))
            with pool.plan([t] * n, H) as p:
                p.append(0, K[t], V[t])
        ten, pos, beg, end = [], [], [], []
        for t in rng.permutation(len(L)):
            for i in range(40 if t == 11 else 3 if t % 4 == 2 else 1):
                at = L[t] - 1 - 2 * i if t != 11 else L[t] - 40 + i
                ten.append(t), pos.append(at), beg.append(0), end.append(at + 1)
            if t % 5 == 3:
                ten.append(t), pos.append(L[t] - 1), beg.append(7), end.append(7)
        ten, pos, beg, end = (np.array(a) for a in (ten, pos, beg, end))
        lo = np.maximum(beg, pos - window + 1) if window else beg
        info = np.stack([pos, np.where(lo < end, lo, 0), np.where(lo < end, end, 0), ten], 1)
        units = R.partition(info, H, kv, ctx.num_sms, cache == "F16")
        small = units[units[:, 0] == 0]
        assert np.bincount(small[:, 1]).max() >= 2 and (cache == "F32" or (units[:, 0] == 1).any())
        n = len(ten)
        q = (torch.randn(n, H, hd, device="cuda", generator=g) * 2).to(getattr(torch, typ))
        slopes = torch.tensor(2.0 ** -np.linspace(1, 8, H), dtype=torch.float32, device="cuda") if bias else None
        scale = 1 / np.sqrt(hd)
        with pool.plan(ten, H, positions=pos, begin=beg, end=end, window=window) as p:
            got = p.attention(0, q, scale, softcap=cap, slopes=slopes)
            again = p.attention(0, q, scale, softcap=cap, slopes=slopes)
        assert torch.equal(got, again)
        ref, S = torch.zeros(n, H, hd, dtype=torch.float64, device="cuda"), 0.0
        for r in range(n):
            if lo[r] >= end[r]:
                continue
            k = K[ten[r]][lo[r]:end[r]].double().repeat_interleave(H // kv, 1)
            v = V[ten[r]][lo[r]:end[r]].double().repeat_interleave(H // kv, 1)
            x = torch.einsum("hd,khd->hk", q[r].double(), k) * scale
            s = cap * torch.tanh(x / cap) if cap else x
            if bias:
                far = slopes.double()[:, None] * torch.arange(pos[r] - lo[r], pos[r] - end[r], -1, device="cuda").abs()
                s, x = s - far, x.abs() + far
            w = torch.softmax(s, -1)
            S = max(S, (w * x.abs()).sum(-1).max().item())
            ref[r] = torch.einsum("hk,khd->hd", w, v)
        empty = torch.from_numpy(lo >= end).cuda()
        assert empty.any() and (got[empty] == 0).all()
        rel = ((got.double() - ref).norm() / ref.norm()).item()
        assert rel <= 2.0 ** -21 * (2 + S) + (0.7 * HALF if typ == "float16" else 0), (rel, S)
    finally:
        pool.close()


@pytest.mark.parametrize("typ", ["float32", "float16"])
@pytest.mark.parametrize("rows,V", [(2, 3000), (5, 32000), (70, 40001), (3, 151937)])
def test_long_histories(ctx, typ, rows, V):
    """Histories of some thousand tokens, with repetitions and tokens past the vocabulary. The largest logit of a
    row after its penalties is the greedy token; a token's penalty is applied once for each time that it is there."""
    import torch
    import realm_b200 as rb
    rng = np.random.default_rng(V)
    x = rng.normal(0, 3, (rows, V)).astype(typ)
    prev = [rng.integers(0, V + 50, int(rng.integers(0, 4000))).tolist() + [int(np.argmax(x[r]))] * (r % 3) for r in range(rows)]
    want = []
    for r in range(rows):
        y = x[r].astype(np.float32)
        for t in prev[r]:
            if t < V:
                y[t] = y[t] / np.float32(1.3) if y[t] > 0 else y[t] * np.float32(1.3)
        want.append(int(np.argmax(y)))
    flat = torch.tensor([t for p in prev for t in p], dtype=torch.int32, device="cuda")
    off = torch.tensor(np.concatenate([[0], np.cumsum([len(p) for p in prev])]), dtype=torch.int32, device="cuda")
    u = np.full(rows, 0.5, np.float32)
    for f in (rb.SamplingFilter(0.0, repetition_penalty=1.3), rb.SamplingFilter(0.7, top_k=1, repetition_penalty=1.3)):
        assert rb.sample_filtered(ctx, x, [f] * rows, u, prev=prev).tolist() == want
        dev = rb.sample_filtered(ctx, _cuda(x), rb.pack_filters([f] * rows, "cuda"), _cuda(u), prev=(flat, off))
        assert dev.tolist() == want

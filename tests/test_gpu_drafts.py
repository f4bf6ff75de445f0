"""GPU tests of filtered probabilities and the verification of drafted tokens.

Weights are held in 40-bit fixed point there and differences of probabilities in 44-bit, so the
choice (which tokens are kept, accepted and drawn) is compared exactly with the same
arithmetic in numpy (integers and 64-bit floats); a probability is a quotient of two such
integers rounded to 32 bits once: off by 2^-24 of itself, and 2^-23 for the weight's own
exponential (the device's is off by at most 2 units of 2^-23; a test computes it in torch on the device).
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------
# filtered probabilities
# ---------------------------------------------------------------------------
def ref_probs(logits, f, prev=None):
    """One row: kept weights (integers) over their sum."""
    import torch
    x = logits.float().cuda().clone()
    if prev is not None and f.repetition_penalty != 1.0:
        for t in prev:
            if t < len(x):
                p = torch.tensor(f.repetition_penalty, device="cuda")
                x[t] = x[t] / p if x[t] > 0 else x[t] * p
    x = torch.where(x.isnan(), torch.full_like(x, -float("inf")), x)
    if not (x > -float("inf")).any():
        return np.zeros(len(x))
    if not f.temperature >= 1e-7:
        out = np.zeros(len(x))
        out[int(torch.nonzero(x == x.max())[0])] = 1
        return out
    x = x / torch.tensor(f.temperature, dtype=torch.float32, device="cuda")
    w = torch.where(x == x.max(), torch.ones_like(x), torch.exp(x - x.max()))
    w = w.cpu().numpy()
    fix = np.floor(w.astype(np.float64) * 2.0 ** 40).astype(np.int64)
    fix[~(w >= np.float32(min(f.min_p, 1.0)))] = 0
    order = np.argsort(-w, kind="stable")
    order = order[fix[order] > 0]
    if 0 < f.top_k < len(w):
        order = order[:f.top_k]
    if 0 < f.top_p < 1:
        s = np.cumsum(fix[order])
        want = max(1, int(float(s[-1]) * float(np.float32(f.top_p))))
        order = order[s - fix[order] < want]
    out = np.zeros(len(w))
    out[order] = fix[order] / float(fix[order].sum())
    return out


def check_probs(got, logits, filters, prev=None):
    for r, f in enumerate(filters):
        ref = ref_probs(logits[r], f, None if prev is None else prev[r])
        g = got[r].double().cpu().numpy()
        assert ((g > 0) == (ref > 2.0 ** -150)).all(), (r, f, int(((g > 0) != (ref > 0)).sum()))
        assert (np.abs(g - ref) <= 2.0 ** -23 * ref).all(), (r, f)


def rules(n):
    import realm_b200 as rb
    F = rb.SamplingFilter
    all_ = [F(1.0), F(0.7, top_k=40, top_p=0.9, min_p=0.02), F(1.0, top_p=0.95), F(0.0), F(1.3, top_k=1), F(0.5, min_p=0.1),
            F(1.0, top_k=1000), F(2.0, top_p=0.5, min_p=1e-4), F(1.0, min_p=2.0), F(0.8, top_p=0.999), F(1.0, top_p=1e-9)]
    return [all_[i % len(all_)] for i in range(n)]


@pytest.mark.parametrize("typ", ["float32", "float16"])
@pytest.mark.parametrize("n,vocab", [(11, 1), (11, 2), (11, 33), (22, 1000), (11, 32000), (5, 65537), (11, 151937), (3, 262144),
                                     (200, 4001)])
def test_probabilities_of_every_rule(ctx, n, vocab, typ):
    import torch
    import realm_b200 as rb
    g = torch.Generator("cuda").manual_seed(vocab + n)
    x = (torch.randn(n, vocab, device="cuda", generator=g) * 3 +
         2 * torch.randn(n, vocab, device="cuda", generator=g).clamp_min(2)).to(getattr(torch, typ))
    f = rules(n)
    out = rb.filter_probs(ctx, x, rb.pack_filters(f, "cuda"))
    check_probs(out, x, f)


@pytest.mark.parametrize("vocab", [500, 40000])
def test_probabilities_ties_flat_and_odd_rows(ctx, vocab):
    """Equal logits (cuts inside a tie keep the lowest indices), infinities, NaNs, rows without a token."""
    import torch
    import realm_b200 as rb
    x = torch.zeros(8, vocab, device="cuda")
    x[1, ::3] = 1.0
    x[2, :] = -float("inf")
    x[2, 77] = 0.0
    x[3, 5] = float("inf")
    x[4, :] = float("nan")
    x[5, ::2] = float("nan")
    x[6] = torch.randint(0, 4, (vocab,), device="cuda").float()
    x[7, 100:] = -3e38
    for f in rules(11):
        out = rb.filter_probs(ctx, x, rb.pack_filters([f] * 8, "cuda"))
        rows = [0, 1, 2, 4, 5, 6, 7]  # of an infinite logit the others' differences are not numbers
        check_probs(out[rows], x[rows], [f] * 7)
        assert (out[4] == 0).all()


def test_probabilities_history_strides_and_host(ctx):
    import torch
    import realm_b200 as rb
    rng = np.random.default_rng(0)
    n, v = 6, 3001
    x = (rng.normal(0, 3, (n, v))).astype(np.float32)
    prev = [[5, 5, 9000, 7], [], [int(np.argmax(x[2]))] * 3, list(range(100)), [0], [3000]]
    f = [rb.SamplingFilter(0.9, 50, 0.9, 0.01, 1.3)] * 3 + [rb.SamplingFilter(1.0, 0, 0.9, 0.0, 0.8)] * 3
    host = rb.filter_probs(ctx, x, f, prev=prev)
    check_probs(torch.from_numpy(host), torch.from_numpy(x), f, prev)
    flat = torch.tensor([t for p in prev for t in p], dtype=torch.int32, device="cuda")
    off = torch.tensor(np.cumsum([0] + [len(p) for p in prev]), dtype=torch.int32, device="cuda")
    for pad, o in ((3, 1), (5, 2), (8, 0)):
        buf = torch.full((n, v + pad), 9.0, device="cuda")
        res = torch.full((n, v + 7), 9.0, device="cuda")
        buf[:, o:o + v] = torch.from_numpy(x)
        rb.filter_probs(ctx, buf[:, o:o + v], rb.pack_filters(f, "cuda"), prev=(flat, off), out=res[:, o:o + v])
        assert torch.equal(res[:, o:o + v].cpu(), torch.from_numpy(host))
        assert (res[:, :o] == 9).all() and (res[:, o + v:] == 9).all()
    assert rb.filter_probs(ctx, torch.from_numpy(x[:0]).cuda(), rb.pack_filters([], "cuda")).shape == (0, v)
    assert rb.filter_probs(ctx, x[:0], []).shape == (0, v)


def test_probabilities_are_what_sampling_draws_from(ctx):
    import torch
    import realm_b200 as rb
    g = torch.Generator("cuda").manual_seed(3)
    n, v = 40, 20011
    x = torch.randn(n, v, device="cuda", generator=g) * 3
    f = rb.pack_filters(rules(n), "cuda")
    p = rb.filter_probs(ctx, x, f)
    prob = torch.empty(n, device="cuda")
    tok = rb.sample_filtered(ctx, x, f, torch.rand(n, device="cuda", generator=g), probs=prob)
    at = p.gather(1, tok.long()[:, None])[:, 0]
    assert ((at - prob).abs() <= 2.0 ** -23 * prob).all()


# ---------------------------------------------------------------------------
# verification
# ---------------------------------------------------------------------------
def ref_verify(p, q, drafts, u, offsets):
    p = np.clip(np.nan_to_num(p.astype(np.float64), nan=0.0), 0, 1)
    q = None if q is None else np.clip(np.nan_to_num(q.astype(np.float64), nan=0.0), 0, 1)
    n, v = p.shape
    tokens, accepted = np.full(n, -7, np.int64), []
    u64 = u.astype(np.float64)
    for a, b in zip(offsets[:-1], offsets[1:]):
        if a == b:
            accepted.append(0)
            continue
        i = a
        while i < b - 1:
            d = drafts[i]
            pd = p[i, d] if 0 <= d < v else 0.0
            qd = 1.0 if q is None or not 0 <= d < v else q[i, d]
            if not u64[i] * qd < pd:
                break
            i += 1
        r = p[i].copy()
        if i < b - 1:
            if q is None:
                if 0 <= drafts[i] < v:
                    r[drafts[i]] = 0
            else:
                r = r - q[i]
        w = np.floor(np.maximum(r, 0) * 2.0 ** 44).astype(np.int64)
        if w.sum() == 0:
            w = np.floor(p[i] * 2.0 ** 44).astype(np.int64)
        total = int(w.sum())
        if total:
            x = u64[b - 1] * float(total)
            want = 0 if not x > 0 else min(int(x), total - 1) if x < float(total) else total - 1
            token = int(np.searchsorted(np.cumsum(w), want, side="right"))
        else:
            token = -1
        tokens[a:i], tokens[i], tokens[i + 1:b] = drafts[a:i], token, -1
        accepted.append(i - a)
    return tokens, np.array(accepted)


def make(rng, counts, v, spread=0.7, sharp=2.0):
    import torch
    n = int(sum(counts))
    x = torch.from_numpy(rng.normal(0, sharp, (n, v)).astype(np.float32))
    p = torch.softmax(x, -1)
    q = torch.softmax(x + spread * torch.from_numpy(rng.normal(0, 1, (n, v)).astype(np.float32)), -1)
    drafts = np.array([rng.choice(v, p=(w := q[i].double().numpy()) / w.sum()) for i in range(n)], np.int32) if n else np.zeros(0, np.int32)
    u = (rng.integers(0, 2 ** 23, n) / 2 ** 23).astype(np.float32)
    return p.numpy(), q.numpy(), drafts, u, np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)


def run(ctx, p, q, drafts, u, offsets, **kw):
    import torch
    import realm_b200 as rb
    c = lambda a: None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    t, a = rb.verify_drafts(ctx, c(p), c(drafts), c(u), c(offsets), draft_probs=c(q), **kw)
    return t.cpu().numpy(), a.cpu().numpy()


@pytest.mark.parametrize("drawn", [True, False])
@pytest.mark.parametrize("requests,most,v", [(1, 0, 1), (1, 5, 7), (3, 2, 1000), (64, 8, 515), (40, 4, 32000), (5, 8, 151937),
                                             (300, 3, 4099), (2, 1, 262144), (2, 700, 64)])
def test_verification(ctx, requests, most, v, drawn):
    rng = np.random.default_rng(requests + most + v)
    counts = [1 + int(rng.integers(0, most + 1)) for _ in range(requests)]
    counts[0] = 1 + most
    p, q, d, u, off = make(rng, counts, v, sharp=2.0 if v < 30000 else 4.0)
    ref = ref_verify(p, q if drawn else None, d, u, off)
    got = run(ctx, p, q if drawn else None, d, u, off)
    assert (got[1] == ref[1]).all()
    assert (got[0] == ref[0]).all(), np.flatnonzero(got[0] != ref[0])[:5]


def test_requests_without_rows_and_rows_of_no_request(ctx):
    import torch
    rng = np.random.default_rng(1)
    p, q, d, u, off = make(rng, [3, 1, 2, 4], 200)
    off = np.array([0, 0, 3, 3, 4, 6, 6, 6], np.int32)  # the last four rows are nobody's
    tokens = torch.full((10,), 77, dtype=torch.int32, device="cuda")
    got = run(ctx, p, q, d, u, off, tokens=tokens)
    ref = ref_verify(p, q, d, u, off)
    assert (got[1] == ref[1]).all() and (got[0][:6] == ref[0][:6]).all() and (got[0][6:] == 77).all()
    assert run(ctx, p, q, d, u, off[:1])[1].shape == (0,)


def test_odd_values(ctx):
    """q above p everywhere, p of nothing, NaNs, values outside [0, 1], drafts outside the vocabulary, uniforms at both ends."""
    v, n = 300, 10
    p, q = np.full((n, v), 1 / v, np.float32), np.full((n, v), 2 / v, np.float32)
    d = np.array([3, 0, -1, 0, v, 0, 7, 0, 9, 0], np.int32)
    u = np.array([0.75, 0.3, 0.0, 1.0, 0.0, 0.0, 0.999, -1.0, 0.5, np.nan], np.float32)
    off = np.arange(0, 11, 2, dtype=np.int32)
    p[4, 10], p[4, 11] = np.nan, 5.0
    q[8] = np.nan
    ref, got = ref_verify(p, q, d, u, off), run(ctx, p, q, d, u, off)
    assert (got[0] == ref[0]).all() and (got[1] == ref[1]).all()
    ref, got = ref_verify(p, None, d, u, off), run(ctx, p, None, d, u, off)
    assert (got[0] == ref[0]).all() and (got[1] == ref[1]).all()
    none = run(ctx, p * 0, q, d, u, off)  # nothing to draw
    assert (none[1] == 0).all() and (none[0] == -1).all()


def test_offsets_on_the_device_that_are_no_rows(ctx):
    rng = np.random.default_rng(2)
    p, q, d, u, _ = make(rng, [6], 50)
    off = np.array([0, 2, 1, 4, 9, -3, 6], np.int32)
    got = run(ctx, p, q, d, u, off)
    assert got[1].tolist()[1:] == [-1, got[1][2], -1, -1, -1] and got[1][0] in (0, 1)


def test_distribution_of_the_first_token(ctx):
    """Over many requests the first token is distributed as p, whatever q is: chi-square over 12 tokens, 11 degrees
    of freedom, below 50 (chance 6e-7)."""
    rng = np.random.default_rng(3)
    v, n = 12, 20000
    pr, qr = rng.dirichlet(np.ones(v)).astype(np.float32), rng.dirichlet(np.ones(v)).astype(np.float32)
    p, q = np.repeat(pr[None], 2 * n, 0), np.repeat(qr[None], 2 * n, 0)
    d = rng.choice(v, size=2 * n, p=qr.astype(np.float64) / qr.astype(np.float64).sum()).astype(np.int32)
    u = rng.random(2 * n).astype(np.float32)
    tokens, _ = run(ctx, p, q, d, u, np.arange(0, 2 * n + 1, 2, dtype=np.int32))
    seen = np.bincount(tokens[::2], minlength=v)
    want = pr.astype(np.float64) / pr.astype(np.float64).sum() * n
    assert ((seen - want) ** 2 / want).sum() < 50


def test_strides_alignment_aliasing_and_graph():
    import torch
    import realm_b200 as rb
    rng = np.random.default_rng(4)
    p, q, d, u, off = make(rng, [4, 2, 5, 1], 1003)
    ref = ref_verify(p, q, d, u, off)
    c = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), rb.Context(0, stream=side.cuda_stream) as ctx:
        for op, oq in ((0, 0), (1, 1), (2, 3), (4, 0)):
            bp, bq = torch.zeros(12, 1010, device="cuda"), torch.zeros(12, 1009, device="cuda")
            bp[:, op:op + 1003], bq[:, oq:oq + 1003] = c(p), c(q)
            t = c(d)
            out, acc = rb.verify_drafts(ctx, bp[:, op:op + 1003], t, c(u), c(off), draft_probs=bq[:, oq:oq + 1003], tokens=t)
            assert out is t and (t.cpu().numpy() == ref[0]).all() and (acc.cpu().numpy() == ref[1]).all()
        args = [c(p), c(d), c(u), c(off)]
        dq, tok, acc = c(q), torch.empty(12, dtype=torch.int32, device="cuda"), torch.empty(4, dtype=torch.int32, device="cuda")
        rb.verify_drafts(ctx, *args, draft_probs=dq, tokens=tok, accepted=acc)
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            rb.verify_drafts(ctx, *args, draft_probs=dq, tokens=tok, accepted=acc)
        u2 = rng.random(12).astype(np.float32)
        args[2].copy_(c(u2))
        g.replay()
        side.synchronize()
        ref = ref_verify(p, q, d, u2, off)
        assert (tok.cpu().numpy() == ref[0]).all() and (acc.cpu().numpy() == ref[1]).all()
        del g


def test_host_arrays_and_refusals(ctx):
    import torch
    import realm_b200 as rb
    rng = np.random.default_rng(5)
    p, q, d, u, off = make(rng, [3, 2], 100)
    ref = ref_verify(p, q, d, u, off)
    t, a = rb.verify_drafts(ctx, p, d, u, off, draft_probs=q)
    assert (t == ref[0]).all() and (a == ref[1]).all()
    for bad in ([0, 3, 2], [0, 3, 6], [3, 0, 5]):
        with pytest.raises(rb.RealmError) as e:
            rb.verify_drafts(ctx, p, d, u, bad, draft_probs=q)
        assert e.value.code == -3
    with pytest.raises(rb.RealmError, match="weighted index"):
        rb.verify_drafts(ctx, p * 0, d, u, off)
    for kw in (dict(draft_probs=q[:, :99]), dict(draft_probs=q[:4]), dict(draft_probs=q.astype(np.float16)),
               dict(tokens=np.zeros(4, np.int32)), dict(accepted=np.zeros(2, np.int64))):
        with pytest.raises(ValueError):
            rb.verify_drafts(ctx, p, d, u, off, **kw)
    for args in ((p.astype(np.float16), d, u, off), (p[0], d, u, off), (p, d[:4], u, off), (p, d, u[:4], off), (p, d, u, [])):
        with pytest.raises(ValueError):
            rb.verify_drafts(ctx, *args)
    c = lambda x: torch.from_numpy(x).cuda()  # noqa: E731
    with pytest.raises(ValueError):
        rb.verify_drafts(ctx, c(p), d, c(u), c(off))
    with pytest.raises(ValueError):
        rb.verify_drafts(ctx, c(p), c(d).long(), c(u), c(off))
    big = torch.zeros(6, dtype=torch.int32, device="cuda")
    with pytest.raises(rb.RealmError, match="overlaps"):
        rb.verify_drafts(ctx, c(p), big[:5], c(u), c(off), tokens=big[1:])
    with pytest.raises(rb.RealmError, match="overlaps"):
        rb.verify_drafts(ctx, c(p), c(d), c(u), c(off), tokens=big[:5], accepted=big[4:])
    with pytest.raises(rb.RealmError) as e:
        rb.verify_drafts(ctx, np.zeros((1, 262145), np.float32), d[:1], u[:1], [0, 1])
    assert e.value.code == -23
    with pytest.raises(ValueError, match="one filter"):
        rb.filter_probs(ctx, p, [rb.SamplingFilter()] * 4)
    with pytest.raises(ValueError, match="float32"):
        rb.filter_probs(ctx, p, [rb.SamplingFilter()] * 5, out=np.zeros((5, 100), np.float16))
    x = c(p)
    with pytest.raises(rb.RealmError, match="overlaps"):
        rb.filter_probs(ctx, x, rb.pack_filters([rb.SamplingFilter()] * 5, "cuda"), out=x)

"""Cases for the serving operators around the paged key-value cache: rows of a
step go in (per-head norms, position rotation, append), attend over the cache
under a mask, and the step's logits are sampled.

Each case runs in a plain form (elementary torch operations in 32 bits) or,
with `own` set, through realm_b200's public calls:

  append     plan.append(layer, k, v, q=...)    KVPool.plan / RowPlan.append
  attention  plan.attention(layer, q, scale)    RowPlan.attention
  sample     sample_filtered(ctx, logits, ...)
"""
import math

import numpy as np
import torch

own = False

PAGE = 16
TYPES = {"f16": torch.float16, "f32": torch.float32}
BYTES = {"f16": 2, "f32": 4}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one decode step of 64 tenants: one new row each, norms of queries and keys, full rotation
        dict(name="append 64 decode rows", op="append", tenants=64, cached=500, rows=1, heads=32, kv_heads=8,
             head_dim=128, type="f16", cache="f16", norm=True, rotary=128, adjacent=False),
        # whole prompts of four tenants in one call
        dict(name="append 4 prompts of 2047", op="append", tenants=4, cached=0, rows=2047, heads=32, kv_heads=8,
             head_dim=128, type="f16", cache="f16", norm=True, rotary=128, adjacent=False),
        # 32-bit rows and cache, half of each head rotated by adjacent pairs, continuing cached prompts
        dict(name="append f32 adjacent 5x333", op="append", tenants=5, cached=77, rows=333, heads=16, kv_heads=16,
             head_dim=64, type="f32", cache="f32", norm=False, rotary=32, adjacent=True),
        # the smallest call: one tenant's next token after a short prompt, in the framework's own 32-bit rows
        dict(name="decode 1x513 capped f32", op="attention", tenants=1, ctx_min=513, ctx_max=513, rows=1, heads=32,
             kv_heads=8, head_dim=128, type="f32", cache="f16", cap=50.0, bias=False, window=0, mask="causal", span=0),
        # a decode step over tenants of mixed lengths, with a bias that falls with distance
        dict(name="decode 16x512-8192 bias", op="attention", tenants=16, ctx_min=512, ctx_max=8192, rows=1, heads=32,
             kv_heads=8, head_dim=128, type="f16", cache="f16", cap=0.0, bias=True, window=0, mask="causal", span=0),
        # long documents: a few tenants, tens of thousands of cached tokens each
        dict(name="decode 4x65537-131072 capped", op="attention", tenants=4, ctx_min=65537, ctx_max=131072, rows=1,
             heads=64, kv_heads=8, head_dim=128, type="f16", cache="f16", cap=30.0, bias=False, window=0,
             mask="causal", span=0),
        # a sliding-window layer over a 32-bit cache
        dict(name="decode 8x100-3001 window f32", op="attention", tenants=8, ctx_min=100, ctx_max=3001, rows=1,
             heads=16, kv_heads=16, head_dim=64, type="f32", cache="f32", cap=0.0, bias=False, window=1024,
             mask="causal", span=0),
        # packed prompts: several documents in each tenant's prompt that must not see one another, 32-bit rows
        dict(name="prompt 6x200-1500 documents", op="attention", tenants=6, ctx_min=200, ctx_max=1500, rows=1500,
             heads=32, kv_heads=8, head_dim=128, type="f32", cache="f16", cap=30.0, bias=False, window=0,
             mask="document", span=300),
        # prompt chunks after cached context, with a prefix that every row sees and a distance bias
        dict(name="chunk 4x512 after 3500-9001", op="attention", tenants=4, ctx_min=3500, ctx_max=9001, rows=512,
             heads=32, kv_heads=32, head_dim=64, type="f16", cache="f16", cap=0.0, bias=True, window=0,
             mask="prefix", span=3800),
        # the largest: one long prompt, capped scores
        dict(name="prompt 8192 capped", op="attention", tenants=1, ctx_min=8192, ctx_max=8192, rows=8192, heads=32,
             kv_heads=8, head_dim=128, type="f16", cache="f16", cap=50.0, bias=False, window=0, mask="causal", span=0),
        # one request's next token over this repository's vocabulary
        dict(name="sample 1x32000", op="sample", rows=1, vocab=32000, temperature=0.8, top_k=40, top_p=0.9,
             min_p=0.02),
        # a full batch over a large vocabulary, nucleus and min-p only
        dict(name="sample 96x151937", op="sample", rows=96, vocab=151937, temperature=1.0, top_k=0, top_p=0.95,
             min_p=0.001),
    ]


def draw(rng):
    """One more case of the listed ones' ranges."""
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["append", "attention", "attention", "attention", "sample"])
    if op == "sample":
        return dict(op=op, rows=log(1, 96), vocab=log(1000, 151937), temperature=rng.choice([0.5, 0.8, 1.0, 1.3]),
                    top_k=rng.choice([0, 1, 20, 40, 200, 1000]), top_p=rng.choice([1.0, 0.99, 0.95, 0.8]),
                    min_p=rng.choice([0.0, 0.001, 0.02, 0.1]))
    hd = rng.choice([64, 128])
    kv = rng.choice([1, 2, 4, 8, 16])
    heads = kv * rng.choice([1, 2, 3, 4, 6, 8])
    while heads * hd > 8192:
        heads //= 2
    heads = max(kv, heads // kv * kv)
    typ = rng.choice(["f16", "f32"])
    cache = "f32" if typ == "f32" and rng.random() < 0.35 else "f16"
    if op == "append":
        tenants = log(1, 64)
        rows = log(1, max(1, 8188 // tenants))
        return dict(op=op, tenants=tenants, cached=rng.choice([0, 15, 16, rng.randint(1, 500)]), rows=rows,
                    heads=heads, kv_heads=kv, head_dim=hd, type=typ, cache=cache, norm=rng.random() < 0.6,
                    rotary=rng.choice([0, 16, hd // 2, hd]), adjacent=rng.random() < 0.5)
    mask = rng.choice(["causal", "causal", "document", "prefix"])
    cap = rng.choice([0.0, 0.0, 30.0, 50.0])
    bias = rng.random() < 0.3
    tenants = log(1, 32)
    if rng.random() < 0.5:  # decode
        longest = log(16, max(16, min(65536, 2 ** 20 // (tenants * kv))))
        rows = 1
    else:
        # 32-bit caches belong to short contexts
        longest = log(16, 1024 if cache == "f32" else 8192)
        rows = log(2, longest)
        while tenants * rows * longest * heads > 8192 * 8192 * 16:
            tenants, rows = max(1, tenants // 2), max(2, rows * 3 // 4)
            longest = max(rows, longest * 3 // 4)
    return dict(op=op, tenants=tenants, ctx_min=max(1, int(longest * rng.uniform(0.1, 1.0))), ctx_max=longest,
                rows=rows, heads=heads, kv_heads=kv, head_dim=hd, type=typ, cache=cache, cap=cap, bias=bias,
                window=rng.choice([0, 0, 128, 1000]), mask=mask, span=log(8, max(8, longest)))


def _spread(lo, hi, n):
    """n lengths from hi down to lo, evenly apart."""
    return np.array([hi - (hi - lo) * i // max(1, n - 1) for i in range(n)], np.int64)


def _rows(case):
    """The rows of an attention case: tenant, position, first and one past the last key that each sees."""
    lens = _spread(case["ctx_min"], case["ctx_max"], case["tenants"])
    count = np.minimum(case["rows"], lens)
    tenant = np.repeat(np.arange(len(lens)), count)
    rank = np.arange(count.sum()) - np.repeat(np.cumsum(count) - count, count)
    pos = (lens - count)[tenant] + rank
    begin, end = np.zeros_like(pos), pos + 1
    if case["mask"] == "document":  # documents of span, span + 1, ... tokens, another offset for each tenant
        at = pos + 7 * tenant
        begin = np.maximum(0, pos - at % max(1, case["span"]))
    if case["mask"] == "prefix":
        end = np.maximum(end, np.minimum(case["span"], lens)[tenant])
    return lens, count, tenant, pos, begin, end


def _seen(case):
    lens, count, tenant, pos, begin, end = _rows(case)
    lo = np.maximum(begin, pos - case["window"] + 1) if case["window"] else begin
    return lens, tenant, np.minimum(lo, end), end


def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4 * n + 36 * case["rows"], "flops": 0}
    hd, kv, heads = case["head_dim"], case["kv_heads"], case["heads"]
    t, c = BYTES[case["type"]], BYTES[case["cache"]]
    if case["op"] == "append":
        n = case["tenants"] * case["rows"]
        return {"bytes": n * hd * ((2 * heads + 2 * kv) * t + 2 * kv * c) + n * case["rotary"] * 4, "flops": 0}
    lens, tenant, lo, hi = _seen(case)
    keys = 0
    for i in range(case["tenants"]):
        m = (tenant == i) & (hi > lo)
        if m.any():
            edge = np.zeros(lens[i] + 1, np.int64)
            np.add.at(edge, lo[m], 1)
            np.add.at(edge, hi[m], -1)
            keys += int((np.cumsum(edge) > 0).sum())
    return {"bytes": keys * kv * hd * 2 * c + 2 * len(tenant) * heads * hd * t,
            "flops": 4 * int((hi - lo).sum()) * heads * hd}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _pages_of(tenant, page, table):
    """Numbers pages 0, 1, ... in the order in which (tenant, page) first come, after those that `table` has."""
    n = int(table.max()) + 1
    key = np.asarray(tenant) * table.shape[1] + np.asarray(page)
    first, at = np.unique(key, return_index=True)
    new = first[np.argsort(at)]
    new = new[table.reshape(-1)[new] < 0]
    table.reshape(-1)[new] = n + np.arange(len(new))


def _fill_rows(lens):
    """(tenant, position) of every cached token, page by page over the tenants, so that each one's pages lie apart."""
    tenant = np.repeat(np.arange(len(lens)), lens)
    pos = np.arange(lens.sum()) - np.repeat(np.cumsum(lens) - lens, lens)
    order = np.lexsort((pos, tenant, pos // PAGE))
    return tenant[order], pos[order]


def _rope_table(n, rotary):
    """[position][cosines | sines] of the usual geometric frequencies, in 32 bits."""
    f = 10000.0 ** (-np.arange(0, rotary, 2, dtype=np.float64) / rotary)
    a = np.arange(n, dtype=np.float64)[:, None] * f
    return np.concatenate([np.cos(a), np.sin(a)], 1).astype(np.float32)


_ctx = []


def _context():
    import realm_b200 as rb
    if not _ctx:
        _ctx.append(rb.Context(0, stream=torch.cuda.current_stream().cuda_stream))
    return _ctx[0]


class State:
    """What a program has in hand before the call; frees the pool that it holds."""

    pool = None

    def __init__(self, **kw):
        self.__dict__.update(kw)

    def __del__(self):
        if self.pool is not None:
            self.pool.close()


def _gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def prepare(case, seed):
    g = _gen(seed)
    if case["op"] == "sample":
        n = case["rows"]
        # logits as a head gives them: a wide spread, a few tokens far ahead of the rest
        x = torch.randn(n, case["vocab"], device="cuda", generator=g) * 3.0
        x += torch.randn(n, case["vocab"], device="cuda", generator=g).clamp_min(2.0) * 2.0
        u = torch.randint(0, 2 ** 23, (n,), device="cuda", generator=g).float() / 2 ** 23
        s = State(case=case, logits=x, uniforms=u, temperature=torch.full((n, 1), case["temperature"], device="cuda"))
        if own:
            import realm_b200 as rb
            s.ctx = _context()
            f = rb.SamplingFilter(case["temperature"], case["top_k"], case["top_p"], case["min_p"])
            s.filters = rb.pack_filters([f] * n, device="cuda")
            s.tokens = torch.empty(n, dtype=torch.int32, device="cuda")
            s.probs = torch.empty(n, device="cuda")
        return s
    T, hd, kv, heads = case["tenants"], case["head_dim"], case["kv_heads"], case["heads"]
    typ, ctyp = TYPES[case["type"]], TYPES[case["cache"]]
    if case["op"] == "append":
        cached = np.array([case["cached"] * (i + 1) // T for i in range(T)], np.int64)
        lens = cached + case["rows"]
        tenant = np.repeat(np.arange(T), case["rows"])
        pos = np.tile(np.arange(case["rows"]), T) + cached[tenant]
    else:
        lens, count, tenant, pos, begin, end = _rows(case)
        cached = lens
    longest = int(lens.max())
    table = np.full((T, (longest + PAGE - 1) // PAGE), -1, np.int64)
    ft, fp = _fill_rows(cached)
    _pages_of(ft, fp // PAGE, table)
    _pages_of(tenant, pos // PAGE, table)
    n_pages = int(table.max()) + 1
    dev = dict(device="cuda")
    s = State(case=case, table=torch.tensor(np.maximum(table, 0), **dev), tenant=torch.tensor(tenant, **dev),
              pos=torch.tensor(pos, **dev))
    pool = None
    if own:
        import realm_b200 as rb
        ctx = _context()
        pool = ctx.kv_pool(1, kv, hd, rb.F16 if case["cache"] == "f16" else rb.F32, n_pages=n_pages, max_tenants=T,
                           max_seq=longest)
        s.pool = pool
        for t in range(T):
            pool.create(t)
    n = len(tenant)
    if case["op"] == "append":
        # the output of a fused projection: q, k and v are slices of one row
        s.qkv = (torch.randn(n, (heads + 2 * kv) * hd, generator=g, **dev) * 1.5).to(typ)
        s.q_norm = 1 + 0.1 * torch.randn(hd, generator=g, **dev) if case["norm"] else None
        s.k_norm = 1 + 0.1 * torch.randn(hd, generator=g, **dev) if case["norm"] else None
        s.rope = torch.tensor(_rope_table(longest, case["rotary"]), **dev) if case["rotary"] else None
        if own:
            if len(ft):
                zero = torch.zeros(len(ft), kv, hd, dtype=typ, **dev)
                with pool.plan(ft, heads, positions=fp) as fill:
                    fill.append(0, zero, zero)
            s.plan = pool.plan(tenant, heads)
            s.q_out = torch.empty(n, heads, hd, dtype=typ, **dev)
            s.pages = pool.pages()
        else:
            s.pages = torch.zeros(n_pages, 1, 2, kv, PAGE, hd, dtype=ctyp, **dev)
        return s
    pages = torch.randn(n_pages, 1, 2, kv, PAGE, hd, generator=g, dtype=ctyp, **dev)
    # normalised and rotated queries; capped models have larger scores
    s.q = (torch.randn(n, heads, hd, generator=g, **dev) * (2.5 if case["cap"] else 1.2)).to(typ)
    s.slopes = torch.tensor(2.0 ** (-8.0 * np.arange(1, heads + 1) / heads), dtype=torch.float32, **dev) \
        if case["bias"] else None
    s.scale = 1.0 / math.sqrt(hd)
    if own:
        at, off = torch.tensor(table[ft, fp // PAGE], **dev), torch.tensor(fp % PAGE, **dev)
        step = 1 << 16
        with pool.plan(ft, heads, positions=fp) as fill:
            kr = torch.cat([pages[at[i:i + step], 0, 0, :, off[i:i + step]] for i in range(0, len(ft), step)])
            vr = torch.cat([pages[at[i:i + step], 0, 1, :, off[i:i + step]] for i in range(0, len(ft), step)])
            fill.append(0, kr, vr)
        s.plan = pool.plan(tenant, heads, positions=pos, begin=begin, end=end, window=case["window"])
        s.out = torch.empty_like(s.q)
    else:
        s.pages = pages
        R = int(count.max())
        first = np.cumsum(count) - count
        take = np.minimum(np.arange(R)[None], (count - 1)[:, None]) + first[:, None]
        s.take = torch.tensor(take, **dev)  # [T][R]: row of the call, the last one repeated
        s.back = torch.tensor(tenant * R + (np.arange(n) - first[tenant]), **dev)
        s.begin, s.end = torch.tensor(begin, **dev), torch.tensor(end, **dev)
        s.longest = longest
    return s


# ---------------------------------------------------------------------------
# the operators
# ---------------------------------------------------------------------------
def run(s):
    return RUN[own, s.case["op"]](s)


def _append_own(s):
    c = s.case
    H, kv, hd = c["heads"], c["kv_heads"], c["head_dim"]
    x = s.qkv.view(-1, H + 2 * kv, hd)
    s.plan.append(0, x[:, H:H + kv], x[:, H + kv:], q=x[:, :H], q_out=s.q_out, q_norm=s.q_norm, k_norm=s.k_norm,
                  eps=1e-6, rope=s.rope, adjacent=c["adjacent"])
    return s.q_out, s.pages


def _attention_own(s):
    c = s.case
    s.plan.attention(0, s.q, s.scale, softcap=c["cap"], slopes=s.slopes, out=s.out)
    return s.out


def _sample_own(s):
    import realm_b200 as rb
    rb.sample_filtered(s.ctx, s.logits, s.filters, s.uniforms, out=s.tokens, probs=s.probs)
    return s.tokens, s.probs


def _norm(x, w):
    return x if w is None else x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w


def _rotate(x, cs, adjacent):
    rot = cs.shape[1]
    c, n = cs[:, None, :rot // 2], cs[:, None, rot // 2:]
    r = x[..., :rot]
    a, b = (r[..., 0::2], r[..., 1::2]) if adjacent else (r[..., :rot // 2], r[..., rot // 2:])
    a, b = a * c - b * n, b * c + a * n
    r = torch.stack([a, b], -1).flatten(-2) if adjacent else torch.cat([a, b], -1)
    return torch.cat([r, x[..., rot:]], -1)


def _append_plain(s):
    c = s.case
    H, kv, hd = c["heads"], c["kv_heads"], c["head_dim"]
    x = s.qkv.view(-1, H + 2 * kv, hd).float()
    q, k, v = _norm(x[:, :H], s.q_norm), _norm(x[:, H:H + kv], s.k_norm), x[:, H + kv:]
    if s.rope is not None:
        cs = s.rope[s.pos]
        q, k = _rotate(q, cs, c["adjacent"]), _rotate(k, cs, c["adjacent"])
    page, off = s.table[s.tenant, s.pos // PAGE], s.pos % PAGE
    s.pages[page, 0, 0, :, off] = k.to(s.pages.dtype)
    s.pages[page, 0, 1, :, off] = v.to(s.pages.dtype)
    return q.to(s.qkv.dtype), s.pages


def _attention_plain(s):
    c = s.case
    H, kv, hd, T = c["heads"], c["kv_heads"], c["head_dim"], c["tenants"]
    rep, R, L = H // kv, s.take.shape[1], s.longest
    kvs = s.pages[s.table][:, :, 0, :, :, :].permute(2, 0, 3, 1, 4, 5).reshape(2, T, kv, -1, hd)[:, :, :, :L].float()
    q = s.q[s.take].float().view(T, R, kv, rep, hd).permute(0, 2, 3, 1, 4).reshape(T, kv, rep * R, hd)
    x = (torch.matmul(q, kvs[0].transpose(-1, -2)) * s.scale).view(T, kv, rep, R, L)
    if c["cap"]:
        x = c["cap"] * torch.tanh(x / c["cap"])
    at, pos = torch.arange(L, device=x.device), s.pos[s.take][..., None]
    if s.slopes is not None:
        x = x - s.slopes.view(1, kv, rep, 1, 1) * (pos - at).abs().float()[:, None, None]
    lo, hi = s.begin[s.take][..., None], s.end[s.take][..., None]
    if c["window"]:
        lo = torch.maximum(lo, pos - c["window"] + 1)
    seen = ((at >= lo) & (at < hi))[:, None, None]
    x = x.masked_fill(~seen, -math.inf)
    top = x.amax(-1, keepdim=True)
    x = torch.exp(x - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(T, kv, rep * R, L), kvs[1]).view(T, kv, rep, R, hd)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    return o.permute(0, 3, 1, 2, 4).reshape(T * R, H, hd)[s.back].to(s.q.dtype)


def _sample_plain(s):
    """Weights exp((x - max) / t) in 40-bit fixed point, so that no sum depends on its order."""
    c = s.case
    x = s.logits / s.temperature
    w = torch.exp(x - x.amax(-1, keepdim=True))
    order = torch.sort(w, dim=-1, descending=True, stable=True)
    ranked = order.values
    fixed = (ranked.double() * 2.0 ** 40).long()
    keep = ranked >= c["min_p"]
    if c["top_k"]:
        keep = keep & (torch.arange(w.shape[1], device=w.device) < c["top_k"])
    fixed = fixed * keep
    if c["top_p"] < 1.0:
        before = fixed.cumsum(-1) - fixed
        keep = keep & (before < (before[:, -1:] + fixed[:, -1:]).double().mul(float(np.float32(c["top_p"]))).long())
        fixed = fixed * keep
    mass = torch.zeros_like(fixed).scatter_(-1, order.indices, fixed)
    run_ = mass.cumsum(-1)
    total = run_[:, -1:]
    target = (s.uniforms.double()[:, None] * total.double()).long()
    token = (run_ > target).to(torch.uint8).argmax(-1, keepdim=True)
    prob = mass.gather(-1, token).double() / total.double()
    return token[:, 0].int(), prob[:, 0].float()


RUN = {(False, "append"): _append_plain, (False, "attention"): _attention_plain, (False, "sample"): _sample_plain,
       (True, "append"): _append_own, (True, "attention"): _attention_own, (True, "sample"): _sample_own}


# ---------------------------------------------------------------------------
# the same in 64 bits, from the definitions
# ---------------------------------------------------------------------------
def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "sample":
        p = torch.softmax(s.logits.double() / s.temperature.double(), -1)
        top, at = torch.sort(p, dim=-1, descending=True, stable=True)
        top = torch.where(top >= case["min_p"] * top[:, :1], top, 0.0)
        if case["top_k"]:
            top[:, case["top_k"]:] = 0
        top /= top.sum(-1, keepdim=True)
        top = torch.where((top.cumsum(-1) - top) < case["top_p"], top, 0.0)
        p = torch.zeros_like(p).scatter_(-1, at, top / top.sum(-1, keepdim=True))
        token = (p.cumsum(-1) <= s.uniforms.double()[:, None]).sum(-1).clamp_max(case["vocab"] - 1)
        return token.int(), p.gather(-1, token[:, None])[:, 0]
    hd, kv, heads = case["head_dim"], case["kv_heads"], case["heads"]
    if case["op"] == "append":
        x = s.qkv.double().view(-1, heads + 2 * kv, hd)
        parts = {}
        for name, lo, hi, w in (("q", 0, heads, s.q_norm), ("k", heads, heads + kv, s.k_norm)):
            y = x[:, lo:hi].clone()
            if w is not None:
                y = y / torch.sqrt(y.pow(2).sum(-1, keepdim=True) / hd + 1e-6) * w.double()
            if case["rotary"]:
                half = case["rotary"] // 2
                turn = torch.complex(s.rope[s.pos, :half].double(), s.rope[s.pos, half:].double())[:, None]
                i = torch.arange(half, device="cuda")
                i, j = (2 * i, 2 * i + 1) if case["adjacent"] else (i, i + half)
                z = torch.complex(y[..., i], y[..., j]) * turn
                y[..., i], y[..., j] = z.real, z.imag
            parts[name] = y
        pages = torch.zeros(s.pages.shape, dtype=torch.float64, device="cuda")
        at = s.table[s.tenant, s.pos // PAGE]
        pages[at, 0, 0, :, s.pos % PAGE] = parts["k"]
        pages[at, 0, 1, :, s.pos % PAGE] = x[:, heads + kv:]
        return parts["q"], pages
    lens, tenant, lo, hi = _seen(case)
    out = torch.zeros(s.q.shape, dtype=torch.float64, device="cuda")
    lo, hi = torch.tensor(lo, device="cuda"), torch.tensor(hi, device="cuda")
    for t in range(case["tenants"]):
        of = torch.tensor(np.flatnonzero(tenant == t), device="cuda")
        kvs = s.pages[s.table[t], 0].double().permute(1, 2, 0, 3, 4).reshape(2, kv, -1, hd)[:, :, :int(lens[t])]
        key = torch.arange(kvs.shape[2], device="cuda")
        for part in of.split(max(1, (1 << 26) // kvs.shape[2])):
            dark = (key < lo[part, None]) | (key >= hi[part, None])
            for h in range(heads):
                x = s.q[part, h].double() @ kvs[0, h * kv // heads].T / math.sqrt(hd)
                if case["cap"]:
                    x = torch.tanh(x / case["cap"]) * case["cap"]
                if s.slopes is not None:
                    x -= (s.pos[part, None] - key).abs() * s.slopes[h].double()
                x = torch.softmax(x.masked_fill_(dark, -math.inf), -1).nan_to_num_(0.0)
                out[part, h] = x @ kvs[1, h * kv // heads]
    return out

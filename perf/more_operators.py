"""Cases for the operators of a step in which every tenant has an adapter of its own
and drafted tokens are verified: low-rank adapters beside a shared projection, the
norms around a block with its gate and residual, the distribution that filtered
sampling draws from, and the verification of drafted tokens.

Each case runs in a plain form (elementary torch operations in 32 bits, in 64 where a
choice is made) or, with `own` set, through realm_b200's public calls:

  adapters   adapters.add(x, slots, y, out=...)         Context.adapters / AdapterSet
  norm       residual_norm(ctx, y, x, ...)
  probs      filter_probs(ctx, logits, filters, ...)
  verify     verify_drafts(ctx, probs, drafts, ...)
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f16": torch.float16, "f32": torch.float32}
BYTES = {"f16": 2, "f32": 4}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # the smallest: one tenant's next token through a square projection, in Weight.matmul's 32-bit rows
        dict(name="adapters 1 row", op="adapters", rows=1, tenants=1, k=4096, n=4096, rank_min=16, rank_max=16,
             type="f32", mixed=False, bare=0.0),
        # a decode step: most rows are of different tenants, ranks differ, some tenants have no adapter
        dict(name="adapters 48 rows of 31 tenants", op="adapters", rows=48, tenants=31, k=4096, n=11008, rank_min=8,
             rank_max=64, type="f32", mixed=True, bare=0.15),
        # short prompts and single tokens of odd sizes in one call, rows off 16 bytes
        dict(name="adapters 701 rows odd", op="adapters", rows=701, tenants=13, k=2072, n=1001, rank_min=5,
             rank_max=24, type="f32", mixed=True, bare=0.1),
        # long prompts of a few tenants, 16-bit rows
        dict(name="adapters 8192 rows of prompts", op="adapters", rows=8192, tenants=4, k=4096, n=4096, rank_min=64,
             rank_max=64, type="f16", mixed=False, bare=0.0),
        # prompts through a wide projection in 32-bit rows, up to the largest ranks
        dict(name="adapters 4096 rows wide", op="adapters", rows=4096, tenants=9, k=11008, n=4096, rank_min=8,
             rank_max=128, type="f32", mixed=False, bare=0.1),
        # between two blocks of one decoded token
        dict(name="norm 1x4096", op="norm", rows=1, dim=4096, type="f32", stream="f32", post=True, gate="none",
             scale=1.0, pre=True),
        # between two blocks of a prompt: 16-bit blocks on a 32-bit residual stream, learned gate
        dict(name="norm 8192x4096 gate", op="norm", rows=8192, dim=4096, type="f16", stream="f32", post=True,
             gate="shared", scale=0.25, pre=True),
        # odd sizes, gates of each row, no norm behind the block
        dict(name="norm 333x5001 gates", op="norm", rows=333, dim=5001, type="f32", stream="f32", post=False,
             gate="rows", scale=1.0, pre=True),
        # one tenant's draft step over this repository's vocabulary
        dict(name="probs 1x32000", op="probs", rows=1, vocab=32000, temperature=0.8, top_k=40, top_p=0.9, min_p=0.02,
             type="f32"),
        # the target's rows of a batch with four drafted tokens each, nucleus only
        dict(name="probs 160x151937", op="probs", rows=160, vocab=151937, temperature=1.0, top_k=0, top_p=0.95,
             min_p=0.0, type="f32"),
        # one request, tokens drafted by looking them up in its own history (no probabilities)
        dict(name="verify 1x6 looked up", op="verify", requests=1, drafts_min=6, drafts_max=6, vocab=32000, sampled=False,
             sharp=3.0),
        # a batch of requests with zero to eight tokens from a draft model
        dict(name="verify 64x0-8", op="verify", requests=64, drafts_min=0, drafts_max=8, vocab=151937, sampled=True,
             sharp=2.5),
    ]


def draw(rng):
    """One more case of the listed ones' ranges."""
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["adapters", "adapters", "adapters", "norm", "probs", "verify"])
    if op == "adapters":
        rows = log(1, 8192)
        k, n = log(256, 11008), log(256, 11008)
        if rng.random() < 0.6:
            k = max(256, k // 64 * 64)
        if rng.random() < 0.6:
            n = max(256, n // 64 * 64)
        typ = rng.choice(["f16", "f32"])
        lo = log(4, 128)
        c = dict(op=op, rows=rows, tenants=log(1, 64), k=k, n=n, rank_min=lo,
                 rank_max=lo if rng.random() < 0.5 else log(lo, 128), type=typ, mixed=rng.random() < 0.5,
                 bare=rng.choice([0.0, 0.0, 0.2]))
        while True:
            c["tenants"] = min(c["tenants"], c["rows"])
            if work(c)["bytes"] <= 3.3e8:
                return c
            c["rows"] = c["rows"] * 3 // 4
    if op == "norm":
        dim = log(64, 16384)
        if rng.random() < 0.6:
            dim = max(64, dim // 64 * 64)
        typ = rng.choice(["f16", "f32"])
        return dict(op=op, rows=log(1, max(1, min(8192, 20000000 // dim))), dim=dim, type=typ,
                    stream=rng.choice(["f32", typ]), post=rng.random() < 0.7, gate=rng.choice(["none", "shared", "rows"]),
                    scale=rng.choice([1.0, 0.25, 1.5]), pre=rng.random() < 0.8)
    if op == "probs":
        return dict(op=op, rows=log(1, 160), vocab=log(1000, 151937), temperature=rng.choice([0.5, 0.8, 1.0, 1.3]),
                    top_k=rng.choice([0, 1, 20, 40, 200, 1000]), top_p=rng.choice([1.0, 0.99, 0.95, 0.8]),
                    min_p=rng.choice([0.0, 0.001, 0.02, 0.1]), type=rng.choice(["f32", "f32", "f16"]))
    lo = rng.randint(0, 8)
    return dict(op=op, requests=log(1, 64), drafts_min=lo, drafts_max=rng.randint(lo, 8), vocab=log(1000, 151937),
                sampled=rng.random() < 0.7, sharp=rng.choice([1.0, 2.5, 4.0]))


def _ranks(case):
    t = case["tenants"]
    return [case["rank_min"] + (case["rank_max"] - case["rank_min"]) * i // max(1, t - 1) for i in range(t)]


def _slots(case):
    """The slot of every row, -1 for tenants without an adapter: requests one after the other, or all mixed."""
    rows, t = case["rows"], case["tenants"]
    of = np.arange(rows) * 7 % t if case["mixed"] else np.arange(rows) * t // rows
    bare = np.array([(i * 37 % 100) < 100 * case["bare"] and i > 0 for i in range(t)])
    return np.where(bare[of], -1, of)


def _offsets(case):
    """First row of every request, and their number: drafted tokens and one more row each."""
    lo, hi = case["drafts_min"], case["drafts_max"]
    count = [1 + lo + i * 5 % (hi - lo + 1) for i in range(case["requests"])]
    return np.concatenate([[0], np.cumsum(count)]).astype(np.int64)


def work(case):
    if case["op"] == "adapters":
        t, k, n = BYTES[case["type"]], case["k"], case["n"]
        slots, ranks = _slots(case), _ranks(case)
        used = sorted(set(slots[slots >= 0].tolist()))
        have = int((slots >= 0).sum())
        # y is read and out written for all rows, x read for those with an adapter
        return {"bytes": have * k * t + 2 * len(slots) * n * t + sum(ranks[a] for a in used) * (k + n) * 2 + 4 * len(slots),
                "flops": 2 * sum(ranks[a] for a in slots.tolist() if a >= 0) * (k + n)}
    if case["op"] == "norm":
        n = case["rows"] * case["dim"]
        t, r = BYTES[case["type"]], BYTES[case["stream"]]
        gate = {"none": 0, "shared": case["dim"] * t, "rows": n * t}[case["gate"]]
        return {"bytes": n * (t + 2 * r) + (n * t if case["pre"] else 0) + gate + 4 * case["dim"] * (case["post"] + case["pre"]),
                "flops": 0}
    if case["op"] == "probs":
        return {"bytes": case["rows"] * (case["vocab"] * (BYTES[case["type"]] + 4) + 20), "flops": 0}
    # a request's token is drawn from one row at least
    return {"bytes": case["requests"] * case["vocab"] * 4 + int(_offsets(case)[-1]) * 20, "flops": 0}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
_ctx = []


def _context():
    import realm_b200 as rb
    if not _ctx:
        _ctx.append(rb.Context(0, stream=torch.cuda.current_stream().cuda_stream))
    return _ctx[0]


class State:
    """What a program has in hand before the call; frees the adapters that it holds."""

    adapters = None

    def __init__(self, **kw):
        self.__dict__.update(kw)

    def __del__(self):
        if self.adapters is not None:
            self.adapters.close()


def _logits(g, rows, vocab, spread):
    """As a head gives them: a wide spread, a few tokens far ahead of the rest."""
    x = torch.randn(rows, vocab, device="cuda", generator=g) * spread
    return x + torch.randn(rows, vocab, device="cuda", generator=g).clamp_min(2.0) * 2.0


def _uniform(g, n):
    return torch.randint(0, 2 ** 23, (n,), device="cuda", generator=g).float() / 2 ** 23


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    dev = dict(device="cuda")
    if case["op"] == "adapters":
        typ, rows, k, n = TYPES[case["type"]], case["rows"], case["k"], case["n"]
        ranks = _ranks(case)
        s = State(case=case, x=torch.randn(rows, k, generator=g, **dev).to(typ),
                  y=torch.randn(rows, n, generator=g, **dev).to(typ),
                  # trained adapters: down of a random projection's size, up grown from zero
                  down=[(torch.randn(r, k, generator=g, **dev) / math.sqrt(k)).half() for r in ranks],
                  up=[(torch.randn(n, r, generator=g, **dev) * 0.1).half() for r in ranks],
                  scales=[2.0 if r % 2 else 1.0 + 1.0 / r for r in ranks],
                  slots=torch.tensor(_slots(case), dtype=torch.int32, **dev))
        if own:
            s.adapters = _context().adapters(n, k, case["tenants"], max(ranks))
            for a, (d, u, f) in enumerate(zip(s.down, s.up, s.scales)):
                s.adapters.set(a, d, u, f)
            s.out = torch.empty_like(s.y)
        else:
            at = _slots(case)
            s.of = [(a, torch.tensor(np.flatnonzero(at == a), **dev)) for a in sorted(set(at[at >= 0].tolist()))]
        return s
    if case["op"] == "norm":
        typ, stream, rows, dim = TYPES[case["type"]], TYPES[case["stream"]], case["rows"], case["dim"]
        s = State(case=case, y=(torch.randn(rows, dim, generator=g, **dev) * 0.7).to(typ),
                  x=(torch.randn(rows, dim, generator=g, **dev) * 3.0).to(stream),
                  post=1 + 0.1 * torch.randn(dim, generator=g, **dev) if case["post"] else None,
                  pre=1 + 0.1 * torch.randn(dim, generator=g, **dev) if case["pre"] else None, gate=None)
        if case["gate"] != "none":
            s.gate = torch.randn(*([rows] if case["gate"] == "rows" else []), dim, generator=g, **dev).to(typ)
        if own:
            s.ctx = _context()
            s.x_out = torch.empty_like(s.x)
            s.out = torch.empty_like(s.y) if case["pre"] else None
        return s
    if case["op"] == "probs":
        n = case["rows"]
        s = State(case=case, logits=_logits(g, n, case["vocab"], 3.0).to(TYPES[case["type"]]),
                  temperature=torch.full((n, 1), case["temperature"], **dev))
        if own:
            import realm_b200 as rb
            s.ctx = _context()
            f = rb.SamplingFilter(case["temperature"], case["top_k"], case["top_p"], case["min_p"])
            s.filters = rb.pack_filters([f] * n, device="cuda")
            s.out = torch.empty(n, case["vocab"], **dev)
        return s
    at = _offsets(case)
    rows, vocab = int(at[-1]), case["vocab"]
    logits = _logits(g, rows, vocab, case["sharp"])
    s = State(case=case, probs=torch.softmax(logits, -1), uniforms=_uniform(g, rows), draft_probs=None,
              offsets=torch.tensor(at, dtype=torch.int32, **dev))
    if case["sampled"]:  # by a smaller model whose logits are near the target's; the last row of a request has no draft
        s.draft_probs = torch.softmax(logits + 0.7 * torch.randn(rows, vocab, generator=g, **dev), -1)
        pick = s.draft_probs
    else:
        pick = s.probs
    u = torch.rand(rows, 1, generator=g, **dev)
    s.drafts = (pick.double().cumsum(-1) <= u).sum(-1).clamp_max(vocab - 1).int()
    if own:
        s.ctx = _context()
        s.tokens = torch.full((rows,), -1, dtype=torch.int32, **dev)
        s.accepted = torch.empty(case["requests"], dtype=torch.int32, **dev)
    else:
        s.first, s.last = s.offsets[:-1].long(), s.offsets[1:].long() - 1
        s.request = torch.tensor(np.repeat(np.arange(case["requests"]), np.diff(at)), **dev)
    return s


# ---------------------------------------------------------------------------
# the operators
# ---------------------------------------------------------------------------
def run(s):
    return RUN[own, s.case["op"]](s)


def _adapters_own(s):
    s.adapters.add(s.x, s.slots, s.y, out=s.out)
    return s.out


def _norm_own(s):
    import realm_b200 as rb
    c = s.case
    rb.residual_norm(s.ctx, s.y, s.x, post_norm=s.post, gate=s.gate, scale=c["scale"], pre_norm=s.pre, eps=1e-6,
                     x_out=s.x_out, out=s.out)
    return (s.x_out, s.out) if c["pre"] else (s.x_out,)


def _probs_own(s):
    import realm_b200 as rb
    rb.filter_probs(s.ctx, s.logits, s.filters, out=s.out)
    return s.out


def _verify_own(s):
    import realm_b200 as rb
    rb.verify_drafts(s.ctx, s.probs, s.drafts, s.uniforms, s.offsets, draft_probs=s.draft_probs, tokens=s.tokens,
                     accepted=s.accepted)
    return s.tokens, s.accepted


def _adapters_plain(s):
    out = s.y.float()
    out = out.clone() if out is s.y else out
    for a, rows in s.of:
        v = torch.matmul(s.x[rows].float(), s.down[a].float().T)
        out[rows] += s.scales[a] * torch.matmul(v, s.up[a].float().T)
    return out.to(s.y.dtype)


def _rms(x, w):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w


def _norm_plain(s):
    c = s.case
    z = s.y.float()
    if s.post is not None:
        z = _rms(z, s.post)
    if s.gate is not None:
        z = z * s.gate.float()
    h = s.x.float() + c["scale"] * z
    if s.pre is None:
        return (h.to(s.x.dtype),)
    return h.to(s.x.dtype), _rms(h, s.pre).to(s.y.dtype)


def _probs_plain(s):
    """Weights exp((x - max) / t) in 40-bit fixed point, so that no sum depends on its order."""
    c = s.case
    x = s.logits.float() / s.temperature
    w = torch.exp(x - x.amax(-1, keepdim=True))
    order = torch.sort(w, dim=-1, descending=True, stable=True)
    ranked = order.values
    fixed = (ranked.double() * 2.0 ** 40).long()
    keep = ranked >= float(np.float32(c["min_p"]))
    if c["top_k"]:
        keep = keep & (torch.arange(w.shape[1], device=w.device) < c["top_k"])
    fixed = fixed * keep
    if c["top_p"] < 1.0:
        run_ = fixed.cumsum(-1)
        keep = run_ - fixed < run_[:, -1:].double().mul(float(np.float32(c["top_p"]))).long()
        fixed = fixed * keep
    p = (fixed.double() / fixed.sum(-1, keepdim=True).double()).float()
    return torch.zeros_like(w).scatter_(-1, order.indices, p)


def _verify_plain(s):
    """The tests in 64 bits (products of 32-bit values, exact); the draw's weights in 44-bit fixed point."""
    rows, vocab = s.probs.shape
    at = torch.arange(rows, device="cuda")
    d = s.drafts.long()
    p = s.probs[at, d].double()
    q = torch.ones_like(p) if s.draft_probs is None else s.draft_probs[at, d].double()
    refused = ~(s.uniforms.double() * q < p) | (at == s.last[s.request])
    # the first refused row of each request; its last row always is
    stop = torch.where(refused, at, torch.full_like(at, rows))
    stop = torch.full_like(s.last, rows).scatter_reduce_(0, s.request, stop, "amin")
    r = s.probs[stop].double()
    inner = (stop < s.last)[:, None]
    if s.draft_probs is None:
        r = torch.where(inner & (torch.arange(vocab, device="cuda") == d[stop][:, None]), 0.0, r)
    else:
        r = torch.where(inner, r - s.draft_probs[stop].double(), r)
    fixed = (r.clamp(0.0, 1.0) * 2.0 ** 44).long()
    sums = fixed.cumsum(-1)
    total = sums[:, -1:]
    want = torch.minimum((s.uniforms[s.last].double()[:, None] * total.double()).long(), total - 1)
    token = (sums <= want).sum(-1).int()
    tokens = torch.where(at < stop[s.request], s.drafts, -1)
    tokens[stop] = token
    return tokens, (stop - s.first).int()


RUN = {(False, "adapters"): _adapters_plain, (False, "norm"): _norm_plain, (False, "probs"): _probs_plain,
       (False, "verify"): _verify_plain, (True, "adapters"): _adapters_own, (True, "norm"): _norm_own,
       (True, "probs"): _probs_own, (True, "verify"): _verify_own}


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
    if case["op"] == "adapters":
        out = s.y.double()
        for row in torch.arange(case["rows"], device="cuda").split(1024):
            for a in set(s.slots[row].tolist()) - {-1}:
                of = row[s.slots[row] == a]
                out[of] += (s.x[of].double() @ s.down[a].double().T) @ (s.up[a].double().T * s.scales[a])
        return out
    if case["op"] == "norm":
        y, x = s.y.double(), s.x.double()
        if s.post is not None:
            y = y / torch.sqrt(y.pow(2).sum(-1, keepdim=True) / case["dim"] + 1e-6) * s.post.double()
        if s.gate is not None:
            y = y * s.gate.double()
        x = x + y * case["scale"]
        if s.pre is None:
            return (x,)
        return x, x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / case["dim"] + 1e-6) * s.pre.double()
    if case["op"] == "probs":
        p = torch.softmax(s.logits.double() / s.temperature.double(), -1)
        top, at = torch.sort(p, dim=-1, descending=True, stable=True)
        top = torch.where(top >= case["min_p"] * top[:, :1], top, 0.0)
        if case["top_k"]:
            top[:, case["top_k"]:] = 0
        top /= top.sum(-1, keepdim=True)
        top = torch.where((top.cumsum(-1) - top) < case["top_p"], top, 0.0)
        return torch.zeros_like(p).scatter_(-1, at, top / top.sum(-1, keepdim=True))
    tokens, accepted = [], []
    at = _offsets(case).tolist()
    u = s.uniforms.double().tolist()
    for a, b in zip(at[:-1], at[1:]):
        i = a
        while i < b - 1:
            d = int(s.drafts[i])
            q = 1.0 if s.draft_probs is None else float(s.draft_probs[i, d])
            if u[i] * q >= float(s.probs[i, d]):
                break
            i += 1
        r = s.probs[i].double()
        if i < b - 1:
            if s.draft_probs is None:
                r[int(s.drafts[i])] = 0
            else:
                r = (r - s.draft_probs[i].double()).clamp_min(0)
        sums = r.cumsum(0)
        token = min(int((sums <= u[b - 1] * sums[-1]).sum()), case["vocab"] - 1)
        tokens += s.drafts[a:i].tolist() + [token] + [-1] * (b - 1 - i)
        accepted.append(i - a)
    return (torch.tensor(tokens, dtype=torch.int32, device="cuda"),
            torch.tensor(accepted, dtype=torch.int32, device="cuda"))

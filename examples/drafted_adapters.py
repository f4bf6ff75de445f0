"""Drafted decoding of tenants with adapters of their own over one shared, quantised model.

Built from the library's operators: the shared projections (Weight.matmul) with every row's
low-rank adapter beside them (AdapterSet.add), norms before and after each block in one pass
(residual_norm), the paged cache with rotation and attention (KVPool.plan), the distribution that is
sampled from (filter_probs) and the verification of drafted tokens (verify_drafts).

Each step a drafter proposes a few tokens a tenant, either a smaller model or what followed
the last tokens in the tenant's own text before; the target runs over all of them at once and keeps those
that it would have drawn itself. Rejected tokens stay in the cache until the next step
overwrites them.

    python examples/drafted_adapters.py
"""
from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import realm_b200 as rb  # noqa: E402

CONFIG = dict(layers=4, hidden=512, heads=8, kv_heads=2, head_dim=64, ffn=1024, vocab=8192, rank=16, residual=0.5,
              max_seq=512, theta=10000.0)


class Decoder:
    """A decoder with a norm on either side of each block. Tenants take a slot of its adapters each."""

    def __init__(self, ctx: rb.Context, cfg: dict, max_tenants: int, seed: int = 0):
        self.ctx, self.cfg = ctx, cfg
        g = torch.Generator("cuda").manual_seed(seed)
        rng = np.random.default_rng(seed)

        def weight(n, k):
            blocks = ctx.quantize(rb.Q4_K, rng.normal(0, 1 / math.sqrt(k), (n, k)).astype(np.float32))
            return ctx.upload_weight(rb.Q4_K, n, k, blocks)

        def norm():
            return 1 + 0.1 * torch.randn(cfg["hidden"], device="cuda", generator=g)

        H, kv, hd, D = cfg["heads"], cfg["kv_heads"], cfg["head_dim"], cfg["hidden"]
        # before the layers: models of one seed share these and their first layers
        self.embedding = torch.randn(cfg["vocab"], D, device="cuda", generator=g)
        self.out_norm = norm()
        self.head = weight(cfg["vocab"], D)
        shapes = dict(qkv=((H + 2 * kv) * hd, D), o=(D, H * hd), up=(2 * cfg["ffn"], D), down=(D, cfg["ffn"]))
        self.layers = []
        for _ in range(cfg["layers"]):
            layer = {name: weight(n, k) for name, (n, k) in shapes.items()}
            layer["adapters"] = {name: ctx.adapters(n, k, max_tenants, cfg["rank"]) for name, (n, k) in shapes.items()}
            layer["norms"] = [norm() for _ in range(4)]
            self.layers.append(layer)
        self.rope = rb.rope_table(cfg["max_seq"], hd, theta=cfg["theta"], device="cuda")
        self.pool = ctx.kv_pool(cfg["layers"], kv, hd, rb.F16, n_pages=max_tenants * ((cfg["max_seq"] + 15) // 16),
                                max_tenants=max_tenants, max_seq=cfg["max_seq"])
        self.has_adapter = set()

    def load_adapter(self, tenant: int, seed: int, rank: int):
        """A random adapter of every projection."""
        g = torch.Generator("cuda").manual_seed(seed)
        for layer in self.layers:
            for a in layer["adapters"].values():
                down = torch.randn(rank, a.k, device="cuda", generator=g) / math.sqrt(a.k)
                up = torch.randn(a.n, rank, device="cuda", generator=g) * 0.3
                a.set(tenant, down.half(), up.half(), scale=1.0 / math.sqrt(rank))
        self.has_adapter.add(tenant)

    def _matmul(self, layer, name, x, slots):
        """Any number of rows, 64 at a time, and what their adapters add."""
        w = layer[name]
        out = torch.empty(len(x), w.n, device="cuda")
        for i in range(0, len(x), 64):
            part = x[i:i + 64].contiguous()
            w.matmul(part, len(part), out=out[i:i + 64])
        return layer["adapters"][name].add(x, slots, out)

    def step(self, tenants, tokens, positions):
        """Feeds one token per row, a tenant's rows one after the other; returns every row's logits."""
        ctx, cfg = self.ctx, self.cfg
        H, kv, hd, scale = cfg["heads"], cfg["kv_heads"], cfg["head_dim"], cfg["residual"]
        slots = torch.tensor([t if t in self.has_adapter else -1 for t in tenants], dtype=torch.int32, device="cuda")
        x = self.embedding[torch.as_tensor(np.asarray(tokens, np.int64), device="cuda")]
        zero = torch.zeros_like(x)
        x, h = rb.residual_norm(ctx, zero, x, pre_norm=self.layers[0]["norms"][0])
        with self.pool.plan(tenants, H, positions=positions) as plan:
            for i, layer in enumerate(self.layers):
                after = self.layers[i + 1]["norms"][0] if i + 1 < len(self.layers) else self.out_norm
                qkv = self._matmul(layer, "qkv", h, slots).view(len(x), H + 2 * kv, hd)
                q = plan.append(i, qkv[:, H:H + kv], qkv[:, H + kv:], q=qkv[:, :H], rope=self.rope)
                a = plan.attention(i, q, 1 / math.sqrt(hd)).view(len(x), H * hd)
                o = self._matmul(layer, "o", a, slots)
                x, h = rb.residual_norm(ctx, o, x, post_norm=layer["norms"][1], scale=scale, pre_norm=layer["norms"][2])
                gate, up = self._matmul(layer, "up", h, slots).chunk(2, -1)
                y = self._matmul(layer, "down", torch.nn.functional.silu(gate) * up, slots)
                x, h = rb.residual_norm(ctx, y, x, post_norm=layer["norms"][3], scale=scale, pre_norm=after)
        logits = torch.empty(len(x), cfg["vocab"], device="cuda")
        for i in range(0, len(x), 64):
            part = h[i:i + 64].contiguous()
            self.head.matmul(part, len(part), out=logits[i:i + 64])
        return logits

    def close(self):
        for layer in self.layers:
            for name, a in layer["adapters"].items():
                a.close()
                layer[name].free()
        self.head.free()
        self.pool.close()


class Lookup:
    """Proposes what followed the text's last two tokens where they stood before."""

    def propose(self, texts, count, sampling, uniforms):
        out = []
        for text in texts:
            got = []
            for i in range(len(text) - 3, -1, -1):
                if text[i:i + 2] == text[-2:]:
                    got = text[i + 2:i + 2 + count]
                    break
            out.append(got)
        return out, None


class DraftModel:
    """A smaller decoder, whose proposals are drawn from its own distribution."""

    def __init__(self, model: Decoder):
        self.model, self.seen = model, {}

    def propose(self, texts, count, sampling, uniforms):
        m, n = self.model, len(texts)
        filters = rb.pack_filters([sampling] * n, "cuda")
        tenants, tokens, positions = [], [], []
        for t, text in enumerate(texts):  # what it has not run over yet; the last token at least
            first = min(self.seen.get(t, 0), len(text) - 1)
            tenants += [t] * (len(text) - first)
            tokens += text[first:]
            positions += range(first, len(text))
            self.seen[t] = len(text)
        out, probs = [[] for _ in texts], []
        last = np.cumsum(np.bincount(tenants, minlength=n)) - 1
        logits = m.step(tenants, tokens, positions)[torch.as_tensor(last, device="cuda")]
        for i in range(count):
            probs.append(rb.filter_probs(m.ctx, logits, filters))
            drawn = rb.sample_filtered(m.ctx, logits, filters, uniforms[i]).tolist()
            for t in range(n):
                out[t].append(drawn[t])
            if i + 1 < count:
                logits = m.step(list(range(n)), drawn, [len(text) + i for text in texts])
        return out, probs


def generate(model: Decoder, prompts, n_tokens: int, sampling: rb.SamplingFilter, drafter, count: int = 4, seed: int = 1):
    """At least n_tokens tokens for each prompt; returns them and how many drafts were accepted of how many."""
    n, g = len(prompts), torch.Generator("cuda").manual_seed(seed)
    for t in range(n):
        model.pool.create(t)
    texts, seen, new = [list(p) for p in prompts], [0] * n, [0] * n
    proposed = accepted = 0
    while min(new) < n_tokens:
        drafts, probs = drafter.propose(texts, count, sampling, torch.rand(count, n, device="cuda", generator=g))
        tenants, tokens, positions, rows = [], [], [], []
        for t, text in enumerate(texts):  # rows of the cache's missing tokens, then of the drafts
            feed = text[seen[t]:] + drafts[t]
            rows.append(np.arange(len(feed) - len(drafts[t]) - 1, len(feed)) + len(tokens))
            tenants += [t] * len(feed)
            tokens += feed
            positions += range(seen[t], seen[t] + len(feed))
        logits = model.step(tenants, tokens, positions)[torch.as_tensor(np.concatenate(rows), device="cuda")]
        p = rb.filter_probs(model.ctx, logits, rb.pack_filters([sampling] * len(logits), "cuda"))
        offsets = np.concatenate([[0], np.cumsum([len(r) for r in rows])]).astype(np.int32)
        given = torch.tensor([d for ds in drafts for d in ds + [-1]], dtype=torch.int32, device="cuda")
        q = None
        if probs is not None:  # row i of request t: draft i's distribution
            q = torch.zeros_like(p)
            for i, row in enumerate(probs):
                q[torch.as_tensor(offsets[:-1] + i, device="cuda").long()] = row
        u = torch.rand(len(logits), device="cuda", generator=g)
        out, kept = rb.verify_drafts(model.ctx, p, given, u, torch.as_tensor(offsets, device="cuda"), draft_probs=q)
        out, kept = out.tolist(), kept.tolist()
        for t, text in enumerate(texts):
            got = out[offsets[t]:offsets[t] + kept[t] + 1]
            seen[t] = len(text) + kept[t]  # the drawn token is not in the cache yet
            text += got
            new[t] += len(got)
            proposed, accepted = proposed + len(drafts[t]), accepted + kept[t]
    return [text[len(p):] for text, p in zip(texts, prompts)], accepted, proposed


def main():
    with rb.Context(0, stream=torch.cuda.current_stream().cuda_stream) as ctx:
        model = Decoder(ctx, CONFIG, max_tenants=3)
        small = Decoder(ctx, dict(CONFIG, layers=1), max_tenants=3)
        model.load_adapter(0, seed=5, rank=16)
        model.load_adapter(2, seed=6, rank=8)  # tenant 1 has the shared model alone
        rng = np.random.default_rng(0)
        prompts = [(rng.integers(0, CONFIG["vocab"], n).tolist() * 2) for n in (20, 5, 33)]
        for t in range(3):
            small.pool.create(t)
        for name, drafter in (("looked up", Lookup()), ("drafted", DraftModel(small))):
            tokens, accepted, proposed = generate(model, prompts, 12, rb.SamplingFilter(0.7, top_k=50, top_p=0.95), drafter)
            for p, t in zip(prompts, tokens):
                print(f"prompt of {len(p):3d} tokens -> {t}")
            print(f"{name}: {accepted} of {proposed} accepted")
            for t in range(3):
                model.pool.destroy(t)
        model.close()
        small.close()


if __name__ == "__main__":
    main()

"""A small decoder whose layers the fused model path does not cover, built from the
library's operators: quantised projections (Weight.matmul), per-head norms of queries
and keys with the position rotation and the paged append (RowPlan.append), attention
with capped scores that is local in every other layer (RowPlan.attention), and
min-p sampling over a large vocabulary (sample_filtered).

Weights are random. Several tenants share one paged cache: their prompts go in with one
plan a step (the rows of all of them), then every step decodes one token each.

    python examples/local_global_decode.py
"""
from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import realm_b200 as rb  # noqa: E402

CONFIG = dict(layers=4, hidden=512, heads=8, kv_heads=2, head_dim=64, ffn=1024, vocab=65537, window=24, softcap=50.0,
              final_cap=30.0, max_seq=512, theta=10000.0)


class Decoder:
    def __init__(self, ctx: rb.Context, cfg: dict, max_tenants: int, seed: int = 0):
        self.ctx, self.cfg = ctx, cfg
        g = torch.Generator("cuda").manual_seed(seed)
        rng = np.random.default_rng(seed)

        def weight(n, k):
            blocks = ctx.quantize(rb.Q4_K, rng.normal(0, 1 / math.sqrt(k), (n, k)).astype(np.float32))
            return ctx.upload_weight(rb.Q4_K, n, k, blocks)

        def norm(n):
            return 1 + 0.1 * torch.randn(n, device="cuda", generator=g)

        H, kv, hd, D = cfg["heads"], cfg["kv_heads"], cfg["head_dim"], cfg["hidden"]
        self.layers = [dict(qkv=weight((H + 2 * kv) * hd, D), o=weight(D, H * hd), up=weight(2 * cfg["ffn"], D),
                            down=weight(D, cfg["ffn"]), attn_norm=norm(D), ffn_norm=norm(D), q_norm=norm(hd),
                            k_norm=norm(hd)) for _ in range(cfg["layers"])]
        self.embedding = torch.randn(cfg["vocab"], D, device="cuda", generator=g)
        self.out_norm = norm(D)
        self.head = weight(cfg["vocab"], D)
        self.rope = rb.rope_table(cfg["max_seq"], hd, theta=cfg["theta"], device="cuda")
        self.pool = ctx.kv_pool(cfg["layers"], kv, hd, rb.F16, n_pages=max_tenants * ((cfg["max_seq"] + 15) // 16),
                                max_tenants=max_tenants, max_seq=cfg["max_seq"])

    def _matmul(self, w, x):
        """Any number of rows, 64 at a time."""
        out = torch.empty(len(x), w.n, device="cuda")
        for i in range(0, len(x), 64):
            part = x[i:i + 64].contiguous()
            out[i:i + 64] = w.matmul(part, len(part), out=torch.empty(len(part), w.n, device="cuda"))
        return out

    @staticmethod
    def _norm(x, w):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w

    def step(self, tenants, tokens):
        """Feeds one token per row (a tenant's rows at its next positions); returns every row's logits."""
        cfg, H, kv, hd = self.cfg, self.cfg["heads"], self.cfg["kv_heads"], self.cfg["head_dim"]
        x = self.embedding[torch.as_tensor(np.asarray(tokens, np.int64), device="cuda")] * math.sqrt(cfg["hidden"])
        pos = self._positions(tenants)
        # one plan for the global layers, one for the local ones
        with self.pool.plan(tenants, H, positions=pos) as full, \
                self.pool.plan(tenants, H, positions=pos, window=cfg["window"]) as local:
            for i, layer in enumerate(self.layers):
                qkv = self._matmul(layer["qkv"], self._norm(x, layer["attn_norm"])).view(len(x), H + 2 * kv, hd)
                plan = local if i % 2 == 0 else full
                q = plan.append(i, qkv[:, H:H + kv], qkv[:, H + kv:], q=qkv[:, :H], q_norm=layer["q_norm"],
                                k_norm=layer["k_norm"], rope=self.rope)
                a = plan.attention(i, q, 1 / math.sqrt(hd), softcap=cfg["softcap"])
                x = x + self._matmul(layer["o"], a.view(len(x), H * hd))
                gate, up = self._matmul(layer["up"], self._norm(x, layer["ffn_norm"])).chunk(2, -1)
                x = x + self._matmul(layer["down"], torch.nn.functional.silu(gate) * up)
        logits = self._matmul(self.head, self._norm(x, self.out_norm))
        return cfg["final_cap"] * torch.tanh(logits / cfg["final_cap"])

    def _positions(self, tenants):
        seen, pos = {}, []
        for t in tenants:
            pos.append(self.pool.len(t) + seen.get(t, 0))
            seen[t] = seen.get(t, 0) + 1
        return pos

    def close(self):
        for layer in self.layers:
            for w in ("qkv", "o", "up", "down"):
                layer[w].free()
        self.head.free()
        self.pool.close()


def generate(model: Decoder, prompts, n_tokens: int, sampling: rb.SamplingFilter, seed: int = 1):
    """Tokens for each prompt: all prompts in one step, then one token each a step."""
    for t in range(len(prompts)):
        model.pool.create(t)
    tenants = [t for t, p in enumerate(prompts) for _ in p]
    last = np.cumsum([len(p) for p in prompts]) - 1
    logits = model.step(tenants, [tok for p in prompts for tok in p])[torch.as_tensor(last, device="cuda")]
    filters = rb.pack_filters([sampling] * len(prompts), "cuda")
    out = []
    for i in range(n_tokens):
        u = torch.tensor([rb.sampling_uniform(seed, i * len(prompts) + t) for t in range(len(prompts))], device="cuda")
        out.append(rb.sample_filtered(model.ctx, logits.contiguous(), filters, u).cpu().numpy())
        if i + 1 < n_tokens:
            logits = model.step(list(range(len(prompts))), out[-1])
    return np.stack(out, 1)


def main():
    # the context works on torch's current stream: no events between the two
    with rb.Context(0, stream=torch.cuda.current_stream().cuda_stream) as ctx:
        model = Decoder(ctx, CONFIG, max_tenants=3)
        rng = np.random.default_rng(0)
        prompts = [rng.integers(0, CONFIG["vocab"], n).tolist() for n in (97, 5, 33)]
        tokens = generate(model, prompts, 16, rb.SamplingFilter(0.8, top_k=50, top_p=0.95, min_p=0.05))
        for p, t in zip(prompts, tokens):
            print(f"prompt of {len(p):3d} tokens -> {t.tolist()}")
        model.close()


if __name__ == "__main__":
    main()

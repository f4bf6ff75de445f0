"""The decoder of examples/local_global_decode.py: feeding a sequence at once, in
chunks or token by token gives the same logits, and the same seed the same tokens."""
import importlib.util
import os

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("local_global_decode",
                                                  os.path.join(ROOT, "examples", "local_global_decode.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_chunks_and_single_tokens_agree(ctx, example):
    import torch
    cfg = dict(example.CONFIG, vocab=1000, layers=3)
    model = example.Decoder(ctx, cfg, max_tenants=3)
    try:
        rng = np.random.default_rng(3)
        seq = rng.integers(0, cfg["vocab"], 90).tolist()
        for t in range(3):
            model.pool.create(t)
        whole = model.step([0] * 90, seq)
        parts = torch.cat([model.step([1] * n, seq[s:s + n]) for s, n in ((0, 37), (37, 50), (87, 3))])
        # rows of two tenants in one step: a chunk of tenant 2 beside a repeated token of tenant 0
        mixed = model.step([2] * 60 + [0], seq[:60] + [7])[:60]
        single = torch.cat([model.step([2], [tok]) for tok in seq[60:]])
        # the projections' and the attention's sums run in other orders: fp32 rounding, and
        # fp16 roundings of cached keys and values that a last-bit difference may turn over
        tol = 2e-3 + 1e-3 * whole.abs()
        assert ((whole - parts).abs() <= tol).all()
        assert ((whole[:60] - mixed).abs() <= tol[:60]).all()
        assert ((whole[60:] - single).abs() <= tol[60:]).all()
    finally:
        model.close()


def test_generation_is_reproducible(ctx, example):
    import realm_b200 as rb
    cfg = dict(example.CONFIG, layers=2)
    model = example.Decoder(ctx, cfg, max_tenants=2)
    try:
        prompts = [[5, 9, 1000, 65536], list(range(40))]
        s = rb.SamplingFilter(0.9, top_k=100, top_p=0.9, min_p=0.01)
        a = example.generate(model, prompts, 6, s)
        b = example.generate(model, prompts, 6, s)
        assert (a == b).all() and a.shape == (2, 6) and (a < cfg["vocab"]).all()
        greedy = example.generate(model, prompts, 3, rb.SamplingFilter(0.0))
        top1 = example.generate(model, prompts, 3, rb.SamplingFilter(1.0, top_k=1))
        assert (greedy == top1).all()
    finally:
        model.close()

"""The loop of examples/drafted_adapters.py: whatever is drafted, the tokens are the target's own."""
import importlib.util
import os

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("drafted_adapters", os.path.join(ROOT, "examples", "drafted_adapters.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


class Fixed:
    """Proposes the next tokens of given texts, every third of them wrong."""

    def __init__(self, texts, vocab):
        self.texts, self.vocab = texts, vocab

    def propose(self, texts, count, sampling, uniforms):
        out = []
        for whole, text in zip(self.texts, texts):
            n = len(text)
            out.append([(whole[i] + (i % 3 == 0)) % self.vocab for i in range(n, min(n + count, len(whole)))])
        return out, None


@pytest.mark.parametrize("drafter", ["none", "lookup", "model", "fixed"])
def test_greedy_tokens_are_the_targets_own(ctx, example, drafter):
    import torch
    import realm_b200 as rb
    cfg = dict(example.CONFIG, vocab=1000, layers=3)
    model, small = example.Decoder(ctx, cfg, max_tenants=4), example.Decoder(ctx, dict(cfg, layers=1), max_tenants=3)
    try:
        model.load_adapter(0, seed=5, rank=16)
        model.load_adapter(2, seed=6, rank=5)
        rng = np.random.default_rng(0)
        prompts = [rng.integers(0, cfg["vocab"], n).tolist() * 2 for n in (9, 2, 30)]
        for t in range(3):
            small.pool.create(t)
        d = {"none": Fixed(prompts, cfg["vocab"]), "lookup": example.Lookup(), "model": example.DraftModel(small)}
        if drafter == "fixed":
            base, _, _ = example.generate(model, prompts, 20, rb.SamplingFilter(0.0), d["none"])
            for t in range(3):
                model.pool.destroy(t)
            d["fixed"] = Fixed([p + b for p, b in zip(prompts, base)], cfg["vocab"])
        tokens, accepted, proposed = example.generate(model, prompts, 20, rb.SamplingFilter(0.0), d[drafter])
        if drafter == "fixed":
            assert 0 < accepted < proposed
        for t, (p, new) in enumerate(zip(prompts, tokens)):
            assert len(new) >= 20
            # the whole text at once: every token leads its row, but for roundings of other sums and cached fp16 values
            text = p + new
            model.pool.clear(t)
            rows = model.step([t] * (len(text) - 1), text[:-1], list(range(len(text) - 1)))[len(p) - 1:]
            lead = rows.gather(1, torch.tensor(new, device="cuda")[:, None])[:, 0]
            assert (rows.max(-1).values - lead <= 2e-2).all()
        # adapters matter: the same text without one has other logits
        bare = model.pool
        bare.create(3)
        text = prompts[0]
        other = model.step([3] * len(text), text, list(range(len(text))))
        model.pool.clear(0)
        own = model.step([0] * len(text), text, list(range(len(text))))
        assert (other - own).abs().max() > 0.05
    finally:
        model.close()
        small.close()


def test_sampled_run_and_seed(ctx, example):
    import realm_b200 as rb
    cfg = dict(example.CONFIG, vocab=1000, layers=2)
    rng = np.random.default_rng(1)
    prompts = [rng.integers(0, cfg["vocab"], n).tolist() for n in (4, 17)]
    runs = []
    for _ in range(2):
        model, small = example.Decoder(ctx, cfg, max_tenants=2), example.Decoder(ctx, dict(cfg, layers=1), max_tenants=2)
        try:
            model.load_adapter(1, seed=3, rank=4)
            for t in range(2):
                small.pool.create(t)
            runs.append(example.generate(model, prompts, 10, rb.SamplingFilter(0.8, 40, 0.95), example.DraftModel(small), seed=9)[0])
        finally:
            model.close()
            small.close()
    assert runs[0] == runs[1] and all(0 <= t < cfg["vocab"] for ts in runs[0] for t in ts)


def test_main_runs(example, capsys):
    example.main()
    assert "accepted" in capsys.readouterr().out

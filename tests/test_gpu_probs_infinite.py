"""GPU tests of filtered probabilities of rows with infinite logits: the whole weight is theirs."""
import numpy as np
import pytest

from test_gpu_drafts import check_probs, rules

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("typ", ["float32", "float16"])
@pytest.mark.parametrize("vocab", [1, 9, 500, 40000, 151937])
def test_infinite_logits(ctx, vocab, typ):
    import torch
    import realm_b200 as rb
    t = getattr(torch, typ)
    inf = float("inf")
    x = torch.randn(6, vocab, device="cuda").to(t)
    x[0, vocab // 2] = inf
    x[1, vocab // 3:] = inf
    x[2, ::2] = -inf
    x[2, vocab - 1] = inf
    x[3, :] = inf
    x[4, :], x[4, vocab // 2] = float("nan"), inf
    x[5, ::3] = torch.finfo(t).max
    x[5, 0] = inf
    for f in rules(11):
        out = rb.filter_probs(ctx, x, rb.pack_filters([f] * 6, "cuda"))
        check_probs(out, x, [f] * 6)
        host = rb.filter_probs(ctx, x.cpu().numpy(), [f] * 6)
        assert np.array_equal(host, out.cpu().numpy())
    history = [[vocab // 2], [], [0, vocab - 1], [5], [vocab // 2] * 3, [0]]
    f = [rb.SamplingFilter(0.9, 50, 0.9, 0.01, 1.3)] * 6
    check_probs(torch.from_numpy(rb.filter_probs(ctx, x.cpu().numpy(), f, prev=history)), x, f, history)

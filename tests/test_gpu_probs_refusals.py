"""GPU tests of what filter_probs refuses to write over."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def test_probabilities_over_their_own_arguments(ctx):
    import torch
    import realm_b200 as rb
    n, v = 5, 1000
    x = torch.randn(n, v, device="cuda")
    f = rb.pack_filters([rb.SamplingFilter(0.9, 40, 0.9, 0.0, 1.2)] * n, "cuda")
    prev = torch.arange(n, dtype=torch.int32, device="cuda"), torch.arange(n + 1, dtype=torch.int32, device="cuda")
    buf = torch.full((n * v + 200,), 7.0, device="cuda")
    for at in (0, 1000, n * v - 4):  # filters within the rows, and over their end
        buf[:] = 7.0
        g = buf.view(torch.uint8)[at * 4:at * 4 + f.numel()].view(f.shape)
        g.copy_(f)
        before = buf.clone()
        with pytest.raises(rb.RealmError, match="overlaps"):
            rb.filter_probs(ctx, x, g, out=buf[:n * v].view(n, v))
        assert torch.equal(buf.view(torch.int32), before.view(torch.int32))
    buf[:] = 7.0
    off = buf.view(torch.int32)[500:500 + n + 1]
    off.copy_(prev[1])
    with pytest.raises(rb.RealmError, match="overlaps"):
        rb.filter_probs(ctx, x, f, prev=(prev[0], off), out=buf[:n * v].view(n, v))
    want = rb.filter_probs(ctx, x, f, prev=prev)
    side = buf.view(torch.uint8)[4 * n * v:4 * n * v + f.numel()].view(f.shape)  # beside the rows
    side.copy_(f)
    assert torch.equal(rb.filter_probs(ctx, x, side, prev=prev, out=buf[:n * v].view(n, v)), want)

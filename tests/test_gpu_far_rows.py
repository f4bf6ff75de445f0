"""Rows so far apart that their offsets pass 32 bits: the same results as side by side."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def apart(t, ld):
    """The rows of t, ld elements apart, in memory that holds nothing else."""
    import torch
    buf = torch.empty((len(t) - 1) * ld + t.shape[1], dtype=t.dtype, device="cuda")
    far = buf.as_strided(t.shape, (ld, 1))
    far.copy_(t)
    return far


@pytest.mark.parametrize("rows,ld", [(3, 3 << 30), (40, 3 << 26), (500, 9 << 20)])
def test_adapters(ctx, rows, ld):
    import torch
    g = torch.Generator("cuda").manual_seed(rows)
    x, y = torch.randn(rows, 192, device="cuda", generator=g).half(), torch.randn(rows, 136, device="cuda", generator=g).half()
    with ctx.adapters(136, 192, 2, 16) as s:
        for i in range(2):
            s.set(i, torch.randn(9, 192, device="cuda", generator=g).half(), torch.randn(136, 9, device="cuda", generator=g).half())
        at = (torch.arange(rows, device="cuda") % 3 - 1).int()
        near = s.add(x, at, y, out=torch.empty_like(y))
        far_x, far_y = apart(x, ld), apart(y, ld)
        assert torch.equal(s.add(far_x, at, y, out=torch.empty_like(y)), near)
        assert torch.equal(s.add(x, at, far_y), near)
        torch.cuda.empty_cache()


def test_norms(ctx):
    import torch
    import realm_b200 as rb
    g = torch.Generator("cuda").manual_seed(1)
    y, x, w = torch.randn(4, 320, device="cuda", generator=g).half(), torch.randn(4, 320, device="cuda", generator=g), torch.rand(320, device="cuda")
    near = rb.residual_norm(ctx, y, x, post_norm=w, pre_norm=w)
    far = rb.residual_norm(ctx, apart(y, 3 << 30), apart(x, 3 << 29), post_norm=w, pre_norm=w)
    assert torch.equal(near[0], far[0]) and torch.equal(near[1], far[1])
    torch.cuda.empty_cache()


def test_probabilities_and_verification(ctx):
    import torch
    import realm_b200 as rb
    g = torch.Generator("cuda").manual_seed(2)
    x = torch.randn(4, 5000, device="cuda", generator=g) * 3
    f = rb.pack_filters([rb.SamplingFilter(1.0, 0, 0.9, 0.0), rb.SamplingFilter(0.8, 40)] * 2, "cuda")
    p = rb.filter_probs(ctx, x, f)
    far = apart(x, 3 << 29)
    assert torch.equal(rb.filter_probs(ctx, far, f), p)
    rb.filter_probs(ctx, x, f, out=far)
    assert torch.equal(far, p)
    drafts = p.argmax(-1).int()
    u, off = torch.rand(4, device="cuda", generator=g), torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    a, b = rb.verify_drafts(ctx, p, drafts, u, off, draft_probs=p.roll(1, 0)), \
        rb.verify_drafts(ctx, far, drafts, u, off, draft_probs=apart(p.roll(1, 0), 3 << 29))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    torch.cuda.empty_cache()

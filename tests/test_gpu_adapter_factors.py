"""GPU tests of adapters whose fp32 factors lie outside the range of fp16.

A factor is held in fp16 after a power of two, at most 2^126, that brings its largest element to [2^14, 2^15), so what a
row adds is compared with the formula of the factors as they are then held: within the bounds of
test_gpu_adapters.py, which know nothing of the factors' size.
"""
import numpy as np
import pytest

from test_gpu_adapters import check

pytestmark = pytest.mark.gpu


def held(f):
    """f [..] float32 as fp16 behind a power of two, in 64 bits."""
    import torch
    most = f.abs()[f.isfinite()].max().item()
    if most == 0:
        return f.double()
    e = min(14 - (np.frexp(most)[1] - 1), 126)
    return torch.from_numpy(np.ldexp(np.ldexp(f.double().numpy(), e).astype(np.float16).astype(np.float64), -e))


@pytest.mark.parametrize("size_down,size_up", [(1e6, 1e-9), (1e-9, 1e6), (1e30, 1e-30), (1e-7, 1e-7), (1e-33, 1e30), (300.0, 0.01)])
@pytest.mark.parametrize("rows", [3, 40, 500])
def test_fp32_factors_of_any_size(ctx, rows, size_down, size_up):
    import torch
    rng = np.random.default_rng(rows)
    k, n, ranks = 520, 200, [16, 7]
    x = torch.from_numpy(rng.normal(0, 1, (rows, k)).astype(np.float32))
    y = torch.zeros(rows, n)
    # elements of unlike sizes, some far below the largest
    f = lambda s, *d: torch.from_numpy((rng.normal(0, 1, d) * 10.0 ** -rng.integers(0, 4, d)).astype(np.float32) * np.float32(s))  # noqa: E731
    down, up = [f(size_down / 20, r, k) for r in ranks], [f(size_up, n, r) for r in ranks]
    slots = rng.integers(-1, 2, rows).astype(np.int32)
    scales = [0.3, -1.7]
    with ctx.adapters(n, k, 2, 16) as s, ctx.adapters(n, k, 2, 16) as host:
        for i in range(2):
            s.set(i, down[i].cuda(), up[i].cuda(), scales[i])
            host.set(i, down[i].numpy(), up[i].numpy(), scales[i])
        at = torch.from_numpy(slots).cuda()
        out = s.add(x.cuda(), at, y.cuda())
        assert torch.equal(out, host.add(x.cuda(), at, y.cuda()))
        check(out, x, y, [held(d) for d in down], [held(u) for u in up], [float(np.float32(c)) for c in scales], slots, rows > 384)


@pytest.mark.parametrize("rows", [3, 40, 500])
def test_fp32_factors_at_the_ends(ctx, rows):
    """Zeros, the largest and the smallest numbers, infinities, and a slot that had another adapter before."""
    import torch
    k, n = 96, 72
    x, y = torch.ones(rows, k, device="cuda"), torch.full((rows, n), 0.5, device="cuda")
    at = torch.zeros(rows, dtype=torch.int32, device="cuda")
    with ctx.adapters(n, k, 1, 8) as s:
        def add(down, up, scale=1.0):
            s.set(0, down.cuda(), up.cuda(), scale)
            return s.add(x, at, y, out=torch.empty_like(y))
        d, u = torch.ones(8, k), torch.ones(n, 8)
        assert (add(d, u) == 0.5 + 8 * k).all()
        assert torch.equal(add(d * 0, u), y) and torch.equal(add(d, u * 0), y)
        assert (add(d * 2.0 ** 120, u * 2.0 ** -119) == 0.5 + 16 * k).all()
        assert (add(d * 2.0 ** -140, u * 2.0 ** 127, 2.0 ** 13) == 0.5 + 8 * k).all()
        assert (add(d * 2.0 ** -130, u * 2.0 ** -130) == 0.5).all()
        big = torch.zeros(n, 8)
        big[:, 1] = 3e38
        v = torch.zeros(8, k)
        v[0], v[1, 5] = 1.0, 0.0
        assert torch.equal(add(v, big), y)  # nothing times much
        v[1, 5] = float("inf")
        assert not add(v, big).isfinite().any()
        assert (add(d, u) == 0.5 + 8 * k).all()

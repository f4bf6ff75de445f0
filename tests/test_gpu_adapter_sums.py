"""GPU tests of adapters' sums: what is small beside y, chains on the tensor core, and captured calls whose adapters change."""
import numpy as np
import pytest

from test_gpu_adapters import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 16, 17, 60, 300, 500])
def test_small_parts_beside_a_large_y(ctx, rows):
    """128 parts of 2^-25 beside y = 1: each of them alone is lost to a rounding at y's size, their sum 2^-18 is not."""
    import torch
    k, n, rank = 128, 96, 128
    down = torch.eye(128, device="cuda").half()
    up = torch.full((n, rank), 2.0 ** -12, device="cuda").half()
    with ctx.adapters(n, k, 1, rank) as s:
        s.set(0, down, up, 2.0 ** -13)
        out = s.add(torch.ones(rows, k, device="cuda"), torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.ones(rows, n, device="cuda"))
        assert (out == 1 + 2.0 ** -18).all(), float(out.max() - 1)


def test_sums_on_the_tensor_core_stay_short(ctx):
    """fp32 rows sum 128 elements of k there: the large parts are 16 instructions, each of which cuts off 0.72 u
    (u = 2^-24; half a step on average over values within a power of two) of a running sum that grows like a root, 2/3 of its
    end: 7.7 u of v, all to the same side. The second product adds four of its own, 1.9 u. 256 elements would be 17 u."""
    import torch
    g = torch.Generator("cuda").manual_seed(0)
    rows, k, n, rank = 1024, 11008, 512, 64
    x = torch.randn(rows, k, device="cuda", generator=g)
    down, up = (torch.randn(rank, k, device="cuda", generator=g) / k ** 0.5).half(), torch.randn(n, rank, device="cuda", generator=g).half()
    with ctx.adapters(n, k, 1, rank) as s:
        s.set(0, down, up)
        out = s.add(x, torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.zeros(rows, n, device="cuda"))
    ref = (x.double() @ down.double().T) @ up.double().T
    e = (out.double() - ref).pow(2).mean().sqrt() / ref.pow(2).mean().sqrt()
    assert e <= 13 * 2.0 ** -24, float(e) * 2 ** 24


@pytest.mark.parametrize("rows", [4, 60, 500])
def test_replayed_after_its_adapter_was_replaced(rows):
    """A captured call takes what set() and clear() have put into the slots since."""
    import torch
    import realm_b200 as rb
    rng = np.random.default_rng(rows)
    k, n = 256, 136
    x, y = (torch.from_numpy(rng.normal(0, 1, (rows, w)).astype(np.float32)) for w in (k, n))
    sets = [(torch.from_numpy((rng.normal(0, 1, (r, k)) / 16).astype(np.float16)),
             torch.from_numpy(rng.normal(0, 1, (n, r)).astype(np.float16)), 0.5 + r) for r in (3, 40, 16)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), rb.Context(0, stream=side.cuda_stream) as c, c.adapters(n, k, 2, 40) as s:
        xc, yc, out = x.cuda(), y.cuda(), torch.empty(rows, n, device="cuda")
        at = torch.ones(rows, dtype=torch.int32, device="cuda")
        s.add(xc, at, yc, out=out)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            s.add(xc, at, yc, out=out)
        for down, up, scale in sets:
            for d, u in ((down.cuda(), up.cuda()), (down.float().numpy(), up.float().numpy())):
                s.set(1, d, u, scale)
                graph.replay()
                side.synchronize()
                check(out, x, y, [down], [up], [scale], np.zeros(rows, int), rows > 384)
                s.clear(1)
                graph.replay()
                side.synchronize()
                assert torch.equal(out, yc)
        del graph

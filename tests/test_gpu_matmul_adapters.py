"""GPU tests of a projection with adapters as one call: what it refuses leaves `out` as it was, and tensors are not waited for."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
N, K, ROWS = 256, 512, 5


@pytest.fixture(scope="module")
def blocks():
    import realm_b200 as rb
    with rb.Context(0) as c:
        return c.quantize(rb.Q4_K, np.random.default_rng(0).normal(0, 0.03, (N, K)).astype(np.float32))


def loaded(c):
    import torch
    g = torch.Generator("cuda").manual_seed(1)
    s = c.adapters(N, K, 3, 16)
    s.set(0, torch.randn(8, K, device="cuda", generator=g) / 20, torch.randn(N, 8, device="cuda", generator=g), 0.5)
    s.set(2, torch.randn(16, K, device="cuda", generator=g) / 20, torch.randn(N, 16, device="cuda", generator=g), 2.0)
    return s


def test_refused_slots_leave_out_alone(ctx, blocks):
    import torch
    import realm_b200 as rb
    w, s = ctx.upload_weight(rb.Q4_K, N, K, blocks), loaded(ctx)
    x, out = np.ones((ROWS, K), np.float32), np.full((ROWS, N), 7, np.float32)
    xc, oc = torch.ones(ROWS, K, device="cuda"), torch.full((ROWS, N), 7.0, device="cuda")
    good = torch.tensor([0, 2, -1, 0, 2], dtype=torch.int32, device="cuda")
    errors = (ValueError, rb.RealmError, AssertionError)
    for slots in ([0, 2, -1, 0], [0, 2, -1, 0, 1], [0, 2, -1, 0, 3], [0, 2, -1, 0, -2], [0.5] * 5, [2 ** 40] * 5, good):
        with pytest.raises(errors):
            w.matmul(x, ROWS, out=out, adapters=s, slots=slots)
        assert (out == 7).all(), slots
    for slots in (good.cpu(), good.long(), good[:4], good.cpu().numpy()):
        with pytest.raises(errors):
            w.matmul(xc, ROWS, out=oc, adapters=s, slots=slots)
        assert (oc == 7).all(), slots
    s.close()
    with pytest.raises(rb.RealmError) as e:
        w.matmul(xc, ROWS, out=oc, adapters=s, slots=good)
    assert e.value.code == -20 and (oc == 7).all()
    w.free()


def test_refused_tensors_leave_out_alone(ctx, blocks):
    """Types and shapes other than the product's, a mix of memories, x and out that overlap."""
    import torch
    import realm_b200 as rb
    w, s = ctx.upload_weight(rb.Q4_K, N, K, blocks), loaded(ctx)
    x, out = np.ones((ROWS, K), np.float32), np.full((ROWS, N), 7, np.float32)
    xc, oc = torch.ones(ROWS, K, device="cuda"), torch.full((ROWS, N), 7.0, device="cuda")
    good = torch.tensor([0, 2, -1, 0, 2], dtype=torch.int32, device="cuda")
    errors = (ValueError, rb.RealmError, AssertionError)
    for a, o in ((xc.half(), oc), (xc.half(), oc.half()), (xc, oc.half()), (xc.double(), oc.double()), (xc[:4], oc), (xc, oc[:, :100]),
                 (xc, oc[:, ::2]), (x, oc), (xc, out)):
        with pytest.raises(errors):
            w.matmul(a, ROWS, out=o, adapters=s, slots=good)
        assert (oc == 7).all() and (out == 7).all() and (o == 7).all()
    both = torch.full((ROWS * (K + N),), 7.0, device="cuda")
    with pytest.raises(rb.RealmError, match="overlaps"):
        w.matmul(both[:ROWS * K].view(ROWS, K), ROWS, out=both[ROWS * K - 8:][:ROWS * N].view(ROWS, N), adapters=s, slots=good)
    assert (both == 7).all()
    s.close()
    w.free()


def test_tensors_on_other_streams(ctx, blocks):
    """The context has a stream of its own: x comes from torch's stream behind much work, and out is read there."""
    import torch
    import realm_b200 as rb
    w, s = ctx.upload_weight(rb.Q4_K, N, K, blocks), loaded(ctx)
    slots = torch.tensor([0, 2, -1, 0, 2], dtype=torch.int32, device="cuda")
    x = torch.randn(ROWS, K, device="cuda")
    want = w.matmul(x, ROWS, out=torch.empty(ROWS, N, device="cuda"), adapters=s, slots=slots).clone()
    a = torch.randn(4096, 4096, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(20):
            a = a @ a / 64
        late = x + 0 * a[:ROWS, :K].nan_to_num(0, 0, 0)
        got = w.matmul(late, ROWS, out=torch.empty(ROWS, N, device="cuda"), adapters=s, slots=slots).clone()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    s.close()
    w.free()


def test_captured_and_replayed(blocks):
    import torch
    import realm_b200 as rb
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), rb.Context(0, stream=side.cuda_stream) as c:
        w, s = c.upload_weight(rb.Q4_K, N, K, blocks), loaded(c)
        x, out = torch.randn(ROWS, K, device="cuda"), torch.empty(ROWS, N, device="cuda")
        slots = torch.tensor([0, 2, -1, 0, 2], dtype=torch.int32, device="cuda")
        w.matmul(x, ROWS, out=out, adapters=s, slots=slots)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            w.matmul(x, ROWS, out=out, adapters=s, slots=slots)
        for seed in range(3):
            g = torch.Generator("cuda").manual_seed(seed)
            x.copy_(torch.randn(ROWS, K, device="cuda", generator=g))
            slots.copy_(torch.randint(-1, 3, (ROWS,), device="cuda", generator=g).int())
            graph.replay()
            got = out.clone()
            want = w.matmul(x, ROWS, out=torch.empty(ROWS, N, device="cuda"), adapters=s, slots=slots)
            side.synchronize()
            assert torch.equal(got, want)
        del graph
        s.close()
        w.free()

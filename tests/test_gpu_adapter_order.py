"""GPU test of the order of set() and clear() with captured calls that are replayed on torch's stream,
while the context has a stream of its own."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [3, 500])
@pytest.mark.parametrize("how", ["clear", "host", "tensors"])
def test_changes_come_after_replays_before_them(rows, how):
    import torch
    import realm_b200 as rb
    k, n = 128, 96
    d, u = torch.ones(4, k, device="cuda").half(), torch.ones(n, 4, device="cuda").half()
    x, y, at = torch.ones(rows, k, device="cuda"), torch.zeros(rows, n, device="cuda"), torch.zeros(rows, dtype=torch.int32, device="cuda")
    a = torch.randn(4096, 4096, device="cuda") / 64
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), rb.Context(0) as c, c.adapters(n, k, 1, 4) as s:
        out = torch.empty_like(y)
        s.set(0, d, u)
        s.add(x, at, y, out=out)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            s.add(x, at, y, out=out)
        for _ in range(3):
            s.set(0, d, u)
            side.synchronize()
            b = a
            for _ in range(30):  # long enough for the host to come to the change
                b = b @ a
            graph.replay()
            first = out.clone()
            if how == "clear":
                s.clear(0)
            elif how == "host":
                s.set(0, d.cpu().numpy(), u.cpu().numpy(), 2.0)
            else:
                s.set(0, d, u, 2.0)
            graph.replay()
            second = out.clone()
            side.synchronize()
            assert (first == 4 * k).all() and (second == (0 if how == "clear" else 8 * k)).all()
        del graph

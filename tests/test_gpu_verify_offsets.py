"""GPU tests of verification where the offsets in device memory are not those of separate rows."""
import numpy as np
import pytest

from test_gpu_drafts import make, ref_verify, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("drawn", [True, False])
@pytest.mark.parametrize("v", [50, 5003, 40001])
def test_valid_requests_beside_bad_ones(ctx, v, drawn):
    """Requests whose offsets fall or pass the rows get -1, those between them, on rows of their own, what they get alone."""
    import torch
    rng = np.random.default_rng(v)
    p, q, d, u, _ = make(rng, [12], v)
    off = np.array([0, 3, 99, 3, 5, -4, 5, 9, 7, 13, 9, 12], np.int32)
    rows = {0: (0, 3), 3: (3, 5), 6: (5, 9), 10: (9, 12)}
    tokens = torch.full((12,), 77, dtype=torch.int32, device="cuda")
    got = run(ctx, p, q if drawn else None, d, u, off, tokens=tokens)
    for r in range(11):
        if r not in rows:
            assert got[1][r] == -1, r
            continue
        a, b = rows[r]
        ref = ref_verify(p[a:b], q[a:b] if drawn else None, d[a:b], u[a:b], [0, b - a])
        assert got[1][r] == ref[1][0] and (got[0][a:b] == ref[0]).all(), r


@pytest.mark.parametrize("drawn", [True, False])
@pytest.mark.parametrize("nothing", [True, False])
@pytest.mark.parametrize("v", [50, 5003, 40001, 151937])
def test_requests_that_share_rows_in_place(ctx, v, nothing, drawn):
    """Tokens written over the drafts that another request reads: the calls end, and stay within the requests' rows."""
    import torch
    import realm_b200 as rb
    rng = np.random.default_rng(v)
    n = 24
    p = torch.softmax(3 * torch.randn(n, v, device="cuda"), -1) * (0 if nothing else 1)
    q = torch.softmax(3 * torch.randn(n, v, device="cuda"), -1) if drawn else None
    off = torch.tensor([0, 18, 1, 17, 2, 18, 4, 20, 0, 20], dtype=torch.int32, device="cuda")
    u = torch.rand(n, device="cuda")
    for _ in range(20):
        drafts = torch.from_numpy(rng.integers(-2, v + 2, n).astype(np.int32)).cuda()
        drafts[20:] = 77
        t, a = rb.verify_drafts(ctx, p, drafts, u, off, draft_probs=q, tokens=drafts)
        ctx.sync()
        t, a = t.cpu().numpy(), a.cpu().numpy()
        assert (a[1::2] == -1).all() and (a[::2] >= 0).all() and (a[::2] < [18, 16, 16, 16, 20]).all()
        assert (t[20:] == 77).all() and t[:20].min() >= -2 and t[:20].max() < v + 2

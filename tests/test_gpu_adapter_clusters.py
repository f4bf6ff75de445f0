"""GPU test of adapters' calls of few rows with the clusters that a part of a GPU can have."""
import numpy as np
import pytest

from test_gpu_adapters import check, load, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("typ", ["float32", "float16"])
@pytest.mark.parametrize("rows,k,n", [(1, 4096, 512), (16, 1000, 301), (3, 7, 5)])
def test_portable_clusters(ctx, rows, k, n, typ):
    import torch
    from realm_b200 import _lib
    rng = np.random.default_rng(rows)
    x, y, down, up, scales = make(rng, rows, k, n, [3, 64, 17], getattr(torch, typ))
    slots = rng.integers(-1, 3, rows).astype(np.int32)
    at = torch.from_numpy(slots).cuda()
    with load(ctx, n, k, down, up, scales) as s:
        assert _lib.rb_test_adapters_portable(ctx.handle, s.handle) == 16  # a whole GPU
        check(s.add(x.cuda(), at, y.cuda()), x, y, down, up, scales, slots, False)
        assert _lib.rb_test_adapters_portable(ctx.handle, s.handle) == 8

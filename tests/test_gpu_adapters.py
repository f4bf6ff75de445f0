"""GPU tests of low-rank adapters against the formula in 64 bits.

Bounds, with u = 2^-24 and S = |y| + |scale| sum_j |up_j| sum_i |down_ji| |x_i|, the value
that every rounding is relative to at most:
- single rows: a sum of k products in fp32 runs over at most k / 32 + 64 terms one after the
  other (each of a cluster's CTAs has a part of k, spread over at least four lanes), one of rank
  products over rank, plus the sums of parts and y: (k / 32 + rank + 80) u S.
- tiles: x and v keep 22 bits (2 * 2^-22 S), the tensor core cuts off at most 2 u at each of the 64
  instructions of a chain (fp32 rows; 64 of 16 products for fp16 ones), and of the 2 rank / 16 of the second product,
  and k / 256 + 8 chains and parts are added: (128 + 4 rank / 16 + k / 256 + 16) u S + 2^-21 S.
- fp16 rows: the result is rounded once more, 2^-11 of it.
S is far above a sum of random signs; for those the root mean square error is held as well: the parts
that are cut off, 2^-24 of sums that grow like a root, give 64 u times 2/3 of the sum, and all
roundings a few u: 6e-6 of the root mean square of what is added (fp32 rows), plus y's own u.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def make(rng, rows, k, n, ranks, typ, scales=None):
    import torch
    x = torch.from_numpy(rng.normal(0, 1, (rows, k)).astype(np.float32)).to(typ)
    y = torch.from_numpy(rng.normal(0, 1, (rows, n)).astype(np.float32)).to(typ)
    down = [torch.from_numpy((rng.normal(0, 1, (r, k)) / np.sqrt(k)).astype(np.float16)) for r in ranks]
    up = [torch.from_numpy(rng.normal(0, 0.3, (n, r)).astype(np.float16)) for r in ranks]
    return x, y, down, up, scales or [1.0 + 0.25 * i for i in range(len(ranks))]


def load(ctx, n, k, down, up, scales, max_rank=None, n_slots=None):
    s = ctx.adapters(n, k, n_slots or len(down), max_rank or max(d.shape[0] for d in down))
    for i, (d, u, f) in enumerate(zip(down, up, scales)):
        s.set(i, d.cuda(), u.cuda(), f)
    return s


def reference(x, y, down, up, scales, slots):
    """(result, S of the bounds, what is added)"""
    import torch
    ref, mag = y.double().cuda(), y.double().abs().cuda()
    add = torch.zeros_like(ref)
    for a in set(int(s) for s in slots) - {-1}:
        rows = torch.from_numpy(np.flatnonzero(np.asarray(slots) == a)).cuda()
        xa, d, u = x.double().cuda()[rows], down[a].double().cuda(), up[a].double().cuda()
        add[rows] = scales[a] * ((xa @ d.T) @ u.T)
        mag[rows] += abs(scales[a]) * ((xa.abs() @ d.abs().T) @ u.abs().T)
    return ref + add, mag, add


def check(got, x, y, down, up, scales, slots, tile):
    import torch
    ref, mag, add = reference(x, y, down, up, scales, slots)
    k, rank = x.shape[1], max(d.shape[0] for d in down)
    few = (k / 32 + rank + 80) * U
    bound = max(few, (128 + rank / 4 + k / 256 + 16) * U + 2.0 ** -21) if tile else few
    tol = bound * mag
    if x.dtype == torch.float16:
        tol = tol + 2.0 ** -11 * ref.abs() + 2.0 ** -25
    err = (got.double() - ref).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (int(bad.sum()), float(err.max()), bad.nonzero()[:4].tolist())
    slots = torch.as_tensor(np.asarray(slots)).cuda()
    if (slots >= 0).any() and x.dtype == torch.float32:
        e, a, yy = (t[slots >= 0].pow(2).mean().sqrt() for t in (err, add, y.double().cuda()))
        assert e <= 6e-6 * a + U * yy, (float(e), float(a))
    # rows without an adapter: bit for bit
    assert torch.equal(got[slots < 0], y.cuda()[slots < 0])


SMALL = [(1, 64, 64), (1, 4096, 4096), (3, 65, 33), (5, 1, 1), (16, 2072, 1001), (17, 256, 520), (33, 1000, 7), (64, 4096, 512),
         (41, 11008, 130), (64, 7, 4097), (65, 64, 64), (130, 33, 65), (384, 256, 264)]
TILE = [(385, 64, 64), (385, 1, 1), (400, 33, 65), (512, 4096, 256), (701, 2072, 1001), (700, 320, 136), (1000, 1000, 131),
        (513, 11008, 72), (450, 64, 4100), (2049, 128, 384), (3000, 520, 24)]


@pytest.mark.parametrize("typ", ["float32", "float16"])
@pytest.mark.parametrize("rows,k,n", SMALL + TILE)
def test_rows_of_mixed_adapters(ctx, rows, k, n, typ):
    import torch
    rng = np.random.default_rng(rows * 31 + k + n)
    ranks = [1, 5, 16, 64, 33, 8]
    x, y, down, up, scales = make(rng, rows, k, n, ranks, getattr(torch, typ))
    slots = rng.integers(-1, len(ranks), rows).astype(np.int32)
    if rows > 64:  # prompts: runs of rows, beside single ones
        slots[rows // 8:rows // 2], slots[rows // 2:rows // 4 * 3] = 3, 4
    with load(ctx, n, k, down, up, scales) as s:
        out = s.add(x.cuda(), torch.from_numpy(slots).cuda(), y.cuda())
        check(out, x, y, down, up, scales, slots, rows > 384)
        other = torch.full_like(out, 7.0)
        s.add(x.cuda(), torch.from_numpy(slots).cuda(), y.cuda(), out=other)
        assert torch.equal(out, other)


@pytest.mark.parametrize("typ", ["float32", "float16"])
@pytest.mark.parametrize("rows", [1, 20, 64, 400, 1500])
@pytest.mark.parametrize("rank,max_rank", [(128, 128), (65, 128), (8, 128), (64, 64), (2, 3)])
def test_ranks(ctx, rows, rank, max_rank, typ):
    import torch
    rng = np.random.default_rng(rows + rank)
    k, n = 1096, 600
    x, y, down, up, scales = make(rng, rows, k, n, [rank, rank], getattr(torch, typ))
    slots = (np.arange(rows) * 3 // (rows + 1) - 1).astype(np.int32)[::-1].copy()
    with load(ctx, n, k, down, up, scales, max_rank=max_rank) as s:
        out = s.add(x.cuda(), torch.from_numpy(slots).cuda(), y.cuda())
        check(out, x, y, down, up, scales, slots, rows > 384)


@pytest.mark.parametrize("rows", [64, 65, 500, 8192, 8193, 9000])
def test_many_slots_and_spans(ctx, rows):
    """More slots than rows have, all rows of one, every row of another, and calls of more than 8192 rows."""
    import torch
    rng = np.random.default_rng(rows)
    k, n, slots_n = 128, 64, 300  # (500 rows go one by one then)
    x, y, down, up, scales = make(rng, rows, k, n, [4] * slots_n, torch.float32, [1.0] * slots_n)
    with load(ctx, n, k, down, up, scales) as s:
        for slots in (np.full(rows, 299), np.arange(rows) % slots_n, np.full(rows, -1), np.arange(rows) // 130 % 7):
            slots = slots.astype(np.int32)
            out = s.add(x.cuda(), torch.from_numpy(slots).cuda(), y.cuda())
            check(out, x, y, down, up, scales, slots, rows > 1024)


@pytest.mark.parametrize("rows", [9, 50, 401])
@pytest.mark.parametrize("typ", ["float32", "float16"])
def test_strides_and_alignment(ctx, rows, typ):
    """x, y and out as slices of wider rows, at every offset that their type allows."""
    import torch
    rng = np.random.default_rng(rows)
    k, n = 264, 200
    x, y, down, up, scales = make(rng, rows, k, n, [16, 9], getattr(torch, typ))
    slots = rng.integers(-1, 2, rows).astype(np.int32)
    st = torch.from_numpy(slots).cuda()
    with load(ctx, n, k, down, up, scales) as s:
        for ox, oy, width in ((0, 264, 464), (1, 267, 470), (8, 273, 481), (3, 270, 479)):
            buf = torch.full((rows, width), 5.0, dtype=x.dtype, device="cuda")
            buf[:, ox:ox + k], buf[:, oy:oy + n] = x.cuda(), y.cuda()
            s.add(buf[:, ox:ox + k], st, buf[:, oy:oy + n])
            check(buf[:, oy:oy + n], x, y, down, up, scales, slots, rows > 384)
            assert torch.equal(buf[:, ox:ox + k], x.cuda())
            rest = torch.ones(width, dtype=torch.bool, device="cuda")
            rest[ox:ox + k] = rest[oy:oy + n] = False
            assert (buf[:, rest] == 5.0).all()
            out = torch.full((rows, n + ox), 5.0, dtype=x.dtype, device="cuda")
            s.add(x.cuda(), st, y.cuda(), out=out[:, ox:])
            check(out[:, ox:], x, y, down, up, scales, slots, rows > 384)
            assert (out[:, :ox] == 5.0).all()


@pytest.mark.parametrize("rows", [7, 40, 500])
def test_rows_do_not_reach_one_another(ctx, rows):
    """Rows without an adapter may hold anything, also in x; a row's infinities and NaNs stay in it."""
    import torch
    rng = np.random.default_rng(rows)
    k, n = 200, 136
    x, y, down, up, scales = make(rng, rows, k, n, [12], torch.float32)
    slots = np.zeros(rows, np.int32)
    slots[2::5] = -1
    x[2::5] = float("nan")
    y[2] = float("inf")
    clean = x.clone(), y.clone()
    x[3], x[5, 7] = float("nan"), float("inf")
    with load(ctx, n, k, down, up, scales) as s:
        st = torch.from_numpy(slots).cuda()
        out = s.add(x.cuda(), st, y.cuda())
        other = s.add(clean[0].cuda(), st, clean[1].cuda())
        same = torch.ones(rows, dtype=torch.bool)
        same[[3, 5]] = False
        assert torch.equal(out[same.cuda()], other[same.cuda()])
        assert out[3].isnan().all() and not out[5].isfinite().any()
        assert torch.equal(out[2], y[2].cuda())


@pytest.mark.parametrize("rows", [3, 30, 450])
@pytest.mark.parametrize("size", [1e-20, 1e-6, 300.0, 1e15])
def test_sizes_of_x(ctx, rows, size):
    """What is added is as exact for small and large rows, and for rows whose elements differ by much."""
    import torch
    rng = np.random.default_rng(rows)
    k, n = 512, 256
    x, y, down, up, scales = make(rng, rows, k, n, [16, 64], torch.float32)
    x = x * size
    x[:, ::7] *= 1e-3
    x[0, 5] *= 1e4
    y = y * 0
    slots = (np.arange(rows) % 2).astype(np.int32)
    with load(ctx, n, k, down, up, scales) as s:
        out = s.add(x.cuda(), torch.from_numpy(slots).cuda(), y.cuda())
        check(out, x, y, down, up, scales, slots, rows > 384)


def test_slots_are_replaced_and_emptied(ctx):
    """Calls in stream order: before set() the old adapter, after clear() none, and none for slots that do not exist."""
    import torch
    rng = np.random.default_rng(0)
    for rows in (5, 400):
        x, y, down, up, scales = make(rng, rows, 300, 260, [8, 24], torch.float32)
        xc, yc = x.cuda(), y.cuda()
        with ctx.adapters(260, 300, 3, 24) as s:
            at = torch.full((rows,), 1, dtype=torch.int32, device="cuda")
            outs = [s.add(xc, at, yc, out=torch.empty_like(yc))]
            s.set(1, down[0].cuda(), up[0].cuda(), scales[0])
            outs.append(s.add(xc, at, yc, out=torch.empty_like(yc)))
            s.set(1, down[1].cuda(), up[1].cuda(), scales[1])
            outs.append(s.add(xc, at, yc, out=torch.empty_like(yc)))
            s.set(1, down[0].float().numpy(), up[0].float().numpy(), scales[0])  # fp32 of the same values, from the host
            outs.append(s.add(xc, at, yc, out=torch.empty_like(yc)))
            s.clear(1)
            outs.append(s.add(xc, at, yc, out=torch.empty_like(yc)))
            wild = torch.tensor([-2 ** 31, 3, 2 ** 31 - 1, 2, -7], dtype=torch.int32, device="cuda").repeat(rows // 5)
            outs.append(s.add(xc, wild, yc, out=torch.empty_like(yc)))
        check(outs[1], x, y, down[:1], up[:1], scales[:1], np.zeros(rows, int), rows > 384)
        check(outs[2], x, y, down[1:], up[1:], scales[1:], np.zeros(rows, int), rows > 384)
        assert torch.equal(outs[1], outs[3])
        for i in (0, 4, 5):
            assert torch.equal(outs[i], yc)


@pytest.mark.parametrize("rows", [4, 500])
def test_captured_and_replayed_with_other_slots(rows):
    import torch
    import realm_b200 as rb
    rng = np.random.default_rng(1)
    x, y, down, up, scales = make(rng, rows, 512, 384, [16, 8, 32], torch.float32)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side), rb.Context(0, stream=side.cuda_stream) as c:
        with load(c, 384, 512, down, up, scales) as s:
            xc, yc = x.cuda(), y.cuda()
            at, out = torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.empty_like(yc)
            s.add(xc, at, yc, out=out)
            side.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                s.add(xc, at, yc, out=out)
            for _ in range(3):
                slots = rng.integers(-1, 3, rows).astype(np.int32)
                at.copy_(torch.from_numpy(slots))
                g.replay()
                side.synchronize()
                check(out, x, y, down, up, scales, slots, rows > 384)
            del g


def test_repeated_calls_give_the_same_bits(ctx):
    import torch
    rng = np.random.default_rng(2)
    for rows in (30, 1200):
        x, y, down, up, scales = make(rng, rows, 2048, 1024, [64, 20, 128], torch.float32)
        at = torch.from_numpy(rng.integers(0, 3, rows).astype(np.int32)).cuda()
        with load(ctx, 1024, 2048, down, up, scales) as s:
            first = s.add(x.cuda(), at, y.cuda())
            for _ in range(5):
                assert torch.equal(first, s.add(x.cuda(), at, y.cuda()))


def test_host_arrays(ctx):
    import torch
    rng = np.random.default_rng(3)
    for rows, typ in ((6, torch.float32), (400, torch.float16)):
        x, y, down, up, scales = make(rng, rows, 136, 72, [8, 16], typ)
        slots = rng.integers(-1, 2, rows)
        with ctx.adapters(72, 136, 2, 16) as s:
            for i in range(2):
                s.set(i, down[i].numpy(), up[i].numpy(), scales[i])
            out = y.numpy().copy()
            assert s.add(x.numpy(), slots, out) is out
            check(torch.from_numpy(out).cuda(), x, y, down, up, scales, slots, rows > 384)
            wide = np.full((rows, 100), 9, out.dtype)
            s.add(x.numpy(), slots, y.numpy(), out=wide[:, 4:76])
            assert (wide[:, 4:76] == out).all() and (wide[:, :4] == 9).all() and (wide[:, 76:] == 9).all()


def test_beside_a_quantised_projection(ctx):
    """Weight.matmul with adapters is the product plus what each row's adapter adds."""
    import torch
    import realm_b200 as rb
    rng = np.random.default_rng(4)
    n, k = 512, 1024
    w = ctx.upload_weight(rb.Q4_K, n, k, ctx.quantize(rb.Q4_K, rng.normal(0, 0.03, (n, k)).astype(np.float32)))
    for rows in (3, 400):
        x, _, down, up, scales = make(rng, rows, k, n, [8, 16], torch.float32)
        slots = rng.integers(-1, 2, rows).astype(np.int32)
        with load(ctx, n, k, down, up, scales) as s:
            base = w.matmul(x.numpy(), rows)
            both = w.matmul(x.numpy(), rows, adapters=s, slots=slots)
            check(torch.from_numpy(both).cuda(), x, torch.from_numpy(base), down, up, scales, slots, rows > 384)
            out = torch.empty(rows, n, device="cuda")
            w.matmul(x.cuda(), rows, out=out, adapters=s, slots=torch.from_numpy(slots).cuda())
            assert torch.equal(out.cpu(), torch.from_numpy(both))
            with pytest.raises(ValueError, match="together"):
                w.matmul(x.numpy(), rows, adapters=s)
        with ctx.adapters(n, k + 64, 1, 8) as s, pytest.raises(ValueError, match="projection"):
            w.matmul(x.numpy(), rows, adapters=s, slots=slots)
    w.free()


def test_refusals(ctx):
    import torch
    import realm_b200 as rb
    from realm_b200 import _lib
    for n, k, slots, rank in ((0, 4, 1, 1), (4, 0, 1, 1), (4, 4, 0, 1), (4, 4, 4097, 1), (4, 4, 1, 0), (4, 4, 1, 129),
                              (2 ** 20 + 1, 4, 1, 1)):
        with pytest.raises(rb.RealmError) as e:
            ctx.adapters(n, k, slots, rank)
        assert e.value.code == -23
    with pytest.raises(ValueError, match="n_slots"):
        ctx.adapters(4, 4, -1, 1)
    s = ctx.adapters(64, 128, 2, 8)
    d, u = np.ones((8, 128), np.float32), np.ones((64, 8), np.float32)
    for args, code in (((2, d, u), -2), ((0, np.ones((9, 128), np.float32), np.ones((64, 9), np.float32)), -23),
                       ((0, d, u, float("inf")), -3)):
        with pytest.raises(rb.RealmError) as e:
            s.set(*args)
        assert e.value.code == code
    for a, b in ((d[:, :127], u), (d, u[:63]), (d, np.ones((64, 7), np.float32)), (d, u.astype(np.float16)), (d[0], u)):
        with pytest.raises(ValueError):
            s.set(0, a, b)
    s.set(0, d, u)
    x, y = np.ones((3, 128), np.float32), np.ones((3, 64), np.float32)
    for slots in ([0, 1, 0], [0, 2, 0], [0, -2, 0]):  # empty, beyond, not -1
        with pytest.raises(rb.RealmError) as e:
            s.add(x, np.array(slots), y)
        assert e.value.code == -2 and (y == 1).all()
    for slots in ([0, 0], [0.0, 0.5, 0.0], [2 ** 40, 0, 0]):
        with pytest.raises(ValueError, match="slots"):
            s.add(x, np.array(slots), y)
    xc, yc, at = torch.ones(3, 128, device="cuda"), torch.ones(3, 64, device="cuda"), torch.zeros(3, dtype=torch.int32).cuda()
    for bad in ((xc.half(), at, yc), (xc, at.long(), yc), (xc, at.cpu(), yc), (xc.cpu().numpy(), at, yc), (xc, at, yc[:2]),
                (xc[:, :64], at, yc), (xc.double(), at, yc.double())):
        with pytest.raises(ValueError):
            s.add(*bad)
    buf = torch.ones(3, 192, device="cuda")
    with pytest.raises(rb.RealmError, match="overlaps"):
        s.add(buf[:, :128], at, buf[:, 100:164])
    with pytest.raises(rb.RealmError, match="overlaps"):
        s.add(xc, at, buf[:, :64], out=buf[:, 32:96])
    big = torch.ones(4, 64, device="cuda")
    with pytest.raises(rb.RealmError, match="overlaps"):
        s.add(xc, at, big[:3], out=big[1:])
    ro = np.ones((3, 64), np.float32)
    ro.flags.writeable = False
    with pytest.raises(ValueError, match="read-only"):
        s.add(x, np.zeros(3, int), ro)
    # empty calls
    assert s.add(xc[:0], at[:0], yc[:0]).shape == (0, 64)
    assert s.add(x[:0], np.zeros(0, int), y[:0]).shape == (0, 64)
    s.close()
    with pytest.raises(rb.RealmError) as e:
        s.add(xc, at, yc)
    assert e.value.code == -20
    assert _lib.rb_adapters_destroy(ctx.handle, 1 << 20) == -20


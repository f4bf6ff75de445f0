"""GPU tests of the norms around a block against the formula in 64 bits.

Bounds, u = 2^-24: a sum of dim squares in fp32, no more than 32 terms one after the other in a thread and a
tree of at most 10 more steps, is off by 42 u of itself, its root's inverse by 21 u and four roundings; so z by 32 u of
itself, h by 32 u |scale gate z| + 2 u (|x| + |scale gate z|), out by the errors of h times |w2| f and 32 u of
itself. Results of 16 bits are rounded once more, 2^-11 of them (2^-25 where they are subnormal).
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def inputs(rng, n, dim, typ, stream, gate):
    import torch
    f = lambda *s: torch.from_numpy(rng.normal(0, 1, s).astype(np.float32)).cuda()  # noqa: E731
    g = None if gate == "none" else f(dim).to(typ) if gate == "shared" else f(n, dim).to(typ)
    return (f(n, dim) * 2).to(typ), (f(n, dim) * 3).to(stream), 1 + 0.2 * f(dim), 1 + 0.2 * f(dim), g


def check(y, x, post, pre, gate, scale, eps, x_out, out):
    import torch
    z = y.double()
    if post is not None:
        z = z / torch.sqrt(z.pow(2).mean(-1, keepdim=True) + eps) * post.double()
    if gate is not None:
        z = z * gate.double()
    z = z * scale
    h = x.double() + z
    eh = 34 * U * z.abs() + 2 * U * x.double().abs()
    half = lambda t, v: 2.0 ** -11 * v.abs() + 2.0 ** -25 if t.dtype == torch.float16 else 0  # noqa: E731
    assert ((x_out.double() - h).abs() <= eh + half(x_out, h)).all()
    if pre is None:
        assert out is None
        return
    f = pre.double() / torch.sqrt(h.pow(2).mean(-1, keepdim=True) + eps)
    ref = h * f
    # a change of h changes the root by at most the mean of the changes
    tol = eh * f.abs() + ref.abs() * (32 * U + (eh * h.abs()).mean(-1, keepdim=True) / (h.pow(2).mean(-1, keepdim=True) + eps))
    assert ((out.double() - ref).abs() <= tol + half(out, ref)).all()


@pytest.mark.parametrize("dim", [1, 7, 8, 64, 100, 255, 1000, 1024, 4096, 4104, 5001, 8192, 12288, 16384, 20001, 32768])
@pytest.mark.parametrize("typ,stream", [("float32", "float32"), ("float16", "float32"), ("float16", "float16"), ("float32", "float16")])
@pytest.mark.parametrize("post,gate,pre", [(True, "shared", True), (False, "rows", True), (True, "none", False), (False, "none", False)])
def test_formula(ctx, dim, typ, stream, post, gate, pre):
    import torch
    import realm_b200 as rb
    rng = np.random.default_rng(dim)
    for n in (1, 5, 67):
        y, x, w1, w2, g = inputs(rng, n, dim, getattr(torch, typ), getattr(torch, stream), gate)
        w1, w2 = w1 if post else None, w2 if pre else None
        x_out, out = rb.residual_norm(ctx, y, x, post_norm=w1, gate=g, scale=0.75, pre_norm=w2, eps=1e-5)
        check(y, x, w1, w2, g, 0.75, 1e-5, x_out, out)
        # in place: the same bits
        a, b = y.clone(), x.clone()
        rb.residual_norm(ctx, a, b, post_norm=w1, gate=g, scale=0.75, pre_norm=w2, eps=1e-5, x_out=b, out=a if pre else None)
        assert torch.equal(b, x_out) and (torch.equal(a, out) if pre else torch.equal(a, y))


def test_many_rows(ctx):
    import torch
    import realm_b200 as rb
    rng = np.random.default_rng(1)
    for n, dim in ((70001, 64), (9001, 513)):
        y, x, w1, w2, g = inputs(rng, n, dim, torch.float16, torch.float32, "rows")
        x_out, out = rb.residual_norm(ctx, y, x, post_norm=w1, gate=g, scale=-1.5, pre_norm=w2)
        check(y, x, w1, w2, g, -1.5, 1e-6, x_out, out)


def test_rows_apart_and_unaligned(ctx):
    """Slices of wider rows side by side in one buffer, at offsets on and off 16 bytes; what lies between stays."""
    import torch
    import realm_b200 as rb
    rng = np.random.default_rng(2)
    n, dim = 33, 200
    y, x, w1, w2, g = inputs(rng, n, dim, torch.float32, torch.float32, "rows")
    for pad in (8, 1, 3):
        buf = torch.full((n, 5 * (dim + pad)), 9.0, device="cuda")
        part = [buf[:, i * (dim + pad):i * (dim + pad) + dim] for i in range(5)]
        part[0][:], part[1][:], part[2][:] = y, x, g
        rb.residual_norm(ctx, part[0], part[1], post_norm=w1, gate=part[2], scale=0.5, pre_norm=w2, x_out=part[3], out=part[4])
        check(y, x, w1, w2, g, 0.5, 1e-6, part[3], part[4])
        assert torch.equal(part[0], y) and torch.equal(part[1], x) and torch.equal(part[2], g)
        for i in range(5):
            assert (buf[:, i * (dim + pad) + dim:(i + 1) * (dim + pad)] == 9.0).all()


def test_rows_do_not_reach_one_another(ctx):
    import torch
    import realm_b200 as rb
    rng = np.random.default_rng(3)
    for dim in (32, 100, 4096):
        y, x, w1, w2, _ = inputs(rng, 9, dim, torch.float32, torch.float32, "none")
        clean = rb.residual_norm(ctx, y, x, post_norm=w1, pre_norm=w2)
        y[2], x[5, 0], y[7] = float("nan"), float("inf"), 0.0
        x_out, out = rb.residual_norm(ctx, y, x, post_norm=w1, pre_norm=w2)
        for r in (0, 1, 3, 4, 6, 8):
            assert torch.equal(x_out[r], clean[0][r]) and torch.equal(out[r], clean[1][r])
        assert x_out[2].isnan().all() and torch.equal(x_out[7], x[7])
        zero = rb.residual_norm(ctx, y[7:8] * 0, x[7:8] * 0, post_norm=w1, pre_norm=w2)  # nothing at all
        assert (zero[0] == 0).all() and (zero[1] == 0).all()


def test_host_arrays_and_empty(ctx):
    import torch
    import realm_b200 as rb
    rng = np.random.default_rng(4)
    y, x, w1, w2, g = inputs(rng, 6, 130, torch.float16, torch.float32, "shared")
    dev = rb.residual_norm(ctx, y, x, post_norm=w1, gate=g, scale=2.0, pre_norm=w2)
    c = [t.cpu().numpy() for t in (y, x, w1, g, w2)]
    host = rb.residual_norm(ctx, c[0], c[1], post_norm=c[2], gate=c[3], scale=2.0, pre_norm=c[4])
    assert (host[0] == dev[0].cpu().numpy()).all() and (host[1] == dev[1].cpu().numpy()).all()
    a, b = rb.residual_norm(ctx, y[:0], x[:0], pre_norm=w2)
    assert a.shape == b.shape == (0, 130)


def test_another_stream_and_graph():
    import torch
    import realm_b200 as rb
    rng = np.random.default_rng(5)
    y, x, w1, w2, _ = inputs(rng, 40, 1024, torch.float16, torch.float32, "none")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), rb.Context(0, stream=side.cuda_stream) as c:
        x_out, out = torch.empty_like(x), torch.empty_like(y)
        rb.residual_norm(c, y, x, post_norm=w1, pre_norm=w2, x_out=x_out, out=out)
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            rb.residual_norm(c, y, x, post_norm=w1, pre_norm=w2, x_out=x_out, out=out)
        y.mul_(1.7)
        g.replay()
        side.synchronize()
        check(y, x, w1, w2, None, 1.0, 1e-6, x_out, out)
        del g


def test_refusals(ctx):
    import torch
    import realm_b200 as rb
    y, x, w = torch.ones(4, 64, device="cuda"), torch.ones(4, 64, device="cuda"), torch.ones(64, device="cuda")
    for kw in (dict(pre_norm=w[:63]), dict(post_norm=w.half()), dict(gate=w.half()), dict(gate=torch.ones(3, 64).cuda()),
               dict(gate=torch.ones(4, 64)), dict(out=y.clone()), dict(x_out=x.half()), dict(pre_norm=w, out=y.half()),
               dict(x_out=np.ones((4, 64), np.float32))):
        with pytest.raises(ValueError):
            rb.residual_norm(ctx, y, x, **kw)
    for bad in ((y[:3], x), (y.double(), x), (y[0], x[0]), (y.int(), x), (y.t(), x.t())):
        with pytest.raises(ValueError):
            rb.residual_norm(ctx, *bad)
    for kw in (dict(scale=float("nan")), dict(eps=-1.0), dict(eps=float("inf"))):
        with pytest.raises(rb.RealmError) as e:
            rb.residual_norm(ctx, y, x, **kw)
        assert e.value.code == -3
    with pytest.raises(rb.RealmError) as e:
        rb.residual_norm(ctx, torch.ones(1, 32769, device="cuda"), torch.ones(1, 32769, device="cuda"))
    assert e.value.code == -23
    buf = torch.ones(5, 64, device="cuda")
    for kw in (dict(x_out=y), dict(pre_norm=w, out=x), dict(pre_norm=w, x_out=buf[:4], out=buf[1:]),
               dict(gate=buf[:4], x_out=buf[1:]), dict(post_norm=buf[0], x_out=buf[:4])):
        with pytest.raises(rb.RealmError, match="overlaps"):
            rb.residual_norm(ctx, y, x, **kw)
    with pytest.raises(rb.RealmError, match="overlaps"):
        rb.residual_norm(ctx, y, buf[:4], x_out=buf[1:])
    ro = np.ones((4, 64), np.float32)
    ro.flags.writeable = False
    with pytest.raises(ValueError, match="read-only"):
        rb.residual_norm(ctx, np.ones((4, 64), np.float32), np.ones((4, 64), np.float32), x_out=ro)

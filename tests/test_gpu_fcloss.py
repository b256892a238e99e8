"""The fully connected softmax loss against its formulas in 64 bits.

Tolerances.  u = 2^-24 bounds a single-precision rounding.  Predictions are sums of D products: exact fp32 sums in blocks are off by about
u * sqrt(D) / 3 of their 2-norm, the split operands by 2^-22 of every factor; for D <= 4096 both stay below 2e-6 of the 2-norm of |x||f|.  An error e
of a prediction changes exp(z - lse) by e of itself, so that derivatives, sums over such terms, are within 1e-5 in the 2-norm (predictions
here have a spread of 1.5 to 3, |z| <= 15: e <= 15 * 2^-22).  The loss and lse, of order 10, are off by u of themselves and by the average of e:
2e-6.  With both operands rounded to 11 bits (plain TF32) an error of 2^-11 * sqrt(2 / 3) of the spread replaces 2e-6: 2e-3 for derivatives.
"""
import numpy as np
import pytest

TOL, TOL_LSE, TOL_TF32 = 1e-5, 2e-6, 2e-3

# images, inputs (H, W, C), classes
SIZES = [(1, (1, 1, 1), 1), (1, (1, 1, 16), 10), (3, (2, 2, 5), 7), (8, (1, 1, 129), 1000), (9, (1, 1, 64), 513), (17, (3, 1, 33), 300), (33, (1, 1, 128), 129),
         (64, (1, 1, 256), 1000), (129, (1, 1, 65), 257), (130, (1, 1, 1000), 2051), (257, (1, 1, 72), 511), (300, (1, 1, 200), 33), (1, (1, 1, 2048), 3001),
         (5, (1, 1, 1023), 4099), (16, (1, 1, 512), 640), (1029, (1, 1, 320), 1500)]


def _inputs(n, hwc, k, seed=0, skip=True, spread=2.0):
    rng = np.random.default_rng(seed)
    d = int(np.prod(hwc))
    x = rng.standard_normal((n, d)).astype(np.float32)
    f = (rng.standard_normal((k, d)) * spread / np.sqrt(d)).astype(np.float32)
    b = rng.standard_normal(k).astype(np.float32)
    c = rng.integers(1, k + 1, n).astype(np.float32)
    if skip and n > 2:
        c[rng.random(n) < 0.2] = 0
        c[0] = 0
    return x, f, b, c


def _up(mat, x, f, b, c, hwc):
    """As the engine takes them: H x W x C x N, memory one image (one class) after the other."""
    import torch
    t = lambda a: torch.from_numpy(a).cuda().view(a.shape[0], hwc[2], hwc[1], hwc[0]).permute(3, 2, 1, 0)          # noqa: E731
    return t(x), t(f), None if b is None else torch.from_numpy(b).cuda().view(-1, 1), torch.from_numpy(c).cuda()


def _down(t):
    return t.permute(3, 2, 1, 0).reshape(t.shape[3], -1).cpu().numpy()


def _oracle(x, f, b, c, dzdy=1.0):
    real = c > 0
    x = np.where(real[:, None], x, 0).astype(np.float64)
    f = f.astype(np.float64)
    z = x @ f.T + (0 if b is None else b.astype(np.float64))
    top = z.max(1, keepdims=True)
    with np.errstate(invalid="ignore"):
        lse = np.where(real, (top + np.log(np.exp(z - top).sum(1, keepdims=True)))[:, 0], 0)
    at = np.maximum(c.astype(int) - 1, 0)
    rows = np.arange(len(c))
    loss = (np.where(real, lse - z[rows, at], 0)).sum() / len(c)
    dz = np.exp(z - lse[:, None])
    dz[rows, at] -= 1
    dz = np.where(real[:, None], dz, 0) * (dzdy / len(c))
    return loss, lse, dz @ f, dz.T @ x, dz.sum(0)


def _rel(a, r):
    a, r = np.asarray(a, np.float64).ravel(), np.asarray(r, np.float64).ravel()
    assert a.shape == r.shape
    return np.linalg.norm(a - r) / max(np.linalg.norm(r), 1e-30)


def _check(nn, mat, x, f, b, c, hwc, tol=TOL, tol_lse=TOL_LSE, dzdy=1.0, ctx=None):
    xd, fd, bd, cd = _up(mat, x, f, b, c, hwc)
    loss, lse, dx, df, db = _oracle(x, f, b, c, dzdy)
    gl, gs = nn.vl_nnfcsoftmaxloss(xd, fd, bd, cd, ctx=ctx)
    assert abs(float(gl) - loss) <= tol_lse * max(abs(loss), 10)
    assert np.abs(gs.cpu().numpy() - lse).max() <= tol_lse * max(np.abs(lse).max(), 10)
    out = []
    for kept in (gs, None):
        gx, gf, gb = nn.vl_nnfcsoftmaxloss(xd, fd, bd, cd, dzdy, lse=kept, ctx=ctx)
        # one class: the exact derivative is 0, and a probability of 1 is off by the error of a prediction
        floor = 1e-30 if f.shape[0] > 1 else 1e6
        for got, want in ((_down(gx), dx), (_down(gf), df)) + (() if b is None else ((gb.cpu().numpy(), db),)):
            assert np.isfinite(got).all()
            assert _rel(got, want) <= tol or np.abs(got - want.reshape(got.shape)).max() <= 1e-30 * floor * tol, (x.shape, f.shape)
        out.append((gx, gf, gb))
    return out


def test_the_oracles_gradient_against_differences():
    x, f, b, c = (a.astype(np.float64) for a in _inputs(5, (1, 1, 4), 6, 1))
    _, _, dx, df, db = _oracle(x, f, b, c, 1.5)
    rng = np.random.default_rng(2)
    ux, uf, ub = rng.standard_normal(x.shape), rng.standard_normal(f.shape), rng.standard_normal(b.shape)
    h = 1e-5
    g = lambda t: 1.5 * _oracle(x + t * ux, f + t * uf, b + t * ub, c)[0]                              # noqa: E731
    assert abs((g(h) - g(-h)) / (2 * h) - ((dx * ux).sum() + (df * uf).sum() + (db * ub).sum())) < 1e-7


@pytest.mark.gpu
@pytest.mark.parametrize("n,hwc,k", SIZES)
@pytest.mark.parametrize("bias", [True, False])
def test_forward_and_backward(gpu, n, hwc, k, bias):
    nn, mat, _ = gpu
    x, f, b, c = _inputs(n, hwc, k)
    _check(nn, mat, x, f, b if bias else None, c, hwc, dzdy=0.7)


@pytest.mark.gpu
@pytest.mark.parametrize("precision,tol,tol_lse", [("FP32", TOL, TOL_LSE), ("TF32", TOL_TF32, TOL_TF32)])
@pytest.mark.parametrize("n,hwc,k", [(3, (2, 2, 5), 7), (65, (1, 1, 200), 300), (300, (1, 1, 72), 1031)])
def test_the_other_arithmetics(gpu, precision, tol, tol_lse, n, hwc, k):
    from matconvnet_b200 import capi
    nn, mat, _ = gpu
    ctx = capi.Context(precision=getattr(capi, "PRECISION_" + precision))
    _check(nn, mat, *_inputs(n, hwc, k), hwc, tol=tol, tol_lse=tol_lse, ctx=ctx)


@pytest.mark.gpu
@pytest.mark.parametrize("n,d,k", [(4, 40, 50), (200, 136, 700)])
def test_skipped_images_may_hold_anything(gpu, n, d, k):
    nn, mat, _ = gpu
    x, f, b, c = _inputs(n, (1, 1, d), k, 3)
    c[1], c[n - 1] = 0, 0
    a = _check(nn, mat, x, f, b, c, (1, 1, d))
    x[0], x[1], x[n - 1] = np.inf, np.nan, 3e38
    for p, q in zip(a, _check(nn, mat, x, f, b, c, (1, 1, d))):
        for s, t in zip(p, q):
            assert (s == t).all()
    # nothing but skipped images: all is zero
    c[:] = 0
    xd, fd, bd, cd = _up(mat, x, f, b, c, (1, 1, d))
    loss, lse = nn.vl_nnfcsoftmaxloss(xd, fd, bd, cd)
    assert float(loss) == 0 and (lse == 0).all()
    for t in nn.vl_nnfcsoftmaxloss(xd, fd, bd, cd, 1.0):
        assert (t == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("n,d,k", [(4, 40, 50), (200, 136, 700)])
def test_classes_that_a_bias_takes_out(gpu, n, d, k):
    """A bias of -inf, or of the type's lowest value, leaves a class without a share and the others as if it were not there."""
    nn, mat, _ = gpu
    x, f, b, c = _inputs(n, (1, 1, d), k, 4)
    c[c > k - 5] = 1
    b[k - 5:k - 2], b[k - 2:] = -np.inf, np.finfo(np.float32).min
    loss, lse, dx, df, db = _oracle(x, f[:k - 5], b[:k - 5], c)
    xd, fd, bd, cd = _up(mat, x, f, b, c, (1, 1, d))
    gl, gs = nn.vl_nnfcsoftmaxloss(xd, fd, bd, cd)
    assert abs(float(gl) - loss) <= TOL_LSE * 10 and np.abs(gs.cpu().numpy() - lse).max() <= TOL_LSE * max(np.abs(lse).max(), 10)
    gx, gf, gb = nn.vl_nnfcsoftmaxloss(xd, fd, bd, cd, 1.0, lse=gs)
    assert _rel(_down(gx), dx) <= TOL and _rel(_down(gf)[:k - 5], df) <= TOL and _rel(gb.cpu().numpy()[:k - 5], db) <= TOL
    assert (_down(gf)[k - 5:] == 0).all() and (gb[k - 5:] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("n,d,k", [(4, 40, 50), (200, 136, 700)])
def test_predictions_far_apart(gpu, n, d, k):
    """Predictions of some hundreds: the largest has all the share.  z is off by 2^-22 * |z|, 1e-4 of a share at most."""
    nn, mat, _ = gpu
    x, f, b, c = _inputs(n, (1, 1, d), k, 5, spread=150.0)
    _check(nn, mat, x, f, b, c, (1, 1, d), tol=1e-3, tol_lse=1e-5)


@pytest.mark.gpu
@pytest.mark.parametrize("n,d,k", [(4, 40, 50), (200, 136, 700)])
def test_scales_of_data_and_filters(gpu, n, d, k):
    """Powers of two on one side and their inverses on the other change nothing but the derivatives' scale."""
    nn, mat, _ = gpu
    x, f, b, c = _inputs(n, (1, 1, d), k, 6)
    base = _check(nn, mat, x, f, b, c, (1, 1, d))
    for e in (-40, 40):
        s = np.float32(2.0 ** e)
        far = _check(nn, mat, x * s, f / s, b, c, (1, 1, d))
        for p, q in zip(base, far):
            assert (p[0] == q[0] * s).all() and (p[1] == q[1] / s).all() and (p[2] == q[2]).all()


@pytest.mark.gpu
def test_labels_above_the_classes_are_skipped_and_reported(gpu):
    from matconvnet_b200 import capi
    nn, mat, _ = gpu
    for n, d, k in ((4, 40, 50), (200, 136, 700)):
        ctx = capi.Context()
        x, f, b, c = _inputs(n, (1, 1, d), k, 7)
        xd, fd, bd, cd = _up(mat, x, f, b, c, (1, 1, d))
        want = nn.vl_nnfcsoftmaxloss(xd, fd, bd, cd, ctx=ctx), nn.vl_nnfcsoftmaxloss(xd, fd, bd, cd, 1.0, ctx=ctx)
        assert ctx.device_status() == 0
        cd[0] = k + 1
        for call, ref in ((lambda: nn.vl_nnfcsoftmaxloss(xd, fd, bd, cd, ctx=ctx), want[0]), (lambda: nn.vl_nnfcsoftmaxloss(xd, fd, bd, cd, 1.0, ctx=ctx), want[1])):
            got = call()
            with pytest.raises(capi.VlbError, match="label"):
                ctx.device_status()
            assert all((p == q).all() for p, q in zip(got, ref))


@pytest.mark.gpu
def test_some_derivatives_only_and_into_given_tensors(gpu):
    nn, mat, _ = gpu
    import torch
    for n, d, k in ((4, 40, 50), (200, 136, 700)):
        x, f, b, c = _inputs(n, (1, 1, d), k, 8)
        xd, fd, bd, cd = _up(mat, x, f, b, c, (1, 1, d))
        dx, df, db = nn.vl_nnfcsoftmaxloss(xd, fd, bd, cd, 1.0)
        for flag, at in (("no_der_data", 0), ("no_der_filters", 1), ("no_der_biases", 2)):
            got = nn.vl_nnfcsoftmaxloss(xd, fd, bd, cd, 1.0, **{flag: True})
            assert got[at] is None and all((p == q).all() for i, (p, q) in enumerate(zip(got, (dx, df, db))) if i != at)
        flat = torch.full((k * d + k + 8,), 7.0, device="cuda")
        pad = (k * d + 3) // 4 * 4
        out = flat[:k * d], flat[pad:pad + k]
        got = nn.vl_nnfcsoftmaxloss(xd, fd, bd, cd, 1.0, der_out=out)
        assert got[1].data_ptr() == out[0].data_ptr() and (out[0].view(k, d) == df.permute(3, 2, 1, 0).reshape(k, d)).all()
        assert (out[1] == db.view(-1)).all() and (flat[pad + k:] == 7).all()


@pytest.mark.gpu
def test_the_same_every_time_in_a_graph_and_on_another_stream(gpu):
    import torch
    nn, mat, _ = gpu
    for n, d, k in ((4, 40, 50), (200, 136, 700)):
        x, f, b, c = _inputs(n, (1, 1, d), k, 9)
        xd, fd, bd, cd = _up(mat, x, f, b, c, (1, 1, d))

        def call():
            loss, lse = nn.vl_nnfcsoftmaxloss(xd, fd, bd, cd)
            return (loss, lse) + nn.vl_nnfcsoftmaxloss(xd, fd, bd, cd, 1.0, lse=lse)

        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kept = call()
        x2, f2, _, c2 = _inputs(n, (1, 1, d), k, 10)
        for t, a in zip((xd, fd, cd), _up(mat, x2, f2, b, c2, (1, 1, d))[:2] + (torch.from_numpy(c2).cuda(),)):
            t.copy_(a)
        want = [t.clone() for t in call()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all((p == q).all() for p, q in zip(kept, want))
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got = call()
        s.synchronize()
        assert all((p == q).all() for p, q in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("n,d,k", [(40, 512, 20003), (700, 64, 9000)])
def test_in_pieces_of_classes(gpu, n, d, k):
    """Bit 5 of the test switches refuses scratch that a call can do without: the smallest pieces."""
    from matconvnet_b200 import capi
    nn, mat, _ = gpu
    ctx = capi.Context()
    ctx.check(ctx.lib.vlb_ctx_set_test_switch(ctx.handle, 32))
    x, f, b, c = _inputs(n, (1, 1, d), k, 12)
    c[3] = k
    before = ctx.launches
    _check(nn, mat, x, f, b, c, (1, 1, d), ctx=ctx)
    pieces = ctx.launches - before
    ctx.check(ctx.lib.vlb_ctx_set_test_switch(ctx.handle, 0))
    before = ctx.launches
    _check(nn, mat, x, f, b, c, (1, 1, d), ctx=ctx)
    assert pieces > ctx.launches - before


@pytest.mark.gpu
def test_more_images_than_go_through_at_once(gpu):
    nn, mat, _ = gpu
    _check(nn, mat, *_inputs(16384 + 77, (1, 1, 40), 90, 13), (1, 1, 40))


@pytest.mark.gpu
@pytest.mark.parametrize("n,d,k", [(2100, 130, 2300), (513, 1030, 900), (1, 50000, 20), (17, 30000, 40)])
def test_larger_tiles_and_long_rows(gpu, n, d, k):
    nn, mat, _ = gpu
    _check(nn, mat, *_inputs(n, (1, 1, d), k, 14), (1, 1, d))


@pytest.mark.gpu
def test_an_image_or_class_is_as_exact_beside_far_larger_ones(gpu):
    """Values keep their digits down to 2^-28 of the largest of 64 neighbouring images (classes), whatever the others are: images and classes 2^14
    smaller than every other one, each against itself, and one image in each of some blocks of 64 whose values make all others vanish beside it."""
    nn, mat, _ = gpu
    n, d, k = 200, 136, 300
    x, f, b, c = _inputs(n, (1, 1, d), k, 15)
    c[c == 0] = 1
    small = np.arange(n) % 2 == 0
    x[small] *= np.float32(2.0 ** -14)
    xd, fd, bd, cd = _up(mat, x, f, b, c, (1, 1, d))
    _, lse, dx, df, _ = _oracle(x, f, b, c)
    gl, gs = nn.vl_nnfcsoftmaxloss(xd, fd, bd, cd)
    assert np.abs(gs.cpu().numpy() - lse).max() <= TOL_LSE * 10
    gx, gf, _ = nn.vl_nnfcsoftmaxloss(xd, fd, bd, cd, 1.0, lse=gs)
    got = _down(gx)
    for i in range(n):
        assert _rel(got[i], dx[i]) <= TOL
    # half of the classes with filters 2^14 smaller: their derivatives are sums over the same images
    x, f, b, c = _inputs(n, (1, 1, d), k, 16)
    f[::2] *= np.float32(2.0 ** -14)
    xd, fd, bd, cd = _up(mat, x, f, b, c, (1, 1, d))
    _, lse, dx, df, db = _oracle(x, f, b, c)
    gx, gf, gb = nn.vl_nnfcsoftmaxloss(xd, fd, bd, cd, 1.0)
    got = _down(gf)
    for i in range(k):
        assert _rel(got[i], df[i]) <= TOL
    assert _rel(_down(gx), dx) <= TOL and _rel(gb.cpu().numpy(), db) <= TOL
    # images 0 and 130 are 2^60 times as large: what the blocks of 64 without them hold keeps its digits
    x, f, b, c = _inputs(n, (1, 1, d), k, 18)
    c[c == 0] = 1
    huge = [0, 130]
    x[huge] *= np.float32(2.0 ** 60)
    xd, fd, bd, cd = _up(mat, x, f, b, c, (1, 1, d))
    _, lse, dx, _, _ = _oracle(x, f, b, c)
    gl, gs = nn.vl_nnfcsoftmaxloss(xd, fd, bd, cd)
    gx, _, _ = nn.vl_nnfcsoftmaxloss(xd, fd, bd, cd, 1.0, lse=gs)
    got, sums = _down(gx), gs.cpu().numpy()
    for i in list(range(64, 128)) + list(range(192, n)):
        assert abs(sums[i] - lse[i]) <= TOL_LSE * 10 and _rel(got[i], dx[i]) <= TOL


@pytest.mark.gpu
def test_two_contexts_on_two_streams_at_once(gpu):
    import torch
    from matconvnet_b200 import capi
    nn, mat, _ = gpu
    work = []
    for i, (n, d, k) in enumerate([(300, 200, 3000), (4, 512, 2000), (900, 72, 700)]):
        data = _up(mat, *_inputs(n, (1, 1, d), k, 20 + i), (1, 1, d))
        ctx = capi.Context()
        want = nn.vl_nnfcsoftmaxloss(*data, ctx=ctx) + nn.vl_nnfcsoftmaxloss(*data, 1.0, ctx=ctx)
        work.append((data, ctx, want, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for data, ctx, _, stream in work:
            with torch.cuda.stream(stream):
                got.append(nn.vl_nnfcsoftmaxloss(*data, ctx=ctx) + nn.vl_nnfcsoftmaxloss(*data, 1.0, ctx=ctx))
        torch.cuda.synchronize()
        for g, (_, ctx, want, _) in zip(got, work):
            assert all((p == q).all() for p, q in zip(g, want)) and ctx.device_status() == 0


@pytest.mark.gpu
def test_a_wait_that_runs_out(gpu):
    """Nothing is loaded, so no wait is ever answered: the kernels give up, say so and leave everything as the next call needs it."""
    from matconvnet_b200 import capi
    nn, mat, _ = gpu
    for n, d, k in ((64, 2048, 200), (2100, 130, 2300)):
        ctx = capi.Context()
        data = _up(mat, *_inputs(n, (1, 1, d), k, 17), (1, 1, d))
        call = lambda: nn.vl_nnfcsoftmaxloss(*data, ctx=ctx) + nn.vl_nnfcsoftmaxloss(*data, 1.0, ctx=ctx)       # noqa: E731
        want = call()
        assert ctx.device_status() == 0
        try:
            ctx.check(ctx.lib.vlb_ctx_set_wait_limit(ctx.handle, 200000))
            ctx.check(ctx.lib.vlb_ctx_set_test_switch(ctx.handle, 1))
            call()
            with pytest.raises(capi.VlbError, match="TIMEOUT|Timeout|timeout"):
                ctx.device_status()
        finally:
            ctx.check(ctx.lib.vlb_ctx_set_test_switch(ctx.handle, 0))
            ctx.check(ctx.lib.vlb_ctx_set_wait_limit(ctx.handle, 0))
        assert all((p == q).all() for p, q in zip(call(), want)) and ctx.device_status() == 0


@pytest.mark.gpu
def test_strides_and_alignment(gpu):
    import torch
    nn, mat, _ = gpu
    x, f, b, c = _inputs(70, (1, 1, 100), 260, 11)
    xd, fd, bd, cd = _up(mat, x, f, b, c, (1, 1, 100))
    want = nn.vl_nnfcsoftmaxloss(xd, fd, bd, cd, 1.0)
    off = torch.empty(f.size + 1, device="cuda")[1:].view(260, 100, 1, 1).permute(3, 2, 1, 0)
    off.copy_(fd)
    xr = torch.from_numpy(np.ascontiguousarray(x.T)).cuda().view(1, 1, 100, 70)             # row-major: copied
    got = nn.vl_nnfcsoftmaxloss(xr, off, bd, cd, 1.0)
    for p, q in zip(got, want):
        assert _rel(p.cpu().numpy(), q.cpu().numpy()) <= TOL


@pytest.mark.gpu
def test_refusals(gpu):
    nn, mat, _ = gpu
    x, f, b, c = _up(mat, *_inputs(6, (1, 1, 8), 9), (1, 1, 8))
    with pytest.raises(TypeError):
        nn.vl_nnfcsoftmaxloss(x.cpu(), f, b, c)
    with pytest.raises(TypeError):
        nn.vl_nnfcsoftmaxloss(x, f.bfloat16(), b, c)
    with pytest.raises(TypeError):
        nn.vl_nnfcsoftmaxloss(x, f, b, c.long())
    with pytest.raises(ValueError, match="FILTERS"):
        nn.vl_nnfcsoftmaxloss(x, f[:, :, :7], b, c)
    with pytest.raises(ValueError, match="BIASES"):
        nn.vl_nnfcsoftmaxloss(x, f, b[:8], c)
    with pytest.raises(ValueError, match="label"):
        nn.vl_nnfcsoftmaxloss(x, f, b, c[:5])
    with pytest.raises(ValueError, match="LSE"):
        nn.vl_nnfcsoftmaxloss(x, f, b, c, 1.0, lse=c[:5])
    with pytest.raises(RuntimeError, match="bad shape"):
        nn.vl_nnfcsoftmaxloss(x[:, :, :, :0], f, b, c[:0])
    with pytest.raises(RuntimeError, match="bad shape"):
        nn.vl_nnfcsoftmaxloss(x, f[:, :, :, :0], None, c)


@pytest.mark.gpu
@pytest.mark.parametrize("hwc,n,k", [((1, 1, 1), 3, 2**31 - 1), ((1, 1, 1), 2**31 - 1, 3), ((1, 1, 2**31 - 1), 3, 3), ((2**16, 2**16, 2), 3, 3), ((2**16, 2**15, 2**16), 3, 3)])
def test_sizes_that_counters_do_not_hold_are_refused(gpu, hwc, n, k):
    ctx = gpu[2]
    # refused before anything is looked at
    some = 256
    assert ctx.lib.vlb_fc_softmaxloss_forward(ctx.handle, some, None, some, some, None, some, *hwc, n, k) == 7
    assert ctx.lib.vlb_fc_softmaxloss_backward(ctx.handle, None, None, None, some, some, None, some, None, 1.0, *hwc, n, k) == 7
    ctx.lib.vlb_ctx_reset_error(ctx.handle)

"""Layer normalisation against its formulas in 64 bits.

Tolerances.  A value is rounded by at most u = 2^-24 of it.  Y = g*(x - m)*r + b is within a few roundings of the exact value once m and r are:
the mean of C values carries at most (log2(C) + 8) * u of the mean of their magnitudes when partial sums of at most eight values are added in a
tree, the variance twice that.  With values of spread s around an offset o the difference x - m is off by u * (|o| + s) * 20 at most, so that in
units of the output (spread 1) an element is within 20 * u * (1 + |o|/s) * |g| + 4 * u * |Y|; TOL below is that bound with |o|/s <= 4,
|g| <= 2: 1.2e-5 of the largest output for single elements, and 2e-6 in the 2-norm, where roundings average out (20 u (1 + 4) / sqrt(12) = 1.7e-6).
The sums over positions add P terms of unit size whose roundings are independent: relative to the 2-norm of the result u * sqrt(20) < 3e-7, and
2e-6 with the moments' own errors.
"""
import numpy as np
import pytest

from conftest import rel_l2

TOL_L2, TOL_MAX = 2e-6, 1.2e-5

SHAPES = [(1, 1, 1, 1), (1, 1, 1, 7), (1, 1, 5, 1), (1, 1, 64, 33), (1, 1, 1024, 1), (1, 1, 1000, 257), (1, 1, 1023, 64), (1, 1, 4096, 70),
          (1, 1, 4099, 5), (1, 1, 8192, 19), (1, 1, 12289, 6), (1, 1, 70001, 3), (1, 1, 260, 5000), (1, 1, 64, 40000), (1, 1, 63, 3000),
          (2, 1, 3, 4), (7, 5, 33, 3), (28, 28, 96, 2), (35, 47, 90, 2), (3, 3, 1031, 5), (1, 9, 512, 40), (64, 64, 17, 1), (5, 1, 6001, 2), (2, 2, 200, 700), (4, 1, 300, 9), (2, 6, 700, 3), (3, 1, 250, 2)]


def _inputs(shape, seed=0, offset=0.5):
    rng = np.random.default_rng(seed)
    c = shape[2]
    x = np.asfortranarray((rng.standard_normal(shape) + offset).astype(np.float32))
    dy = np.asfortranarray(rng.standard_normal(shape).astype(np.float32))
    return x, rng.uniform(0.5, 2, (c, 1)).astype(np.float32), rng.standard_normal((c, 1)).astype(np.float32), dy


def _forward(x, g, b, eps):
    x, g, b = (a.astype(np.float64) for a in (x, g, b))
    m, v = x.mean(2, keepdims=True), x.var(2, keepdims=True)
    return g.reshape(1, 1, -1, 1) * (x - m) / np.sqrt(v + eps) + b.reshape(1, 1, -1, 1)


def _backward(x, g, dy, eps):
    x, g, dy = (a.astype(np.float64) for a in (x, g, dy))
    m, r = x.mean(2, keepdims=True), 1 / np.sqrt(x.var(2, keepdims=True) + eps)
    xh, gd = (x - m) * r, g.reshape(1, 1, -1, 1) * dy
    dx = r * (gd - gd.mean(2, keepdims=True) - xh * (gd * xh).mean(2, keepdims=True))
    return dx, (dy * xh).sum((0, 1, 3))[:, None], dy.sum((0, 1, 3))[:, None]


def _close(got, want, scale=None):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape
    scale = np.abs(want).max() if scale is None else scale
    assert np.abs(got - want).max() <= TOL_MAX * max(scale, 1e-30)
    assert np.linalg.norm(got - want) <= TOL_L2 * max(np.linalg.norm(want), scale * np.sqrt(want.size), 1e-30)


def test_the_oracles_gradient_against_differences():
    x, g, b, dy = (a.astype(np.float64) for a in _inputs((2, 3, 7, 2), 3))
    dx, dg, db = _backward(x, g, dy, 1e-3)
    rng = np.random.default_rng(4)
    ux, ug, ub = rng.standard_normal(x.shape), rng.standard_normal(g.shape), rng.standard_normal(b.shape)
    h = 1e-5
    # central differences in 64 bits: h^2 of truncation and 1e-16 / h of rounding
    f = lambda t: (_forward(x + t * ux, g + t * ug, b + t * ub, 1e-3) * dy).sum()                    # noqa: E731
    assert abs((f(h) - f(-h)) / (2 * h) - ((dx * ux).sum() + (dg * ug).sum() + (db * ub).sum())) < 1e-6


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_and_backward(gpu, shape):
    nn, mat, _ = gpu
    x, g, b, dy = _inputs(shape)
    xd, gd, bd, dyd = (mat.from_numpy(a) for a in (x, g, b, dy))
    y = nn.vl_nnlayernorm(xd, gd, bd, epsilon=1e-3)
    _close(mat.to_numpy(y), _forward(x, g, b, 1e-3))
    dx, dg, db = nn.vl_nnlayernorm(xd, gd, bd, dyd, epsilon=1e-3)
    rx, rg, rb = _backward(x, g, dy, 1e-3)
    _close(mat.to_numpy(dx), rx, scale=max(np.abs(rx).max(), 1.0))          # (one channel: the exact derivative is 0)
    positions = shape[0] * shape[1] * shape[3]
    _close(mat.to_numpy(dg), rg, scale=max(np.abs(rg).max(), np.sqrt(positions)))
    _close(mat.to_numpy(db), rb, scale=max(np.abs(rb).max(), np.sqrt(positions)))


# a shape of every kernel for maps, with and without 16-byte accesses, and more tiles than blocks run at one time
MAPS = [(2, 2, 24, 9), (3, 7, 30, 11), (4, 4, 60, 7), (3, 1, 64, 50), (8, 2, 128, 3), (4, 1, 256, 11), (6, 2, 512, 5), (8, 4, 1000, 30), (4, 2, 1500, 5), (3, 3, 2048, 6),
        (4, 3, 2049, 3), (16, 16, 40, 700), (13, 11, 120, 220), (8, 8, 300, 200), (9, 7, 300, 200), (8, 8, 700, 80)]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", MAPS)
def test_maps_of_every_kind(gpu, shape):
    test_forward_and_backward(gpu, shape)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(4, 4, 200, 9), (7, 3, 200, 9), (1, 1, 300, 40)])
def test_the_derivative_of_the_data_or_of_the_parameters_alone(gpu, shape):
    import ctypes
    import torch
    nn, mat, ctx = gpu
    x, g, b, dy = _inputs(shape, 2)
    xd, gd, bd, dyd = (mat.from_numpy(a) for a in (x, g, b, dy))
    want = nn.vl_nnlayernorm(xd, gd, bd, dyd)
    ptr = lambda t: ctypes.c_void_p(t.data_ptr())                                        # noqa: E731
    ctx.check(ctx.lib.vlb_ctx_set_stream(ctx.handle, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)))
    for asked in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1), (1, 0, 1)):
        got = [mat.from_numpy(np.asfortranarray(np.full(tuple(t.shape), 7, np.float32))) for t in want]
        ctx.check(ctx.lib.vlb_lnorm_backward(ctx.handle, *(ptr(t) if a else None for t, a in zip(got, asked)), ptr(xd), ptr(gd), ptr(dyd), *shape, 1e-5))
        for t, full, a in zip(got, want, asked):
            assert (t == full).all() if a else (t == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 1, 513, 9), (5, 3, 40, 4)])
def test_values_far_from_zero_and_outputs_asked_for(gpu, shape):
    """An offset of 1000 spreads: the differences from the mean keep what the inputs hold (2^-24 * 1000 of a spread, 6e-5, is in the inputs
    themselves); sums of squares without the mean would lose it all."""
    nn, mat, _ = gpu
    x, g, b, dy = _inputs(shape, 5, offset=1000.0)
    xd, gd, bd, dyd = (mat.from_numpy(a) for a in (x, g, b, dy))
    y = mat.to_numpy(nn.vl_nnlayernorm(xd, gd, bd))
    ref = _forward(x, g, b, 1e-5)
    # the mean, about 1000, is off by at most 2^-24 * 1000 * a few: 2e-4 of a spread
    assert np.abs(y - ref).max() < 2 * 2e-4 + 1e-5
    out = [mat.empty((shape[2], 1)), mat.empty((shape[2], 1))]
    dx, dg, db = nn.vl_nnlayernorm(xd, gd, bd, dyd, der_out=out)
    assert dg.data_ptr() == out[0].data_ptr() and db.data_ptr() == out[1].data_ptr()
    again = nn.vl_nnlayernorm(xd, gd, bd, dyd)
    for p, q in zip((dx, dg, db), again):
        assert (mat.to_numpy(p) == mat.to_numpy(q)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 1, 260, 6), (3, 5, 70, 2)])
def test_infinities_and_not_a_numbers_stay_at_their_position(gpu, shape):
    nn, mat, _ = gpu
    x, g, b, dy = _inputs(shape, 7)
    ref = mat.to_numpy(nn.vl_nnlayernorm(*(mat.from_numpy(a) for a in (x, g, b))))
    bad = x.copy(order="F")
    bad[0, 0, 3, 0], bad[-1, -1, 5, -1] = np.nan, np.inf
    y = mat.to_numpy(nn.vl_nnlayernorm(*(mat.from_numpy(a) for a in (bad, g, b))))
    hit = np.zeros(shape, bool)
    hit[0, 0, :, 0] = hit[-1, -1, :, -1] = True
    assert np.isnan(y[0, 0, :, 0]).all() and np.isnan(y[-1, -1, :, -1]).all()
    assert (y[~hit] == ref[~hit]).all()
    dx = mat.to_numpy(nn.vl_nnlayernorm(*(mat.from_numpy(a) for a in (bad, g, b, dy)))[0])
    rx = mat.to_numpy(nn.vl_nnlayernorm(*(mat.from_numpy(a) for a in (x, g, b, dy)))[0])
    assert np.isnan(dx[hit]).all() and (dx[~hit] == rx[~hit]).all()


@pytest.mark.gpu
def test_constant_channels_give_the_shift(gpu):
    nn, mat, _ = gpu
    x, g, b, _ = _inputs((1, 1, 300, 4), 8)
    x[:] = 3.0
    y = mat.to_numpy(nn.vl_nnlayernorm(*(mat.from_numpy(a) for a in (x, g, b))))
    # 300 * 3 and its mean are exact in single precision
    assert (y == b.reshape(1, 1, -1, 1)).all()


@pytest.mark.gpu
def test_views_strides_and_a_stream_of_its_own(gpu):
    import torch
    nn, mat, _ = gpu
    x, g, b, dy = _inputs((6, 4, 50, 3), 9)
    xd, gd, bd, dyd = (mat.from_numpy(a) for a in (x, g, b, dy))
    want = [mat.to_numpy(t) for t in (nn.vl_nnlayernorm(xd, gd, bd),) + nn.vl_nnlayernorm(xd, gd, bd, dyd)]
    rows = torch.from_numpy(np.ascontiguousarray(x)).cuda()               # row-major: copied
    off = torch.empty(x.size + 1, device="cuda")[1:]                        # 4-byte aligned
    off = off.view(3, 50, 4, 6).permute(3, 2, 1, 0)
    off.copy_(xd)
    s = torch.cuda.Stream()
    for v in (rows, off):
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            got = (nn.vl_nnlayernorm(v, gd, bd),) + nn.vl_nnlayernorm(v, gd, bd, dyd)
        s.synchronize()
        for p, q in zip(got, want):
            assert rel_l2(mat.to_numpy(p), q) < TOL_L2


@pytest.mark.gpu
def test_in_a_graph(gpu):
    import torch
    nn, mat, _ = gpu
    for shape in ((1, 1, 512, 40), (6, 4, 50, 3)):
        x, g, b, dy = _inputs(shape, 10)
        xd, gd, bd, dyd = (mat.from_numpy(a) for a in (x, g, b, dy))
        nn.vl_nnlayernorm(xd, gd, bd, dyd)                                   # scratch grows outside the capture
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y, grads = nn.vl_nnlayernorm(xd, gd, bd), nn.vl_nnlayernorm(xd, gd, bd, dyd)
        x2, _, _, dy2 = _inputs(shape, 11)
        xd.copy_(mat.from_numpy(x2))
        dyd.copy_(mat.from_numpy(dy2))
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip((y,) + tuple(grads), (nn.vl_nnlayernorm(xd, gd, bd),) + nn.vl_nnlayernorm(xd, gd, bd, dyd)):
            assert (mat.to_numpy(p) == mat.to_numpy(q)).all()


@pytest.mark.gpu
def test_refusals(gpu):
    import torch
    nn, mat, ctx = gpu
    x, g, b, dy = (mat.from_numpy(a) for a in _inputs((2, 2, 8, 3)))
    with pytest.raises(TypeError):
        nn.vl_nnlayernorm(x.cpu(), g, b)
    with pytest.raises(TypeError):
        nn.vl_nnlayernorm(x.half(), g, b)
    with pytest.raises(ValueError, match="G is not the same"):
        nn.vl_nnlayernorm(x, g[:7], b)
    with pytest.raises(ValueError, match="B is not the same"):
        nn.vl_nnlayernorm(x, g, b[:7])
    with pytest.raises(ValueError, match="DZDY"):
        nn.vl_nnlayernorm(x, g, b, dy[:, :, :, :2])
    with pytest.raises(ValueError, match="DG"):
        nn.vl_nnlayernorm(x, g, b, dy, der_out=(torch.empty(7, device="cuda"), None))
    with pytest.raises(RuntimeError, match="epsilon"):
        nn.vl_nnlayernorm(x, g, b, epsilon=-1.0)
    with pytest.raises(RuntimeError, match="epsilon"):
        nn.vl_nnlayernorm(x, g, b, epsilon=float("nan"))
    with pytest.raises(RuntimeError, match="bad shape"):
        nn.vl_nnlayernorm(x[:, :, :, :0], g, b)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 1, 2**31 - 1, 1), (1, 1, 2**30, 1), (1, 1, 1, 2**31 - 1), (2**16, 2**15, 4, 1), (2**31 - 1, 2**31 - 1, 4, 4), (2**16, 2**16, 4, 2**31 - 1)])
def test_sizes_that_counters_do_not_hold_are_refused(gpu, shape):
    ctx = gpu[2]
    some = 256                               # refused before anything is looked at
    assert ctx.lib.vlb_lnorm_forward(ctx.handle, some, some, some, some, *shape, 1e-5) == 7
    assert ctx.lib.vlb_lnorm_backward(ctx.handle, some, None, None, some, some, some, *shape, 1e-5) == 7
    ctx.lib.vlb_ctx_reset_error(ctx.handle)

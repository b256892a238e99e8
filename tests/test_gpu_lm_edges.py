"""The operators of language models' training steps at the ends of what they take: long rows, dimensions beyond 32 bits, scratch that grows or is not to be had,
waits that run out, contexts of another device."""
import ctypes

import numpy as np
import pytest

import test_gpu_fcloss as fcloss
import test_gpu_lnorm as lnorm
import test_gpu_muon as muon

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,cols", [(1, 1200000), (3, 1054400), (3, 1605602), (3, 1605632), (1605632, 3)])
def test_muon_on_rows_of_more_than_a_million_columns(gpu, rows, cols):
    """After a call that leaves not-a-numbers in the scratch: a place of it that is read without having been written shows.

    Tolerance.  The matrix X X' of at most three rows is a sum of 25088 chains of 64 products: a chain is off by at most 12 * 2^-24 (additions that truncate), products by
    2^-22 of random sign, the sums of at most 392 chains by 2^-24 * sqrt(392 / 3): together below 2e-6 of an element.  The singular values of these gradients are within
    a factor of two of one another, where the polynomial's derivative is at most 1.2 or so: five steps stay below the 2e-5 of the other sizes."""
    nn = gpu[0]
    shape = (1, 1, cols, rows)
    w, m, g = muon._inputs(shape, 30)
    g[:] = np.nan
    nn.solver_update_("muon", muon._up(w, shape), {"s1": muon._up(m, shape), "t": 1}, muon._up(g, shape), 0.5, 0.0, 0.1, muon.OPTS)
    muon._check(nn, [shape], seed=31)


@pytest.mark.parametrize("shape", [(1, 1, 2050, 3), (1, 1, 5003, 300), (7, 7, 512, 130), (1, 1, 130, 25088), (1, 1, 65600, 40)])
def test_muon_on_rows_and_columns_of_some_thousands(gpu, shape):
    """Sums of up to 65600 products, in chains of 64 of which at most 1025 follow one another: rounded by less than one sum of 4096 is bounded by in test_gpu_muon.py."""
    muon._check(gpu[0], [shape], seed=35)


LONG = 2 ** 32 + 5                          # what a 32-bit number has of it is 5


def test_dimensions_beyond_32_bits_are_refused(gpu):
    """Tensors without elements, so that nothing has to be held: each dimension in turn is LONG and another one 0."""
    import torch
    nn = gpu[0]
    some = torch.zeros(5, 1, device="cuda")
    empty = lambda *s: torch.empty(s, device="cuda")                                                # noqa: E731
    for at in range(4):
        shape = [0 if i == (at + 1) % 4 else 1 for i in range(4)]
        shape[at] = LONG
        x = empty(*shape)
        assert x.numel() == 0
        with pytest.raises(ValueError, match="too large"):
            nn.vl_nnlayernorm(x, some, some)
        with pytest.raises(ValueError, match="too large"):
            nn.vl_nnlayernorm(x, some, some, x)
        for dzdy in (None, 1.0):
            with pytest.raises(ValueError, match="too large"):
                nn.vl_nnfcsoftmaxloss(x, empty(1, 1, 1, 5), None, some, dzdy)
    for dzdy in (None, 1.0):
        with pytest.raises(ValueError, match="F is too large"):
            nn.vl_nnfcsoftmaxloss(empty(0, 1, 1, 5), empty(0, 1, 1, LONG), None, some, dzdy)
    with pytest.raises(ValueError, match="too large"):
        nn.vl_nnlayernorm(empty(1, 0, 3, 2 ** 20, 2 ** 12), some, some)                             # (trailing dimensions count as the fourth)


def test_more_positions_than_32_bits_hold_are_refused(gpu):
    """17 GB of them.  Five positions would be computed and the others left as they were found."""
    import torch
    nn = gpu[0]
    if torch.cuda.mem_get_info()[0] < 60e9:
        pytest.skip("needs room for two tensors of 17 GB")
    one = torch.zeros(1, 1, device="cuda")
    x = torch.empty(LONG, device="cuda").view(1, 1, 1, LONG)
    try:
        with pytest.raises(ValueError, match="too large"):
            nn.vl_nnlayernorm(x, one, one)
    finally:
        del x
        torch.cuda.empty_cache()


def test_layer_normalisation_whose_waits_run_out(gpu):
    """No row comes, so no wait is ever answered: the kernel gives up, says so and leaves everything as the next call needs it."""
    from matconvnet_b200 import capi
    nn, mat, _ = gpu
    for shape in ((1, 1, 64, 5000), (1, 1, 1024, 900), (1, 1, 8192, 200)):
        ctx = capi.Context()
        x, g, b, dy = (mat.from_numpy(a) for a in lnorm._inputs(shape, 6))
        want = nn.vl_nnlayernorm(x, g, b, dy, ctx=ctx)
        assert ctx.device_status() == 0
        try:
            ctx.check(ctx.lib.vlb_ctx_set_wait_limit(ctx.handle, 200000))
            ctx.check(ctx.lib.vlb_ctx_set_test_switch(ctx.handle, 1))
            nn.vl_nnlayernorm(x, g, b, dy, ctx=ctx)
            with pytest.raises(capi.VlbError, match="TIMEOUT|Timeout|timeout"):
                ctx.device_status()
        finally:
            ctx.check(ctx.lib.vlb_ctx_set_test_switch(ctx.handle, 0))
            ctx.check(ctx.lib.vlb_ctx_set_wait_limit(ctx.handle, 0))
        assert all((p == q).all() for p, q in zip(nn.vl_nnlayernorm(x, g, b, dy, ctx=ctx), want)) and ctx.device_status() == 0


def _fcloss_data(n, d, k, seed):
    import torch
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x, f = torch.randn(n, d, device="cuda", generator=gen), torch.randn(k, d, device="cuda", generator=gen) * (2 / d ** 0.5)
    b = torch.randn(k, 1, device="cuda", generator=gen)
    c = torch.randint(0, k + 1, (n,), device="cuda", generator=gen).float()
    up = lambda t: t.view(t.shape[0], t.shape[1], 1, 1).permute(3, 2, 1, 0)                         # noqa: E731
    return x, f, b, c, up(x), up(f)


@pytest.mark.parametrize("n,d,k", [(16384 + 300, 40, 15000)])
def test_fcloss_in_pieces_of_classes_and_of_images(gpu, n, d, k):
    """With the smallest pieces: dX is added up over pieces of classes, dF over pieces of images, the parts of a log-sum-exp over the former.  Tolerances as in
    test_gpu_fcloss.py; sums in 64 bits on the device."""
    import torch
    from matconvnet_b200 import capi
    nn = gpu[0]
    x, f, b, c, xd, fd = _fcloss_data(n, d, k, 40)
    xs, fs, bs = x.double(), f.double(), b.double().view(-1)
    real, at = c > 0, (c.long() - 1).clamp(min=0)
    lse, dx, df, db, loss = torch.zeros(n, device="cuda", dtype=torch.float64), torch.zeros_like(xs), torch.zeros_like(fs), torch.zeros_like(bs), 0.0
    for i in range(0, n, 4096):
        p = slice(i, min(n, i + 4096))
        z = xs[p] @ fs.T + bs
        lse[p] = torch.logsumexp(z, 1) * real[p]
        loss += ((torch.logsumexp(z, 1) - z.gather(1, at[p, None])[:, 0]) * real[p]).sum() / n
        z = (z - torch.logsumexp(z, 1, keepdim=True)).exp()
        z.scatter_add_(1, at[p, None], -torch.ones_like(z[:, :1]))
        z *= real[p, None] / n
        dx[p] = z @ fs
        df += z.T @ xs[p]
        db += z.sum(0)
    ctx = capi.Context()
    ctx.check(ctx.lib.vlb_ctx_set_test_switch(ctx.handle, 32))
    gl, gs = nn.vl_nnfcsoftmaxloss(xd, fd, b, c, ctx=ctx)
    assert abs(float(gl) - float(loss)) <= fcloss.TOL_LSE * 10 and float((gs - lse).abs().max()) <= fcloss.TOL_LSE * 10
    rel = lambda a, r: float((a.double() - r).norm() / r.norm())                                    # noqa: E731
    for kept in (gs, None):
        gx, gf, gb = nn.vl_nnfcsoftmaxloss(xd, fd, b, c, 1.0, lse=kept, ctx=ctx)
        for got, want in ((gx.permute(3, 2, 1, 0).reshape(n, d), dx), (gf.permute(3, 2, 1, 0).reshape(k, d), df), (gb.view(-1), db)):
            assert rel(got, want) <= fcloss.TOL


def test_fcloss_scratch_is_what_a_call_needs(gpu):
    """Many images and classes of few features.  What the products' epilogues leave of a piece of classes -- 8 bytes for an image and 64 classes -- goes by the piece, and
    is not taken where the log-sum-exp are given."""
    from matconvnet_b200 import capi
    nn = gpu[0]
    n, d, k = 8192, 8, 300000
    _, _, b, c, xd, fd = _fcloss_data(n, d, k, 41)
    pairs, parts = 4 * 64 * n, n * 2 * (-(-k // 128)) * 8
    assert parts > 300e6
    ctx = capi.Context()
    ctx.check(ctx.lib.vlb_ctx_set_test_switch(ctx.handle, 32))              # the smallest pieces: 16 MB for pairs, as much for parts
    want = nn.vl_nnfcsoftmaxloss(xd, fd, b, c, ctx=ctx)
    assert ctx.workspace_bytes < 2 * (16 << 20) + (64 << 20) + pairs + (1 << 20)
    whole = nn.vl_nnfcsoftmaxloss(xd, fd, b, c, ctx=gpu[2])
    for p, q in zip(want, whole):
        assert float((p - q).abs().max()) <= 2 * fcloss.TOL_LSE * 15        # (lse near log(k) + 2, either side off by TOL_LSE of it)
    # one piece, backward: pairs of X, F and the derivative of the predictions, its sums over 32 images, 64 MB for parts of sums
    n, d, k = 4096, 8, 20032
    _, _, b, c, xd, fd = _fcloss_data(n, d, k, 42)
    lse = nn.vl_nnfcsoftmaxloss(xd, fd, b, c)[1]
    need = 4 * 64 * (n + k) + 4 * n * k + 4 * (n // 32) * k + (64 << 20)
    parts = n * 2 * (-(-k // 128)) * 8
    ctx = capi.Context()
    nn.vl_nnfcsoftmaxloss(xd, fd, b, c, 1.0, lse=lse, ctx=ctx)
    assert need <= ctx.workspace_bytes < need + parts // 2


@pytest.mark.parametrize("precision", ["3XTF32", "FP32"])
def test_muon_whose_scratch_is_not_to_be_had_changes_nothing(gpu, precision):
    """Sixteen banks and one behind them whose scratch no device has: the call is refused before the first of them is touched.  (Nothing looks at the last one's tensors.)"""
    import torch
    from matconvnet_b200 import capi
    ctx = capi.Context(precision=getattr(capi, "PRECISION_" + precision))
    w, s1, g = (torch.randn(17, 64, 40, device="cuda") for _ in range(3))
    u = (capi.MuonParam * 17)()
    for i in range(17):
        u[i] = capi.MuonParam(w[i].data_ptr(), s1[i].data_ptr(), g[i].data_ptr(), 64, 40, 0.0, 0.1)
    u[16] = capi.MuonParam(256, 512, 768, 2 ** 20, 2 ** 20, 0.0, 0.1)
    o = capi.MuonOpts(0.95, 1e-7, 3.4445, -4.7750, 2.0315, 1, 5)
    before = w.clone(), s1.clone()
    torch.cuda.synchronize()
    for alone in (False, True):              # the first banks in shared launches, and none of them in the same launch as another
        if alone:
            for i in range(1, 16):
                u[i] = u[0]
        assert ctx.lib.vlb_muon_update_many(ctx.handle, 17, u, 1.0, ctypes.byref(o)) == capi.ERROR_NAMES.index("VLE_OutOfGPUMemeory")
        ctx.lib.vlb_ctx_reset_error(ctx.handle)
        torch.cuda.synchronize()
        assert (w == before[0]).all() and (s1 == before[1]).all()


def test_a_context_of_another_device_is_refused(gpu):
    """Its scratch and its status word are not this device's.  The number of the device is the first word of a context."""
    from matconvnet_b200 import capi
    nn, mat, _ = gpu
    x, g, b, dy = (mat.from_numpy(a) for a in lnorm._inputs((1, 1, 40, 50), 1))
    c = mat.from_numpy(np.ones(50, np.float32))
    ctx = capi.Context()
    device = ctypes.c_int.from_address(ctx.handle.value)
    calls = [lambda: nn.vl_nnlayernorm(x, g, b, ctx=ctx), lambda: nn.vl_nnlayernorm(x, g, b, dy, ctx=ctx), lambda: nn.vl_nnfcsoftmaxloss(x, dy, None, c, ctx=ctx),
             lambda: nn.vl_nnfcsoftmaxloss(x, dy, None, c, 1.0, ctx=ctx), lambda: nn.solver_update_("muon", x, {}, dy, 1.0, 0.0, 0.1, ctx=ctx)]
    assert device.value == 0
    device.value = 1
    try:
        for call in calls:
            with pytest.raises(capi.VlbError, match="device"):
                call()
    finally:
        device.value = 0
    for call in calls:
        call()
    assert ctx.device_status() == 0


def test_muon_on_a_bank_of_one_filter_whose_derivative_has_a_fourth_dimension(gpu):
    """A bank FH x FW x FC is one of a single filter; its derivative, as vl_nnconv returns it, is FH x FW x FC x 1."""
    import torch
    nn, mat, _ = gpu
    w, m, g = muon._inputs((3, 3, 8, 1), 50)
    three = lambda a: torch.from_numpy(a.copy()).cuda().view(8, 3, 3).permute(2, 1, 0)               # noqa: E731
    want, got, one, two = muon._up(w, (3, 3, 8, 1)), three(w), {}, {}
    for _ in range(2):
        nn.solver_update_("muon", want, one, muon._up(g, (3, 3, 8, 1)), 1.0, 0.0, 0.1, muon.OPTS)
        nn.solver_update_("muon", got, two, muon._up(g, (3, 3, 8, 1)), 1.0, 0.0, 0.1, muon.OPTS)
    assert got.shape == (3, 3, 8) and two["t"] == 2 and (got == want[..., 0]).all() and (two["s1"] == one["s1"][..., 0]).all()
    with pytest.raises(ValueError, match="shape"):
        nn.solver_update_("muon", got, two, muon._up(g, (3, 3, 8, 1)).reshape(8, 3, 3, 1), 1.0, 0.0, 0.1, muon.OPTS)


def test_muon_steps_beyond_reason_are_refused(gpu):
    from matconvnet_b200 import capi
    nn, _, ctx = gpu
    w, _, g = muon._inputs((1, 1, 6, 8), 60)
    for steps in (2 ** 32 + 5, 2 ** 16):      # (32 bits of the first are 5)
        v, state = muon._up(w, (1, 1, 6, 8)), {}
        with pytest.raises(ValueError, match="steps"):
            nn.solver_update_("muon", v, state, muon._up(g, (1, 1, 6, 8)), 1.0, 0.0, 0.1, dict(muon.OPTS, steps=steps))
        assert (muon._down(v) == w).all() and not state
    v, s1, d = (muon._up(a, (1, 1, 6, 8)) for a in (w, w, g))
    u = capi.MuonParam(v.data_ptr(), s1.data_ptr(), d.data_ptr(), 8, 6, 0.0, 0.1)
    for steps in (2 ** 31 - 1, 2 ** 16):
        o = capi.MuonOpts(0.95, 1e-7, 3.4445, -4.7750, 2.0315, 1, steps)
        assert ctx.lib.vlb_muon_update_many(ctx.handle, 1, ctypes.byref(u), 1.0, ctypes.byref(o)) == 7
        ctx.lib.vlb_ctx_reset_error(ctx.handle)
        assert (muon._down(v) == w).all()


@pytest.mark.parametrize("n,d,k", [(4, 40, 50), (200, 136, 700)])
def test_fcloss_with_scales_of_data_and_filters_far_from_one(gpu, n, d, k):
    """As at 2^40 in test_gpu_fcloss.py: powers of two on one side and their inverses on the other change nothing but the derivatives' scale."""
    nn, mat, _ = gpu
    x, f, b, c = fcloss._inputs(n, (1, 1, d), k, 6)
    base = fcloss._check(nn, mat, x, f, b, c, (1, 1, d))
    for e in (-80, 80):
        s = np.float32(2.0 ** e)
        far = fcloss._check(nn, mat, x * s, f / s, b, c, (1, 1, d))
        for p, q in zip(base, far):
            assert (p[0] == q[0] * s).all() and (p[1] == q[1] / s).all() and (p[2] == q[2]).all()


@pytest.mark.parametrize("n,d,k", [(155, 441, 4385), (639, 274, 5051), (415, 187, 9123), (2949, 1523, 1968)])
def test_fcloss_whose_derivatives_have_fewer_tiles_than_there_are_places(gpu, n, d, k):
    """Some places have no tile of either derivative, and nothing to wait for.  (The images' derivative is a long sum and is cut; the tiles go to the places by what they take.)"""
    from matconvnet_b200 import capi
    nn, mat, _ = gpu
    ctx = capi.Context()
    fcloss._check(nn, mat, *fcloss._inputs(n, (1, 1, d), k, 70), (1, 1, d), ctx=ctx)
    assert ctx.device_status() == 0


def test_muon_whose_products_have_fewer_tiles_than_there_are_places(gpu):
    from matconvnet_b200 import capi
    ctx = capi.Context()
    muon._check(gpu[0], [(1, 1, 167, 18), (1, 1, 82, 249), (1, 1, 70, 5), (1, 1, 4, 42), (1, 1, 7, 460), (1, 1, 96, 3), (3, 3, 9, 187), (1, 1, 2, 15), (3, 3, 64, 563), (1, 1, 2674, 650),
                         (1, 1, 6, 50), (1, 1, 83, 52), (1, 1, 20, 1), (3, 3, 16, 6), (1, 1, 2, 1), (1, 1, 43, 142), (1, 1, 312, 3), (3, 3, 2, 4)], ctx=ctx, seed=71)
    assert ctx.device_status() == 0

"""The Muon solver against its formulas in 64 bits.

Tolerances.  The polynomial's derivative on the interval of singular values (0 to 1.2) is at most a = 3.44 and mostly about 1, so that five steps
carry an error of the first by at most 3.44^5 = 485, and that only along singular values which started that much smaller; the others by about 1.
A step's products are off by 2^-22 per factor and by the roundings of sums of n products, about 2^-24 * sqrt(n) / 3 of |A||X|: 5e-7 for n up to
4096.  Measured in the 2-norm of the orthogonalised matrix, five such errors and their growth stay below 2e-5 unless most singular values are
tiny.  With operands of 11 bits (plain TF32) 2^-12 replaces 5e-7: 2e-2.  The momentum, momentum*M + (gradMult*G + decay*W), takes three
products and two sums, each rounded by at most 2^-24 of magnitudes that the sum of the three terms' magnitudes bounds, and the factors themselves are
rounded to single precision, 2^-24 of their terms: together at most 6 * 2^-24 of that sum, under 2^-21 of it (and not of the result: terms can cancel).
"""
import numpy as np
import pytest

TOL, TOL_TF32 = 2e-5, 2e-2
OPTS = dict(momentum=0.9, nesterov=True, steps=5, a=3.4445, b=-4.7750, c=2.0315, epsilon=1e-7)

SHAPES = [(1, 1, 1, 1), (1, 1, 5, 1), (1, 1, 1, 6), (1, 1, 3, 4), (3, 3, 3, 64), (3, 3, 64, 64), (1, 1, 129, 1000), (1, 1, 1000, 129), (5, 5, 7, 130), (1, 1, 256, 256),
          (1, 1, 65, 2000), (3, 3, 57, 300), (1, 1, 513, 640), (1, 1, 700, 1100), (1, 1, 1300, 1090), (1, 1, 128, 2048), (1, 1, 2048, 128), (1, 1, 128, 2049), (1, 1, 2000, 64)]


def _inputs(shape, seed=0):
    rng = np.random.default_rng(seed)
    k, n = shape[3], int(np.prod(shape[:3]))
    rank = max(1, min(k, n) // 4)
    g = rng.standard_normal((k, rank)) @ rng.standard_normal((rank, n)) * 1e-2 + rng.standard_normal((k, n)) * 1e-2
    return [a.astype(np.float32) for a in (rng.standard_normal((k, n)) * 0.05, rng.standard_normal((k, n)) * 1e-2, g)]


def _orthogonalise(u, o):
    x = u / (np.linalg.norm(u) + o["epsilon"])
    flip = x.shape[0] > x.shape[1]
    x = x.T if flip else x
    for _ in range(o["steps"]):
        p = x @ x.T
        x = o["a"] * x + (o["b"] * p + o["c"] * p @ p) @ x
    return x.T if flip else x


def _oracle(w, m, g, gm, decay, lr, o):
    w, m, g = (a.astype(np.float64) for a in (w, m, g))
    d = gm * g + decay * w
    m = o["momentum"] * m + d
    x = _orthogonalise(d + o["momentum"] * m if o["nesterov"] else m, o)
    return x, m, w - lr * np.sqrt(max(1.0, w.shape[0] / w.shape[1])) * x


def _up(a, shape):
    import torch
    return torch.from_numpy(a.copy()).cuda().view(shape[3], shape[2], shape[1], shape[0]).permute(3, 2, 1, 0)


def _down(t):
    return t.permute(3, 2, 1, 0).reshape(t.shape[3], -1).cpu().numpy().astype(np.float64)


def _rel(a, r):
    return np.linalg.norm(a - r) / max(np.linalg.norm(r), 1e-30)


def _check(nn, shapes, o=OPTS, tol=TOL, ctx=None, seed=0):
    """From W = 0 without decay the step is the orthogonalised matrix itself; and a step as it is in training."""
    for zero in (True, False):
        items, want = [], []
        for i, shape in enumerate(shapes):
            w, m, g = _inputs(shape, seed + i)
            decay = 0.0 if zero else 1e-3
            w = w * 0 if zero else w
            lr = 1.0 if zero else 0.02 * (i + 1)
            terms = o["momentum"] * np.abs(m.astype(np.float64)) + 0.5 * np.abs(g) + decay * np.abs(w)
            want.append(_oracle(w, m, g, 0.5, decay, lr, o) + (terms,))
            items.append((_up(w, shape), {"s1": _up(m, shape), "t": 2}, _up(g, shape), decay, lr))
        nn.solver_update_many_("muon", items, 0.5, o, ctx=ctx)
        for (w, state, _, _, lr), (x, m, ref, terms), shape in zip(items, want, shapes):
            scale = lr * np.sqrt(max(1.0, shape[3] / np.prod(shape[:3])))
            assert state["t"] == 3
            assert (np.abs(_down(state["s1"]) - m) <= 2 ** -21 * terms).all()
            # W itself is rounded once more, by 2^-24 of its elements
            assert np.linalg.norm(_down(w) - ref) <= tol * scale * np.linalg.norm(x) + 2 ** -23 * np.linalg.norm(ref), shape


def test_the_update_is_near_the_orthogonal_factor():
    """The oracle itself: singular values of a well-conditioned matrix end near 1 (the published coefficients leave them between 0.6 and 1.3)."""
    rng = np.random.default_rng(0)
    s = np.linalg.svd(_orthogonalise(rng.standard_normal((30, 60)), OPTS), compute_uv=False)
    assert 0.6 < s.min() and s.max() < 1.3


def test_refusals_that_need_no_gpu():
    import torch
    from matconvnet_b200 import nn
    w = torch.zeros(1, 1, 4, 4)
    with pytest.raises(TypeError):
        nn.solver_update_many_("muon", [(w, {}, w, 0.0, 0.1)], 1.0)
    with pytest.raises(ValueError):
        nn.solver_update_many_("muons", [], 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES)
def test_one_bank(gpu, shape):
    _check(gpu[0], [shape])


@pytest.mark.gpu
def test_many_banks_at_once(gpu):
    _check(gpu[0], SHAPES + [(3, 3, 64, 64)] * 7)


@pytest.mark.gpu
@pytest.mark.parametrize("change", [dict(nesterov=False), dict(steps=0), dict(steps=1), dict(steps=3, a=1.5, b=-0.5, c=0.0), dict(momentum=0.0), dict(epsilon=1.0)])
@pytest.mark.parametrize("shape", [(1, 1, 40, 30), (1, 1, 300, 520)])
def test_options(gpu, change, shape):
    _check(gpu[0], [shape], dict(OPTS, **change))


@pytest.mark.gpu
@pytest.mark.parametrize("precision,tol", [("FP32", TOL), ("TF32", TOL_TF32)])
def test_the_other_arithmetics(gpu, precision, tol):
    from matconvnet_b200 import capi
    _check(gpu[0], [(3, 3, 64, 64), (1, 1, 300, 520), (1, 1, 520, 300)], tol=tol, ctx=capi.Context(precision=getattr(capi, "PRECISION_" + precision)))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 1, 40, 30), (1, 1, 300, 520)])
def test_gradients_of_any_size(gpu, shape):
    """The matrix is normalised: a power of two on gradient and momentum leaves the step as it is, as far as epsilon allows."""
    nn = gpu[0]
    _, m, g = _inputs(shape, 3)
    o = dict(OPTS, epsilon=0.0)
    steps = []
    for e in (0, 60, -60):
        s = np.float32(2.0 ** e)
        w = _up(m * 0, shape)
        nn.solver_update_("muon", w, {"s1": _up(m * s, shape), "t": 1}, _up(g * s, shape), 1.0, 0.0, 1.0, o)
        steps.append(_down(w))
    assert (steps[0] == steps[1]).all() and (steps[0] == steps[2]).all()
    # nothing to orthogonalise: nothing happens
    w = _up(m, shape)
    nn.solver_update_("muon", w, {}, _up(g * 0, shape), 1.0, 0.0, 1.0, OPTS)
    assert (_down(w) == m).all()


@pytest.mark.gpu
def test_banks_that_go_through_all_steps_in_one_launch_take_any_number_of_neighbours(gpu):
    _check(gpu[0], [(3, 3, 3, 64), (1, 1, 128, 100), (1, 1, 5, 900), (1, 1, 2000, 33), (1, 1, 1, 1)] * 4)


@pytest.mark.gpu
def test_a_wait_that_runs_out(gpu):
    """Nothing is loaded, so no wait is ever answered: the kernels give up, say so and leave everything as the next call needs it."""
    from matconvnet_b200 import capi
    nn = gpu[0]
    for shape in ((1, 1, 40, 30), (1, 1, 300, 520), (1, 1, 1300, 1090)):
        ctx = capi.Context()
        data = _inputs(shape, 6)

        def call():
            w, m, g = (_up(a, shape) for a in data)
            nn.solver_update_("muon", w, {"s1": m, "t": 1}, g, 1.0, 0.0, 0.1, OPTS, ctx=ctx)
            return _down(w)

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
        assert (call() == want).all() and ctx.device_status() == 0


@pytest.mark.gpu
def test_a_not_a_number_stays_in_its_bank(gpu):
    nn = gpu[0]
    shapes = [(1, 1, 40, 30), (1, 1, 300, 520), (1, 1, 30, 40)]
    items, ref = [], []
    for i, s in enumerate(shapes):
        w, m, g = _inputs(s, i)
        ref.append(_oracle(w, m, g, 1.0, 0.0, 0.1, OPTS)[2])
        if i == 1:
            g[0, 0] = np.nan
        items.append((_up(w, s), {"s1": _up(m, s), "t": 1}, _up(g, s), 0.0, 0.1))
    nn.solver_update_many_("muon", items, 1.0, OPTS)
    assert np.isnan(_down(items[1][0])).all()
    for i in (0, 2):
        assert _rel(_down(items[i][0]), ref[i]) < TOL


@pytest.mark.gpu
def test_weights_that_two_items_share_take_both_steps(gpu):
    nn = gpu[0]
    for shape in ((1, 1, 40, 30), (1, 1, 300, 520)):
        w0, m, g = _inputs(shape, 4)
        g2 = _inputs(shape, 5)[2]
        w, s1, s2 = _up(w0, shape), {"s1": _up(m, shape), "t": 1}, {"s1": _up(m, shape), "t": 1}
        nn.solver_update_many_("muon", [(w, s1, _up(g, shape), 0.1, 0.1), (w, s2, _up(g2, shape), 0.1, 0.1)], 1.0, OPTS)
        v, t1, t2 = _up(w0, shape), {"s1": _up(m, shape), "t": 1}, {"s1": _up(m, shape), "t": 1}
        nn.solver_update_("muon", v, t1, _up(g, shape), 1.0, 0.1, 0.1, OPTS)
        nn.solver_update_("muon", v, t2, _up(g2, shape), 1.0, 0.1, 0.1, OPTS)
        assert (_down(w) == _down(v)).all() and (_down(s2["s1"]) == _down(t2["s1"])).all()


@pytest.mark.gpu
def test_a_new_state_that_two_items_share_takes_both_steps(gpu):
    nn = gpu[0]
    shape = (1, 1, 40, 30)
    w0, _, g = _inputs(shape, 4)
    g2 = _inputs(shape, 5)[2]
    w, state, v, one = _up(w0, shape), {}, _up(w0, shape), {}
    nn.solver_update_many_("muon", [(w, state, _up(g, shape), 0.1, 0.1), (w, state, _up(g2, shape), 0.1, 0.1)], 1.0, OPTS)
    for d in (g, g2):
        nn.solver_update_("muon", v, one, _up(d, shape), 1.0, 0.1, 0.1, OPTS)
    assert state["t"] == 2 and (_down(w) == _down(v)).all() and (_down(state["s1"]) == _down(one["s1"])).all()
    with pytest.raises(ValueError):
        other = {}
        nn.solver_update_many_("muon", [(w, other, _up(g, shape), 0.1, 0.1), (w.reshape(1, 1, 30, 40), other, _up(g, shape).reshape(1, 1, 30, 40), 0.1, 0.1)], 1.0, OPTS)


@pytest.mark.gpu
def test_in_a_graph_and_from_an_empty_state(gpu):
    import torch
    nn = gpu[0]
    shapes = [(3, 3, 16, 40), (1, 1, 300, 260)]
    data = [_inputs(s, i) for i, s in enumerate(shapes)]
    make = lambda: [(_up(w, s), {"s1": _up(m, s), "t": 1}, _up(g, s), 1e-3, 0.02) for (w, m, g), s in zip(data, shapes)]      # noqa: E731
    want = make()
    for _ in range(3):
        nn.solver_update_many_("muon", want, 1.0, OPTS)
    torch.cuda.synchronize()
    got = make()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        nn.solver_update_many_("muon", got, 1.0, OPTS)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for p, q in zip(got, want):
        assert (p[0] == q[0]).all() and (p[1]["s1"] == q[1]["s1"]).all()
    state = {}
    w, m, g = data[0]
    nn.solver_update_("muon", _up(w, shapes[0]), state, _up(g, shapes[0]), 1.0, 0.0, 0.1)
    assert state["t"] == 1 and (_down(state["s1"]) == g.astype(np.float64)).all()


@pytest.mark.gpu
def test_refusals(gpu):
    import torch
    nn, mat, _ = gpu
    w, m, g = (_up(a, (1, 1, 6, 8)) for a in _inputs((1, 1, 6, 8)))
    state = {"s1": m, "t": 1}
    before = w.clone()
    for bad, kind in (((w.cpu(), state, g, 0.0, 0.1), TypeError), ((w, state, g.half(), 0.0, 0.1), TypeError),
                      ((w, state, g[:, :, :5], 0.0, 0.1), ValueError), ((w, state, g.reshape(1, 1, 8, 6), 0.0, 0.1), ValueError),
                      ((w.contiguous(), state, g, 0.0, 0.1), ValueError), ((w, {"s1": m.reshape(1, 1, 8, 6), "t": 1}, g, 0.0, 0.1), ValueError),
                      ((w[:, :, :, :0], {}, g[:, :, :, :0], 0.0, 0.1), RuntimeError)):
        with pytest.raises(kind):
            nn.solver_update_many_("muon", [(w, state, g, 0.0, 0.1), bad], 1.0)
    for opts in (dict(steps=-1), dict(epsilon=-1.0), dict(epsilon=float("nan"))):
        with pytest.raises(ValueError):
            nn.solver_update_("muon", w, state, g, 1.0, 0.0, 0.1, opts)
    assert (w == before).all() and state["t"] == 1
    nn.solver_update_many_("muon", [], 1.0)
    assert torch.cuda.is_available()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", [(2**31 - 1, 1), (1, 2**31 - 1)])
def test_sizes_that_counters_do_not_hold_are_refused(gpu, rows, cols):
    import ctypes
    from matconvnet_b200 import capi
    ctx = gpu[2]
    u = capi.MuonParam(256, 256, 256, rows, cols, 0.0, 0.1)              # refused before anything is looked at
    o = capi.MuonOpts(0.95, 1e-7, 3.4445, -4.7750, 2.0315, 1, 5)
    assert ctx.lib.vlb_muon_update_many(ctx.handle, 1, ctypes.byref(u), 1.0, ctypes.byref(o)) == 7
    ctx.lib.vlb_ctx_reset_error(ctx.handle)

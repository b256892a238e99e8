"""The operators of language models' training steps at the ends of what they take: long rows, dimensions beyond 32 bits, scratch that grows or is not to be had,
waits that run out, contexts of another device."""
import numpy as np
import pytest

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

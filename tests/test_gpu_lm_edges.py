"""The operators of language models' training steps at the ends of what they take: long rows, dimensions beyond 32 bits, scratch that grows or is not to be had,
waits that run out, contexts of another device."""
import numpy as np
import pytest

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

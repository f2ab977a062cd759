"""Layer norm where a row's infinity comes first, last or between, and with an epsilon that swallows every variance: the
definition's results, the same from each of its kernels."""
import numpy as np
import pytest

import sequence_reference as ref
from parity import assert_bits_equal

pytestmark = pytest.mark.gpu

COLS = [1, 3, 8, 33, 200, 700, 1500, 3000, 7000, 10000, 20000, 50000, 70000]


def data(seed, *shape):
    return np.random.default_rng(seed).standard_normal(shape).astype(np.float32)


@pytest.mark.parametrize("cols", COLS)
def test_mean_of_a_row_with_infinities(cols, gc):
    x, gamma, beta = data(1, 9, cols), data(2, cols), data(3, cols)
    clean = [t.toArray().copy() for t in gc.layerNorm(1, 1e-5).calculateOutput(*(gc.createRaw(list(a.shape), a) for a in (x, gamma, beta)))]
    means = {1: np.inf, 2: -np.inf, 3: np.inf, 4: -np.inf, 5: np.nan, 6: np.nan}
    x[1, 0], x[2, 0], x[3, cols // 2], x[4, cols - 1], x[6, 0] = np.inf, -np.inf, np.inf, -np.inf, np.nan
    x[5, 0] = np.inf
    if cols > 1:
        x[5, cols - 1] = -np.inf
    else:
        means[5] = np.inf
    got = [t.toArray() for t in gc.layerNorm(1, 1e-5).calculateOutput(*(gc.createRaw(list(a.shape), a) for a in (x, gamma, beta)))]
    for row, mean in means.items():
        assert got[1][row] == mean or (np.isnan(mean) and np.isnan(got[1][row])), (row, got[1][row], mean)
        assert np.isnan(got[2][row]) and np.isnan(got[0][row]).all(), row
    for row in (0, 7, 8):
        for a, b in zip(got, clean):
            assert_bits_equal(a[row:row + 1], b[row:row + 1], "the other rows")


@pytest.mark.parametrize("cols", COLS)
def test_infinite_epsilon(cols, gc):
    """1 / sqrt(var + inf) is 0: the result is beta, and nothing of the gradient but beta's is left."""
    x, gamma, beta, go = data(1, 5, cols), data(2, cols), data(3, cols), data(4, 5, cols)
    raw = [gc.createRaw(list(a.shape), a) for a in (x, gamma, beta, go)]
    norm = gc.layerNorm(1, np.inf)
    out, _, std = norm.calculateOutput(raw[0], raw[1], raw[2])
    assert (std.toArray() == 0).all()
    assert (out.toArray() == np.broadcast_to(beta, x.shape)).all()
    grad_in, grad_gamma, grad_beta = norm.calculateGrads(raw[0], raw[1], raw[3])
    assert (grad_in.toArray() == 0).all() and (grad_gamma.toArray() == 0).all()
    ref.assert_within(grad_beta.toArray(), ref.f64(go).sum(0), 3 * ref.U * np.abs(ref.f64(go)).sum(0), "grad of beta")

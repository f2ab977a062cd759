"""The weights' gradients of a layer norm at the top of the 32-bit element range, where single rows tell: the output's gradient
is zero but in a few rows, the first, the last and some between, and each of these must count once, in its own columns."""
import numpy as np
import pytest

import sequence_reference as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows, cols", [(134217727, 16), (33554431, 63), (2097151, 1023), (524287, 4095), (262143, 8191), (32767, 65535), (2147, 1000003)],
                         ids=lambda v: str(v))
def test_every_row_counts_once(rows, cols, gc):
    rng = np.random.default_rng(cols)
    weight = np.zeros((rows, 1), np.float32)
    some = np.unique(np.concatenate([[0, 1, rows // 2, (1 << 30) // cols, rows - 2, rows - 1], rng.integers(0, rows, 40)]))
    weight[some, 0] = rng.integers(1, 9, some.size)
    # multiples of 1/64 whose sums are exact in a float, so that every row has the same normalised values
    shift = (rng.integers(-32, 33, (rows, 1)) / 8).astype(np.float32)
    c = (rng.integers(-256, 257, cols) / 64).astype(np.float32)
    c[:2] = 4, -4
    x = gc.createRaw([rows, 1], shift).plus(gc.createRaw([cols], c))
    go = gc.createRaw([rows, 1], weight).plus(gc.createRawFill([cols], 0.0))
    _, grad_gamma, grad_beta = gc.layerNorm(1, 0.0).calculateGrads(x, None, go, False, True, True)
    total = float(weight.sum(dtype=np.float64))
    assert (grad_beta.toArray() == total).all(), "whole numbers, exact in any order"
    c64 = c.astype(np.float64)
    xh = (c64 - c64.mean()) / c64.std()
    # the bound of ref.layer_norm_grad_bounds for such rows: terms of two roundings in double, in pieces rounded to float
    # once; the statistics are sums of cols doubles of d = x - x[0], which is at most 8
    e_std = (3 * cols + 8) * ref.W * 64 / c64.var()
    e_mean = 2 * cols * ref.W * 8 + 4 * ref.W * 8
    bound = total * (np.abs(xh) * (6 * ref.U + 2 * e_std) + e_mean / c64.std()) + 1e-44
    ref.assert_within(grad_gamma.toArray(), total * xh, bound, "gradient of gamma")

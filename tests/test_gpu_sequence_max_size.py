"""The layers over sequences at the top of the 32-bit element range, each kernel family once. Rows (channels) do not depend on
one another, so the last ones have to come out as in a call on them alone; x[i, j] = r[i] + c[j] is built on the device."""
import numpy as np
import pytest

from kten_amd.host_mirror.shape_functions import ALL
from parity import assert_bits_equal

pytestmark = pytest.mark.gpu

MAX = 2 ** 31 - 1


def outer_sum(ops, rows, cols, seed):
    rng = np.random.default_rng(seed)
    return ops.createRaw([rows, 1], rng.standard_normal((rows, 1)).astype(np.float32)).plus(
        ops.createRaw([cols], rng.standard_normal(cols).astype(np.float32)))


def last(raw, rows):
    return raw.get([(raw.shape[0] - rows, raw.shape[0] - 1)] + [ALL] * (raw.dimensions - 1))


@pytest.mark.parametrize("rows, cols", [(134217727, 16), (2097151, 1023), (524287, 4095), (32767, 65535)])
def test_layer_norm(rows, cols, gc):
    x, gamma, beta = outer_sum(gc, rows, cols, 1), gc.createRaw([cols], np.full(cols, 0.5, np.float32)), gc.createRaw([cols], np.arange(cols, dtype=np.float32))
    few = last(x, 3)
    norm = gc.layerNorm(1, 1e-5)
    out = norm.calculateOutput(x, gamma, beta)[0]
    assert_bits_equal(last(out, 3).toArray(), norm.calculateOutput(few, gamma, beta)[0].toArray(), "the last rows")
    grad_in, grad_gamma, grad_beta = norm.calculateGrads(x, gamma, out)
    some = norm.calculateGrads(few, gamma, last(out, 3), True, False, False)[0].toArray()
    # another number of rows may take another split of a row: its f64 sums (of terms up to cols) are off by cols roundings each,
    # and the float result by one
    got = last(grad_in, 3).toArray()
    assert (np.abs(got - some) <= 2.0 ** -23 * np.abs(some) + 16 * cols ** 2 * 2.0 ** -53).all()
    # the gradient of beta is the sum of the output's rows: two roundings here, one there, of at most rows * cols
    assert (np.abs(grad_beta.toArray() - out.sum(0).toArray()) <= 2.0 ** -22 * rows * cols).all()
    assert np.isfinite(grad_gamma.toArray()).all()


def test_layer_norm_of_one_row(gc):
    x = gc.createRawFill([1, MAX], 1.0)
    x.set([(0, 0), (MAX - 2, MAX - 1)], gc.createRaw([1, 2], np.array([[3.0, -1.0]], np.float32)))     # mean 1, variance 8 / MAX
    out, mean, std = gc.layerNorm(1, 0.0).calculateOutput(x)
    want = np.sqrt(MAX / 8.0)
    assert mean.toArray()[0] == 1.0 and abs(std.toArray()[0] / want - 1) < 1e-6
    tail = out.get([(0, 0), (MAX - 4, MAX - 1)]).toArray().reshape(-1)
    assert np.allclose(tail, [0, 0, 2 * want, -2 * want], rtol=1e-6, atol=0)


def test_dropout(gc):
    x = gc.createRawFill([MAX], 1.0)
    out = gc.dropout(0.25, 99, 7).calculateOutput(x, x)
    first = (MAX // 4 - 1000) * 4                     # from here on with the counter that belongs there
    tail = out.get([(first, MAX - 1)]).toArray()
    one = gc.createRawFill([MAX - first], 1.0)
    assert_bits_equal(tail, gc.dropout(0.25, 99, 7 + first // 4).calculateOutput(one, one).toArray(), "the last values")
    assert abs(float(out.mean().toArray()[0]) - 2.0) < 1e-3


@pytest.mark.parametrize("outer, steps, inner", [(4194303, 2, 255), (32767, 1023, 64), (60000, 1100, 32), (2097151, 1023, 1), (1000000, 700, 3)],
                         ids=["walk", "tiles", "tiles in turn", "narrow", "narrow rows of three"])
def test_recurrence(outer, steps, inner, gc):
    x = outer_sum(gc, outer, steps * inner, 3).reshape([outer, steps, inner])
    few = last(x, 4)
    op = gc.gatedRecurrence(1)
    out, final = op.calculateOutput(x, x)
    few_out, few_final = op.calculateOutput(few, few)
    assert_bits_equal(last(out, 4).toArray(), few_out.toArray(), "states of the last rows")
    assert_bits_equal(last(final, 4).toArray(), few_final.toArray(), "last states of the last rows")
    gate, into, _ = op.calculateGrads(x, x, None, out, x, None, True, True, False)
    few_gate, few_into, _ = op.calculateGrads(few, few, None, few_out, few, None, True, True, False)
    assert_bits_equal(last(gate, 4).toArray(), few_gate.toArray(), "gradient of the gate")
    assert_bits_equal(last(into, 4).toArray(), few_into.toArray(), "gradient of the input")


@pytest.mark.parametrize("steps, inner", [(8388607, 256), (MAX, 1)], ids=["tiles", "narrow"])
def test_one_sequence(steps, inner, gc):
    """With a decay of 0.5 the states of the last steps do not feel what was before the last few hundred."""
    gate = gc.createRawFill([steps, inner], 0.5)
    x = gc.createRawFill([steps, inner], 1.0)
    tail = np.random.default_rng(5).standard_normal((6000, inner)).astype(np.float32)
    x.set([(steps - 6000, steps - 1), (0, inner - 1)], gc.createRaw([6000, inner], tail))
    op = gc.gatedRecurrence(0, False)
    out, final = op.calculateOutput(gate, x)
    got = out.get([(steps - 6001, steps - 1), (0, inner - 1)]).toArray()
    want, h = np.empty((6000, inner)), np.full(inner, 2.0)
    for t in range(6000):
        h = 0.5 * h + tail[t]
        want[t] = h
    assert (got[0] == 2.0).all()
    # a rounding to float of states that tiles hand on to 2^-41 of themselves
    assert (np.abs(got[1:] - want) <= 2.0 ** -24 * np.abs(want) + 2.0 ** -38 * 16).all()
    assert_bits_equal(final.toArray().reshape(-1), got[-1], "the last state")
    # backwards the gradient is 2 - 0.5^(steps - 1 - t) for an output gradient of ones
    gc.release(x)
    ones = gc.createRawFill([steps, inner], 1.0)
    into, start = op.calculateGrads(gate, gate, None, out, ones, None, False, True, True)[1:]
    ends = into.get([(steps - 3, steps - 1), (0, inner - 1)]).toArray()
    assert (ends == np.array([[1.75], [1.5], [1.0]])).all()
    assert (into.get([(0, 2), (0, inner - 1)]).toArray() == 2.0).all() and (start.toArray() == 1.0).all()

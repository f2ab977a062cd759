"""What a gated recurrence's backward pass does not read need not be there, in the Python wrapper as in the entry point."""
import numpy as np
import pytest

import sequence_reference as ref
from kten_amd import abi
from parity import assert_bits_equal

pytestmark = pytest.mark.gpu


def data(seed, *shape):
    return np.random.default_rng(seed).standard_normal(shape).astype(np.float32)


@pytest.mark.parametrize("shape", [(2, 3, 5), (2, 300, 70), (1, 5000, 3)], ids=lambda s: "x".join(map(str, s)))
def test_gradients_without_what_they_do_not_read(shape, gc):
    n, t, c = shape
    gate, x, go, state = data(1, *shape) * np.float32(0.4), data(2, *shape), data(3, *shape), data(4, n, c)
    raw = [gc.createRaw(list(a.shape), a) for a in (gate, x, go, state)]
    for sigmoid in (False, True):
        op = gc.gatedRecurrence(1, sigmoid)
        out = op.calculateOutput(raw[0], raw[1], raw[3])[0]
        whole = [g.toArray() for g in op.calculateGrads(raw[0], raw[1], raw[3], out, raw[2], raw[3])]
        if not sigmoid:                                # a given gate's gradient needs no input
            got = op.calculateGrads(raw[0], None, raw[3], out, raw[2], raw[3])
            for a, b in zip(got, whole):
                assert_bits_equal(a.toArray(), b, "without the input")
        got = op.calculateGrads(raw[0], None, None, None, raw[2], raw[3], False, True, True)
        assert got[0] is None
        for a, b in zip(got[1:], whole[1:]):
            assert_bits_equal(a.toArray(), b, "without input, output and first state")
            assert a.shape == list(b.shape)
    op = gc.gatedRecurrence(1, True)
    with pytest.raises(ValueError):
        op.calculateGrads(raw[0], None, raw[3], out, raw[2])         # a sigmoid gate's does
    with pytest.raises(ValueError):
        gc.gatedRecurrence(1, False).calculateGrads(raw[0], raw[1], raw[3], None, raw[2])


def test_a_given_gate_keeps_no_input_for_its_backward_pass(hip):
    gate, x, state = hip.create([2, 40, 6], True, data(1, 2, 40, 6)), hip.create([2, 40, 6], True, data(2, 2, 40, 6)), hip.create([2, 6], True, data(3, 2, 6))
    f = (x * 2.0).gatedRecurrence(1, gate, state, sigmoidGate=False)
    f.forward()
    assert [None if r is None else r.shape for r in f.saved] == [[2, 40, 6], None, [2, 6], [2, 40, 6]]
    weights = data(4, 2, 40, 6)
    (f * hip.create([2, 40, 6], False, weights)).sum().backward()
    g64, x64, s64 = (ref.f64(t.getRawValue().toArray()) for t in (gate, x, state))
    h = ref.recurrence(g64, 2 * x64, s64, False)[0]
    want = ref.recurrence_grads(g64, 2 * x64, s64, h, weights, None, False)
    for leaf, w, factor in ((gate, want[0], 1.0), (x, want[1], 2.0), (state, want[2], 1.0)):
        got = leaf.grad().toArray()
        # the states and the gradient that comes in are floats: a few half steps of the largest result each
        assert np.abs(got - factor * w).max() <= 64 * ref.U * np.abs(factor * w).max()

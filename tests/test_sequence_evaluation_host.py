"""Dropout outside training takes and refuses the operands that it takes and refuses in training (CPU)."""
import numpy as np
import pytest

import sequence_reference as ref
from kten_amd.host_mirror.autograd import CounterGenerator


@pytest.mark.parametrize("training", [True, False])
@pytest.mark.parametrize("shape", [[3], [1, 3], [2, 1], [2, 3, 1], [6]], ids=str)
def test_residual_of_another_shape(shape, training):
    """One that would broadcast too: the result has the input's shape, in training and outside."""
    ops = ref.SequenceOracleOperations()
    x, residual = ops.create([2, 3], True, np.ones((2, 3), np.float32)), ops.create(shape, False, np.ones(shape, np.float32))
    generator = CounterGenerator(1)
    with pytest.raises(ValueError, match="residual"):
        x.dropout(0.1, generator, training=training, residual=residual)
    assert generator.offset == 0


def test_residual_of_the_same_shape():
    ops = ref.SequenceOracleOperations()
    x, residual = (ops.create([2, 3], True, np.full((2, 3), v, np.float32)) for v in (1, 2))
    out = x.dropout(0.9, CounterGenerator(1), training=False, residual=residual)
    assert np.array_equal(out.toArray(), np.full((2, 3), 3, np.float32))
    out.sum().backward()
    for leaf in (x, residual):
        assert np.array_equal(leaf.grad().toArray(), np.ones((2, 3), np.float32))

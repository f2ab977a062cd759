"""The layers over sequences on the CPU: the definitions the device is held to (the generator's published answers, the
gradients against differences), the autograd functions above them, and what the host refuses before a device is asked."""
import ctypes

import numpy as np
import pytest

import sequence_reference as ref
from kten_amd.host_mirror.autograd import CounterGenerator


@pytest.fixture()
def ops():
    return ref.SequenceOracleOperations()


def data(seed, *shape):
    return np.random.default_rng(seed).standard_normal(shape).astype(np.float32)


def test_generator_gives_the_published_words():
    """The three known answers its authors publish with it (counter, key -> words)."""
    for low, high, key, words in [(0, 0, 0, (0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8)),
                                  (2 ** 64 - 1, 2 ** 64 - 1, 2 ** 64 - 1, (0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd)),
                                  (0x85a308d3243f6a88, 0x0370734413198a2e, 0x299f31d0a4093822, (0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1))]:
        assert tuple(int(w) for w in ref.random_words(key, np.array([low], dtype=np.uint64), high)[0]) == words


def test_share_of_kept_values():
    for p in (0.0, 0.1, 0.5, 0.9):
        n = 1 << 18
        share = ref.kept(n, p, 1234, 77).mean()
        assert abs(share - (1 - p)) <= 5 * np.sqrt(p * (1 - p) / n) + 2.0 ** -32      # five standard deviations
    assert not ref.kept(100, 1.0, 1, 2).any()


def differences(f, arrays, step=1e-5):
    """Central differences of the scalar f(*arrays) in float64."""
    grads = []
    for k, a in enumerate(arrays):
        if a is None:
            grads.append(None)
            continue
        g = np.zeros(a.size)
        for i in range(a.size):
            v = []
            for s in (step, -step):
                b = a.copy().reshape(-1); b[i] += s
                v.append(f(*[b.reshape(a.shape) if j == k else c for j, c in enumerate(arrays)]))
            g[i] = (v[0] - v[1]) / (2 * step)
        grads.append(g.reshape(a.shape))
    return grads


@pytest.mark.parametrize("affine", [True, False])
def test_layer_norm_gradients_against_differences(affine):
    x, go = ref.f64(data(1, 3, 5)), ref.f64(data(2, 3, 5))
    gamma, beta = (ref.f64(data(3, 5)), ref.f64(data(4, 5))) if affine else (None, None)
    want = differences(lambda x, g, b: (ref.layer_norm(x, g, b, 1e-2)[0] * go).sum(), [x, gamma, beta])
    got = ref.layer_norm_grads(x, gamma, go, 1e-2)
    for g, w in zip(got, want):
        if w is not None:
            assert np.allclose(g, w, atol=1e-7)


@pytest.mark.parametrize("sigmoid", [True, False])
@pytest.mark.parametrize("with_initial", [True, False])
def test_recurrence_gradients_against_differences(sigmoid, with_initial):
    gate, x, go = (ref.f64(data(s, 2, 6, 3)) for s in (5, 6, 7))
    gf = ref.f64(data(8, 2, 3))
    initial = ref.f64(data(9, 2, 3)) if with_initial else None

    def loss(gate, x, initial):
        h, final = ref.recurrence(gate, x, initial, sigmoid)
        return (h * go).sum() + (final * gf).sum()

    want = differences(loss, [gate, x, initial])
    got = ref.recurrence_grads(gate, x, initial, ref.recurrence(gate, x, initial, sigmoid)[0], go, gf, sigmoid)
    for g, w in zip(got, want):
        if w is not None:
            assert np.allclose(g, w, atol=1e-7)


# ---------------------------------------------------------------- the autograd functions

def block(ops, arrays, p=0.25, training=True, generator=None):
    """x + dropout(recurrence(layer norm(x))): the residual block, and its leaves."""
    x, gamma, beta, gate, initial = (ops.create(list(a.shape), True, a) for a in arrays)
    generator = generator or CounterGenerator(99, 7)
    h = x.layerNorm(-1, 1e-3, gamma, beta).gatedRecurrence(1, gate, initial)
    return h.dropout(p, generator, training, residual=x), [x, gamma, beta, gate, initial], h


def block64(arrays, weights, p=0.25):
    x, gamma, beta, gate, initial = (ref.f64(a) for a in arrays)
    n, t, c = x.shape
    y = ref.layer_norm(x.reshape(-1, c), gamma, beta, 1e-3)[0].reshape(x.shape)
    h, _ = ref.recurrence(gate, y, initial, True)
    keep = ref.kept(x.size, p, 99, 7).reshape(x.shape)
    return ((x + keep * h / (1 - p)) * ref.f64(weights)).sum()


def test_block_gradients_against_differences(ops):
    arrays = [data(1, 2, 4, 3), data(2, 3), data(3, 3), data(4, 2, 4, 3), data(5, 2, 3)]
    weights = data(6, 2, 4, 3)
    out, leaves, _ = block(ops, arrays)
    loss = (out * ops.create([2, 4, 3], False, weights)).sum()
    loss.backward()
    want = differences(lambda *a: block64(a, weights), [ref.f64(a) for a in arrays], 1e-4)
    assert abs(loss.item() - block64(arrays, weights)) < 1e-4
    for leaf, w in zip(leaves, want):
        # floats between the operators: a few 2^-24 of values of order 10
        assert np.allclose(leaf.grad().toArray(), w, atol=2e-5), (leaf.grad().toArray(), w)


def test_operand_in_two_places_gets_both_gradients(ops):
    x = ops.create([2, 5], True, data(1, 2, 5))
    f = x * 2.0                                     # a function, which hears of its uses
    (f.dropout(0.5, CounterGenerator(3), residual=f)).sum().backward()
    keep = ref.kept(10, 0.5, 3, 0).reshape(2, 5)
    assert np.allclose(x.grad().toArray(), 2.0 * (1 + 2 * keep))
    y = ops.create([2, 5], True, data(2, 2, 5))
    (y * 1.0).gatedRecurrence(1, y * 1.0, sigmoidGate=False).sum().backward()
    z = ops.create([2, 5], True, data(2, 2, 5))
    f = z * 1.0
    f.gatedRecurrence(1, f, sigmoidGate=False).sum().backward()
    assert np.allclose(z.grad().toArray(), y.grad().toArray(), atol=1e-6)


def test_generator_is_advanced_by_what_a_layer_takes(ops):
    g = CounterGenerator(5, 2 ** 64 - 2)
    x = ops.create([9], False, np.ones(9, np.float32))
    first = x.dropout(0.5, g)
    assert g.offset == 1                            # three counters from 2^64 - 2 on
    second = x.dropout(0.5, g)
    assert g.offset == 4
    for layer, offset in ((first, 2 ** 64 - 2), (second, 1)):
        layer.forward()
        assert np.array_equal(layer.toArray() != 0, ref.kept(9, 0.5, 5, offset))
    g = CounterGenerator(5)
    assert x.dropout(0.5, g, training=False) is x and g.offset == 0
    assert np.array_equal(x.dropout(0.5, g, training=False, residual=x).toArray(), np.full(9, 2, np.float32))


def test_stretches_of_a_sequence_join_at_the_final_state(ops):
    gate, x = data(1, 2, 7, 3), data(2, 2, 7, 3)
    whole = ops.create([2, 7, 3], False, x).gatedRecurrence(1, ops.create([2, 7, 3], False, gate))
    a = ops.create([2, 4, 3], False, x[:, :4]).gatedRecurrence(1, ops.create([2, 4, 3], False, gate[:, :4]))
    b = ops.create([2, 3, 3], False, x[:, 4:]).gatedRecurrence(1, ops.create([2, 3, 3], False, gate[:, 4:]), a.finalState)
    assert np.allclose(np.concatenate([a.toArray(), b.toArray()], 1), whole.toArray(), atol=1e-6)


def test_shapes_the_layers_refuse(ops):
    x = ops.create([2, 4, 3], True, data(1, 2, 4, 3))
    other = ops.create([2, 4, 2], False, data(2, 2, 4, 2))
    with pytest.raises(ValueError, match="Gamma and beta"):
        x.layerNorm(-1, gamma=ops.create([4], True, data(3, 4)))
    with pytest.raises(ValueError, match="Gamma and beta"):
        x.layerNorm(1, beta=ops.create([3], True, data(3, 3)))
    with pytest.raises(ValueError):
        x.layerNorm(3)
    with pytest.raises(ValueError, match="residual"):
        x.dropout(0.1, CounterGenerator(1), residual=other)
    with pytest.raises(ValueError, match="same shape"):
        x.gatedRecurrence(1, other)
    with pytest.raises(ValueError, match="initial state"):
        x.gatedRecurrence(1, x, initial=ops.create([3], False, data(4, 3)))
    with pytest.raises(ValueError):
        x.gatedRecurrence(3, x)


class _Library:
    """Stands in for the device library: counts what would be launched."""
    def __init__(self): self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append(name)
            if name == "kth_alloc":
                args[1]._obj.value = len(self.calls)
            return 0
        return call


def test_operations_refuse_before_the_device_is_asked():
    from kten_amd.hip_raw_tensor import HipDropout, HipGatedRecurrence, HipLayerNorm, HipRawTensor, HipTensorOperations
    ops = HipTensorOperations.__new__(HipTensorOperations)
    ops.lib, ops.alive, ops._collector = _Library(), True, None
    x, row, rows = ops.createRaw([4, 6]), ops.createRaw([6]), ops.createRaw([4])
    ops.lib.calls.clear()
    norm, recur = ops.layerNorm(-1, 1e-5), ops.gatedRecurrence(1)
    assert isinstance(norm, HipLayerNorm) and isinstance(recur, HipGatedRecurrence)
    for f in (lambda: norm.calculateOutput(x, gamma=rows), lambda: norm.calculateOutput(x, beta=rows), lambda: norm.calculateGrads(x, rows, x),
              lambda: norm.calculateGrads(x, None, row), lambda: ops.layerNorm(2, 1e-5).calculateOutput(x),
              lambda: ops.dropout(0.5, 1).calculateOutput(x, row), lambda: ops.dropout(-0.1, 1), lambda: ops.dropout(1.5, 1),
              lambda: ops.dropout(float("nan"), 1), lambda: ops.dropout(0.5, -1), lambda: ops.dropout(0.5, 1, 1 << 64),
              lambda: recur.calculateOutput(x, row), lambda: recur.calculateOutput(x, x, row), lambda: recur.step(x, x, row),
              lambda: recur.calculateGrads(x, x, row, x, x), lambda: recur.calculateGrads(x, x, rows, row, x),
              lambda: recur.calculateGrads(x, x, rows, x, row), lambda: recur.calculateGrads(x, x, rows, x, x, row)):
        with pytest.raises(ValueError):
            f()
    assert norm.calculateGrads(x, None, x, False, False, False) == (None, None, None)
    assert recur.calculateGrads(x, x, None, x, x, None, False, False, False) == (None, None, None)
    assert not [c for c in ops.lib.calls if c != "kth_release"], ops.lib.calls
    rows.release()
    with pytest.raises(RuntimeError, match="released"):
        recur.calculateOutput(x, x, rows)

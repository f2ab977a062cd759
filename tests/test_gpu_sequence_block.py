"""The layers over sequences together, as a model uses them: x + dropout(recurrence(layer norm(x))) forward and backward
through the autograd layer on the device, against float64; and the same block fed one token at a time."""
import numpy as np
import pytest

import sequence_reference as ref
from kten_amd.host_mirror.autograd import CounterGenerator
from parity import assert_bits_equal

pytestmark = pytest.mark.gpu


def data(seed, *shape):
    return np.random.default_rng(seed).standard_normal(shape).astype(np.float32)


@pytest.mark.parametrize("shape", [(2, 9, 33), (4, 300, 64), (1, 5000, 130), (3, 257, 512)], ids=lambda s: "x".join(map(str, s)))
def test_block_forward_and_backward(shape, hip):
    n, t, c = shape
    p, eps, seed, offset = 0.1, 1e-5, 2024, 2 ** 32 - 3
    arrays = [data(1, *shape), data(2, c), data(3, c), data(4, *shape) + np.float32(1), data(5, n, c)]
    weights = data(6, *shape)
    x, gamma, beta, gate, initial = (hip.create(list(a.shape), True, a) for a in arrays)
    w = hip.create(list(shape), False, weights)
    generator = CounterGenerator(seed, offset)
    h = x.layerNorm(-1, eps, gamma, beta).gatedRecurrence(1, gate, initial)
    out = h.dropout(p, generator, residual=x)
    assert generator.offset == offset + (n * t * c + 3) // 4
    (out * w).sum().backward()

    x64, g64, b64, gate64, i64 = (ref.f64(a) for a in arrays)
    flat = x64.reshape(-1, c)
    y, mean, std = ref.layer_norm(flat, g64, b64, np.float32(eps))
    states, _ = ref.recurrence(gate64, y.reshape(shape), i64, True)
    keep = ref.kept(x64.size, p, seed, offset).reshape(shape) / (1.0 - p)
    go = ref.f64(weights)
    grad_gate, grad_y, grad_initial = ref.recurrence_grads(gate64, y.reshape(shape), i64, states, go * keep, None, True)
    grad_x, grad_gamma, grad_beta = ref.layer_norm_grads(flat, g64, grad_y.reshape(-1, c), np.float32(eps))
    want = {"x": go + grad_x.reshape(shape), "gamma": grad_gamma, "beta": grad_beta, "gate": grad_gate, "initial": grad_initial}
    # Floats between the operators: each hands on values that are off by a few 2^-24 of the largest (32 covers the chain of
    # three operators forward and three backward), and a weight's gradient sums rows of them.
    for name, leaf in zip(("x", "gamma", "beta", "gate", "initial"), (x, gamma, beta, gate, initial)):
        got = leaf.grad().toArray()
        scale = np.abs(want[name]).max() if name in ("x", "gate", "initial") else np.abs(grad_y).sum((0, 1)).max() * 4
        assert np.abs(got - want[name]).max() <= 64 * ref.U * scale, name


def test_block_one_token_at_a_time_gives_the_sequence(gc):
    n, t, c = 3, 20, 96
    x, gate, initial = data(1, n, t, c), data(2, n, t, c), data(3, n, c)
    norm, recur = gc.layerNorm(-1, 1e-5), gc.gatedRecurrence(1)
    whole_norm = norm.calculateOutput(gc.createRaw([n, t, c], x))[0]
    whole = recur.calculateOutput(gc.createRaw([n, t, c], gate), whole_norm, gc.createRaw([n, c], initial))[0].toArray()
    state = gc.createRaw([n, c], initial)
    bound = ref.recurrence_bound(gate, whole_norm.toArray(), initial, True)
    for i in range(t):
        y = norm.calculateOutput(gc.createRaw([n, 1, c], x[:, i]))[0]
        assert_bits_equal(y.toArray()[:, 0], whole_norm.toArray()[:, i], "a token's layer norm does not depend on its neighbours")
        h = recur.step(gc.createRaw([n, 1, c], gate[:, i]), y, state)
        ref.assert_within(h.toArray()[:, 0], whole[:, i], 3 * bound[:, i], f"token {i}")


def test_passes_add_up_with_numbers_of_their_own(hip):
    """Two backward passes over one graph shape add up in the leaves; the second draws other numbers."""
    x = hip.create([4, 50], True, data(1, 4, 50))
    generator = CounterGenerator(11)
    for _ in range(2):
        x.dropout(0.5, generator).sum().backward()
    keep = [ref.kept(200, 0.5, 11, o).reshape(4, 50) * np.float32(2) for o in (0, 50)]
    assert_bits_equal(x.grad().toArray(), keep[0] + keep[1], "both passes' gradients")


def test_final_state_starts_the_next_stretch(hip):
    gate, x = data(1, 2, 70, 33), data(2, 2, 70, 33)
    make = lambda a: hip.create(list(a.shape), False, a)
    whole = make(x).gatedRecurrence(1, make(gate)).toArray()
    first = make(x[:, :41]).gatedRecurrence(1, make(gate[:, :41]))
    second = make(x[:, 41:]).gatedRecurrence(1, make(gate[:, 41:]), first.finalState)
    got = np.concatenate([first.toArray(), second.toArray()], 1)
    ref.assert_within(got, whole, 3 * ref.recurrence_bound(gate, x, None, True), "two stretches")

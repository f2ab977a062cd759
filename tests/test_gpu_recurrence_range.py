"""Products of given gates that leave the range of a double and come back: the states are those of the definition, worked out
step by step in float64, whichever kernel takes the call. All gates and inputs are powers of two or small multiples, so every
product is exact and the results are compared as bits."""
import numpy as np
import pytest

import sequence_reference as ref
from parity import assert_bits_equal

pytestmark = pytest.mark.gpu


def segments(*pairs):
    """[(gate, steps), ...] one after another."""
    return np.concatenate([np.full(n, g, np.float64) for g, n in pairs])


# gates of a channel, the state it begins with, inputs by step
PATTERNS = [
    ("lost over a tile, then gates above one", segments((1, 256), (2.0 ** -8, 256), (16, 255)), 5.0, {}),
    ("the same off the tiles' borders", segments((1, 37), (2.0 ** -8, 300), (16, 255)), -5.0, {}),
    ("decayed and grown again", segments((2.0 ** -8, 100), (256, 100)), 5.0, {}),
    ("through the subnormal doubles", segments((1, 3), (2.0 ** -8, 130), (256, 130)), 5.0, {}),
    ("lost within a few steps", segments((1, 5), (2.0 ** -100, 12), (2.0 ** 100, 12)), 5.0, {}),
    ("grown past a float and back", segments((16, 256), (1.0 / 16, 256)), 2.0 ** -100, {}),
    ("gates below zero", segments((-2.0 ** -8, 301), (-16, 251)), 5.0, {}),
    ("an infinite state stays infinite", segments((1, 9), (2.0 ** -8, 700)), np.inf, {}),
    ("and keeps its sign through negative gates", segments((1, 9), (-2.0 ** -8, 333)), -np.inf, {}),
    ("a new state after the old one was lost", segments((2.0 ** -8, 400), (1, 1), (4, 50)), 5.0, {400: 3.0}),
    ("a closed gate between", segments((2.0 ** -8, 200), (0, 1), (16, 250)), 5.0, {200: 1.0}),
    ("nothing before a growth", segments((16, 400)), 0.0, {}),
    ("lost, then grown past a double", segments((2.0 ** -8, 256), (2.0 ** 8, 300)), 5.0, {}),
    ("lost and grown again by as much", segments((2.0 ** -10, 200), (2.0 ** 10, 200)), 5.0, {}),
    ("just lost and grown again", segments((2.0 ** -8, 140), (2.0 ** 8, 140)), 5.0, {}),
    ("grown past a double and back", segments((16, 300), (1.0 / 16, 300)), 5.0, {}),
    ("grown past a double, then a closed gate", segments((16, 300), (0, 1), (1, 50)), 5.0, {}),
    ("up and down and up", segments((2.0 ** 8, 100), (2.0 ** -8, 220), (2.0 ** 8, 230)), 1.0, {}),
    ("lost within a few steps, and a new state", segments((1, 2), (2.0 ** -120, 20), (2.0 ** 120, 19)), 5.0, {9: 1.0}),
]


def arrays(outer, steps, inner, late):
    """Channel i takes pattern i % len(PATTERNS); `late`: how many steps of gate 1 come before it."""
    gate, x, state = np.ones((outer * inner, steps)), np.zeros((outer * inner, steps)), np.zeros(outer * inner)
    for i in range(outer * inner):
        _, g, s, inputs = PATTERNS[i % len(PATTERNS)]
        g = g[:steps - late]
        gate[i, late:late + len(g)] = g
        state[i] = s
        for t, u in inputs.items():
            if late + t < steps:
                x[i, late + t] = u
    shape = lambda a: np.ascontiguousarray(a.reshape(outer, inner, steps).transpose(0, 2, 1)).astype(np.float32)
    return shape(gate), shape(x), state.reshape(outer, inner).astype(np.float32)


# tiles of 64 channels, the narrow kernel with rows that fit a workgroup and with tiles, the walk
SHAPES = [(1, 1024, 64, 0), (1, 1300, 65, 111), (1, 1300, 70, 156), (2, 6000, 64, 5000), (1, 7000, 64, 3950), (1, 900, 20, 0), (20, 1200, 1, 0),
          (20, 1200, 2, 5), (7, 5000, 3, 3500), (20, 9000, 1, 7000), (20, 9000, 1, 3900), (1, 32, 64, 0), (2, 8, 20, 0)]


def names(outer, inner):
    return [PATTERNS[i % len(PATTERNS)][0] for i in range(outer * inner)]


def compare(got, want, outer, inner, what):
    with np.errstate(over="ignore"):
        want = want.astype(np.float32)
    bad = ~((got == want) | (np.isnan(got) & np.isnan(want)))
    if bad.any():
        o, t, c = (int(v[0]) for v in np.nonzero(bad))
        raise AssertionError(f"{what}, {names(outer, inner)[o * inner + c]!r}: step {t}: got {got[o, t, c]!r}, want {want[o, t, c]!r}")


@pytest.mark.parametrize("outer, steps, inner, late", SHAPES, ids=lambda v: str(v))
def test_forward(outer, steps, inner, late, gc):
    gate, x, state = arrays(outer, steps, inner, late)
    with np.errstate(over="ignore", invalid="ignore"):
        want = ref.recurrence(gate, x, state, False)[0]
    out, final = gc.gatedRecurrence(1, False).calculateOutput(*(gc.createRaw(list(a.shape), a) for a in (gate, x, state)))
    got = out.toArray()
    compare(got, want, outer, inner, "states")
    assert_bits_equal(final.toArray().reshape(outer, inner), got[:, -1], "last states")


@pytest.mark.parametrize("outer, steps, inner, late", SHAPES, ids=lambda v: str(v))
def test_backward(outer, steps, inner, late, gc):
    """The same towards the first step: gradients that only the end of the sequence gives."""
    gate, x, state = arrays(outer, steps, inner, late)
    gate, x = np.ascontiguousarray(gate[:, ::-1]), np.ascontiguousarray(x[:, ::-1])
    zero = np.zeros_like(gate)
    with np.errstate(over="ignore", invalid="ignore"):
        _, into, start = ref.recurrence_grads(gate, zero, None, zero, x, state, False)
    raw = [gc.createRaw(list(a.shape), a) for a in (gate, zero, x, state)]
    got = gc.gatedRecurrence(1, False).calculateGrads(raw[0], raw[1], None, raw[1], raw[2], raw[3], False, True, True)
    compare(got[1].toArray(), into, outer, inner, "gradient of the input")
    compare(got[2].toArray().reshape(outer, 1, inner), start[:, None], outer, inner, "gradient of the first state")


@pytest.mark.parametrize("outer, steps, inner", [(1, 2000, 70), (1, 9000, 2), (13, 3000, 1)], ids=lambda v: str(v))
def test_sigmoid_gates_that_forget(outer, steps, inner, gc):
    """Long strong decay of logits, then open gates: finite states are lost, infinite ones are not."""
    gate = np.full((outer, steps, inner), 40.0, np.float32)
    gate[:, 100:900] = -30.0
    zero = np.zeros_like(gate)
    for value in (3.0, np.inf):
        state = np.full((outer, inner), value, np.float32)
        out, _ = gc.gatedRecurrence(1).calculateOutput(*(gc.createRaw(list(a.shape), a) for a in (gate, zero, state)))
        want = ref.recurrence(gate, zero, state, True)[0]
        bound = ref.recurrence_bound(gate, zero, state, True) if np.isfinite(value) else np.zeros_like(want)
        got = out.toArray()
        if np.isfinite(value):
            ref.assert_within(got, want, bound, "states")
        else:
            assert (got == np.inf).all()


@pytest.mark.parametrize("outer, steps, inner", [(8, 60, 64), (64, 250, 1024), (3, 600, 65), (1, 5000, 64), (40, 100, 20), (500, 200, 1), (2, 9000, 3)], ids=lambda v: str(v))
def test_state_in_place_where_several_waves_read_it(outer, steps, inner, gc):
    """The last step's state is written over the first while the waves of the sequence's first tile may still be at work."""
    rng = np.random.default_rng(steps)
    gate, x = (gc.createRaw([outer, steps, inner], rng.standard_normal((outer, steps, inner)).astype(np.float32)) for _ in range(2))
    state = gc.createRaw([outer, inner], rng.standard_normal((outer, inner)).astype(np.float32))
    apart = state.copy()
    op = gc.gatedRecurrence(1)
    for _ in range(10):
        out, apart = op.calculateOutput(gate, x, apart)
        assert_bits_equal(op.step(gate, x, state).toArray(), out.toArray(), "states")
        assert_bits_equal(state.toArray(), apart.toArray(), "the state in place")

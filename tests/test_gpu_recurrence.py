"""The gated linear recurrence on the device against its definition in float64, within bounds counted from the roundings
(sequence_reference.py): one step to long sequences, channels from one to many, axes in any place, gates near both ends,
absent operands, single steps that go on from a state, and refusals."""
import numpy as np
import pytest

import sequence_reference as ref
from kten_amd import abi
from parity import assert_bits_equal

pytestmark = pytest.mark.gpu


def data(seed, *shape):
    return np.random.default_rng(seed).standard_normal(shape).astype(np.float32)


def gates(seed, shape, sigmoid):
    """Logits around 2, or decays from a tenth to nearly one."""
    g = data(seed, *shape) * np.float32(1.5) + np.float32(2.0)
    return g if sigmoid else (1.0 / (1.0 + np.exp(-g))).astype(np.float32)


def check(ops, gate, x, initial, go, gf, sigmoid, requires=(True, True, True)):
    o, t, c = x.shape
    raw = [None if a is None else ops.createRaw(list(a.shape), a) for a in (gate, x, initial, go, gf)]
    op = ops.gatedRecurrence(1, sigmoid)
    out, final = op.calculateOutput(raw[0], raw[1], raw[2])
    want, bound = ref.recurrence(gate, x, initial, sigmoid)[0], ref.recurrence_bound(gate, x, initial, sigmoid)
    h = out.toArray()
    what = f"{'sigmoid' if sigmoid else 'given'} {x.shape}"
    ref.assert_within(h, want, bound, "states, " + what)
    assert_bits_equal(final.toArray().reshape(o, c), h[:, -1], "final state, " + what)
    if initial is None:
        requires = (requires[0], requires[1], requires[2])
    got = op.calculateGrads(raw[0], raw[1], raw[2], out, raw[3], raw[4], *requires)
    want = ref.recurrence_grads(gate, x, initial, h, go, gf, sigmoid)
    bound = ref.recurrence_grad_bounds(gate, x, initial, h, go, gf, sigmoid)
    for g, w, b, need, name in zip(got, want, bound, requires, ("gradGate", "gradIn", "gradInitial")):
        assert (g is not None) == need
        if need:
            ref.assert_within(g.toArray(), w, b, f"{name}, {what}")


def run(ops, shape, sigmoid, with_state=True, seed=0, requires=(True, True, True)):
    o, t, c = shape
    seed = seed + o * 7 + t * 3 + c
    check(ops, gates(seed, shape, sigmoid), data(seed + 1, *shape), data(seed + 2, o, c) if with_state else None, data(seed + 3, *shape),
          data(seed + 4, o, c) if with_state else None, sigmoid, requires)


SHAPES = [(1, 1, 1), (64, 1, 1024), (3, 1, 5), (1, 2, 1), (2, 3, 4), (1, 7, 64), (1, 8, 65), (3, 9, 63), (2, 15, 130), (1, 16, 256), (2, 17, 257), (4, 31, 100),
          (1, 32, 1), (5, 33, 2), (1, 63, 3), (2, 64, 17), (1, 65, 33), (7, 100, 12), (1, 127, 64), (2, 128, 128), (1, 129, 200), (3, 255, 70),
          (1, 256, 512), (1, 257, 1000), (2, 511, 63), (1, 512, 4), (1, 1000, 1), (8, 1023, 20), (2, 1025, 96), (1, 2048, 64), (1, 4096, 16), (1, 4099, 65),
          (2, 5000, 8), (1, 8191, 31), (1, 20000, 5), (1, 30011, 1), (3, 1999, 331), (300, 40, 3), (2000, 5, 1), (1, 3, 5000), (700, 2, 33)]


@pytest.mark.parametrize("sigmoid", [True, False], ids=["sigmoid", "given"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_forward_and_backward(shape, sigmoid, gc):
    run(gc, shape, sigmoid)


@pytest.mark.parametrize("sigmoid", [True, False], ids=["sigmoid", "given"])
@pytest.mark.parametrize("shape", [(4, 1, 40), (2, 50, 70), (1, 3000, 64), (1, 3000, 3)], ids=lambda s: "x".join(map(str, s)))
def test_absent_operands_and_results(shape, sigmoid, gc):
    run(gc, shape, sigmoid, with_state=False)
    for requires in ((True, False, False), (False, True, False), (False, False, True), (True, True, False), (False, True, True)):
        run(gc, shape, sigmoid, requires=requires)


@pytest.mark.parametrize("shape", [(1, 66000, 2), (1, 40000, 64), (2, 20001, 65)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("sigmoid", [True, False], ids=["sigmoid", "given"])
def test_long_sequences(shape, sigmoid, gc):
    run(gc, shape, sigmoid)


def test_gates_at_both_ends(gc):
    """Decays so near one that 1 - a is lost in a float, and gates that close or open altogether."""
    shape = (2, 3000, 70)
    x, go = data(1, *shape), data(2, *shape)
    state = data(3, 2, 70)
    for level in (12.0, 17.0, 30.0, 88.0, 110.0, np.inf, -12.0, -30.0, -88.0, -110.0, -np.inf):
        gate = np.full(shape, level, np.float32)
        check(gc, gate, x, state, go, state, True)
    mixed = np.where(data(4, *shape) > 0, np.float32(200), np.float32(-200))
    check(gc, mixed, x, state, go, state, True)
    for value in (0.0, 1.0, -1.0, -0.5, 1e-30):
        check(gc, np.full(shape, value, np.float32), x, state, go, state, False)


def test_growing_states(gc):
    """Gates above one are a user's own: the states overflow to infinity where the definition's do."""
    gate, x = np.full((1, 600, 65), 1.5, np.float32), np.ones((1, 600, 65), np.float32)
    out, final = gc.gatedRecurrence(1, False).calculateOutput(gc.createRaw([1, 600, 65], gate), gc.createRaw([1, 600, 65], x))
    with np.errstate(over="ignore"):
        want = ref.recurrence(gate, x, None, False)[0].astype(np.float32)
    got = out.toArray()
    assert np.isinf(got[0, -1]).all()
    assert np.allclose(got[np.isfinite(want)], want[np.isfinite(want)], rtol=1e-6) and (np.isinf(got) == np.isinf(want)).all()


@pytest.mark.parametrize("shape", [(2, 40, 70), (1, 4000, 70), (1, 4000, 3)], ids=lambda s: "x".join(map(str, s)))
def test_nan_stays_in_its_channel_and_after_its_step(shape, gc):
    gate, x, go = gates(1, shape, True), data(2, *shape), data(3, *shape)
    state = data(4, shape[0], shape[2])
    op = gc.gatedRecurrence(1)
    t = shape[1] // 2
    clean = op.calculateOutput(*(gc.createRaw(list(a.shape), a) for a in (gate, x, state)))[0].toArray()
    for which in (gate, x):
        keep = which[0, t, 1]
        which[0, t, 1] = np.nan
        raw = [gc.createRaw(list(a.shape), a) for a in (gate, x, state)]
        out = op.calculateOutput(*raw)[0]
        got = out.toArray()
        assert np.isnan(got[0, t:, 1]).all()
        got[0, t:, 1] = clean[0, t:, 1]
        assert_bits_equal(got, clean, "the other channels, and the steps before")
        which[0, t, 1] = keep
    gate[0, t, 1] = -np.inf                          # a closed gate forgets everything before it
    x[0, t - 1, 1] = np.nan
    got = op.calculateOutput(*(gc.createRaw(list(a.shape), a) for a in (gate, x, state)))[0].toArray()
    assert np.isnan(got[0, t - 1:, 1]).all()         # 0 x NaN: the formula's result


@pytest.mark.parametrize("shape", [(2, 8, 70), (1, 4000, 70), (1, 4000, 3)], ids=lambda s: "x".join(map(str, s)))
def test_infinite_gate_and_infinite_input(shape, gc):
    """An infinite gate leaves its channel infinite or NaN from its step on, an infinite input infinite while the decay lasts
    (0.5 here); steps before and other channels keep their bits."""
    gate, x, state = np.full(shape, 0.5, np.float32), data(2, *shape), data(4, shape[0], shape[2])
    op = gc.gatedRecurrence(1, False)
    t = shape[1] // 2
    clean = op.calculateOutput(*(gc.createRaw(list(a.shape), a) for a in (gate, x, state)))[0].toArray()
    for which in (gate, x):
        keep = which[0, t, 1]
        which[0, t, 1] = np.inf
        got = op.calculateOutput(*(gc.createRaw(list(a.shape), a) for a in (gate, x, state)))[0].toArray()
        if which is x:
            assert (got[0, t:, 1] == np.inf).all()
        else:
            assert np.isinf(got[0, t, 1]) and not np.isfinite(got[0, t:, 1]).any()
        got[0, t:, 1] = clean[0, t:, 1]
        assert_bits_equal(got, clean, "the other channels, and the steps before")
        which[0, t, 1] = keep
    # the same towards the first step for an infinite gradient
    zero = np.zeros(shape, np.float32)
    zero[0, t, 1] = np.inf
    grad = op.calculateGrads(*(gc.createRaw(list(a.shape), a) for a in (gate, x, state, clean, zero)))
    want = np.zeros(shape, np.float32)
    want[0, :t + 1, 1] = np.inf
    assert_bits_equal(grad[1].toArray(), want, "gradIn")
    want = np.zeros(state.shape, np.float32)
    want[0, 1] = np.inf
    assert_bits_equal(grad[2].toArray().reshape(state.shape), want, "gradInitial")


def test_axes(gc):
    full = data(1, 4, 5, 6, 7)
    gate, go = gates(2, full.shape, True), data(3, *full.shape)
    for axis in (0, 1, 2, 3, -1):
        a = axis % 4
        state_shape = [d for i, d in enumerate(full.shape) if i != a]
        initial = data(4, *state_shape)
        raw = {k: gc.createRaw(list(v.shape), v) for k, v in dict(gate=gate, x=full, initial=initial, go=go).items()}
        op = gc.gatedRecurrence(axis)
        out, final = op.calculateOutput(raw["gate"], raw["x"], raw["initial"])
        o, i = int(np.prod(full.shape[:a])), int(np.prod(full.shape[a + 1:]))
        view = lambda v: v.reshape(o, full.shape[a], i)
        s = initial.reshape(o, i)
        assert out.shape == list(full.shape) and final.shape == state_shape
        ref.assert_within(out.toArray(), ref.recurrence(view(gate), view(full), s, True)[0], ref.recurrence_bound(view(gate), view(full), s, True), "states")
        grads = op.calculateGrads(raw["gate"], raw["x"], raw["initial"], out, raw["go"])
        args = (view(gate), view(full), s, view(out.toArray()), view(go), None, True)
        for g, w, b in zip(grads, ref.recurrence_grads(*args), ref.recurrence_grad_bounds(*args)):
            ref.assert_within(g.toArray(), w, b, "gradient")
    flat = data(5, 50)
    out, final = gc.gatedRecurrence(0).calculateOutput(gc.createRaw([50], flat), gc.createRaw([50], flat))
    assert final.shape == [1] and final.toArray()[0] == out.toArray()[-1]


@pytest.mark.parametrize("sigmoid", [True, False], ids=["sigmoid", "given"])
@pytest.mark.parametrize("channels", [(3, 5), (64, 256)], ids=lambda s: "x".join(map(str, s)))
def test_single_steps_go_on_from_the_state(channels, sigmoid, gc):
    o, c = channels
    steps = 6
    gate, x, initial = gates(1, (o, steps, c), sigmoid), data(2, o, steps, c), data(3, o, c)
    op = gc.gatedRecurrence(1, sigmoid)
    state = gc.createRaw([o, c], initial)
    before = state.copy()
    whole = ref.recurrence(gate, x, initial, sigmoid)[0]
    bound = ref.recurrence_bound(gate, x, initial, sigmoid)
    for t in range(steps):
        out = op.step(gc.createRaw([o, 1, c], gate[:, t]), gc.createRaw([o, 1, c], x[:, t]), state)
        assert_bits_equal(out.toArray().reshape(o, c), state.toArray(), "the state is the step's result")
        # the state is rounded to float between the calls: u of it each time, which decays with it: 3 u of the magnitudes again
        ref.assert_within(out.toArray(), whole[:, t], 2 * bound[:, t], f"step {t}")
    assert_bits_equal(before.toArray(), initial, "a copy of the state made before the steps")


@pytest.mark.parametrize("shape", [(2, 3000, 65), (1, 20000, 3)], ids=lambda s: "x".join(map(str, s)))
def test_state_updated_in_place_over_many_steps(shape, gc):
    gate, x, initial = gates(1, shape, True), data(2, *shape), data(3, shape[0], shape[2])
    op = gc.gatedRecurrence(1)
    raw = [gc.createRaw(list(a.shape), a) for a in (gate, x, initial)]
    out, final = op.calculateOutput(*raw)
    again = op.step(*raw)
    assert_bits_equal(again.toArray(), out.toArray(), "states")
    assert_bits_equal(raw[2].toArray(), final.toArray(), "the state in place")


def test_put_off_operands_and_longer_stores(gc):
    shape = (2, 30, 40)
    x = data(1, *shape)
    gate = gc.createRawFill(list(shape), 0.5)
    state, long = gc.createRawFill([2, 40], 2.0), gc.createRawFill([2 * 30 * 40 + 9], 7.0)
    rx = gc.createRaw(list(shape), x)
    abi.check(gc.lib.kth_gated_recurrence_forward(gate.storeReference, rx.copy().storeReference, abi.shape_array(shape), 3, 1, abi.KTH_GATE_GIVEN,
                                                  state.storeReference, long.storeReference, state.storeReference))
    g, s = np.full(shape, 0.5, np.float32), np.full((2, 40), 2.0, np.float32)
    got = long.toArray()
    ref.assert_within(got[:2400], ref.recurrence(g, x, s, False)[0], ref.recurrence_bound(g, x, s, False), "states")
    assert (got[2400:] == 7.0).all()
    assert_bits_equal(state.toArray(), got[:2400].reshape(shape)[:, -1], "the state in place of a constant")


def test_the_same_call_gives_the_same_bits(gc):
    for shape in ((4, 3000, 64), (1, 30000, 16), (1, 9000, 600), (1, 50000, 1)):
        raw = [gc.createRaw(list(a.shape), a) for a in (gates(1, shape, True), data(2, *shape), data(3, shape[0], shape[2]), data(4, *shape))]
        op = gc.gatedRecurrence(1)
        first = None
        for _ in range(4):
            out, final = op.calculateOutput(raw[0], raw[1], raw[2])
            got = [t.toArray() for t in (out, final, *op.calculateGrads(raw[0], raw[1], raw[2], out, raw[3]))]
            first = first or got
            for a, b in zip(got, first):
                assert_bits_equal(a, b, "the same call again")


@pytest.mark.parametrize("sigmoid", [True, False], ids=["sigmoid", "given"])
@pytest.mark.parametrize("shape", [(20000, 33, 8), (9000, 60, 15), (70000, 11, 4), (3, 100000, 7), (40, 5000, 4), (257, 300, 31), (1, 200, 31), (5, 9, 1), (300000, 9, 1),
                                   (12, 40, 6), (2, 4097, 1), (1, 65536, 1)], ids=lambda s: "x".join(map(str, s)))
def test_every_kernel_at_its_borders(shape, sigmoid, gc):
    run(gc, shape, sigmoid)


def test_thousands_of_calls_in_a_row(gc):
    """Tiles hand states on through words that carry the call's number, of which there are 4095 before they start again;
    calls of other sizes, which need more words, come between."""
    small = [gc.createRaw(list(a.shape), a) for a in (gates(1, (1, 300, 65), True), data(2, 1, 300, 65))]
    narrow = [gc.createRaw(list(a.shape), a) for a in (gates(3, (1, 9000, 2), True), data(4, 1, 9000, 2))]
    large = [gc.createRaw(list(a.shape), a) for a in (gates(5, (2, 3000, 130), True), data(6, 2, 3000, 130))]
    op = gc.gatedRecurrence(1)
    want = {}
    for i in range(4300):
        for name, raw in (("small", small), ("narrow", narrow if i % 50 == 0 else None), ("large", large if i in (100, 4200) else None)):
            if raw is None:
                continue
            out, final = op.calculateOutput(*raw)
            if i < 3 or i % 500 == 0 or i in (100, 4200) or 4090 < i < 4100:
                got = out.toArray()
                want.setdefault(name, got)
                assert_bits_equal(got, want[name], f"call {i}, {name}")
            out.release(); final.release()


def test_two_threads_at_once(gc):
    """Calls from several threads follow one another: each gets its own results."""
    import threading
    made = []
    for k in range(2):
        shape = (2, 2000 + 500 * k, 65)
        raw = [gc.createRaw(list(a.shape), a) for a in (gates(k, shape, True), data(k + 5, *shape))]
        made.append((raw, gc.gatedRecurrence(1).calculateOutput(*raw)[0].toArray()))
    errors = []

    def work(k):
        raw, want = made[k]
        h = [t.storeReference for t in raw]
        out = outs[k]
        for _ in range(60):
            if gc.lib.kth_gated_recurrence_forward(h[0], h[1], abi.shape_array(raw[0].shape), 3, 1, 1, 0, out.storeReference, 0) != 0:
                errors.append(k)

    outs = [gc.createRaw(m[0][0].shape) for m in made]
    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads: t.start()
    for t in threads: t.join()
    assert not errors
    for k in range(2):
        assert_bits_equal(outs[k].toArray(), made[k][1], f"thread {k}")


def test_refusals(gc):
    g, x, state = gc.createRaw([2, 4, 3], data(1, 2, 4, 3)), gc.createRaw([2, 4, 3], data(2, 2, 4, 3)), gc.createRaw([2, 3], data(3, 2, 3))
    out, final, short = gc.createRawFill([2, 4, 3], 9.0), gc.createRawFill([2, 3], 9.0), gc.createRaw([5])
    grads = [gc.createRawFill([2, 4, 3], 9.0) for _ in range(2)] + [gc.createRawFill([2, 3], 9.0)]
    h = lambda t: 0 if t is None else t.storeReference
    shape = abi.shape_array([2, 4, 3])
    launches = gc.getMetrics()["launches"]

    def forward(a=g, b=x, s=shape, dims=3, axis=1, mode=1, i=state, o=out, f=final):
        return gc.lib.kth_gated_recurrence_forward(h(a), h(b), s, dims, axis, mode, h(i), h(o), h(f))

    def backward(a=g, b=x, s=shape, dims=3, axis=1, mode=1, i=state, o=out, go=x, gf=state, gg=grads[0], gi=grads[1], g0=grads[2]):
        return gc.lib.kth_gated_recurrence_backward(h(a), h(b), s, dims, axis, mode, h(i), h(o), h(go), h(gf), h(gg), h(gi), h(g0))

    A, S = abi.KTH_E_ARGUMENT, abi.KTH_E_SHAPE
    for got, want in [(forward(mode=2), A), (forward(mode=-1), A), (forward(axis=3), A), (forward(axis=-1), A), (forward(dims=0), A), (forward(dims=11), A),
                      (forward(s=None), A), (forward(s=abi.shape_array([2, 0, 3])), A), (forward(s=abi.shape_array([2048, 1024, 1024])), A),
                      (forward(a=None), A), (forward(b=None), A), (forward(o=None), A), (forward(a=short), S), (forward(b=short), S), (forward(i=short), S),
                      (forward(o=short), S), (forward(f=short), S), (forward(o=g), A), (forward(o=x), A), (forward(f=out), A),
                      (forward(o=state, i=state, s=abi.shape_array([2, 1, 3]), f=None), A), (forward(f=x), A),
                      (backward(mode=7), A), (backward(axis=4), A), (backward(a=None), A), (backward(go=None), A), (backward(o=None), A), (backward(b=None), A),
                      (backward(go=short), S), (backward(gf=short), S), (backward(i=short), S), (backward(o=short), S), (backward(gg=short), S),
                      (backward(gi=short), S), (backward(g0=short), S), (backward(gg=g), A), (backward(gi=x), A), (backward(gi=grads[0]), A),
                      (backward(g0=state), A), (backward(gg=out), A)]:
        assert got == want, (got, want, abi.last_error())
    dead = gc.createRaw([2, 4, 3]); handle = dead.storeReference; dead.release()
    assert gc.lib.kth_gated_recurrence_forward(handle, h(x), shape, 3, 1, 1, 0, h(out), 0) == abi.KTH_E_HANDLE
    assert backward(gg=None, gi=None, g0=None) == 0
    assert gc.getMetrics()["launches"] == launches, "a refused call launches nothing"
    assert (out.toArray() == 9.0).all() and (final.toArray() == 9.0).all()
    # what the gate's gradient needs is not needed without it
    assert backward(b=None, o=None, i=None, gg=None) == 0
    assert backward(b=None, mode=0) == 0

"""A recurrence whose tiles give up waiting for one another (a limit of no looks at all): every kernel ends, what lies behind the
first tile is NaN, the next blocking call says so once, and the call after that is right again."""
import ctypes

import numpy as np
import pytest

import sequence_reference as ref
from kten_amd import abi
from parity import assert_bits_equal

pytestmark = pytest.mark.gpu

LOOKS = 1 << 22


def data(seed, *shape):
    return np.random.default_rng(seed).standard_normal(shape).astype(np.float32)


@pytest.fixture()
def impatient(gc):
    """A function that sets the limit; the default is back afterwards, and nothing is left to report."""
    yield gc.lib.kth_recurrence_wait_limit
    abi.check(gc.lib.kth_recurrence_wait_limit(LOOKS))
    gc.lib.kth_sync()


# steps of a tile: tiles of 64 channels, and the narrow kernel's (inner 1 and 3)
CASES = [((1, 2000, 64), 256, 128), ((3, 700, 100), 256, 128), ((1, 5000, 65), 256, 128), ((1, 9000, 1), 4096, 4096), ((2, 4000, 3), 1360, 1360)]


@pytest.mark.parametrize("sigmoid", [True, False], ids=["sigmoid", "given"])
@pytest.mark.parametrize("shape, forward_steps, backward_steps", CASES, ids=lambda v: str(v))
def test_given_up(shape, forward_steps, backward_steps, sigmoid, gc, impatient):
    n, t, c = shape
    gate, x, state, go = data(1, *shape), data(2, *shape), data(3, n, c), data(4, *shape)
    if not sigmoid:
        gate = np.abs(gate) / (1 + np.abs(gate))
    raw = [gc.createRaw(list(a.shape), a) for a in (gate, x, state, go)]
    op = gc.gatedRecurrence(1, sigmoid)
    out, final = op.calculateOutput(*raw[:3])
    right = out.toArray()
    grads = [g.toArray() for g in op.calculateGrads(raw[0], raw[1], raw[2], out, raw[3])]

    abi.check(impatient(0))
    lost = op.calculateOutput(*raw[:3])[0]
    assert gc.lib.kth_sync() == abi.KTH_E_DEVICE and b"gave up waiting" in gc.lib.kth_last_error()
    assert gc.lib.kth_sync() == abi.KTH_OK, "reported once"
    got = lost.toArray()
    assert_bits_equal(got[:, :forward_steps], right[:, :forward_steps], "the first tile")
    assert np.isnan(got[:, forward_steps:]).all()
    _, lost, start = op.calculateGrads(raw[0], raw[1], raw[2], out, raw[3])
    with pytest.raises(RuntimeError, match="gave up waiting"):
        lost.toArray()
    got = lost.toArray()
    assert_bits_equal(got[:, t - backward_steps:], grads[1][:, t - backward_steps:], "the gradient of the last steps, the first tile backward")
    assert np.isnan(got[:, :t - backward_steps]).all() and np.isnan(start.toArray()).all()

    abi.check(impatient(LOOKS))
    out, again = op.calculateOutput(*raw[:3])
    assert_bits_equal(out.toArray(), right, "the call after that")
    for g, want in zip(op.calculateGrads(raw[0], raw[1], raw[2], out, raw[3]), grads):
        assert_bits_equal(g.toArray(), want, "and its gradients")


@pytest.mark.parametrize("shape, steps", [((1, 2000, 64), 256), ((1, 9000, 1), 4096)], ids=lambda v: str(v))
def test_given_up_by_tiles_whose_waves_take_turns(shape, steps, gc, impatient):
    gate, x = np.full(shape, 0.4, np.float32), data(2, *shape)
    for k in range(8):                               # up by 2^24 and down again
        gate[:, k::32], gate[:, k + 8::32] = 8.0, 0.125
    raw = [gc.createRaw(list(a.shape), a) for a in (gate, x)]
    right = gc.gatedRecurrence(1, False).calculateOutput(*raw)[0].toArray()
    abi.check(impatient(0))
    lost = gc.gatedRecurrence(1, False).calculateOutput(*raw)[0]
    assert gc.lib.kth_sync() == abi.KTH_E_DEVICE
    assert_bits_equal(lost.toArray()[:, :steps], right[:, :steps], "the first tile")
    assert np.isnan(lost.toArray()[:, steps:]).all()


def test_every_blocking_call_reports(gc, impatient):
    raw = [gc.createRaw([1, 600, 64], data(k, 1, 600, 64)) for k in (1, 2)]
    value, flag = ctypes.c_float(), ctypes.c_int()
    host = np.empty(64, np.float32)
    abi.check(impatient(0))
    for blocking in (lambda: gc.lib.kth_sync(), lambda: gc.lib.kth_read_scalar(raw[0].storeReference, 0, ctypes.byref(value)),
                     lambda: gc.lib.kth_contains_nan(raw[0].storeReference, 64, ctypes.byref(flag)),
                     lambda: gc.lib.kth_download(host.ctypes.data_as(ctypes.c_void_p), raw[0].storeReference, 0, 64)):
        gc.gatedRecurrence(1).calculateOutput(*raw)
        assert blocking() == abi.KTH_E_DEVICE and blocking() == abi.KTH_OK


def test_sequences_of_one_tile_wait_for_nobody(gc, impatient):
    abi.check(impatient(0))
    for shape in ((2, 256, 64), (64, 1, 128), (300, 64, 1)):
        gate, x = data(1, *shape), data(2, *shape)
        out = gc.gatedRecurrence(1).calculateOutput(*(gc.createRaw(list(a.shape), a) for a in (gate, x)))[0]
        ref.assert_within(out.toArray(), ref.recurrence(gate, x, None, True)[0], ref.recurrence_bound(gate, x, None, True), str(shape))


def test_a_mark_that_is_pending_does_not_disturb_who_need_not_wait_long(gc, impatient):
    """Calls behind one that gave up, before the host has asked: waits that end soon are not given up for it."""
    raw = [gc.createRaw([1, 1000, 64], data(k, 1, 1000, 64)) for k in (1, 2)]
    right = gc.gatedRecurrence(1).calculateOutput(*raw)[0].toArray()
    abi.check(impatient(0))
    gc.gatedRecurrence(1).calculateOutput(*raw)
    abi.check(impatient(LOOKS))
    out = gc.gatedRecurrence(1).calculateOutput(*raw)[0]
    assert gc.lib.kth_sync() == abi.KTH_E_DEVICE
    got = out.toArray()
    assert_bits_equal(got[:, :256], right[:, :256], "the first tile")
    assert ((got == right) | np.isnan(got)).all()

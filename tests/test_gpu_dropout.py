"""Dropout on the device against the published generator in numpy, bit for bit: which values are kept, their scale, the
residual, counters past 32 bits and round the end, sizes that are no multiple of four, and refusals."""
import ctypes

import numpy as np
import pytest

import sequence_reference as ref
from kten_amd import abi
from parity import assert_bits_equal

pytestmark = pytest.mark.gpu


def data(seed, *shape):
    return np.random.default_rng(seed).standard_normal(shape).astype(np.float32)


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 7, 8, 63, 1023, 1024, 2047, 2048, 2049, 2051, 4096, 100003, 1 << 20, (1 << 20) + 3])
def test_bits(n, residual, gc):
    x, y = data(n, n), data(n + 1, n) if residual else None
    op = gc.dropout(0.3, 0x123456789ABCDEF0 + n, 5 * n)
    got = op.calculateOutput(gc.createRaw([n], x), gc.createRaw([n], y) if residual else None)
    assert_bits_equal(got.toArray(), ref.dropout(x, 0.3, 0x123456789ABCDEF0 + n, 5 * n, y), f"dropout of {n}")


@pytest.mark.parametrize("p", [0.0, 2.0 ** -33, 1e-4, 0.1, 0.5, 0.75, 0.999999, 1.0 - 2.0 ** -53, 1.0])
def test_probabilities(p, gc):
    x = data(7, 30011)
    x[5], x[6], x[7], x[8] = np.nan, np.inf, -np.inf, 1e-45
    got = gc.dropout(p, 42, 9).calculateOutput(gc.createRaw([30011], x)).toArray()
    assert_bits_equal(got, ref.dropout(x, p, 42, 9), f"p = {p}")
    keep = ref.kept(30011, p, 42, 9)
    assert (got[~keep] == 0).all(), "what is dropped is zero, whatever it was"
    if p == 0.0:
        assert_bits_equal(got, x, "nothing dropped")


@pytest.mark.parametrize("seed,offset", [(0, 0), (2 ** 64 - 1, 2 ** 64 - 100), (2 ** 63, 2 ** 32 - 50), (1, 2 ** 32 - 1), (2 ** 32, 2 ** 63)])
def test_seeds_and_counters(seed, offset, gc):
    x = data(3, 4003)
    assert_bits_equal(gc.dropout(0.5, seed, offset).calculateOutput(gc.createRaw([4003], x)).toArray(), ref.dropout(x, 0.5, seed, offset), "counters")


def test_gradient_is_the_same_call(gc):
    go = data(1, 3, 1001)
    op = gc.dropout(0.2, 77, 3)
    assert_bits_equal(op.calculateGrad(gc.createRaw([3, 1001], go)).toArray(), ref.dropout(go, 0.2, 77, 3), "gradient")
    pieces = gc.dropout(0.2, 77, 3 + 250).calculateOutput(gc.createRaw([1, 2003], go.reshape(1, -1)[:, 1000:]))
    assert_bits_equal(pieces.toArray(), ref.dropout(go, 0.2, 77, 3).reshape(1, -1)[:, 1000:], "the rest of a tensor from its own counter")


def test_results_over_their_operands_and_put_off_values(gc):
    x, y = data(1, 5003), data(2, 5003)
    lib = gc.lib
    want = ref.dropout(x, 0.4, 5, 6, y)
    a, b = gc.createRaw([5003], x), gc.createRaw([5003], y)
    kept_a, kept_b = a.copy(), b.copy()
    abi.check(lib.kth_dropout(a.storeReference, 5003, 0.4, 5, 6, b.storeReference, a.storeReference))
    assert_bits_equal(a.toArray(), want, "over the input")
    assert_bits_equal(kept_a.toArray(), x, "a copy made before")
    abi.check(lib.kth_dropout(kept_a.storeReference, 5003, 0.4, 5, 6, b.storeReference, b.storeReference))
    assert_bits_equal(b.toArray(), want, "over the residual")
    assert_bits_equal(kept_b.toArray(), y, "a copy made before")
    # the same store as input and residual, a constant, and a result inside a longer store that is owed one
    abi.check(lib.kth_dropout(kept_a.storeReference, 5003, 0.4, 5, 6, kept_a.storeReference, a.storeReference))
    assert_bits_equal(a.toArray(), ref.dropout(x, 0.4, 5, 6, x), "its own residual")
    ones, long = gc.createRawFill([5003], 1.0), gc.createRawFill([6000], 8.0)
    abi.check(lib.kth_dropout(ones.storeReference, 5003, 0.4, 5, 6, 0, long.storeReference))
    assert_bits_equal(long.toArray()[:5003], ref.dropout(np.ones(5003, np.float32), 0.4, 5, 6), "a constant")
    assert (long.toArray()[5003:] == 8.0).all()
    same = gc.createRawFill([5003], 2.0)
    abi.check(lib.kth_dropout(same.storeReference, 5003, 0.4, 5, 6, 0, same.storeReference))
    assert_bits_equal(same.toArray(), ref.dropout(np.full(5003, 2, np.float32), 0.4, 5, 6), "a constant over itself")


def test_refusals(gc):
    a, b = gc.createRaw([16], data(1, 16)), gc.createRawFill([16], 3.0)
    launches = gc.getMetrics()["launches"]
    f = lambda i=a.storeReference, n=16, p=0.5, r=0, o=b.storeReference: gc.lib.kth_dropout(i, n, p, 1, 2, r, o)
    for p in (-1e-9, 1.0000001, float("nan"), float("inf")):
        assert f(p=p) == abi.KTH_E_ARGUMENT
    assert f(n=17) == abi.KTH_E_ARGUMENT and f(n=2 ** 63) == abi.KTH_E_ARGUMENT
    short = gc.createRaw([8])
    assert f(r=short.storeReference) == abi.KTH_E_ARGUMENT and f(o=short.storeReference) == abi.KTH_E_ARGUMENT
    for bad in (0, 2 ** 40):
        assert f(i=bad) == abi.KTH_E_HANDLE and f(o=bad) == abi.KTH_E_HANDLE
    assert f(r=2 ** 40) == abi.KTH_E_HANDLE
    assert f(n=0) == 0
    assert gc.getMetrics()["launches"] == launches
    assert (b.toArray() == 3.0).all()

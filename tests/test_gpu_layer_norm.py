"""Layer normalisation on the device against its definition in float64, within bounds counted from the roundings
(sequence_reference.py): every width a kernel is chosen by, rows from one to many, operands absent, values that are hard on
one-pass statistics, results over their inputs, and refusals."""
import numpy as np
import pytest

import sequence_reference as ref
from kten_amd import abi
from parity import assert_bits_equal

pytestmark = pytest.mark.gpu

EPS = 1e-5


def data(seed, *shape):
    return np.random.default_rng(seed).standard_normal(shape).astype(np.float32)


def check_forward(ops, x, gamma, beta, eps=EPS):
    rows, cols = x.shape
    raw = [None if a is None else ops.createRaw(list(a.shape), a) for a in (x, gamma, beta)]
    got = ops.layerNorm(1, eps).calculateOutput(*raw)
    want = ref.layer_norm(x, gamma, beta, np.float32(eps))
    for g, w, b, what in zip(got, want, ref.layer_norm_bounds(x, gamma, beta, np.float32(eps)), ("output", "currentMean", "currentStd")):
        ref.assert_within(g.toArray(), w, b, f"{what} of {x.shape}")


def check_backward(ops, x, gamma, go, eps=EPS, requires=(True, True, True)):
    raw = [None if a is None else ops.createRaw(list(a.shape), a) for a in (x, gamma, go)]
    got = ops.layerNorm(1, eps).calculateGrads(raw[0], raw[1], raw[2], *requires)
    want, bound = ref.layer_norm_grads(x, gamma, go, np.float32(eps)), ref.layer_norm_grad_bounds(x, gamma, go, np.float32(eps))
    for g, w, b, need, what in zip(got, want, bound, requires, ("gradIn", "gradGamma", "gradBeta")):
        assert (g is not None) == need
        if need:
            ref.assert_within(g.toArray(), w, b, f"{what} of {x.shape}")


# widths around every size at which another kernel or another number of registers takes over, odd ones, one column
SHAPES = [(1, 1), (5, 1), (3, 2), (7, 3), (300, 4), (1000, 5), (257, 8), (33, 17), (65, 31), (4097, 32), (9, 63), (100, 64), (101, 65), (50, 127),
          (64, 128), (1, 129), (40, 255), (41, 256), (42, 257), (37, 511), (19, 512), (23, 513), (11, 1000), (64, 1024), (13, 1025), (8, 2047),
          (7, 2048), (9, 2049), (5, 4095), (600, 4096), (3, 4097), (4, 6000), (2, 8191), (3, 8192), (2, 8193), (1, 12289), (3, 16383), (2, 16384),
          (2, 16385), (3, 20001), (2, 32768), (1, 40003), (2, 65536), (1, 100003), (5000, 768), (20000, 33), (1, 1 << 20), (2500, 300)]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{s[0]}x{s[1]}")
def test_forward_and_backward(shape, gc):
    rows, cols = shape
    seed = rows * 31 + cols
    x = data(seed, rows, cols) * np.float32(1.7) + np.float32(0.3)
    gamma, beta, go = data(seed + 1, cols), data(seed + 2, cols), data(seed + 3, rows, cols)
    check_forward(gc, x, gamma, beta)
    check_backward(gc, x, gamma, go)


@pytest.mark.parametrize("shape", [(70000, 16), (131073, 7), (40000, 130)], ids=lambda s: f"{s[0]}x{s[1]}")
def test_many_rows(shape, gc):
    x, go = data(1, *shape), data(2, *shape)
    gamma, beta = data(3, shape[1]), data(4, shape[1])
    check_forward(gc, x, gamma, beta)
    check_backward(gc, x, gamma, go)


@pytest.mark.parametrize("shape", [(64, 16385), (300, 20003), (65, 36864), (64, 36865), (63, 40000), (520, 17000), (64, 65536), (100, 65533), (64, 65537), (515, 33001)],
                         ids=lambda s: f"{s[0]}x{s[1]}")
def test_long_rows(shape, gc):
    x, go = data(1, *shape) + np.float32(0.5), data(2, *shape)
    gamma, beta = data(3, shape[1]), data(4, shape[1])
    check_forward(gc, x, gamma, beta)
    check_forward(gc, x, None, None)
    check_backward(gc, x, gamma, go)
    # the result over its input, with the statistics left out
    raw = [gc.createRaw(list(a.shape), a) for a in (x, gamma, beta)]
    want = gc.layerNorm(1, EPS).calculateOutput(*raw)[0].toArray()
    abi.check(gc.lib.kth_layer_norm_forward(raw[0].storeReference, abi.shape_array(shape), 2, 1, EPS, raw[1].storeReference, raw[2].storeReference,
                                            raw[0].storeReference, 0, 0))
    assert_bits_equal(raw[0].toArray(), want, "in place")


@pytest.mark.parametrize("shape", [(37, 60), (37, 300), (20, 1500), (10, 5000), (6, 20000)], ids=lambda s: f"{s[0]}x{s[1]}")
def test_absent_operands_and_results(shape, gc):
    x, go, gamma, beta = data(1, *shape), data(2, *shape), data(3, shape[1]), data(4, shape[1])
    for g, b in ((None, None), (gamma, None), (None, beta)):
        check_forward(gc, x, g, b)
    for requires in ((True, False, False), (False, True, False), (False, False, True), (True, True, False), (False, True, True)):
        check_backward(gc, x, gamma if requires[1] else None, go, requires=requires)
    # no statistics asked for
    rx, out = gc.createRaw(list(shape), x), gc.createRaw(list(shape))
    abi.check(gc.lib.kth_layer_norm_forward(rx.storeReference, abi.shape_array(shape), 2, 1, EPS, 0, 0, out.storeReference, 0, 0))
    assert_bits_equal(out.toArray(), gc.layerNorm(1, EPS).calculateOutput(rx)[0].toArray(), "output without statistics")


@pytest.mark.parametrize("cols", [24, 200, 900, 3000, 9000, 20000])
def test_values_that_are_hard_on_the_statistics(cols, gc):
    x = data(cols, 8, cols)
    x[0] += 1000.0                                   # a mean far from zero
    x[1, 0] = 1e5                                    # the first value, which the sums are taken around, far from the rest
    x[2] = 3.25                                      # no variance
    x[3] = 0.0
    x[4] *= np.float32(1e-20)                        # squares below the smallest float
    x[5] *= np.float32(1e18)                         # squares above the largest
    x[6, -1] = -1e6
    go, gamma, beta = data(cols + 1, 8, cols), data(cols + 2, cols), data(cols + 3, cols)
    check_forward(gc, x, gamma, beta)
    check_backward(gc, x, gamma, go)
    # without an epsilon the rows without variance give beta, and a gradient of zero
    check_forward(gc, x[2:4], gamma, beta, 0.0)
    grads = gc.layerNorm(1, 0.0).calculateGrads(*(gc.createRaw(list(a.shape), a) for a in (x[2:4], gamma, go[2:4])))
    assert not grads[0].toArray().any() and not grads[1].toArray().any()


@pytest.mark.parametrize("cols", [5, 24, 900, 9000, 20000])
def test_rows_of_subnormal_values_without_epsilon(cols, gc):
    """1 / sqrt(var) is beyond fp32's range there, the normalised values are not."""
    x = (np.random.default_rng(cols).integers(-200, 200, (3, cols)) * 2.0 ** -149).astype(np.float32)
    gamma, beta = data(cols + 2, cols), data(cols + 3, cols)
    out, mean, std = gc.layerNorm(1, 0.0).calculateOutput(*(gc.createRaw(list(a.shape), a) for a in (x, gamma, beta)))
    ref.assert_within(out.toArray(), ref.layer_norm(x, gamma, beta, 0.0)[0], ref.layer_norm_bounds(x, gamma, beta, 0.0)[0], "output")
    assert np.isinf(std.toArray()).all()


@pytest.mark.parametrize("cols", [24, 900, 9000, 20000])
def test_infinities_and_nan_stay_in_their_rows(cols, gc):
    x, go = data(cols, 6, cols), data(cols + 1, 6, cols)
    clean = gc.layerNorm(1, EPS).calculateOutput(gc.createRaw([6, cols], x))[0].toArray()
    clean_grad = gc.layerNorm(1, EPS).calculateGrads(gc.createRaw([6, cols], x), None, gc.createRaw([6, cols], go))[0].toArray()
    x[1, 3], x[4, cols - 1] = np.nan, np.inf
    go[2, 5] = np.nan
    out = gc.layerNorm(1, EPS).calculateOutput(gc.createRaw([6, cols], x))[0].toArray()
    assert np.isnan(out[1]).all() and np.isnan(out[4, -1])
    keep = [0, 2, 3, 5]
    assert_bits_equal(out[keep], clean[keep], "the other rows")
    grad = gc.layerNorm(1, EPS).calculateGrads(gc.createRaw([6, cols], x), None, gc.createRaw([6, cols], go))[0].toArray()
    assert np.isnan(grad[1]).all() and np.isnan(grad[2]).all()
    assert_bits_equal(grad[[0, 3, 5]], clean_grad[[0, 3, 5]], "the other rows' gradient")


def test_axes_and_trailing_dims(gc):
    x, go = data(1, 3, 4, 5, 6), data(2, 3, 4, 5, 6)
    for axis in (0, 1, 2, 3, -1, -3):
        a = axis % 4
        weights = x.shape[a:]
        gamma, beta = data(3, *weights), data(4, *weights)
        raw = {k: gc.createRaw(list(v.shape), v) for k, v in dict(x=x, go=go, gamma=gamma, beta=beta).items()}
        op = gc.layerNorm(axis, EPS)
        out, mean, std = op.calculateOutput(raw["x"], raw["gamma"], raw["beta"])
        cols = int(np.prod(weights))
        flat = x.reshape(-1, cols)
        assert out.shape == [3, 4, 5, 6] and mean.shape == (list(x.shape[:a]) or [1])
        ref.assert_within(out.toArray(), ref.layer_norm(flat, gamma.ravel(), beta.ravel(), np.float32(EPS))[0],
                          ref.layer_norm_bounds(flat, gamma.ravel(), beta.ravel(), np.float32(EPS))[0], "output")
        grads = op.calculateGrads(raw["x"], raw["gamma"], raw["go"])
        assert [g.shape for g in grads] == [[3, 4, 5, 6], list(weights), list(weights)]
        for g, w, b in zip(grads, ref.layer_norm_grads(flat, gamma.ravel(), go.reshape(-1, cols), np.float32(EPS)),
                           ref.layer_norm_grad_bounds(flat, gamma.ravel(), go.reshape(-1, cols), np.float32(EPS))):
            ref.assert_within(g.toArray(), w, b, "gradient")


@pytest.mark.parametrize("shape", [(50, 33), (50, 700), (20, 5000), (3, 30000)], ids=lambda s: f"{s[0]}x{s[1]}")
def test_results_over_their_inputs(shape, gc):
    x, go, gamma = data(1, *shape), data(2, *shape), data(3, shape[1])
    op = gc.layerNorm(1, EPS)
    rx, rgo, rga = (gc.createRaw(list(a.shape), a) for a in (x, go, gamma))
    want_out = op.calculateOutput(rx, rga)[0].toArray()
    want = [g.toArray() for g in op.calculateGrads(rx, rga, rgo)]
    weights = [gc.createRaw([shape[1]]) for _ in range(2)]
    abi.check(gc.lib.kth_layer_norm_backward(rx.storeReference, abi.shape_array(shape), 2, 1, EPS, rga.storeReference, rgo.storeReference,
                                             rgo.storeReference, weights[0].storeReference, weights[1].storeReference))
    for g, w in zip((rgo, *weights), want):
        assert_bits_equal(g.toArray(), w, "gradients, that of the input over that of the output")
    copy = rx.copy()                                 # put off until rx is written
    abi.check(gc.lib.kth_layer_norm_forward(rx.storeReference, abi.shape_array(shape), 2, 1, EPS, rga.storeReference, 0, rx.storeReference, 0, 0))
    assert_bits_equal(rx.toArray(), want_out, "output over its input")
    assert_bits_equal(copy.toArray(), x, "a copy of the input made before")


def test_constants_copies_and_sums_that_were_put_off(gc):
    x = data(1, 40, 64)
    gamma, beta = gc.createRawFill([64], 1.5), gc.createRawFill([64], -0.5)
    rx = gc.createRaw([40, 64], x)
    out = gc.layerNorm(1, EPS).calculateOutput(rx.copy(), gamma, beta)[0]
    g, b = np.full(64, 1.5, np.float32), np.full(64, -0.5, np.float32)
    ref.assert_within(out.toArray(), ref.layer_norm(x, g, b, np.float32(EPS))[0], ref.layer_norm_bounds(x, g, b, np.float32(EPS))[0], "constants")
    summed = gc.createRaw([40, 16, 64], data(2, 40, 16, 64))
    small = summed.sum(1)
    values = summed.sum(1).toArray()
    out = gc.layerNorm(1, EPS).calculateOutput(small)[0]
    ref.assert_within(out.toArray(), ref.layer_norm(values, None, None, np.float32(EPS))[0],
                      ref.layer_norm_bounds(values, None, None, np.float32(EPS))[0], "a sum that was put off")
    # a store longer than the result, owed a constant: what lies behind the result keeps it
    long = gc.createRawFill([41 * 64], 7.0)
    abi.check(gc.lib.kth_layer_norm_forward(rx.storeReference, abi.shape_array([40, 64]), 2, 1, EPS, 0, 0, long.storeReference, 0, 0))
    assert (long.toArray()[40 * 64:] == 7.0).all()
    # the gradient of a sum is one constant that was never written out
    ones = gc.createRawFill([40, 64], 1.0)
    check = gc.layerNorm(1, EPS).calculateGrads(rx, None, ones)
    want = ref.layer_norm_grads(x, None, np.ones((40, 64)), np.float32(EPS))
    for a, w, bound in zip(check, want, ref.layer_norm_grad_bounds(x, None, np.ones((40, 64)), np.float32(EPS))):
        ref.assert_within(a.toArray(), w, bound, "gradients of a sum")


def test_the_same_call_gives_the_same_bits(gc):
    for shape in ((3000, 100), (700, 4096), (5, 50000)):
        x, go, gamma = data(1, *shape), data(2, *shape), data(3, shape[1])
        raw = [gc.createRaw(list(a.shape), a) for a in (x, gamma, go)]
        first = [g.toArray() for g in gc.layerNorm(1, EPS).calculateGrads(*raw)]
        for _ in range(3):
            for a, b in zip(gc.layerNorm(1, EPS).calculateGrads(*raw), first):
                assert_bits_equal(a.toArray(), b, "gradients")


def test_refusals(gc):
    x, row, rows = gc.createRaw([4, 6], data(1, 4, 6)), gc.createRaw([6], data(2, 6)), gc.createRaw([4])
    out, short = gc.createRawFill([4, 6], 9.0), gc.createRaw([5])
    h = lambda t: 0 if t is None else t.storeReference
    shape = abi.shape_array([4, 6])
    launches = gc.getMetrics()["launches"]

    def forward(a=x, s=shape, dims=2, axis=1, eps=EPS, g=None, b=None, o=out, m=None, sd=None):
        return gc.lib.kth_layer_norm_forward(h(a), s, dims, axis, eps, h(g), h(b), h(o), h(m), h(sd))

    def backward(a=x, s=shape, dims=2, axis=1, eps=EPS, g=None, go=x, gi=out, gg=None, gb=None):
        return gc.lib.kth_layer_norm_backward(h(a), s, dims, axis, eps, h(g), h(go), h(gi), h(gg), h(gb))

    A, S = abi.KTH_E_ARGUMENT, abi.KTH_E_SHAPE
    for got, want in [(forward(eps=-1.0), A), (forward(eps=float("nan")), A), (forward(axis=2), A), (forward(axis=-1), A), (forward(dims=0), A),
                      (forward(dims=11), A), (forward(s=None), A), (forward(s=abi.shape_array([4, 0])), A), (forward(a=None), A), (forward(o=None), A),
                      (forward(s=abi.shape_array([65536, 65536])), A), (forward(s=abi.shape_array([5, 6])), S), (forward(o=short), S),
                      (forward(g=short), S), (forward(b=short), S), (forward(m=short, s=abi.shape_array([6, 4]), o=out), S), (forward(o=row, g=row, s=abi.shape_array([1, 6])), A),
                      (forward(m=rows, sd=rows), A), (forward(m=out), A), (forward(m=x), A), (backward(eps=-0.5), A), (backward(go=None), A), (backward(a=None), A),
                      (backward(gi=x), A), (backward(gg=row, gb=row), A), (backward(gg=row, g=row), A), (backward(gg=short), S), (backward(go=row), S),
                      (backward(gi=short), S), (backward(axis=5), A)]:
        assert got == want, (got, want, abi.last_error())
    dead = gc.createRaw([4, 6]); handle = dead.storeReference; dead.release()
    assert gc.lib.kth_layer_norm_forward(handle, shape, 2, 1, EPS, 0, 0, h(out), 0, 0) == abi.KTH_E_HANDLE
    assert backward(gi=None) == 0                   # nothing is asked for
    assert gc.getMetrics()["launches"] == launches, "a refused call launches nothing"
    assert (out.toArray() == 9.0).all()

"""Layer norm, dropout and the gated linear recurrence from their definitions in float64 (numpy), each with a bound on what
a correct float kernel may differ by: u = 2^-24 is half a step of a float, w = 2^-53 that of a double.

`SequenceOracleOperations` puts them behind the oracle's raw tensors, so that the autograd layer runs on the CPU."""
import numpy as np

from kten_amd.host_mirror import shape_functions as sf
from oracle.jvm_oracle import JvmOracleOperations

U, W = 2.0 ** -24, 2.0 ** -53
M32 = np.uint64(0xFFFFFFFF)


def f64(a):
    return None if a is None else np.asarray(a, dtype=np.float64)


# ---------------------------------------------------------------- layer norm of [rows, cols]

def layer_norm(x, gamma, beta, eps):
    """out, mean, std = 1 / sqrt(var + eps); a row without variance and without eps has std 0."""
    x = f64(x)
    mean = x.mean(1)
    s = ((x - mean[:, None]) ** 2).mean(1) + eps
    std = np.where(s == 0, 0.0, 1.0 / np.sqrt(np.where(s == 0, 1.0, s)))
    out = (x - mean[:, None]) * std[:, None]
    if gamma is not None:
        out = out * f64(gamma)
    if beta is not None:
        out = out + f64(beta)
    return out, mean, std


def _statistics_error(x, eps):
    """Relative error of std, absolute error of the mean, each before its rounding to float: sums of n doubles of
    d = x - x[0] and d^2 (each term and each addition is off by w of the running sum at most), and their difference."""
    x = f64(x)
    n = x.shape[1]
    d = x - x[:, :1]
    s = ((x - x.mean(1)[:, None]) ** 2).mean(1) + eps
    mean = 2 * n * W * np.abs(d).mean(1) + 4 * W * np.abs(x[:, 0])
    std = (3 * n + 8) * W * (d * d).mean(1) / np.where(s == 0, np.inf, s)
    return std, mean


def layer_norm_bounds(x, gamma, beta, eps):
    """(out, mean, std): (x - mean) rounded, times std rounded, times gamma, plus beta, each step rounded: 4 u of the
    product, u of the sum; and what the statistics are off."""
    out, mean, std = layer_norm(x, gamma, beta, eps)
    e_std, e_mean = _statistics_error(x, eps)
    g = np.ones(x.shape[1]) if gamma is None else np.abs(f64(gamma))
    xh = np.abs(f64(x) - mean[:, None]) * std[:, None]
    b_out = xh * g * (5 * U + 2 * e_std[:, None]) + g * (std * e_mean)[:, None] * 2 + 2 * U * np.abs(out)
    tiny = 1e-44                                     # a step of the smallest floats
    return b_out + tiny, 2 * U * np.abs(mean) + e_mean + tiny, std * (2 * U + 2 * e_std) + tiny


def layer_norm_grads(x, gamma, go, eps):
    x, go = f64(x), f64(go)
    n = x.shape[1]
    _, mean, std = layer_norm(x, None, None, eps)
    xh = (x - mean[:, None]) * std[:, None]
    w = go * f64(gamma) if gamma is not None else go
    grad_in = std[:, None] * (w - w.mean(1)[:, None] - xh * (w * xh).mean(1)[:, None])
    return grad_in, (go * xh).sum(0), go.sum(0)


def layer_norm_grad_bounds(x, gamma, go, eps):
    """grad_in: three terms, each off by a few roundings of itself and by what the statistics and the means of w and w xh
    (sums of n doubles) are off. The weights' gradients: terms of two roundings, summed in pieces rounded to float once."""
    x, go = f64(x), f64(go)
    n = x.shape[1]
    e_std, e_mean = _statistics_error(x, eps)
    _, mean, std = layer_norm(x, None, None, eps)
    xh = (x - mean[:, None]) * std[:, None]
    w = go * f64(gamma) if gamma is not None else go
    d = np.abs(x - x[:, :1])
    terms = np.abs(w) + np.abs(w.mean(1))[:, None] + np.abs(xh * (w * xh).mean(1)[:, None])
    # sum of w (x - mean) from sums over d: n w of sum |w| d, and as much of the correction by the mean
    dot = (3 * n + 8) * W * ((np.abs(w) * d).mean(1) + d.mean(1) * np.abs(w).mean(1)) * std
    off_mean = (std * e_mean)[:, None]
    means = 2 * n * W * np.abs(w).mean(1)[:, None] + np.abs(xh) * (dot[:, None] + off_mean * np.abs(w).mean(1)[:, None])
    b_in = std[:, None] * (6 * U * terms + 4 * e_std[:, None] * terms + means + off_mean * np.abs((w * xh).mean(1))[:, None])
    b_gamma = (np.abs(go) * (np.abs(xh) * (6 * U + 2 * e_std[:, None]) + off_mean)).sum(0)
    return b_in + 1e-44, b_gamma + 1e-44, 3 * U * np.abs(go).sum(0) + 1e-44


# ---------------------------------------------------------------- dropout

def random_words(seed, counters, high=None):
    """[n, 4] 32-bit words of the ten-round 4x32 generator of Salmon, Moraes, Dror and Shaw (2011) for 64-bit counters;
    `high`: the upper 64 bits of the counter (zero in the operator)."""
    c = np.asarray(counters, dtype=np.uint64)
    shift = np.uint64(32)
    w = [c & M32, c >> shift, np.zeros_like(c), np.zeros_like(c)]
    if high is not None:
        w[2], w[3] = np.full_like(c, np.uint64(high) & M32), np.full_like(c, np.uint64(high) >> shift)
    k = [np.uint64(seed & 0xFFFFFFFF), np.uint64(seed >> 32)]
    for _ in range(10):
        p0, p1 = w[0] * np.uint64(0xD2511F53), w[2] * np.uint64(0xCD9E8D57)
        w = [(p1 >> shift) ^ w[1] ^ k[0], p1 & M32, (p0 >> shift) ^ w[3] ^ k[1], p0 & M32]
        k = [(k[0] + np.uint64(0x9E3779B9)) & M32, (k[1] + np.uint64(0xBB67AE85)) & M32]
    return np.stack(w, -1)


def kept(n, p, seed, offset):
    if p == 1.0:
        return np.zeros(n, dtype=bool)
    with np.errstate(over="ignore"):
        counters = np.arange((n + 3) // 4, dtype=np.uint64) + np.uint64(offset)
    return random_words(seed, counters).reshape(-1)[:n] >= np.uint64(int(p * 2.0 ** 32))


def dropout(x, p, seed, offset, residual=None):
    """The bits of the result: one product and at most one sum, in float."""
    x = np.asarray(x, dtype=np.float32)
    scale = np.float32(0.0 if p == 1.0 else 1.0 / (1.0 - p))
    with np.errstate(invalid="ignore", over="ignore"):
        y = np.where(kept(x.size, p, seed, offset).reshape(x.shape), x * scale, np.float32(0.0)).astype(np.float32)
        return y if residual is None else np.asarray(residual, dtype=np.float32) + y


# ---------------------------------------------------------------- gated linear recurrence of [outer, steps, inner]

def coefficients(gate, x, sigmoid):
    """a, b = 1 - a (1 where the gate is given), u."""
    gate, x = f64(gate), f64(x)
    if not sigmoid:
        return gate, np.ones_like(gate), x
    with np.errstate(over="ignore"):
        e = np.exp(-np.abs(gate))
    near, far = 1.0 / (1.0 + e), e / (1.0 + e)
    a, b = np.where(gate >= 0, near, far), np.where(gate >= 0, far, near)
    return a, b, b * x


def scan(a, u, initial, reverse=False):
    """h_t = a_t h_{t-1} + u_t along axis 1 (or from the end: h_t = a_t h_{t+1} + u_t)."""
    h = np.empty(u.shape)
    state = np.zeros(u[:, 0].shape) if initial is None else f64(initial)
    for t in (range(u.shape[1] - 1, -1, -1) if reverse else range(u.shape[1])):
        state = a[:, t] * state + u[:, t]
        h[:, t] = state
    return h


def recurrence(gate, x, initial, sigmoid):
    a, _, u = coefficients(gate, x, sigmoid)
    h = scan(a, u, initial)
    return h, h[:, -1]


def _shift(a):
    """The coefficient of step t + 1 at t; that of the gradient which comes in at the end is 1."""
    return np.concatenate([a[:, 1:], np.ones_like(a[:, :1])], 1)


def recurrence_bound(gate, x, initial, sigmoid):
    """The state is summed in double and may be rounded to float where it is handed on: 3 u of the sum of magnitudes. A
    sigmoid gate is off by 6 u of the smaller of a and b (an exponential, a sum, a quotient and a product), b by 6 u of itself."""
    a, b, u = coefficients(gate, x, sigmoid)
    size = scan(np.abs(a), np.abs(u), None if initial is None else np.abs(f64(initial)))
    first = np.zeros_like(size[:, :1]) if initial is None else np.abs(f64(initial))[:, None]
    before = np.concatenate([first, size[:, :-1]], 1)
    bound = 3 * U * size
    if sigmoid:
        bound = bound + scan(np.abs(a), 6 * U * (np.minimum(a, b) * before + np.abs(u)), None)
    return bound + 1e-44


def recurrence_grads(gate, x, initial, h, go, grad_final, sigmoid):
    a, b, _ = coefficients(gate, x, sigmoid)
    d = scan(_shift(a), f64(go), grad_final, reverse=True)
    first = np.zeros_like(d[:, :1]) if initial is None else f64(initial)[:, None]
    before = np.concatenate([first, f64(h)[:, :-1]], 1)
    if sigmoid:
        return d * (before - f64(x)) * a * b, d * b, a[:, 0] * d[:, 0]
    return d * before, d, a[:, 0] * d[:, 0]


def recurrence_grad_bounds(gate, x, initial, h, go, grad_final, sigmoid):
    a, b, _ = coefficients(gate, x, sigmoid)
    ahead = _shift(a)
    size = scan(np.abs(ahead), np.abs(f64(go)), None if grad_final is None else np.abs(f64(grad_final)), reverse=True)
    off = 3 * U * size
    if sigmoid:
        after = np.concatenate([size[:, 1:], np.zeros_like(size[:, :1])], 1)
        off = off + scan(np.abs(ahead), 6 * U * np.minimum(ahead, 1.0) * np.concatenate([np.minimum(a, b)[:, 1:] / np.maximum(a[:, 1:], 1e-300),
                                                                                         np.zeros_like(a[:, :1])], 1) * after, None, reverse=True)
    first = np.zeros_like(size[:, :1]) if initial is None else f64(initial)[:, None]
    before = np.concatenate([first, f64(h)[:, :-1]], 1)
    a0 = np.abs(a[:, 0])
    b_initial = a0 * off[:, 0] + 8 * U * a0 * size[:, 0] + 1e-44
    if sigmoid:
        f = np.abs(before - f64(x)) * a * b
        return f * off + 18 * U * f * size + 1e-44, b * (off + 8 * U * size) + 1e-44, b_initial
    return np.abs(before) * (off + 2 * U * size) + 1e-44, off + 2 * U * size + 1e-44, b_initial


# ---------------------------------------------------------------- behind the oracle's raw tensors

def _view(raw, *shape):
    return None if raw is None else raw.toArray().reshape(*shape)


class _LayerNorm:
    def __init__(self, axis, epsilon, ops):
        self.axis, self.epsilon, self.ops = axis, epsilon, ops

    def _rows_cols(self, input):
        cols = sf.to_store_size(input.shape[self.axis:])
        return sf.to_store_size(input.shape) // cols, cols

    def calculateOutput(self, input, gamma=None, beta=None):
        r, c = self._rows_cols(input)
        out, mean, std = layer_norm(_view(input, r, c), _view(gamma, c), _view(beta, c), self.epsilon)
        lead = list(input.shape[:self.axis]) or [1]
        return self.ops.createRaw(input.shape, out), self.ops.createRaw(lead, mean), self.ops.createRaw(lead, std)

    def calculateGrads(self, input, gamma, gradOut, *requires):
        r, c = self._rows_cols(input)
        grads = layer_norm_grads(_view(input, r, c), _view(gamma, c), _view(gradOut, r, c), self.epsilon)
        weights = list(input.shape[self.axis:])
        return [self.ops.createRaw(s, g) if need else None for g, s, need in zip(grads, (input.shape, weights, weights), requires)]


class _Dropout:
    def __init__(self, p, seed, offset, ops):
        self.p, self.seed, self.offset, self.ops = p, seed, offset, ops

    def calculateOutput(self, input, residual=None):
        return self.ops.createRaw(input.shape, dropout(input.toArray().reshape(-1), self.p, self.seed, self.offset,
                                                       None if residual is None else residual.toArray().reshape(-1)))

    def calculateGrad(self, gradOut):
        return self.calculateOutput(gradOut)


class _GatedRecurrence:
    def __init__(self, axis, sigmoidGate, ops):
        self.axis, self.sigmoid, self.ops = axis, sigmoidGate, ops

    def _shapes(self, t):
        s = list(t.shape)
        o, i = sf.to_store_size(s[:self.axis]), sf.to_store_size(s[self.axis + 1:])
        return (o, s[self.axis], i), (o, i), s[:self.axis] + s[self.axis + 1:] or [1]

    def calculateOutput(self, gate, input, initial=None):
        full, state, lead = self._shapes(input)
        h, final = recurrence(_view(gate, *full), _view(input, *full), _view(initial, *state), self.sigmoid)
        return self.ops.createRaw(input.shape, h), self.ops.createRaw(lead, final)

    def calculateGrads(self, gate, input, initial, output, gradOut, gradFinal, *requires):
        full, state, lead = self._shapes(gate)
        grads = recurrence_grads(_view(gate, *full), _view(input, *full), _view(initial, *state), _view(output, *full), _view(gradOut, *full),
                                 _view(gradFinal, *state), self.sigmoid)
        return [self.ops.createRaw(s, g) if need else None for g, s, need in zip(grads, (gate.shape, gate.shape, lead), requires)]


class SequenceOracleOperations(JvmOracleOperations):
    def layerNorm(self, axis, epsilon): return _LayerNorm(axis, epsilon, self)
    def dropout(self, p, seed, offset=0): return _Dropout(p, seed, offset, self)
    def gatedRecurrence(self, axis, sigmoidGate=True): return _GatedRecurrence(axis, sigmoidGate, self)


def assert_within(got, want, bound, what):
    got, want, bound = f64(got).reshape(-1), f64(want).reshape(-1), np.broadcast_to(f64(bound), np.shape(want)).reshape(-1)
    assert got.shape == want.shape, f"{what}: {got.shape} values, {want.shape} are wanted"
    bad = ~(np.abs(got - want) <= bound)
    if bad.any():
        i = int(np.argmax(np.where(bad, np.abs(got - want) / bound, 0)))
        raise AssertionError(f"{what}: {np.count_nonzero(bad)} of {got.size} outside their bound; at {i}: got {got[i]!r}, want {want[i]!r}, "
                             f"off by {abs(got[i] - want[i]):.3e}, allowed {bound[i]:.3e}")

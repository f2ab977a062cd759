"""The operators of a residual block over sequences, as they are measured: layer norm, dropout from a counter-based
generator, the gated linear recurrence, each forward and backward. Every case is fp32, as every store of the library is.

`run` computes a case in elementary torch operations, or, where `own` is set, by the library's entry points over stores
that a program holds (inputs and results are stores; torch sees their memory through their device address)."""
import math

import torch

own = False

EPSILON = 1e-5
MASK32 = 0xFFFFFFFF


# ---------------------------------------------------------------- cases

def listed():
    return [
        # one short sequence's tokens through a layer norm: the time is that of a launch
        {"name": "norm small", "op": "norm", "backward": False, "rows": 64, "cols": 1024},
        # a batch whose width is a multiple of nothing
        {"name": "norm odd", "op": "norm", "backward": False, "rows": 8191, "cols": 1021},
        # the shape of the autograd benchmark: a training batch of 16384 tokens
        {"name": "norm large", "op": "norm", "backward": False, "rows": 16384, "cols": 4096},
        # backward of a middling batch, weight gradients included
        {"name": "norm grad", "op": "norm", "backward": True, "rows": 8192, "cols": 768},
        # backward of the benchmark's shape
        {"name": "norm grad large", "op": "norm", "backward": True, "rows": 16384, "cols": 4096},
        # dropout of a few activations (forward of a small batch, or its gradient: the same call)
        {"name": "dropout small", "op": "dropout", "n": 64 * 1024, "p": 0.1, "residual": False},
        # the end of a residual branch: x + dropout(branch)
        {"name": "dropout residual", "op": "dropout", "n": 16384 * 4096, "p": 0.1, "residual": True},
        # one token for each of 64 sequences: the state goes in and comes out
        {"name": "recurrence token", "op": "recurrence", "backward": False, "mode": "sigmoid", "batch": 64, "steps": 1, "width": 1024},
        # training sequences
        {"name": "recurrence", "op": "recurrence", "backward": False, "mode": "sigmoid", "batch": 8, "steps": 2048, "width": 1024},
        # one long document: hardly any parallel work but over the steps
        {"name": "recurrence long", "op": "recurrence", "backward": False, "mode": "given", "batch": 1, "steps": 65536, "width": 512},
        # backward of training sequences of odd sizes
        {"name": "recurrence grad", "op": "recurrence", "backward": True, "mode": "sigmoid", "batch": 5, "steps": 1999, "width": 1001},
        # backward of the long document
        {"name": "recurrence grad long", "op": "recurrence", "backward": True, "mode": "given", "batch": 1, "steps": 65536, "width": 512},
    ]


def _log_between(rng, low, high):
    """A whole number of [low, high], spread over its logarithm; at times a multiple of 64."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if v > 64 and rng.random() < 0.4:
        v -= v % 64
    return min(max(v, low), high)


def draw(rng):
    op = rng.choice(["norm", "norm", "dropout", "recurrence", "recurrence"])
    if op == "norm":
        cols = _log_between(rng, 8, 65536)
        rows = _log_between(rng, 1, min(65536, max(1, (1 << 26) // cols)))
        return {"op": op, "backward": rng.random() < 0.5, "rows": rows, "cols": cols}
    if op == "dropout":
        return {"op": op, "n": _log_between(rng, 1, 1 << 26), "p": round(rng.uniform(0.0, 0.9), 3), "residual": rng.random() < 0.5}
    steps = _log_between(rng, 1, 65536)
    width = _log_between(rng, 1, min(4096, max(1, (1 << 25) // steps)))
    batch = _log_between(rng, 1, min(64, max(1, (1 << 25) // (steps * width))))
    return {"op": op, "backward": rng.random() < 0.5, "mode": rng.choice(["sigmoid", "given"]), "batch": batch, "steps": steps, "width": width}


def work(case):
    if case["op"] == "norm":
        n, r, c = case["rows"] * case["cols"], case["rows"], case["cols"]
        if case["backward"]:
            return {"bytes": 4 * (3 * n + 3 * c), "flops": 18 * n}
        return {"bytes": 4 * (2 * n + 2 * r + 2 * c), "flops": 8 * n}
    if case["op"] == "dropout":
        return {"bytes": 4 * case["n"] * (3 if case["residual"] else 2), "flops": 2 * case["n"]}
    n, s = case["batch"] * case["steps"] * case["width"], case["batch"] * case["width"]
    sigmoid = case["mode"] == "sigmoid"
    if case["backward"]:
        return {"bytes": 4 * ((6 if sigmoid else 5) * n + 3 * s), "flops": (12 if sigmoid else 4) * n}
    return {"bytes": 4 * (3 * n + 2 * s), "flops": (8 if sigmoid else 2) * n}


# ---------------------------------------------------------------- inputs

class _State(dict):
    """A case's tensors by name, and where `own` is set the stores that hold them (in .raw)."""

    def __init__(self, case, seed):
        super().__init__()
        self.case = case
        self.generator = torch.Generator(device="cuda")
        self.generator.manual_seed(seed)
        self.ops, self.raw = None, {}
        if own:
            import kten_amd
            self.ops = kten_amd.platform(0)
            self.ops.sync()             # pooled memory may still be written by the calls before

    def new(self, name, *shape):
        if self.ops is not None:
            self.raw[name] = self.ops.createRaw(list(shape))
            self[name] = torch.as_tensor(self.raw[name], device="cuda")
        else:
            self[name] = torch.empty(shape, device="cuda")
        return self[name]

    def normal(self, name, shape, mean=0.0, std=1.0):
        return self.new(name, *shape).normal_(mean, std, generator=self.generator)

    def uniform(self, name, shape, low, high):
        return self.new(name, *shape).uniform_(low, high, generator=self.generator)

    def handle(self, name):
        return self.raw[name].storeReference


def prepare(case, seed):
    s = _State(case, seed)
    if case["op"] == "norm":
        rows, cols = case["rows"], case["cols"]
        s.normal("x", [rows, cols], 0.25, 1.5)
        s.uniform("gamma", [cols], 0.5, 1.5)
        if case["backward"]:
            s.normal("grad_out", [rows, cols])
            results = [("grad_in", [rows, cols]), ("grad_gamma", [cols]), ("grad_beta", [cols])]
        else:
            s.uniform("beta", [cols], -0.1, 0.1)
            results = [("out", [rows, cols]), ("mean", [rows]), ("std", [rows])]
    elif case["op"] == "dropout":
        s.normal("x", [case["n"]])
        if case["residual"]:
            s.normal("residual", [case["n"]])
        s.seed = (seed * 0x9E3779B97F4A7C15 + 1) & ((1 << 63) - 1)
        s.offset = (seed % 1000) << 32        # a training run is past 2^32 numbers soon
        results = [("out", [case["n"]])]
    else:
        shape = [case["batch"], case["steps"], case["width"]]
        state_shape = [case["batch"], case["width"]]
        if case["mode"] == "sigmoid":
            s.normal("gate", shape, 2.0, 1.5)
        else:                                 # decays from a tenth to nearly one
            s.normal("gate", shape, 2.0, 1.5).sigmoid_()
        s.normal("x", shape)
        s.normal("initial", state_shape)
        if case["backward"]:
            s.normal("grad_out", shape)
            s.normal("grad_final", state_shape)
            a, u = (v.double() for v in _coefficients(s))
            s.new("h", *shape).copy_(_scan(a, u, s["initial"].double()))
            results = [("grad_gate", shape), ("grad_in", shape), ("grad_initial", state_shape)]
        else:
            results = [("out", shape), ("final", state_shape)]
    for name, shape in results:
        if s.ops is not None:
            s.new(name, *shape)
    s.results = [name for name, _ in results]
    s.generator = None
    torch.cuda.synchronize()
    return s


# ---------------------------------------------------------------- one pass

def run(state):
    """The plain form runs on torch's stream. With `own` the calls are queued on the library's, as a program of such calls has
    them: whoever reads the results outside the library, or stops a clock, first waits for the device (torch.cuda.synchronize,
    or the library's sync)."""
    if own:
        return _run_own(state)
    return {"norm": _norm, "dropout": _dropout, "recurrence": _recurrence}[state.case["op"]](state)


def _run_own(s):
    from kten_amd import abi
    case, lib, h = s.case, s.ops.lib, s.handle
    if case["op"] == "norm":
        shape = abi.shape_array([case["rows"], case["cols"]])
        if case["backward"]:
            status = lib.kth_layer_norm_backward(h("x"), shape, 2, 1, EPSILON, h("gamma"), h("grad_out"),
                                                 h("grad_in"), h("grad_gamma"), h("grad_beta"))
        else:
            status = lib.kth_layer_norm_forward(h("x"), shape, 2, 1, EPSILON, h("gamma"), h("beta"), h("out"), h("mean"), h("std"))
    elif case["op"] == "dropout":
        status = lib.kth_dropout(h("x"), case["n"], case["p"], s.seed, s.offset, h("residual") if case["residual"] else 0, h("out"))
    else:
        shape = abi.shape_array([case["batch"], case["steps"], case["width"]])
        mode = abi.KTH_GATE_SIGMOID if case["mode"] == "sigmoid" else abi.KTH_GATE_GIVEN
        if case["backward"]:
            x = h("x") if mode == abi.KTH_GATE_SIGMOID else 0
            status = lib.kth_gated_recurrence_backward(h("gate"), x, shape, 3, 1, mode, h("initial"), h("h"), h("grad_out"),
                                                       h("grad_final"), h("grad_gate"), h("grad_in"), h("grad_initial"))
        else:
            status = lib.kth_gated_recurrence_forward(h("gate"), h("x"), shape, 3, 1, mode, h("initial"), h("out"), h("final"))
    abi.check(status)
    return {name: s[name] for name in s.results}


def _norm(s):
    x, gamma, cols = s["x"], s["gamma"], s.case["cols"]
    mean = x.sum(1) / cols
    centred = x - mean[:, None]
    std = 1.0 / torch.sqrt((centred * centred).sum(1) / cols + EPSILON)
    if not s.case["backward"]:
        return {"out": centred * std[:, None] * gamma + s["beta"], "mean": mean, "std": std}
    normalised = centred * std[:, None]
    weighted = s["grad_out"] * gamma
    mean_w = weighted.sum(1, keepdim=True) / cols
    mean_wn = (weighted * normalised).sum(1, keepdim=True) / cols
    return {"grad_in": std[:, None] * (weighted - mean_w - normalised * mean_wn),
            "grad_gamma": (s["grad_out"] * normalised).sum(0), "grad_beta": s["grad_out"].sum(0)}


def _philox(seed, offset, count, device):
    """Four 32-bit words for each of `count` counters from `offset` on: the ten-round 4x32 generator of Salmon, Moraes, Dror
    and Shaw, "Parallel random numbers: as easy as 1, 2, 3" (2011). 64-bit products wrap, which leaves their bits right."""
    c = torch.arange(count, dtype=torch.int64, device=device) + offset
    w0, w1 = c & MASK32, (c >> 32) & MASK32
    w2 = w3 = torch.zeros_like(c)
    k0, k1 = seed & MASK32, (seed >> 32) & MASK32
    for _ in range(10):
        p0, p1 = w0 * 0xD2511F53, w2 * 0xCD9E8D57
        w0, w1, w2, w3 = ((p1 >> 32) & MASK32) ^ w1 ^ k0, p1 & MASK32, ((p0 >> 32) & MASK32) ^ w3 ^ k1, p0 & MASK32
        k0, k1 = (k0 + 0x9E3779B9) & MASK32, (k1 + 0xBB67AE85) & MASK32
    return torch.stack([w0, w1, w2, w3], 1).reshape(-1)


def _dropout(s):
    n, p = s.case["n"], s.case["p"]
    keep = _philox(s.seed, s.offset, (n + 3) // 4, s["x"].device)[:n] >= int(p * (1 << 32))
    y = torch.where(keep, s["x"] * (1.0 / (1.0 - p)), 0.0)
    return {"out": s["residual"] + y if s.case["residual"] else y}


def _coefficients(s):
    """a and u of h_t = a_t h_{t-1} + u_t. 1 - a is computed as the sigmoid of the negative gate: the difference would lose it."""
    if s.case["mode"] == "given":
        return s["gate"], s["x"]
    return 1.0 / (1.0 + torch.exp(-s["gate"])), s["x"] / (1.0 + torch.exp(s["gate"]))


def _scan(a, u, initial):
    """h_t = a_t h_{t-1} + u_t over dim 1, by doubling: after the k-th pass a step holds the product and the sum of the last 2^k."""
    h = u.clone()
    h[:, 0] += a[:, 0] * initial
    steps, reach = h.shape[1], 1
    while reach < steps:
        h = torch.cat([h[:, :reach], h[:, reach:] + a[:, reach:] * h[:, :-reach]], 1)
        if 2 * reach < steps:
            a = torch.cat([a[:, :reach], a[:, reach:] * a[:, :-reach]], 1)
        reach *= 2
    return h


def _recurrence(s):
    a, u = _coefficients(s)
    initial = s["initial"]
    if not s.case["backward"]:
        h = _scan(a, u, initial)
        return {"out": h, "final": h[:, -1].clone()}
    # the gradient of the state runs backward: d_t = grad_out_t + a_{t+1} d_{t+1}
    ahead = torch.cat([a[:, 1:], torch.ones_like(a[:, :1])], 1)
    d = _scan(ahead.flip(1), s["grad_out"].flip(1), s["grad_final"]).flip(1)
    before = torch.cat([initial[:, None], s["h"][:, :-1]], 1)
    grad_initial = a[:, 0] * d[:, 0]
    if s.case["mode"] == "given":
        return {"grad_gate": d * before, "grad_in": d, "grad_initial": grad_initial}
    b = 1.0 / (1.0 + torch.exp(s["gate"]))
    return {"grad_gate": d * (before - s["x"]) * a * b, "grad_in": d * b, "grad_initial": grad_initial}


# ---------------------------------------------------------------- the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "dropout": _exact_dropout, "recurrence": _exact_recurrence}[case["op"]](s)


def _exact_norm(s):
    x = s["x"].double()
    n = x.shape[1]
    mean = x.mean(1)
    r = (((x - mean.unsqueeze(1)).square().mean(1)) + EPSILON).rsqrt()
    hat = (x - mean.unsqueeze(1)).mul_(r.unsqueeze(1))
    if not s.case["backward"]:
        return {"out": torch.addcmul(s["beta"].double().expand_as(hat), hat, s["gamma"].double().expand_as(hat)), "mean": mean, "std": r}
    go = s["grad_out"].double()
    w = go * s["gamma"].double()
    grad_in = (n * w - w.sum(1, keepdim=True) - hat * torch.mul(w, hat).sum(1, keepdim=True)) * (r / n).unsqueeze(1)
    return {"grad_in": grad_in, "grad_gamma": torch.mul(go, hat).sum(0), "grad_beta": go.sum(0)}


def _times32(x, m):
    """High and low word of the 64-bit product of two 32-bit numbers, in 16-bit halves that never overflow."""
    x0, x1, m0, m1 = x & 0xFFFF, x >> 16, m & 0xFFFF, m >> 16
    low = x0 * m0
    middle = x1 * m0 + (low >> 16)
    other = x0 * m1 + (middle & 0xFFFF)
    return x1 * m1 + (middle >> 16) + (other >> 16), ((other & 0xFFFF) << 16) | (low & 0xFFFF)


def _exact_dropout(s):
    n, p = s.case["n"], s.case["p"]
    counter = s.offset + torch.arange((n + 3) // 4, dtype=torch.int64, device="cuda")
    words = [counter % (1 << 32), counter // (1 << 32), torch.zeros_like(counter), torch.zeros_like(counter)]
    key = [s.seed % (1 << 32), s.seed // (1 << 32)]
    for _ in range(10):
        high0, low0 = _times32(words[0], 0xD2511F53)
        high1, low1 = _times32(words[2], 0xCD9E8D57)
        words = [high1 ^ words[1] ^ key[0], low1, high0 ^ words[3] ^ key[1], low0]
        key = [(key[0] + 0x9E3779B9) % (1 << 32), (key[1] + 0xBB67AE85) % (1 << 32)]
    numbers = torch.stack(words, dim=1).flatten()[:n]
    out = s["x"].double() / (1.0 - p) * (numbers >= int(p * (1 << 32)))
    if s.case["residual"]:
        out += s["residual"]
    return {"out": out}


def _exact_recurrence(s):
    gate, x = s["gate"].double(), s["x"].double()
    sigmoid = s.case["mode"] == "sigmoid"
    a, b = (torch.sigmoid(gate), torch.sigmoid(-gate)) if sigmoid else (gate, None)
    steps = gate.shape[1]
    initial = s["initial"].double()
    if not s.case["backward"]:
        u = b * x if sigmoid else x
        h, state = torch.empty_like(u), initial
        for t in range(steps):
            state = torch.addcmul(u[:, t], a[:, t], state, out=h[:, t])
        return {"out": h, "final": state}
    d = s["grad_out"].double()
    d[:, -1] += s["grad_final"]
    for t in range(steps - 2, -1, -1):
        d[:, t].addcmul_(a[:, t + 1], d[:, t + 1])
    before = torch.cat([initial.unsqueeze(1), s["h"].double()[:, :-1]], 1)
    grad_gate = d * (before - x) * a * b if sigmoid else d * before
    return {"grad_gate": grad_gate, "grad_in": d * b if sigmoid else d, "grad_initial": a[:, 0] * d[:, 0]}

"""Memory of the layers over sequences: the words that the tiles of a recurrence hand states on through count as memory of
the library's, are served from what the pool can give up, and are given up themselves; a call that is refused for want
of memory leaves its results as they were. In child processes: what a session kept from earlier calls would hide it."""
import os
import subprocess
import sys
import textwrap

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

HEAD = textwrap.dedent("""
    import ctypes, sys
    import numpy as np
    sys.path.insert(0, %r)
    import kten_amd
    from kten_amd import abi
    ops = kten_amd.platform(0); lib = ops.lib
    MIB = 1 << 20
    total = ctypes.c_uint64()
    abi.check(lib.kth_device_info(None, 0, ctypes.byref(total), None, None))
    def budget(n):                                       # the library may hold n bytes
        abi.check(lib.kth_set_memory_scale_hint(n / total.value))
    def held():
        m = ops.getMetrics()
        return m["liveBytes"] + m["poolBytes"]
    h = lambda t: t.storeReference
    SHAPE, N = abi.shape_array([2000, 300, 8]), 2000 * 300 * 8      # two tiles forward, three backward: 4 and 6 MB of words
    def forward(gate, x, out):
        return lib.kth_gated_recurrence_forward(h(gate), h(x), SHAPE, 3, 1, abi.KTH_GATE_GIVEN, 0, h(out), 0)
    gate, x = ops.createRawFill([N], 0.5), ops.createRawFill([N], 1.0)
    gate.toArray(); x.toArray()                          # (values in memory, not constants that are still owed)
    want = 2.0 - 0.5 ** np.arange(300.0)
    def right(out):
        got = out.toArray().reshape(2000, 300, 8)
        return (got == want.astype(np.float32)[None, :, None]).all()
""") % ROOT

CASES = {
    "words are counted": """
        out = ops.createRaw([N])
        ops.sync(); before = held()
        abi.check(forward(gate, x, out))
        assert right(out)
        assert held() >= before + 4 * 1000 * 1000, (before, held())
    """,
    "refused without room, and nothing of the result touched": """
        out, grads = ops.createRawFill([N], 9.0), [ops.createRawFill([N], 9.0) for _ in range(2)]
        budget(ops.getMetrics()["liveBytes"] + 64 * 1024)
        launches = ops.getMetrics()["launches"]
        assert forward(gate, x, out) == abi.KTH_E_MEMORY
        assert lib.kth_gated_recurrence_backward(h(gate), 0, SHAPE, 3, 1, abi.KTH_GATE_GIVEN, 0, h(x), h(x), 0, h(grads[0]), h(grads[1]), 0) == abi.KTH_E_MEMORY
        for t in [out] + grads:
            assert (t.toArray() == 9.0).all()
        budget(0.5 * total.value)
        abi.check(forward(gate, x, out))
        assert right(out)
    """,
    "a layer norm without its workspace": """
        rows, cols = 8, 200000
        a = ops.createRaw([rows, cols], np.random.default_rng(1).standard_normal(rows * cols).astype(np.float32))
        go = a.copy(); go.toArray()
        results = [ops.createRawFill([rows, cols], 9.0), ops.createRawFill([cols], 9.0), ops.createRawFill([cols], 9.0)]
        out, mean, std = ops.createRawFill([rows, cols], 9.0), ops.createRawFill([rows], 9.0), ops.createRawFill([rows], 9.0)
        shape = abi.shape_array([rows, cols])
        def backward():
            return lib.kth_layer_norm_backward(h(a), shape, 2, 1, 1e-5, 0, h(go), *(h(t) for t in results))
        budget(ops.getMetrics()["liveBytes"])
        assert backward() == abi.KTH_E_MEMORY
        assert lib.kth_layer_norm_forward(h(a), shape, 2, 1, 1e-5, 0, 0, h(out), h(mean), h(std)) == abi.KTH_E_MEMORY
        for t in results + [out, mean, std]:
            assert (t.toArray() == 9.0).all()
        budget(0.5 * total.value)
        abi.check(backward())
        assert np.isfinite(results[0].toArray()).all() and (results[2].toArray() != 9.0).all()
    """,
    "room is made from the pool, and the words are given up for a store": """
        out = ops.createRaw([N])
        parked = ops.createRaw([16 * MIB // 4]); parked.release()        # 16 MiB that nobody uses
        live = ops.getMetrics()["liveBytes"]
        budget(live + 17 * MIB)
        abi.check(forward(gate, x, out))                                 # fits once the pool is given up
        assert right(out)
        assert held() <= live + 17 * MIB, (held(), live)
        store = ops.createRaw([15 * MIB // 4])                           # fits once the words are
        store.inplaceFill(3.0)
        assert held() <= live + 17 * MIB and (store.toArray() == 3.0).all()
        store.release()
        abi.check(forward(gate, x, out))                                 # and back again
        assert right(out)
    """,
    "longer and longer sequences": """
        for steps in list(range(5000, 40000, 5000)) + [40001]:
            g, u = ops.createRawFill([1, steps, 64], 0.5), ops.createRawFill([1, steps, 64], 1.0)
            o, f = ops.gatedRecurrence(1, False).calculateOutput(g, u)
            assert (f.toArray() == 2.0).all() and (o.toArray()[0, 60:] == 2.0).all() and (o.toArray()[0, 0] == 1.0).all()
            g.release(); u.release(); o.release(); f.release()
        out = ops.createRaw([N])
        abi.check(forward(gate, x, out))
        assert right(out)
        abi.check(lib.kth_shutdown())
    """,
}


@pytest.mark.parametrize("case", CASES)
def test_memory(case):
    done = subprocess.run([sys.executable, "-c", HEAD + textwrap.dedent(CASES[case]) + "\nprint('case ok')"], capture_output=True, text=True, timeout=100)
    assert done.returncode == 0 and "case ok" in done.stdout, done.stdout + done.stderr

"""The layers over sequences in one session of the library after another: what a device granted, and the memory that tiles hand
states on through, belong to a session. In a child process, so that the test session's own library instance stays up."""
import os
import subprocess
import sys
import textwrap

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SESSIONS = textwrap.dedent("""
    import ctypes, sys
    import numpy as np
    sys.path.insert(0, %r)
    from kten_amd import abi
    lib = abi.load()
    def store(values):
        h = ctypes.c_uint64()
        values = np.ascontiguousarray(values, np.float32)
        abi.check(lib.kth_alloc(values.size, ctypes.byref(h)))
        abi.check(lib.kth_upload(h, 0, values.ctypes.data_as(ctypes.c_void_p), values.size))
        return h
    def read(h, n):
        out = np.empty(n, np.float32)
        abi.check(lib.kth_download(out.ctypes.data_as(ctypes.c_void_p), h, 0, n))
        return out
    rng = np.random.default_rng(1)
    first = None
    for session in range(3):
        abi.check(lib.kth_init(0))
        got = []
        for cols in (20000, 36000, 60000):                   # LDS alone up to its end, LDS and registers
            rows = 100
            x = np.random.default_rng(cols).standard_normal((rows, cols)).astype(np.float32)
            h, out = store(x), store(np.zeros_like(x))
            abi.check(lib.kth_layer_norm_forward(h, abi.shape_array([rows, cols]), 2, 1, 0.0, 0, 0, out, 0, 0))
            y = read(out, x.size).reshape(x.shape)
            x64 = x.astype(np.float64)
            want = (x64 - x64.mean(1, keepdims=True)) / x64.std(1, keepdims=True)
            assert np.abs(y - want).max() <= 8 * 2.0 ** -24 * np.abs(want).max(), cols
            got.append(y)
        gate, u = store(np.full((1, 3000, 64), 0.5)), store(np.ones((1, 3000, 64)))
        out = store(np.zeros((1, 3000, 64)))
        abi.check(lib.kth_gated_recurrence_forward(gate, u, abi.shape_array([1, 3000, 64]), 3, 1, abi.KTH_GATE_GIVEN, 0, out, 0))
        h = read(out, 3000 * 64).reshape(3000, 64)
        assert (h[-1] == 2.0).all() and (h[0] == 1.0).all()
        if first is not None:
            assert all(np.array_equal(a, b) for a, b in zip(first, got))
        first = got
        abi.check(lib.kth_shutdown())
    print("sessions ok")
""") % ROOT


def test_sessions():
    done = subprocess.run([sys.executable, "-c", SESSIONS], capture_output=True, text=True, timeout=100)
    assert done.returncode == 0 and "sessions ok" in done.stdout, done.stdout + done.stderr

"""kth_device_address: a store whose memory other code of the process reads and writes. What the library would put off
(constants, whole-store copies, small sums) has to be in memory at once for such a store, in both directions, and index
values in it are checked at every use. The other code is played by plain copies of the HIP runtime the library has loaded."""
import ctypes
import os
import subprocess
import sys

import numpy as np
import pytest

from parity import assert_bits_equal

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture()
def memory(gc):
    """(read, write) of device memory by address, outside the library."""
    path = next(line.split()[-1] for line in open("/proc/self/maps") if "libamdhip64" in line)
    hip = ctypes.CDLL(path)
    hip.hipMemcpy.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int]

    def read(raw, address, first=0):
        gc.sync()
        host = np.empty(raw.size - first, dtype=np.float32)
        assert hip.hipMemcpy(host.ctypes.data, address + 4 * first, host.nbytes, 2) == 0
        return host

    def write(raw, address, values):
        gc.sync()
        host = np.ascontiguousarray(values, dtype=np.float32).reshape(-1)
        assert host.size <= raw.size
        assert hip.hipMemcpy(address, host.ctypes.data, host.nbytes, 1) == 0
    return read, write


def data(shape, seed):
    return np.random.default_rng(seed).standard_normal(shape).astype(np.float32)


def test_what_a_store_was_owed_is_in_memory(gc, memory):
    read, _ = memory
    x = data([64, 48], 1)
    a = gc.createRaw([64, 48], x)
    filled, copied, summed = gc.createRawFill([1000], 2.5), a.copy(), a.sum(0)
    assert_bits_equal(read(filled, filled.deviceAddress()), np.full(1000, 2.5, np.float32), "an owed fill")
    assert_bits_equal(read(copied, copied.deviceAddress()), x.reshape(-1), "a copy that was put off")
    assert_bits_equal(read(summed, summed.deviceAddress()), summed.toArray().reshape(-1), "a sum that was put off")
    small = gc.createRaw([2, 16, 16], data([2, 16, 16], 2))
    chain = small.sum(1)
    assert np.allclose(read(chain, chain.deviceAddress()), small.toArray().astype(np.float64).sum(1).reshape(-1), atol=1e-4)


def test_nothing_is_put_off_for_a_shared_store(gc, memory):
    read, _ = memory
    t = gc.createRaw([4096])
    at = t.deviceAddress()
    t.inplaceFill(3.0)
    assert_bits_equal(read(t, at), np.full(4096, 3.0, np.float32), "inplaceFill")
    lib = gc.lib
    one = np.array([7.0], np.float32)
    assert lib.kth_upload(t.storeReference, 0, one.ctypes.data_as(ctypes.c_void_p), 1) == 0
    assert read(t, at)[0] == 7.0 and read(t, at)[1] == 3.0
    constant = gc.createRawFill([4096], 1.25)
    assert lib.kth_copy(t.storeReference, 0, constant.storeReference, 0, 4096) == 0
    assert_bits_equal(read(t, at), np.full(4096, 1.25, np.float32), "a copied constant")
    assert lib.kth_scalar(2, constant.storeReference, 2.0, 0, t.storeReference, 4096) == 0
    assert_bits_equal(read(t, at), np.full(4096, 2.5, np.float32), "constant times constant")
    from kten_amd import abi
    one_value = gc.createRawFill([1], 0.5)
    assert lib.kth_broadcast_to(one_value.storeReference, abi.shape_array([1]), 1, t.storeReference, abi.shape_array([4096]), 1) == 0
    assert_bits_equal(read(t, at), np.full(4096, 0.5, np.float32), "a broadcast constant")
    x = data([4096], 3)
    source = gc.createRaw([4096], x)
    assert lib.kth_copy(t.storeReference, 0, source.storeReference, 0, 4096) == 0
    assert_bits_equal(read(t, at), x, "a whole-store copy into it")
    assert lib.kth_scalar(4, source.storeReference, 1.0, 0, t.storeReference, 4096) == 0
    assert_bits_equal(read(t, at), x, "pow 1 into it")
    small = gc.createRaw([2, 16, 16], data([2, 16, 16], 4))
    out = gc.createRaw([2, 16])
    out_at = out.deviceAddress()
    assert lib.kth_reduce_axis(7, small.storeReference, out.storeReference, 2, 16, 16) == 0
    assert np.allclose(read(out, out_at), small.toArray().astype(np.float64).sum(1).reshape(-1), atol=1e-4)
    assert t.deviceAddress() == at and out.deviceAddress() == out_at, "the address does not change"


def test_writes_from_outside_do_not_reach_copies_made_before(gc, memory):
    read, write = memory
    x, y = data([3000], 5), data([3000], 6)
    t = gc.createRaw([3000], x)
    at = t.deviceAddress()
    before, powered = t.copy(), t._scalar("pow", 1.0)
    small = gc.createRaw([2, 16, 16], x[:512])
    small_at = small.deviceAddress()
    summed = small.sum(1)
    write(t, at, y)
    write(small, small_at, y[:512])
    assert_bits_equal(before.toArray(), x, "a copy made before the write")
    assert_bits_equal(powered.toArray(), x, "pow 1 made before the write")
    assert np.allclose(summed.toArray(), x[:512].reshape(2, 16, 16).astype(np.float64).sum(1), atol=1e-4)
    assert_bits_equal((t._scalar("times", 2.0)).toArray(), y * np.float32(2), "the call after the write")


def test_index_values_written_from_outside_are_checked(gc, memory):
    _, write = memory
    table = gc.createRaw([10, 4], np.arange(40, dtype=np.float32))
    index = gc.createRaw([3], np.array([1, 2, 3], np.float32))
    at = index.deviceAddress()
    for _ in range(2):
        assert_bits_equal(table.indexSelect(0, index).toArray(), np.arange(40, dtype=np.float32).reshape(10, 4)[1:4], "rows")
    write(index, at, [1, 10, 3])
    with pytest.raises(ValueError, match="out of bounds"):
        table.indexSelect(0, index)
    write(index, at, [9, 0, 3])
    assert_bits_equal(table.indexSelect(0, index).toArray(), np.arange(40, dtype=np.float32).reshape(10, 4)[[9, 0, 3]], "rows")


def test_address_of_a_released_handle_is_refused(gc):
    from kten_amd import abi
    t = gc.createRaw([16])
    h = t.storeReference
    address = ctypes.c_uint64()
    assert gc.lib.kth_device_address(h, None, None) == abi.KTH_E_ARGUMENT
    n = ctypes.c_uint64()
    assert gc.lib.kth_device_address(h, ctypes.byref(address), ctypes.byref(n)) == 0 and n.value == 16 and address.value != 0
    t.release()
    assert gc.lib.kth_device_address(h, ctypes.byref(address), None) == abi.KTH_E_HANDLE
    # the slot's next store starts unshared: its fill is put off again
    launches = gc.getMetrics()["launches"]
    gc.createRawFill([16], 1.0)
    assert gc.getMetrics()["launches"] == launches


SHARED_WITH_TORCH = """
import torch
import numpy as np
import kten_amd
ops = kten_amd.platform(0)
raw = ops.createRaw([37, 5], np.arange(185, dtype=np.float32))
seen = torch.as_tensor(raw, device="cuda")
ops.sync()
assert seen.shape == (37, 5) and seen.data_ptr() == raw.deviceAddress()
assert torch.equal(seen.cpu(), torch.arange(185, dtype=torch.float32).reshape(37, 5))
seen.mul_(2.0)
torch.cuda.synchronize()
assert raw.toArray()[3, 2] == 34.0
raw.plusAssign(1.0)
ops.sync()
assert float(seen[3, 2]) == 35.0
del raw
assert float(seen[3, 2]) == 35.0
print("shared")
"""


def test_torch_sees_the_memory_of_a_store():
    """In a process of its own: torch has to be there first."""
    done = subprocess.run([sys.executable, "-c", SHARED_WITH_TORCH], cwd=ROOT, capture_output=True, text=True, timeout=100)
    assert done.returncode == 0 and "shared" in done.stdout, done.stdout + done.stderr

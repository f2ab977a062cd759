"""The gated recurrence through the C++ host mirror without the tensors that it does not read: its test program passes on the GPU."""
import os
import subprocess

import pytest

BINARY = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "sequence_absent_test")


@pytest.mark.gpu
def test_cpp_absent_tensors():
    assert os.path.exists(BINARY), "tests/cpp/sequence_absent_test is not built (python __graft_entry__.py build)"
    done = subprocess.run([BINARY], capture_output=True, text=True, timeout=120)
    assert done.returncode == 0, done.stdout + done.stderr
    assert " 0 failed" in done.stdout

"""The layers over sequences through the C++ host mirror: its test program passes on the GPU."""
import os
import subprocess

import pytest

BINARY = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "sequence_mirror_test")


@pytest.mark.gpu
def test_cpp_sequence_layers():
    assert os.path.exists(BINARY), "tests/cpp/sequence_mirror_test is not built (python __graft_entry__.py build)"
    done = subprocess.run([BINARY], capture_output=True, text=True, timeout=120)
    print(done.stdout)
    print(done.stderr)
    assert done.returncode == 0, done.stdout + done.stderr
    assert " 0 failed" in done.stdout

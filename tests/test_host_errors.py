"""The host side of the C-ABI where the HIP runtime refuses something (CPU
only): tests/cpp/test_host_errors.cpp defines the runtime's entry points that
libokq.so calls, so that no device is needed or touched."""
import os
import subprocess

import pytest

BINARY = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "_build", "test_host_errors")


@pytest.mark.parametrize("case", ["refused_fills", "missing_workspaces"])
def test_host_errors(case):
    assert os.path.exists(BINARY), f"{BINARY} is not built: run __graft_entry__.build() (make -C tests/cpp)"
    r = subprocess.run([BINARY, case], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr

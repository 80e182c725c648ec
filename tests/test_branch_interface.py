"""The C++ operator interface of layer norm, dropout and differential attention (include/ops)."""
import pathlib
import subprocess

import pytest

ROOT = pathlib.Path(__file__).resolve().parent.parent


@pytest.mark.gpu
def test_interface_program():
    """tests/cpp/branch_ops_test.cpp: known answers, one mask in both directions, refusals as exceptions."""
    binary = ROOT / "tests" / "cpp" / "branch_ops_test.bin"
    assert binary.exists(), "build it with `python -m cgpt_amd.build` (there is no fallback)"
    proc = subprocess.run([str(binary)], capture_output=True, text=True, timeout=120)
    assert proc.returncode == 0, proc.stdout + proc.stderr
    assert proc.stdout == "0 failure(s)\n"

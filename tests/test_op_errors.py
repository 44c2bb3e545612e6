"""Failures at the C entries of the training operators, on the CPU
(tests/cpp/test_op_errors.cu)."""
import os
import shutil
import subprocess

import pytest

from alphazero_b200 import build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _nvcc():
    if os.path.exists(build.NVCC):
        return build.NVCC
    return shutil.which("nvcc")


@pytest.mark.skipif(_nvcc() is None, reason="nvcc not found")
def test_every_exception_becomes_a_code_and_its_own_message(tmp_path):
    exe = str(tmp_path / "test_op_errors")
    r = subprocess.run([_nvcc(), build.GENCODE, "-O1", "-std=c++17", "-o", exe,
                        os.path.join(ROOT, "tests", "cpp", "test_op_errors.cu")], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr

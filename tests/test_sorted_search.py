"""The embedding gradient's search among sorted tokens
(alphazero_b200/csrc/sorted_search.cuh), run on the CPU up to the largest
number of tokens that a call accepts (tests/cpp/test_sorted_search.cu)."""
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
def test_search_stays_inside_the_tokens(tmp_path):
    exe = str(tmp_path / "test_sorted_search")
    r = subprocess.run([_nvcc(), build.GENCODE, "-O2", "-std=c++17", "-o", exe,
                        os.path.join(ROOT, "tests", "cpp", "test_sorted_search.cu")],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr
    assert " 0 failures" in r.stdout

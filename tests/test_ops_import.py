"""alphazero_b200.ops on a torch without CUDA: the import works, calls refuse."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SCRIPT = """
import torch
del torch._C._cuda_getCurrentRawStream  # as a torch built without CUDA has it
from alphazero_b200 import ops
t = torch.zeros(4, 8, dtype=torch.bfloat16)
try:
    ops.linear(t, t)
except TypeError as e:
    assert "CUDA tensor" in str(e)
    print("refused")
"""


def test_imports_without_cuda():
    r = subprocess.run([sys.executable, "-c", SCRIPT], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    assert r.stdout.strip() == "refused"

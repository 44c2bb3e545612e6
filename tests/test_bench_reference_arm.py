"""The reference arm's process maps none of the product's libraries, with a
reference tree to take the positions from or without one."""
import os
import subprocess
import sys

import numpy as np

from alphazero_b200 import host_lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SCRIPT = """
import sys
sys.path[:0] = [%r, %r]
import bench, oracle
x = bench.reference_positions(9, 6, 60)
maps = open("/proc/self/maps").read()
assert "libminigo" not in maps, "a product library is mapped"
assert x.ndim == 2
x.tofile(sys.argv[1])
""" % (ROOT, os.path.join(ROOT, "oracle"))


def test_reference_arm_maps_no_product_library(tmp_path):
    out = str(tmp_path / "positions")
    r = subprocess.run([sys.executable, "-c", SCRIPT, out], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    want = host_lib.random_positions(9, 6, 1000, 60)
    assert np.array_equal(np.fromfile(out, np.float32).reshape(want.shape), want)

"""The residual tower over operands of more than 2^32 elements (8.6 GB of bf16), and its large 16-bit kernels recorded into a graph.  In a
child process: torch has to be loaded before libps_amd."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
TEST_TIMEOUT_S = 240            # the first import of torch on a cold machine can take two minutes


def test_offsets_beyond_32_bits_and_large_graphs():
    here = os.path.dirname(os.path.abspath(__file__))
    r = subprocess.run([sys.executable, "-u", os.path.join(here, "tower_large_child.py")], capture_output=True, text=True, timeout=220)
    assert r.returncode == 0 and "all done" in r.stdout, r.stdout[-3000:] + r.stderr[-3000:]

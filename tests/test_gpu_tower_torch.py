"""The residual tower's Python layers (LnLayer, FcResLayer) on torch tensors: strided views, adopted streams, torch's graphs, autograd's
gradients, refusals.  In a child process: torch brings a HIP runtime of its own, which has to be loaded before libps_amd."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
TEST_TIMEOUT_S = 240            # the first import of torch on a cold machine can take two minutes


def test_layers_on_torch_tensors():
    here = os.path.dirname(os.path.abspath(__file__))
    r = subprocess.run([sys.executable, "-u", os.path.join(here, "tower_torch_child.py")], capture_output=True, text=True, timeout=220)
    assert r.returncode == 0 and "all done" in r.stdout, r.stdout[-3000:] + r.stderr[-3000:]

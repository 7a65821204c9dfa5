"""The residual tower's Python layers where torch works on another stream than the store (a store that has adopted none, a torch stream
entered later): ordered both ways, refused while a graph is recorded.  In a child process: torch has to be loaded before libps_amd."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
TEST_TIMEOUT_S = 240            # the first import of torch on a cold machine can take two minutes


def test_layers_on_other_streams():
    here = os.path.dirname(os.path.abspath(__file__))
    r = subprocess.run([sys.executable, "-u", os.path.join(here, "tower_streams_child.py")], capture_output=True, text=True, timeout=220)
    assert r.returncode == 0 and "all done" in r.stdout, r.stdout[-3000:] + r.stderr[-3000:]

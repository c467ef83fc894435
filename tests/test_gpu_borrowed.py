"""GPU: memory borrowed from torch's tensors — the order of calls with torch's own work."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu


def test_calls_stand_in_torchs_order():
    here = os.path.dirname(os.path.abspath(__file__))
    r = subprocess.run([sys.executable, os.path.join(here, "torch_order_check.py")], capture_output=True, text=True, timeout=110, cwd=os.path.dirname(here))
    assert r.returncode == 0 and "torch order OK" in r.stdout, r.stdout[-2000:] + r.stderr[-2000:]


def test_a_step_in_torchs_graph():
    here = os.path.dirname(os.path.abspath(__file__))
    r = subprocess.run([sys.executable, os.path.join(here, "torch_capture_check.py")], capture_output=True, text=True, timeout=110, cwd=os.path.dirname(here))
    assert r.returncode == 0 and "torch capture OK" in r.stdout, r.stdout[-2000:] + r.stderr[-2000:]

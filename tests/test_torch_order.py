"""GPU: the 8-bit and orthogonalised operators among torch's own work (torch_order.py, a process of its own)."""
import os
import subprocess
import sys

import pytest

from conftest import ROOT


@pytest.mark.gpu
def test_calls_are_in_order_with_torch():
    env = dict(os.environ, HSA_ENABLE_IPC_MODE_LEGACY="0")
    r = subprocess.run([sys.executable, "-u", os.path.join(ROOT, "tests", "torch_order.py")], capture_output=True, text=True, timeout=110, env=env)
    assert r.returncode == 0 and r.stdout.strip().endswith("done"), (r.stdout[-1500:], r.stderr[-2500:])

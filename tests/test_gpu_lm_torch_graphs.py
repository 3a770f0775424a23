"""Several graphs of the serving operators' calls on torch tensors (lm_torch_graphs_main.py, a process for each check)."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.mark.parametrize("check", ["order", "together", "given", "grown"])
def test_graphs(check):
    p = subprocess.run([sys.executable, "-u", os.path.join(HERE, "lm_torch_graphs_main.py"), check], capture_output=True, text=True, timeout=110)
    assert p.returncode == 0 and f"ok {check}" in p.stdout, p.stdout[-1000:] + p.stderr[-3000:]

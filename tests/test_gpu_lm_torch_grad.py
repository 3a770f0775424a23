"""The serving operators and tensors that require gradients (lm_torch_grad_main.py, a process of its own)."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))


def test_grad():
    p = subprocess.run([sys.executable, "-u", os.path.join(HERE, "lm_torch_grad_main.py")], capture_output=True, text=True, timeout=110)
    assert p.returncode == 0 and "ok grad" in p.stdout, p.stdout[-1000:] + p.stderr[-3000:]

"""The serving operators on torch tensors: one decode step against the plain statements, on other streams, in graphs,
and what is refused (lm_torch_main.py, a process for each)."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.mark.parametrize("check", ["step", "streams", "graphs", "refusals"])
def test_torch(check):
    p = subprocess.run([sys.executable, "-u", os.path.join(HERE, "lm_torch_main.py"), check], capture_output=True, text=True, timeout=110)
    assert p.returncode == 0 and f"ok {check}" in p.stdout, p.stdout[-1000:] + p.stderr[-3000:]

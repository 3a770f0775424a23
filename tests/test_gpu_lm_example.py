"""examples/turn_reply.py: speech decoder, page plans, cache, attention and sampling together, its last step's logits
checked against dense attention over the cache read back."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("sessions,reply", [(1, 2), (5, 70)])
def test_turn_reply(sessions, reply):
    p = subprocess.run([sys.executable, "-u", os.path.join(ROOT, "examples", "turn_reply.py"), "--sessions", str(sessions), "--reply", str(reply),
                        "--check"], capture_output=True, text=True, timeout=110)
    assert p.returncode == 0 and "agree" in p.stdout and p.stdout.count("session ") == sessions, p.stdout[-1500:] + p.stderr[-2500:]

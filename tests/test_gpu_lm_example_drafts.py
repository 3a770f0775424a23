"""examples/turn_reply.py over the 8-bit cache, token by token and with drafted tokens: it runs, its logits agree with dense
attention over the cache, and every session has its reply."""
import ast
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("cache,draft", [(8, 0), (8, 3), (4, 2)])
def test_turn_reply(cache, draft):
    p = subprocess.run([sys.executable, os.path.join(ROOT, "examples", "turn_reply.py"), "--sessions", "3", "--reply", "9", "--cache", str(cache),
                        "--draft", str(draft), "--check"], capture_output=True, text=True, timeout=110)
    assert p.returncode == 0, p.stdout[-1000:] + p.stderr[-3000:]
    assert "agree with dense attention" in p.stdout
    replies = [ast.literal_eval(line.split(":", 1)[1].strip()) for line in p.stdout.splitlines() if line.startswith("session ")]
    assert [len(r) for r in replies] == [9] * 3

"""examples/turn_reply.py answers from one distribution with drafted tokens and without: what it bars for lm.verify is what lm.sample's
filters leave out."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

ALIKE = """
import sys
import torch
sys.path.insert(0, sys.argv[1])
import turn_reply as example
lm = example.lm
g = torch.Generator("cuda").manual_seed(5)
i32 = dict(dtype=torch.int32, device="cuda")
for n, V in ((400, 1027), (30, 20011)):
    x = torch.randn(n, V, generator=g, device="cuda") * 3
    x[:, 5] = x[:, 7]                                     # equal logits: the lower index comes first
    settings = dict(temperature=torch.rand(n, generator=g, device="cuda") + 0.4, top_k=torch.randint(1, 90, (n,), generator=g, device="cuda").int(),
                    top_p=torch.rand(n, generator=g, device="cuda"), min_p=torch.rand(n, generator=g, device="cuda") * 0.2)
    settings["top_k"][0], settings["min_p"][1], settings["top_p"][2] = 1, 0.0, 0.0
    u = torch.rand(n, generator=g, device="cuda")
    token, prob, kept = torch.zeros(n, **i32), torch.zeros(n, device="cuda"), torch.zeros(n, **i32)
    lm.sample(x, u, token, prob=prob, kept=kept, **settings)
    allowed = example.barred(x, **settings)
    assert torch.equal((allowed > -torch.inf).sum(-1).int(), kept)
    assert torch.equal(torch.where(allowed > -torch.inf, allowed, x), x)
    out, accepted, p = torch.zeros(n, **i32), torch.zeros(n, **i32), torch.zeros(n, device="cuda")
    lm.verify(allowed, torch.zeros(n, **i32), torch.arange(n + 1, **i32), u, u, out, accepted, max_new=1, temperature=settings["temperature"], prob=p)
    # each side's weights are off by 2^-18 of themselves and 2^-30 of the largest, of kept ones at most 90
    assert torch.equal(out, token) and ((p - prob).abs() <= 2.0 ** -16 * prob + 2.0 ** -22).all()
print("ok alike")
"""


def test_filters_bar_what_the_sampler_leaves_out():
    p = subprocess.run([sys.executable, "-c", ALIKE, os.path.join(ROOT, "examples")], capture_output=True, text=True, timeout=110)
    assert p.returncode == 0 and "ok alike" in p.stdout, p.stdout[-1000:] + p.stderr[-3000:]

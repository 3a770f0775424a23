"""Serving operators on torch tensors that require gradients: they have no backward pass, so with gradients on they refuse
such tensors, inputs and outputs alike, and without they take them.  Started by test_gpu_lm_torch_grad.py."""
import torch

from lm_torch_main import Step
from parakeet_amd import lm

s = Step(20)
s.run()
s.check()
d, o = s.d, s.o
qkv = d["qkv"]
calls = {
    "q": lambda: lm.kv4_attend(d["qkv"][:, :8], d["cache"], d["table"], o["lens"], o["out"], 32, first=o["first"], max_new=3),
    "k": lambda: lm.kv4_store(d["qkv"][:, 8:10], d["qkv"][:, 10:], o["slots"][:s.n], d["cache"], 32),
    "logits": lambda: lm.sample(d["logits"], d["u"], o["token"]),
    "lse": lambda: lm.kv4_attend(qkv[:, :8], d["cache"], d["table"], o["lens"], o["out"], 32, first=o["first"], max_new=3, lse=o["lse"]),
    "prob": lambda: lm.sample(d["logits"], d["u"], o["token"], prob=o["prob"]),
}
for name, call in calls.items():
    where, key = {"q": (d, "qkv"), "k": (d, "qkv"), "logits": (d, "logits"), "lse": (o, "lse"), "prob": (o, "prob")}[name]
    kept = where[key]
    where[key] = kept.clone().requires_grad_()
    try:
        call()
    except ValueError as e:
        assert "gradient" in str(e) and name in str(e), str(e)
    else:
        raise AssertionError(f"{name} taken")
    with torch.no_grad():
        call()
    with torch.inference_mode():
        call()
    where[key] = kept
s.clear()
s.run()
s.check()
torch.cuda.synchronize()
print("ok grad", flush=True)

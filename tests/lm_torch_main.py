"""The serving operators on torch tensors, in a process of its own (torch is imported before the library, so that both use
torch's HIP runtime): started by test_gpu_lm_torch.py with the name of one check."""
import os
import sys

import numpy as np
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path[:0] = [ROOT, os.path.join(ROOT, "tests")]
import __graft_entry__ as graft  # noqa: E402

graft.load_package()
import lm_reference as R  # noqa: E402
from parakeet_amd import lm, pk  # noqa: E402

I32 = dict(dtype=torch.int32, device="cuda")


class Step:
    """One decode step of 5 sessions, a layer's worth: plan, store, attend, sample, everything in tensors that stay."""

    def __init__(self, seed=0, page=32, H=2, Hq=8, D=128, V=20011, long=3000):
        g = np.random.default_rng(seed)
        self.page, self.H, self.Hq, self.D, self.V = page, H, Hq, D, V
        lens = np.array([long, 0, 31, 32, 700], np.int32)
        self.old, self.new = lens, lens + np.array([1, 3, 1, 1, 1], np.int32)
        B, width = 5, -(-long // page) + 1
        held = -(-lens // page)
        self.n_pages = int(held.sum()) + 9
        ids = g.permutation(self.n_pages).astype(np.int32)
        self.table = np.full((B, width), self.n_pages, np.int32)
        at = 0
        for b in range(B):
            self.table[b, :held[b]] = ids[at:at + held[b]]
            at += held[b]
        self.ring = np.roll(np.concatenate([ids[at:], np.full(at, -1, np.int32)]), 4)
        self.state = np.array([4, self.n_pages - at], np.int32)
        self.cache = g.integers(0, 256, (self.n_pages, H, R.record_bytes(page, D)), dtype=np.uint8)
        for b in np.flatnonzero(lens):
            k, v = g.standard_normal((2, lens[b], H, D))
            R.store(self.cache, page, D, k, v, [self.table[b, t // page] * page + t % page for t in range(lens[b])])
        n = int((self.new - self.old).sum())
        self.qkv = R.to_dtype(g.standard_normal((n, Hq + 2 * H, D)), "bf16")
        self.logits = R.to_dtype(g.standard_normal((B, V)) * 2.5, "f32")
        self.u = g.random(B).astype(np.float32)
        self.settings = dict(temperature=np.full(B, 0.8, np.float32), top_k=np.array([40, 0, 7, 0, 0], np.int32),
                             top_p=np.array([0.9, 1.0, 1.0, 0.9, 0.5], np.float32), min_p=np.array([0, 0, 0, 0, 0.05], np.float32))
        self.n = n
        put = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
        self.d = dict(old=put(self.old), new=put(self.new), table=put(self.table), ring=put(self.ring), state=put(self.state),
                      cache=put(self.cache), qkv=put(self.qkv.view(np.int16)).view(torch.bfloat16), logits=put(self.logits), u=put(self.u),
                      **{k: put(v) for k, v in self.settings.items()})
        e = lambda *s: torch.zeros(*s, **I32)  # noqa: E731
        self.o = dict(state_out=e(2), lens=e(B), ok=e(B), first=e(B + 1), slots=e(n + 2), pos=e(n + 2), token=e(B), kept=e(B),
                      prob=torch.zeros(B, device="cuda"), out=torch.zeros(n, Hq, D, dtype=torch.bfloat16, device="cuda"),
                      lse=torch.zeros(n, Hq, device="cuda"))

    def run(self, stream=None):
        d, o, Hq, H = self.d, self.o, self.Hq, self.H
        lm.kv_plan(d["old"], d["new"], d["table"], d["ring"], d["state"], self.page, state_out=o["state_out"], lens=o["lens"], ok=o["ok"],
                   first=o["first"], slots=o["slots"], pos=o["pos"], stream=stream)
        lm.kv4_store(d["qkv"][:, Hq:Hq + H], d["qkv"][:, Hq + H:], o["slots"][:self.n], d["cache"], self.page, stream=stream)
        lm.kv4_attend(d["qkv"][:, :Hq], d["cache"], d["table"], o["lens"], o["out"], self.page, first=o["first"], max_new=3, lse=o["lse"],
                      stream=stream)
        lm.sample(d["logits"], d["u"], o["token"], temperature=d["temperature"], top_k=d["top_k"], top_p=d["top_p"], min_p=d["min_p"],
                  prob=o["prob"], kept=o["kept"], stream=stream)

    def clear(self):
        for t in self.o.values():
            t.zero_()

    def results(self):
        torch.cuda.synchronize()
        return {k: v.clone() for k, v in self.o.items()} | {"cache": self.d["cache"].clone(), "table": self.d["table"].clone()}

    def check(self):
        r = {k: v.float().cpu().numpy() if v.dtype == torch.bfloat16 else v.cpu().numpy() for k, v in self.results().items()}
        want = R.plan(self.old, self.new, self.table, self.ring, self.state, self.page, self.n + 2)
        for k in ("state_out", "lens", "ok", "first", "slots", "pos", "table"):
            assert np.array_equal(r[k], want[k]), k
        cache = self.cache.copy()
        kv = R.to_f64(self.qkv, "bf16")
        R.store(cache, self.page, self.D, kv[:, self.Hq:self.Hq + self.H], kv[:, self.Hq + self.H:], want["slots"][:self.n])
        assert np.array_equal(r["cache"], cache)
        out, lse, tol, ltol = R.attend(kv[:, :self.Hq], cache, want["table"], want["lens"], want["first"], self.page, self.D ** -0.5, 0, "bf16")
        assert (np.abs(r["out"] - out) <= tol).all() and (np.abs(r["lse"] - lse) <= ltol).all()
        for b in range(5):
            s = {k: v[b].item() for k, v in self.settings.items()}
            w = R.sample_bounds(self.logits[b], float(self.u[b]), **s)
            assert r["token"][b] in w["tokens"] and w["kept"][0] <= r["kept"][b] <= w["kept"][1]


def same(a, b):
    for k in a:
        assert torch.equal(a[k], b[k]), k


def step():
    s = Step()
    s.run()
    s.check()


def streams():
    """On a stream of its own, made current or given by its handle, its inputs made there too: the same results."""
    s = Step(1)
    s.run()
    want = s.results()
    side = torch.cuda.Stream()
    for given in (False, True):
        s.clear()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            late = s.d["qkv"].clone()
            torch.cuda._sleep(2_000_000)
            s.d["qkv"].zero_()
            s.d["qkv"].copy_(late)
            if not given:
                s.run()
        if given:
            s.run(stream=side.cuda_stream)
        side.synchronize()
        same(s.results(), want)


def graphs():
    """Captured once and replayed, new inputs in between and eager calls of other shapes beside: every replay as eager."""
    s, other = Step(2), Step(3, page=16, D=64, V=301, long=900)
    s.run()
    other.run()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        s.run()
    for turn in range(5):
        s.d["u"].copy_(torch.rand(5, device="cuda"))
        s.d["logits"].copy_(torch.randn(5, s.V, device="cuda") * (1 + turn))
        s.d["qkv"].copy_(torch.randn(s.d["qkv"].shape, device="cuda").bfloat16())
        s.clear()
        g.replay()
        got = s.results()
        s.clear()
        s.run()
        same(s.results(), got)
        other.run()
        big = torch.randn(3, 60000 + turn, device="cuda")
        token = torch.zeros(3, **I32)
        lm.sample(big, torch.rand(3, device="cuda"), token, top_p=torch.full((3,), 0.9, device="cuda"))
        torch.cuda.synchronize()
        assert (token >= 0).all()
    other.check()


def refusals():
    s = Step(4)
    d, o = s.d, s.o

    def refused(kind, text, f, *a, **k):
        try:
            f(*a, **k)
        except kind as e:
            assert text in str(e), (text, str(e))
            return
        raise AssertionError(f"not refused: {text}")

    plan = dict(state_out=o["state_out"], lens=o["lens"], ok=o["ok"], first=o["first"], slots=o["slots"], pos=o["pos"])
    args = [d["old"], d["new"], d["table"], d["ring"], d["state"], 32]
    refused(ValueError, "on the GPU", lm.kv_plan, *args[:2], d["table"].cpu(), *args[3:], **plan)
    refused(ValueError, "arrays on", lm.kv_plan, d["old"].cpu(), *args[1:], **plan)
    refused(TypeError, "old_len", lm.kv_plan, d["old"].long(), *args[1:], **plan)
    refused(ValueError, "new_len", lm.kv_plan, d["old"], d["new"][:3], *args[2:], **plan)
    refused(ValueError, "first", lm.kv_plan, *args, **dict(plan, first=o["first"][:5]))
    refused(ValueError, "not contiguous", lm.kv_plan, *args, **dict(plan, slots=torch.zeros(20, **I32)[::2]))
    refused(pk.PkError, "pages of 33", lm.kv_plan, *args[:5], 33, **plan)
    refused(TypeError, "not a tensor", lm.kv_plan, None, *args[1:], **plan)
    k = d["qkv"][:, 8:10]
    slots = o["slots"][:s.n]
    refused(ValueError, "kv4_shape", lm.kv4_store, k, k, slots, d["cache"], 31)
    refused(TypeError, "uint8", lm.kv4_store, k, k, slots, d["cache"].view(torch.int8), 32)
    refused(ValueError, "rows of", lm.kv4_store, k[:, :1], k[:, :1], slots, d["cache"], 32)
    refused(ValueError, "not adjacent", lm.kv4_store, k.transpose(1, 2), k.transpose(1, 2), slots, d["cache"], 32)
    refused(TypeError, "f32, f16 or bf16", lm.kv4_load, d["cache"], slots, k.int(), k.int(), 32)
    refused(ValueError, "v (7", lm.kv4_load, d["cache"], slots, k, k.float(), 32)
    q = d["qkv"][:, :8]
    at = [q, d["cache"], d["table"], o["lens"], o["out"], 32]
    refused(ValueError, "query heads", lm.kv4_attend, q[:, :7], *at[1:4], o["out"][:, :7], 32)
    refused(ValueError, "out", lm.kv4_attend, *at[:4], o["out"].half(), 32)
    refused(ValueError, "overlap", lm.kv4_attend, *at[:4], o["out"][:1].expand(s.n, 8, 128), 32)
    refused(pk.PkError, "without first", lm.kv4_attend, *at)
    refused(pk.PkError, "workspace", lm.kv4_attend, *at, first=o["first"], max_new=3, workspace=torch.zeros(64, dtype=torch.uint8, device="cuda"))
    refused(ValueError, "out of range", lm.kv4_attend, *at, first=o["first"], max_new=1 << 40)
    x = d["logits"]
    refused(ValueError, "logits", lm.sample, x[0], d["u"], o["token"])
    refused(ValueError, "not adjacent", lm.sample, x.t(), d["u"], o["token"])
    refused(TypeError, "logits", lm.sample, x.double(), d["u"], o["token"])
    refused(TypeError, "top_k", lm.sample, x, d["u"], o["token"], top_k=d["u"])
    refused(ValueError, "u: shape", lm.sample, x, d["u"][:2], o["token"])
    s.run()
    s.check()


if __name__ == "__main__":
    globals()[sys.argv[1]]()
    torch.cuda.synchronize()
    print("ok", sys.argv[1], flush=True)

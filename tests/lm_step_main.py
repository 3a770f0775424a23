"""Steps with drafted tokens on torch tensors, in a process of its own (torch is imported before the library, so that both use
torch's HIP runtime): started by test_gpu_lm_step.py with the name of one check."""
import os
import sys

import numpy as np
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path[:0] = [ROOT, os.path.join(ROOT, "tests")]
import __graft_entry__ as graft  # noqa: E402

graft.load_package()
import lm_reference as R  # noqa: E402
import lm_step_reference as S  # noqa: E402
from lm_torch_main import same  # noqa: E402
from parakeet_amd import lm, pk  # noqa: E402

I32 = dict(dtype=torch.int32, device="cuda")


class Step:
    """A step of 5 sessions, a layer's worth, everything in tensors that stay: the plan for each session's last token and its
    drafts, the rows into the cache, attention, what stands of the drafts, the plan that cuts the cache back to it."""

    def __init__(self, seed=0, page=32, H=2, Hq=8, D=128, V=2003, dtype=torch.bfloat16, draft=True, long=1500):
        g = torch.Generator().manual_seed(seed)
        self.page, self.H, self.Hq, self.D, self.V = page, H, Hq, D, V
        self.old = torch.tensor([long, 0, 31, 33, 700])
        self.more = torch.tensor([3, 4, 1, 5, 2])
        B, width = 5, -(-long // page) + 1
        held = (self.old + page - 1) // page
        self.n_pages = int(held.sum()) + 9
        ids = torch.randperm(self.n_pages, generator=g)
        table = torch.full((B, width), self.n_pages)
        at = 0
        for b in range(B):
            table[b, :held[b]] = ids[at:at + held[b]]
            at += int(held[b])
        ring = torch.roll(torch.cat([ids[at:], torch.full((at,), -1)]), 4)
        self.n = n = int(self.more.sum())
        i32 = lambda t: t.to(torch.int32).cuda()  # noqa: E731
        e = lambda *s: torch.zeros(*s, **I32)  # noqa: E731
        self.shape = lm.kv8_shape(self.n_pages, H, D, page)
        self.inv = (10000.0 ** (-torch.arange(0, D, 2) / D)).cuda()
        self.w = (1 + 0.2 * torch.randn(2, D, generator=g)).cuda()
        kept = torch.cat([torch.cat([table[b, t // page] * page + t % page for t in [torch.arange(int(self.old[b]))]]) for b in range(B)])
        before = torch.zeros(self.shape, dtype=torch.uint8, device="cuda")
        rows = torch.randn(2, len(kept), H, D, generator=g).to(dtype).cuda()
        lm.kv8_append(rows[0], rows[1], i32(kept), before, page)
        x = torch.randn(n, V, generator=g) * 3
        y = x + torch.randn(n, V, generator=g)
        self.d = dict(old=i32(self.old), new=i32(self.old + self.more), table0=i32(table), ring0=i32(ring), state=i32(torch.tensor([4, self.n_pages - at])),
                      before=before, qkv=torch.randn(n, Hq + 2 * H, D, generator=g).to(dtype).cuda(), logits=x.cuda(), draft=y.cuda() if draft else None,
                      tokens=i32(torch.cat([torch.zeros(1, dtype=torch.long), x.argmax(1)[:-1]])), u=torch.rand(n, generator=g).cuda(),
                      u_draw=torch.rand(B, generator=g).cuda(), temperature=torch.tensor([1.0, 0.7, 0.0, 0.9, 1.3]).cuda())
        self.o = dict(state_out=e(2), state2=e(2), lens=e(B), lens2=e(B), ok=e(B), ok2=e(B), first=e(B + 1), first2=e(B + 1), slots=e(n + 2), pos=e(n + 2),
                      none=e(0), q=torch.zeros(n + 2, Hq, D, dtype=dtype, device="cuda"), out=torch.zeros(n, Hq, D, dtype=dtype, device="cuda"),
                      lse=torch.zeros(n, Hq, device="cuda"), tokens=e(n), accepted=e(B), cut=e(B), prob=torch.zeros(n, device="cuda"),
                      cache=torch.zeros(self.shape, dtype=torch.uint8, device="cuda"), table=e(B, width), ring=e(self.n_pages),
                      turned=torch.zeros(n, Hq + H, D, dtype=dtype, device="cuda"))
        self.scratch = torch.zeros(n + 2, Hq + 2 * H, D, dtype=dtype, device="cuda")

    def run(self, stream=None):
        d, o, Hq, H = self.d, self.o, self.Hq, self.H
        n, page = self.n, self.page
        if stream is None:
            o["table"].copy_(d["table0"])
            o["ring"].copy_(d["ring0"])
            o["cache"].copy_(d["before"])
            self.scratch[:n].copy_(d["qkv"])
        lm.kv_plan(d["old"], d["new"], o["table"], o["ring"], d["state"], page, state_out=o["state_out"], lens=o["lens"], ok=o["ok"], first=o["first"],
                   slots=o["slots"], pos=o["pos"], stream=stream)
        x = self.scratch
        lm.kv8_append(x[:, Hq:Hq + H], x[:, Hq + H:], o["slots"], o["cache"], page, pos=o["pos"], inv_freq=self.inv, eps=1e-6, k_weight=self.w[1],
                      q=x[:, :Hq], q_out=o["q"], q_weight=self.w[0], stream=stream)
        lm.qk_rope(x[:n, :Hq], o["turned"][:, :Hq], o["pos"][:n], self.inv, k=x[:n, Hq:Hq + H], k_out=o["turned"][:, Hq:], eps=1e-6, q_weight=self.w[0],
                   k_weight=self.w[1], stream=stream)
        lm.kv8_attend(o["q"][:n], o["cache"], o["table"], o["lens"], o["out"], page, first=o["first"], max_new=5, lse=o["lse"], stream=stream)
        lm.verify(d["logits"], d["tokens"], o["first"], d["u"], d["u_draw"], o["tokens"], o["accepted"], max_new=5, draft=d["draft"],
                  temperature=d["temperature"], lens=o["lens"], lens_out=o["cut"], prob=o["prob"], stream=stream)
        lm.kv_plan(o["lens"], o["cut"], o["table"], o["ring"], o["state_out"], page, state_out=o["state2"], lens=o["lens2"], ok=o["ok2"],
                   first=o["first2"], slots=o["none"], stream=stream)

    def clear(self):
        for t in self.o.values():
            t.zero_()

    def results(self):
        torch.cuda.synchronize()
        return {k: v.clone() for k, v in self.o.items()}

    def check(self):
        """Every part against its plain statement, from the parts before it."""
        r = self.results()
        f = lambda t: t.double().cpu().numpy()  # noqa: E731
        n, Hq, H, D, page = self.n, self.Hq, self.H, self.D, self.page
        assert r["ok"].all() and torch.equal(r["lens"].cpu(), (self.old + self.more).int())
        assert torch.equal(r["turned"][:, :Hq], r["q"][:n])                       # one rotation, on the way or not
        pos, slots = r["pos"].cpu().numpy(), r["slots"].cpu().numpy()
        want, tol = S.rope(f(self.d["qkv"][:, :Hq]), pos[:n], self.inv.cpu().numpy(), 1e-6, self.w[0].cpu().numpy())
        assert (np.abs(f(r["q"][:n]) - want) <= tol + R.UNIT["bf16"] * (np.abs(want) + tol)).all()
        want, tol = S.rope(f(self.d["qkv"][:, Hq:Hq + H]), pos[:n], self.inv.cpu().numpy(), 1e-6, self.w[1].cpu().numpy())
        cache = r["cache"].cpu().numpy()
        for i, s in enumerate(slots[:n]):
            for h in range(H):
                k, v = S.get_row(cache[s // page, h], s % page, page, D)
                scale = np.abs(S.parts(cache[s // page, h], page, D)[2][s % page // 32])
                assert (np.abs(k - want[i, h]) <= 2.0 ** -4 * np.abs(want[i, h]) + 2.0 ** -10 * scale[0] + 2 * tol[i, h]).all()
                row = f(self.d["qkv"][i, Hq + H + h])
                assert (np.abs(v - row) <= 2.0 ** -4 * np.abs(row) + 2.0 ** -10 * scale[1]).all()
        out, lse, tol, ltol = S.attend(f(r["q"][:n]), cache, r["table"].cpu().numpy(), r["lens"].cpu().numpy(), r["first"].cpu().numpy(), page,
                                       D ** -0.5, 0, "bf16")
        assert (np.abs(f(r["out"]) - out) <= tol).all() and (np.abs(f(r["lse"]) - lse) <= ltol).all()
        first, draft = r["first"].tolist(), self.d["draft"]
        for b in range(5):
            at = slice(first[b], first[b + 1])
            answers, _ = S.verify_bounds(f(self.d["logits"][at]), None if draft is None else f(draft[at]), self.d["tokens"][at].tolist()[1:],
                                         f(self.d["u"][at]), float(self.d["u_draw"][b]), float(self.d["temperature"][b]), 1.0)
            a = int(r["accepted"][b])
            assert (a, int(r["tokens"][first[b] + a])) in answers
            assert int(r["cut"][b]) == int(self.old[b]) + 1 + a == int(r["lens2"][b])
        assert r["ok2"].all() and int(r["state2"][1]) == int(self.d["state"][1]) + int(((self.old + page - 1) // page).sum()) - int(
            ((r["lens2"].cpu() + page - 1) // page).sum())


def step():
    for kw in (dict(), dict(page=64, D=64, V=20011, draft=False), dict(page=256, D=256, H=1, Hq=4, V=50)):
        s = Step(1, **kw)
        s.run()
        s.check()


def streams():
    """On a stream of its own, made current or given by its handle: the same results."""
    s = Step(1)
    s.run()
    want = s.results()
    side = torch.cuda.Stream()
    for given in (False, True):
        s.clear()
        if given:
            s.o["table"].copy_(s.d["table0"])
            s.o["ring"].copy_(s.d["ring0"])
            s.o["cache"].copy_(s.d["before"])
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            late = s.d["qkv"].clone()
            torch.cuda._sleep(2_000_000)
            s.d["qkv"].zero_()
            s.d["qkv"].copy_(late)
            if not given:
                s.run()
            else:
                s.scratch[:s.n].copy_(s.d["qkv"])
        if given:
            s.run(stream=side.cuda_stream)
        side.synchronize()
        same(s.results(), want)


def graphs():
    """Captured once and replayed, new inputs in between and eager calls of other shapes beside: every replay as eager."""
    s, other = Step(2), Step(3, page=64, D=64, V=30011, long=900)
    s.run()
    other.run()
    torch.cuda.synchronize()
    graph = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    for g, x in zip(graph, (s, other)):
        with torch.cuda.graph(g):
            x.run()
    for turn in range(5):
        for x in (s, other):
            x.d["u"].copy_(torch.rand(x.n, device="cuda"))
            x.d["logits"].copy_(torch.randn(x.n, x.V, device="cuda") * (1 + turn))
            x.d["qkv"].copy_(torch.randn(x.d["qkv"].shape, device="cuda").to(x.d["qkv"].dtype))
            x.clear()
        graph[turn % 2].replay()
        graph[1 - turn % 2].replay()
        got = s.results(), other.results()
        for x, y in zip((s, other), got):
            x.clear()
            x.run()
            same(x.results(), y)
    s.check()
    other.check()


def refusals():
    s = Step(4)
    d, o, n = s.d, s.o, s.n
    s.run()
    torch.cuda.synchronize()

    def refused(kind, text, f, *a, **k):
        try:
            f(*a, **k)
        except kind as e:
            assert text in str(e), (text, str(e))
            return
        raise AssertionError(f"not refused: {text}")

    x = s.scratch[:n]
    q, k, v = x[:, :8], x[:, 8:10], x[:, 10:]
    pos, slots = o["pos"][:n], o["slots"][:n]
    refused(ValueError, "on the GPU", lm.qk_rope, q.cpu(), q, pos, s.inv)
    refused(ValueError, "arrays on", lm.qk_rope, q, o["q"][:n], pos.cpu(), s.inv)
    refused(ValueError, "q_out", lm.qk_rope, q, o["q"][:n].half(), pos, s.inv)
    refused(ValueError, "q_out: missing", lm.qk_rope, q, None, pos, s.inv)
    refused(ValueError, "overlap", lm.qk_rope, q, o["q"][:1].expand(n, 8, 128), pos, s.inv)
    refused(TypeError, "pos", lm.qk_rope, q, o["q"][:n], pos.long(), s.inv)
    refused(TypeError, "inv_freq", lm.qk_rope, q, o["q"][:n], pos, s.inv.double())
    refused(pk.PkError, "turned", lm.qk_rope, q, o["q"][:n], pos, s.inv[:60].contiguous())
    refused(pk.PkError, "NULL positions", lm.qk_rope, q, o["q"][:n], None, s.inv)
    refused(ValueError, "q_weight", lm.qk_rope, q, o["q"][:n], pos, s.inv, eps=0.0, q_weight=s.w[0, :64])
    refused(ValueError, "k: rows", lm.qk_rope, q, o["q"][:n], pos, s.inv, k=k[:3], k_out=o["turned"][:3, 8:])
    refused(ValueError, "requires a gradient", lm.qk_rope, q.float().requires_grad_(), o["q"][:n].float(), pos, s.inv)
    refused(ValueError, "kv8_shape", lm.kv8_append, k, v, slots, o["cache"], 31)
    refused(TypeError, "uint8", lm.kv8_append, k, v, slots, o["cache"].view(torch.int8), 32)
    refused(ValueError, "rows of", lm.kv8_append, k[:, :1], v[:, :1], slots, o["cache"], 32)
    refused(ValueError, "not adjacent", lm.kv8_append, k.transpose(1, 2), v.transpose(1, 2), slots, o["cache"], 32)
    refused(ValueError, "q: rows", lm.kv8_append, k, v, slots, o["cache"], 32, q=q[:2], q_out=o["q"][:2])
    refused(ValueError, "slots", lm.kv8_append, k, v, slots[:3], o["cache"], 32)
    refused(TypeError, "f32, f16 or bf16", lm.kv8_load, o["cache"], slots, k.int(), k.int(), 32)
    refused(ValueError, "kv8_shape", lm.kv8_load, o["cache"], slots, k, v, 0)
    at = [q, o["cache"], o["table"], o["lens"], o["out"], 32]
    refused(ValueError, "query heads", lm.kv8_attend, q[:, :7], *at[1:4], o["out"][:, :7], 32)
    refused(pk.PkError, "without first", lm.kv8_attend, *at)
    refused(ValueError, "kv8_shape", lm.kv8_attend, q, torch.zeros(lm.kv4_shape(4, 2, 128, 32), dtype=torch.uint8, device="cuda"), *at[2:])
    ver = [d["logits"], d["tokens"], o["first"], d["u"], d["u_draw"], o["tokens"], o["accepted"]]
    refused(ValueError, "logits", lm.verify, d["logits"][0], *ver[1:])
    refused(ValueError, "not adjacent", lm.verify, d["logits"].t().contiguous().t(), *ver[1:])
    refused(TypeError, "tokens", lm.verify, ver[0], d["tokens"].long(), *ver[2:])
    refused(ValueError, "draft", lm.verify, *ver, draft=d["draft"][:2])
    refused(ValueError, "draft", lm.verify, *ver, draft=d["draft"].half())
    refused(TypeError, "temperature", lm.verify, *ver, temperature=d["tokens"][:5])
    refused(pk.PkError, "lens_out", lm.verify, *ver, lens_out=o["cut"])
    refused(pk.PkError, "tokens are read", lm.verify, *ver[:5], d["tokens"], ver[6])
    refused(pk.PkError, "workspace", lm.verify, *ver, workspace=torch.zeros(64, dtype=torch.uint8, device="cuda"))
    refused(ValueError, "requires a gradient", lm.verify, d["logits"].clone().requires_grad_(), *ver[1:])
    s.run()
    s.check()


if __name__ == "__main__":
    globals()[sys.argv[1]]()
    torch.cuda.synchronize()
    print("ok", sys.argv[1], flush=True)

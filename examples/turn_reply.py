#!/usr/bin/env python3
"""Speech in, an answer out: sessions' turns decoded by the EOU decoder, answered by a small decoder-only model over one
4-bit paged cache.

    python3 examples/turn_reply.py [--sessions 4] [--reply 24] [--check]

Both models have random weights (the decoder's shape is eou-120m's, the answering model's is given below), so the text
means nothing; the calls are those of a voice agent:

    pk.Decoder.decode        frames of each session's turn -> its tokens, until end of turn
    lm.kv_plan               pages and slots for the turn as a prompt, then for one token more of each session a step
    lm.kv4_store             a layer's new key and value rows into the cache
    lm.kv4_attend            attention over it, prompts and single tokens alike
    lm.sample                the next token of every session
    lm.kv_plan (length 0)    the pages of a session that has answered go back to the ring

Products, norms and rotary positions are torch's.  --check reads the cache back (lm.kv4_load) and compares the last
step's logits with dense attention over it in f32.
"""
import argparse
import os
import sys
import tempfile
import time

import torch     # before the library, so that both use torch's HIP runtime

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
import __graft_entry__ as graft  # noqa: E402

graft.load_package()
from parakeet_amd import lm, pk, synth  # noqa: E402

LAYERS, HEADS, KV_HEADS, DIM, PAGE = 4, 8, 2, 64, 64
WIDTH = HEADS * DIM
I32 = dict(dtype=torch.int32, device="cuda")


class Model:
    """A decoder-only transformer of random weights: grouped heads, rotary positions, gated feed-forward."""

    def __init__(self, vocab: int):
        g = torch.Generator("cuda").manual_seed(0)
        w = lambda *s: (torch.randn(*s, generator=g, device="cuda") * s[-1] ** -0.5).bfloat16()  # noqa: E731
        self.embed = w(vocab, WIDTH) * 8
        self.qkv = [w((HEADS + 2 * KV_HEADS) * DIM, WIDTH) for _ in range(LAYERS)]
        self.out = [w(WIDTH, WIDTH) for _ in range(LAYERS)]
        self.up = [w(8 * WIDTH, WIDTH) for _ in range(LAYERS)]
        self.down = [w(WIDTH, 4 * WIDTH) for _ in range(LAYERS)]
        self.head = w(vocab, WIDTH) * 3
        self.inv = 10000.0 ** (-torch.arange(0, DIM, 2, device="cuda") / DIM)

    @staticmethod
    def norm(x):
        f = x.float()
        return (f * torch.rsqrt((f * f).mean(-1, keepdim=True) + 1e-6)).bfloat16()

    def rope(self, x, pos):
        a = pos.clamp(min=0).float()[:, None] * self.inv
        c, s = a.cos()[:, None], a.sin()[:, None]
        u, v = x.float().chunk(2, -1)
        return torch.cat([u * c - v * s, u * s + v * c], -1).bfloat16()

    def forward(self, tokens, pos, attention):
        """tokens, pos [n] -> logits [n, vocab]; attention(layer, q, k, v) -> [n, heads, dim]."""
        x = self.embed[tokens]
        for i in range(LAYERS):
            qkv = (self.norm(x) @ self.qkv[i].T).view(-1, HEADS + 2 * KV_HEADS, DIM)
            qk = self.rope(qkv[:, :HEADS + KV_HEADS], pos)
            x = x + attention(i, qk[:, :HEADS], qk[:, HEADS:], qkv[:, HEADS + KV_HEADS:]).reshape(-1, WIDTH) @ self.out[i].T
            a, b = (self.norm(x) @ self.up[i].T).chunk(2, -1)
            x = x + (torch.nn.functional.silu(a) * b) @ self.down[i].T
        return (self.norm(x) @ self.head.T).float()


class Sessions:
    """The sessions' pages: a table and a ring of free pages on the device, one cache with all layers."""

    def __init__(self, n: int, longest: int, pages: int):
        self.n, self.longest = n, longest
        self.table = torch.zeros(n, -(-longest // PAGE), **I32)
        self.ring = torch.randperm(pages, device="cuda").to(torch.int32)
        self.state = [torch.tensor([0, pages], **I32), torch.zeros(2, **I32)]
        self.lens = [torch.zeros(n, **I32), torch.zeros(n, **I32)]
        self.ok, self.first = torch.zeros(n, **I32), torch.zeros(n + 1, **I32)
        _, heads, size = lm.kv4_shape(pages, KV_HEADS, DIM, PAGE)
        self.cache = torch.zeros(pages, LAYERS, heads, size, dtype=torch.uint8, device="cuda")

    def plan(self, new_len, most: int):
        """new_len tokens in each session; returns slots and positions of the new ones (at most `most`)."""
        slots, pos = torch.zeros(most, **I32), torch.zeros(most, **I32)
        lm.kv_plan(self.lens[0], new_len, self.table, self.ring, self.state[0], PAGE, state_out=self.state[1], lens=self.lens[1],
                   ok=self.ok, first=self.first, slots=slots, pos=pos)
        self.lens.reverse()
        self.state.reverse()
        return slots, pos

    def attention(self, slots, max_new: int, max_len: int):
        def layer(i, q, k, v):
            cache = self.cache[:, i]
            lm.kv4_store(k, v, slots, cache, PAGE)
            out = torch.empty_like(q)
            lm.kv4_attend(q, cache, self.table, self.lens[0], out, PAGE, first=self.first, max_new=max_new, max_len=max_len)
            return out
        return layer

    def dense(self, slots, b: int, n: int):
        """attention over session b's n tokens as the cache holds them, in f32 (for --check)."""
        t = torch.arange(n, device="cuda")
        held = (self.table[b, t // PAGE] * PAGE + t % PAGE).to(torch.int32)

        def layer(i, q, k, v):
            ks, vs = torch.empty(n, KV_HEADS, DIM, device="cuda"), torch.empty(n, KV_HEADS, DIM, device="cuda")
            lm.kv4_load(self.cache[:, i], held, ks, vs, PAGE)
            qq = q.float().view(KV_HEADS, HEADS // KV_HEADS, DIM)
            p = torch.softmax(qq @ ks.permute(1, 2, 0) * DIM ** -0.5, -1)
            return (p @ vs.permute(1, 0, 2)).reshape(1, HEADS, DIM).bfloat16()
        return layer


def turns(n: int):
    """Tokens of n sessions' turns from the EOU decoder (random weights of eou-120m's shape)."""
    with tempfile.TemporaryDirectory() as tmp:
        path = os.path.join(tmp, "eou.gguf")
        synth.make_shape(path, "eou-120m")
        dec = pk.Decoder.from_gguf(path, n_slots=n)
    res = dec.decode([synth.encoder_frames(u, 30 + 25 * u, dec.info.D) for u in range(n)])
    vocab = dec.info.V1
    dec.close()
    return [torch.tensor([int(t) for t in r["tokens"]] or [0]) for r in res], vocab


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--sessions", type=int, default=4)
    ap.add_argument("--reply", type=int, default=24)
    ap.add_argument("--check", action="store_true")
    a = ap.parse_args()
    prompts, vocab = turns(a.sessions)
    model = Model(vocab)
    lens = [len(p) for p in prompts]
    longest = max(lens) + a.reply + 1
    sessions = Sessions(a.sessions, longest, a.sessions * -(-longest // PAGE) + 2)
    print("turns of", lens, "tokens", flush=True)

    gen = torch.Generator("cuda").manual_seed(1)
    settings = dict(temperature=torch.full((a.sessions,), 0.9, device="cuda"), top_k=torch.full((a.sessions,), 50, **I32),
                    top_p=torch.full((a.sessions,), 0.95, device="cuda"), min_p=torch.full((a.sessions,), 0.02, device="cuda"))
    token = torch.zeros(a.sessions, **I32)
    replies = []

    def choose(logits):
        lm.sample(logits, torch.rand(a.sessions, generator=gen, device="cuda"), token, **settings)
        replies.append(token.clone())

    # the turns as prompts, all sessions in one batch
    total = sum(lens)
    slots, pos = sessions.plan(torch.tensor(lens, **I32), total)
    logits = model.forward(torch.cat(prompts).cuda(), pos, sessions.attention(slots, max(lens), max(lens)))
    choose(logits[sessions.first[1:].long() - 1])
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    for step in range(a.reply - 1):
        slots, pos = sessions.plan(sessions.lens[0] + 1, a.sessions)
        logits = model.forward(token.long(), pos, sessions.attention(slots, 1, longest))
        choose(logits)
    torch.cuda.synchronize()
    took = time.perf_counter() - t0
    if a.check:
        for b in range(a.sessions):
            n = lens[b] + a.reply - 1
            want = model.forward(replies[-2][b:b + 1].long(), pos[b:b + 1], sessions.dense(slots, b, n))
            off = ((logits[b] - want[0]).norm() / want.norm()).item()
            assert off < 0.03, (b, off)
        print("logits of the last step agree with dense attention over the cache", flush=True)
    sessions.plan(torch.zeros(a.sessions, **I32), 0)
    assert sessions.state[0][1].item() == sessions.ring.numel() and not sessions.lens[0].any()
    for b, reply in enumerate(torch.stack(replies, 1).tolist()):
        print(f"session {b}: {reply}")
    print(f"{a.sessions * (a.reply - 1) / took:.0f} tokens/s, {took / max(a.reply - 1, 1) * 1e6:.0f} us a step ({LAYERS} layers)")


if __name__ == "__main__":
    main()

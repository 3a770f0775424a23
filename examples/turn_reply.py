#!/usr/bin/env python3
"""Speech in, an answer out: sessions' turns decoded by the EOU decoder, answered by a small decoder-only model over one
paged cache, of 4 bits or of 8.

    python3 examples/turn_reply.py [--sessions 4] [--reply 24] [--cache 4|8] [--draft 0] [--check]

Both models have random weights (the decoder's shape is eou-120m's, the answering model's is given below), so the text
means nothing; the calls are those of a voice agent:

    pk.Decoder.decode        frames of each session's turn -> its tokens, until end of turn
    lm.kv_plan               pages and slots for the turn as a prompt, then for one token more of each session a step
    lm.kv4_store             a layer's new key and value rows into the cache
    lm.kv4_attend            attention over it, prompts and single tokens alike
    lm.sample                the next token of every session
    lm.kv_plan (length 0)    the pages of a session that has answered go back to the ring

Over the 4-bit cache products, norms and rotary positions are torch's.  With --cache 8 queries and keys are normed for each
head and rotated on the way into the cache:

    lm.kv8_append            a layer's new rows into the cache, keys and queries normed and rotated
    lm.kv8_attend            attention over it

and with --draft N each step brings up to N tokens more, guessed from what followed the last token before:

    lm.verify                which of them stand, by the target's own logits, and the token behind them
    lm.kv_plan               cuts the cache back to those that stand

lm.verify has a temperature and no filters: what lm.sample's top-k, top-p and min-p would leave out is barred in the logits
(torch's part), so that replies are drawn from the same distribution with drafts and without.

--check reads the cache back (lm.kv4_load, lm.kv8_load) and compares the last step's logits with dense attention over it in
f32.
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
        self.norms = 1 + 0.1 * torch.randn(LAYERS, 2, DIM, generator=g, device="cuda")     # of queries and keys, with the 8-bit cache

    @staticmethod
    def norm(x):
        f = x.float()
        return (f * torch.rsqrt((f * f).mean(-1, keepdim=True) + 1e-6)).bfloat16()

    def rope(self, x, pos):
        a = pos.clamp(min=0).float()[:, None] * self.inv
        c, s = a.cos()[:, None], a.sin()[:, None]
        u, v = x.float().chunk(2, -1)
        return torch.cat([u * c - v * s, u * s + v * c], -1).bfloat16()

    def forward(self, tokens, pos, attention, turned=True):
        """tokens, pos [n] -> logits [n, vocab]; attention(layer, q, k, v) -> [n, heads, dim], its queries and keys rotated
        unless it does that itself (turned False)."""
        x = self.embed[tokens]
        for i in range(LAYERS):
            qkv = (self.norm(x) @ self.qkv[i].T).view(-1, HEADS + 2 * KV_HEADS, DIM)
            qk = self.rope(qkv[:, :HEADS + KV_HEADS], pos) if turned else qkv[:, :HEADS + KV_HEADS]
            x = x + attention(i, qk[:, :HEADS], qk[:, HEADS:], qkv[:, HEADS + KV_HEADS:]).reshape(-1, WIDTH) @ self.out[i].T
            a, b = (self.norm(x) @ self.up[i].T).chunk(2, -1)
            x = x + (torch.nn.functional.silu(a) * b) @ self.down[i].T
        return (self.norm(x) @ self.head.T).float()


class Sessions:
    """The sessions' pages: a table and a ring of free pages on the device, one cache with all layers."""

    def __init__(self, n: int, longest: int, pages: int, bits: int, model):
        self.n, self.longest, self.bits, self.model = n, longest, bits, model
        self.table = torch.zeros(n, -(-longest // PAGE), **I32)
        self.ring = torch.randperm(pages, device="cuda").to(torch.int32)
        self.state = [torch.tensor([0, pages], **I32), torch.zeros(2, **I32)]
        self.lens = [torch.zeros(n, **I32), torch.zeros(n, **I32)]
        self.ok, self.first = torch.zeros(n, **I32), torch.zeros(n + 1, **I32)
        _, heads, size = (lm.kv4_shape if bits == 4 else lm.kv8_shape)(pages, KV_HEADS, DIM, PAGE)
        self.cache = torch.zeros(pages, LAYERS, heads, size, dtype=torch.uint8, device="cuda")

    def plan(self, new_len, most: int):
        """new_len tokens in each session; returns slots and positions of the new ones (at most `most`)."""
        slots, pos = torch.zeros(most, **I32), torch.zeros(most, **I32)
        lm.kv_plan(self.lens[0], new_len, self.table, self.ring, self.state[0], PAGE, state_out=self.state[1], lens=self.lens[1],
                   ok=self.ok, first=self.first, slots=slots, pos=pos)
        self.lens.reverse()
        self.state.reverse()
        return slots, pos

    def attention(self, slots, pos, max_new: int, max_len: int):
        at = dict(first=self.first, max_new=max_new, max_len=max_len)

        def layer4(i, q, k, v):
            cache = self.cache[:, i]
            lm.kv4_store(k, v, slots, cache, PAGE)
            out = torch.empty_like(q)
            lm.kv4_attend(q, cache, self.table, self.lens[0], out, PAGE, **at)
            return out

        def layer8(i, q, k, v):
            cache, (wq, wk) = self.cache[:, i], self.model.norms[i]
            turned, out = torch.empty_like(q), torch.empty_like(q)
            lm.kv8_append(k, v, slots, cache, PAGE, pos=pos, inv_freq=self.model.inv, eps=1e-6, k_weight=wk, q=q, q_out=turned, q_weight=wq)
            lm.kv8_attend(turned, cache, self.table, self.lens[0], out, PAGE, **at)
            return out
        return layer4 if self.bits == 4 else layer8

    def dense(self, b: int, n: int):
        """attention over session b's n tokens as the cache holds them, in f32 (for --check)."""
        t = torch.arange(n, device="cuda")
        held = (self.table[b, t // PAGE] * PAGE + t % PAGE).to(torch.int32)
        place = torch.full((1,), n - 1, **I32)

        def layer(i, q, k, v):
            ks, vs = torch.empty(n, KV_HEADS, DIM, device="cuda"), torch.empty(n, KV_HEADS, DIM, device="cuda")
            (lm.kv4_load if self.bits == 4 else lm.kv8_load)(self.cache[:, i], held, ks, vs, PAGE)
            if self.bits == 8:
                turned = torch.empty_like(q)
                lm.qk_rope(q, turned, place, self.model.inv, eps=1e-6, q_weight=self.model.norms[i, 0])
                q = turned
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


def barred(logits, temperature, top_k, top_p, min_p):
    """logits [n, vocab] with the tokens that lm.sample's filters leave out at -inf; the settings are the rows'."""
    x = logits.double()
    weight, order = torch.exp((x - x.amax(-1, keepdim=True)) / temperature[:, None]).sort(dim=-1, descending=True, stable=True)
    rank = torch.arange(x.shape[1], device=x.device)
    weight = weight * (rank < top_k[:, None])
    keep = (weight.cumsum(-1) - weight < top_p[:, None] * weight.sum(-1, keepdim=True)) & (weight >= min_p[:, None] * weight[:, :1]) & (weight > 0)
    keep[:, 0] = True
    return logits.masked_fill(~torch.zeros_like(keep).scatter(1, order, keep), float("-inf"))


def guesses(history, most: int):
    """Up to `most` tokens that followed the last token of a session's history when it was there before."""
    for i in range(len(history) - 2, -1, -1):
        if history[i] == history[-1]:
            return history[i + 1:i + 1 + most]
    return []


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--sessions", type=int, default=4)
    ap.add_argument("--reply", type=int, default=24)
    ap.add_argument("--cache", type=int, choices=(4, 8), default=4)
    ap.add_argument("--draft", type=int, default=0)
    ap.add_argument("--check", action="store_true")
    a = ap.parse_args()
    prompts, vocab = turns(a.sessions)
    model = Model(vocab)
    lens = [len(p) for p in prompts]
    longest = max(lens) + a.reply + a.draft + 2
    sessions = Sessions(a.sessions, longest, a.sessions * -(-longest // PAGE) + 2, a.cache, model)
    print("turns of", lens, "tokens", flush=True)

    gen = torch.Generator("cuda").manual_seed(1)
    uniform = lambda n: torch.rand(n, generator=gen, device="cuda")  # noqa: E731
    settings = dict(temperature=torch.full((a.sessions,), 0.9, device="cuda"), top_k=torch.full((a.sessions,), 50, **I32),
                    top_p=torch.full((a.sessions,), 0.95, device="cuda"), min_p=torch.full((a.sessions,), 0.02, device="cuda"))
    token = torch.zeros(a.sessions, **I32)

    def forward(tokens, slots, pos, max_new, max_len):
        return model.forward(tokens, pos, sessions.attention(slots, pos, max_new, max_len), a.cache == 4)

    # the turns as prompts, all sessions in one batch
    total = sum(lens)
    slots, pos = sessions.plan(torch.tensor(lens, **I32), total)
    logits = forward(torch.cat(prompts).cuda(), slots, pos, max(lens), max(lens))
    lm.sample(logits[sessions.first[1:].long() - 1], uniform(a.sessions), token, **settings)
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    if a.draft:
        replies, steps, fed, logits, took = drafted(a, sessions, forward, token, prompts, uniform, settings)
    else:
        got, fed = [token.clone()], token
        for steps in range(1, a.reply):
            fed = token.clone()
            slots, pos = sessions.plan(sessions.lens[0] + 1, a.sessions)
            logits = forward(token.long(), slots, pos, 1, longest)
            lm.sample(logits, uniform(a.sessions), token, **settings)
            got.append(token.clone())
        torch.cuda.synchronize()
        took = time.perf_counter() - t0
        replies, steps = torch.stack(got, 1).tolist(), max(a.reply - 1, 1)
    if a.check and a.reply > 1:
        held = sessions.lens[0].tolist()
        for b in range(a.sessions):
            n = held[b]
            want = model.forward(fed[b:b + 1].long(), torch.tensor([n - 1], **I32), sessions.dense(b, n), a.cache == 4)
            off = ((logits[b] - want[0]).norm() / want.norm()).item()
            assert off < 0.03, (b, off)
        print("logits of the last step agree with dense attention over the cache", flush=True)
    sessions.plan(torch.zeros(a.sessions, **I32), 0)
    assert sessions.state[0][1].item() == sessions.ring.numel() and not sessions.lens[0].any()
    for b, reply in enumerate(replies):
        print(f"session {b}: {reply}")
    made = sum(len(r) - 1 for r in replies)
    print(f"{made / took:.0f} tokens/s, {took / steps * 1e6:.0f} us a step ({LAYERS} layers)")


def drafted(a, sessions, forward, token, prompts, uniform, settings):
    """Steps that bring each session's last token with what was guessed behind it, until all have their reply.  Returns the
    replies, how many steps, and of the last one the tokens that stood last, their logits and the time of all."""
    t0 = time.perf_counter()
    replies = [[t] for t in token.tolist()]
    accepted, cut = torch.zeros(a.sessions, **I32), torch.zeros(a.sessions, **I32)
    steps = 0
    while any(len(r) < a.reply for r in replies):
        brought = []
        for b, reply in enumerate(replies):
            left = a.reply - len(reply)
            brought.append([reply[-1]] + guesses(prompts[b].tolist() + reply, min(a.draft, left - 1)) if left > 0 else [])
        counts = [len(x) for x in brought]
        n = sum(counts)
        tokens = torch.tensor([t for x in brought for t in x], **I32)
        slots, pos = sessions.plan(sessions.lens[0] + torch.tensor(counts, **I32), n)
        first = sessions.first.clone()
        logits = forward(tokens.long(), slots, pos, max(counts), sessions.longest)
        out = torch.zeros(n, **I32)
        own = torch.repeat_interleave(torch.arange(a.sessions, device="cuda"), torch.tensor(counts, device="cuda"), output_size=n)
        allowed = barred(logits, **{k: v[own] for k, v in settings.items()})
        lm.verify(allowed, tokens, first, uniform(n), uniform(a.sessions), out, accepted, max_new=max(counts), temperature=settings["temperature"],
                  lens=sessions.lens[0], lens_out=cut)
        sessions.plan(cut, 0)
        stood = accepted.tolist()
        got = out.tolist()
        at = 0
        for b, c in enumerate(counts):
            replies[b] += got[at:at + stood[b] + 1] if c else []
            at += c
        steps += 1
    last = (first[:-1] + accepted).long().clamp(max=n - 1)
    done = [c > 0 for c in counts]
    if a.check and not all(done):      # a session that ended earlier has no logits of this step: bring its last token once more
        counts = [1] * a.sessions
        fed = torch.tensor([r[-2] for r in replies], **I32)
        sessions.plan(sessions.lens[0] - 1, 0)
        slots, pos = sessions.plan(sessions.lens[0] + 1, a.sessions)
        return replies, steps, fed, forward(fed.long(), slots, pos, 1, sessions.longest), time.perf_counter() - t0
    return replies, steps, tokens[last], logits[last], time.perf_counter() - t0


if __name__ == "__main__":
    main()

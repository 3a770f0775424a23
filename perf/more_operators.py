"""Performance cases of one decode step with drafted tokens (parakeet_amd.lm): what lies between a decoder-only model's
joint QKV product and its next tokens, over a paged cache held in 8 bits.

  rope     norms of queries and keys for each head, with the position rotation (lm.qk_rope)
  append   rows into the 8-bit paged cache, keys normed and rotated on the way, and back out of it (lm.kv8_append, lm.kv8_load)
  attend   attention over that cache, single tokens and whole prompts (lm.kv8_attend)
  verify   drafted tokens against the target's probabilities, from given uniform numbers (lm.verify)

`own` chooses between the plain forms below (elementary torch operations, 32 bits; angles in 64) and the framework's kernels.

The cache.  Values are 8-bit floating point (sign, 4 exponent bits, 3 of fraction, largest 448, one NaN) under one power
of two 2^e for the 32 tokens of a block and one head, K and V each; e is the smallest, -100 .. 119, that puts the block's
largest magnitude at 448 2^e or below.  A page holds `page` tokens; a (page, kv head) record is K codes [page][D] | V codes
[page/8][32][8][D/32] | [page/32] entries of 16 bytes: the K scale and the V scale in f32, negative where the block
holds a NaN, and 8 bytes of zeros.  In the V codes, entry [a][r][i] has the D/32 channels from r D/32 of token 8a + i.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZEOF = {"f32": 4, "f16": 2, "bf16": 2}
BLOCK, E_MIN, E_MAX = 32, -100, 119


# ---- the cases ----

def listed():
    return [
        # one live session's next token, rotation alone, the smaller model width of the speech encoders (512 = 8 x 64)
        dict(name="rope_one", kind="rope", tokens=1, heads=8, kv_heads=8, dim=64, rot=64, dtype="bf16", norm=False, swap=False,
             far=1000),
        # one layer of a batch of prompts, queries and keys normed for each head, far into their sessions
        dict(name="rope_prompts", kind="rope", tokens=16385, heads=32, kv_heads=8, dim=128, rot=128, dtype="bf16", norm=True,
             swap=False, far=200003),
        # the step of 64 sessions with up to four drafted tokens each: short runs inside blocks that already hold rows
        dict(name="append_step", kind="append", requests=64, new=5, heads=32, kv_heads=8, dim=128, rot=128, dtype="bf16",
             page=64, norm=True, swap=False, far=4097),
        # one layer of a batch of prompts of uneven length, queries rotated in the same call
        dict(name="append_prompts", kind="append", requests=12, new=4095, heads=32, kv_heads=8, dim=128, rot=128, dtype="bf16",
             page=64, norm=True, swap=False, far=8191),
        # one live session's next token, a short turn
        dict(name="attend_one", kind="attend", requests=1, new=1, length=733, heads=8, kv_heads=8, dim=64, dtype="bf16",
             page=64, window=0),
        # a server's step: 64 sessions of uneven length, one of them still empty, four drafted tokens beside the last one
        dict(name="attend_sessions", kind="attend", requests=64, new=5, length=4097, heads=32, kv_heads=8, dim=128,
             dtype="bf16", page=64, window=0),
        # two day-long transcripts held as context, few rows and a long axis
        dict(name="attend_long", kind="attend", requests=2, new=1, length=200003, heads=16, kv_heads=2, dim=128,
             dtype="f16", page=128, window=0),
        # prompts of uneven length, some behind what their session already holds
        dict(name="attend_prompts", kind="attend", requests=4, new=2047, length=4095, heads=32, kv_heads=8, dim=128,
             dtype="bf16", page=64, window=0),
        # long prompts through layers that see the last 1,000 tokens, in f16
        dict(name="attend_window", kind="attend", requests=4, new=4001, length=8191, heads=16, kv_heads=4, dim=128,
             dtype="f16", page=32, window=1000),
        # one live session: four tokens guessed from the text, against the speech decoder's own 8193 token logits
        dict(name="verify_one", kind="verify", requests=1, new=5, vocab=8193, pad=5, dtype="f32", draft=False),
        # 256 sessions over the turn-taking model's vocabulary, drafted by a smaller model
        dict(name="verify_sessions", kind="verify", requests=256, new=6, vocab=1027, pad=0, dtype="f32", draft=True),
        # a server's step over a large vocabulary, drafted by a smaller model
        dict(name="verify_large", kind="verify", requests=64, new=5, vocab=128001, pad=0, dtype="bf16", draft=True),
    ]


def draw(rng):
    def log(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    kind = rng.choice(("rope", "append", "append", "attend", "attend", "attend", "verify", "verify"))
    dim = rng.choice((64, 128, 128, 256))
    page = rng.choice((32, 64, 128, 256))
    rot = rng.choice((dim, dim, dim // 2, 32))
    norm, swap = rng.random() < 0.5, rng.random() < 0.3
    kv_heads = rng.choice((1, 2, 3, 4, 8))
    heads = kv_heads * rng.choice((1, 2, 3, 4, 8))
    width = (heads + kv_heads) * dim
    if kind == "rope":
        return dict(kind=kind, tokens=log(1, 16385 * 40 * 128 // width // 2), heads=heads, kv_heads=kv_heads, dim=dim, rot=rot,
                    dtype=rng.choice(("bf16", "f16", "f32")), norm=norm, swap=swap, far=log(16, 2000003))
    if kind == "append":
        requests = log(1, 256)
        new = rng.choice((1, 1, 5, log(1, max(2, 24000 * 40 * 128 // width // requests))))
        return dict(kind=kind, requests=requests, new=new, heads=heads, kv_heads=kv_heads, dim=dim, rot=rot,
                    dtype=rng.choice(("bf16", "f16", "f32")), page=page, norm=norm, swap=swap, far=log(max(new, 16) + 1, 200003))
    dtype = rng.choice(("bf16", "f16"))
    if kind == "attend":
        window = rng.choice((0, 0, 0, log(1, 2000)))
        width = kv_heads * dim
        if rng.random() < 0.6:      # decode steps, one token or a few drafted ones
            requests = log(1, 512)
            return dict(kind=kind, requests=requests, new=rng.choice((1, 1, 1, 2, 5)),
                        length=log(5, max(6, min(200003, 64 * 4097 * 1024 // (2 * width * requests)))), heads=heads,
                        kv_heads=kv_heads, dim=dim, dtype=dtype, page=page, window=window)
        requests = log(1, 16)
        new = log(16, 2047)
        most = int(4 * 2047 * 4095 * 32 * 128 / (4.0 * requests * new * heads * dim))
        return dict(kind=kind, requests=requests, new=new, length=log(new, max(new + 1, min(16384, most))), heads=heads,
                    kv_heads=kv_heads, dim=dim, dtype=dtype, page=page, window=window)
    vocab, new = log(64, 200001), rng.choice((1, 2, 3, 5, 9))
    return dict(kind=kind, requests=log(1, min(512, max(1, 64 * 5 * 128001 // (vocab * new)))), new=new, vocab=vocab,
                pad=rng.choice((0, 0, 5, 64)), dtype=rng.choice(("f32", "f16", "bf16")), draft=rng.random() < 0.6)


# ---- their inputs ----

def _pages(length, page):
    return (length + page - 1) // page


def prepare(case, seed):
    return globals()["_prepare_" + case["kind"]](case, torch.Generator().manual_seed(seed),
                                                 torch.Generator("cuda").manual_seed(seed))


def _inv_freq(case):
    i = torch.arange(0, case["rot"], 2, dtype=torch.float64)
    return (10000.0 ** (-i / case["rot"])).float().cuda()


def _rows_of_model(N, heads, D, dtype, gd):
    """Rows as a joint product leaves them, with channels of uneven size and heads beside each other."""
    x = torch.randn(N, heads, D, generator=gd, device="cuda")
    x *= torch.exp(0.7 * torch.randn(1, heads, D, generator=gd, device="cuda"))
    return x.to(DTYPES[dtype])


def _spread(most, B, g):
    """Lengths of B requests, spread evenly up to `most`, in an order of the seed's, the first as long as allowed."""
    rank = torch.cat([torch.tensor([B]), torch.randperm(B - 1, generator=g) + 1])
    return (most * rank // B).clamp(min=1)


def _norm_weights(case, gd):
    if not case["norm"]:
        return None, None
    w = 1.0 + 0.3 * torch.randn(2, case["dim"], generator=gd, device="cuda")
    return w[0].contiguous(), w[1].contiguous()


def _prepare_rope(case, g, gd):
    N, Hq, H, D = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
    x = _rows_of_model(N, Hq + 2 * H, D, case["dtype"], gd)            # queries and keys, cut out of a joint QKV product
    pos = torch.randint(0, case["far"], (N,), generator=g)
    if N > 8:
        pos[N - N // 8:] = -1                                          # padding: rows that are left as they are
    wq, wk = _norm_weights(case, gd)
    return dict(kind="rope", q=x[:, :Hq], k=x[:, Hq:Hq + H], pos=pos.to(torch.int32).cuda(), inv_freq=_inv_freq(case), wq=wq, wk=wk,
                eps=1e-6 if case["norm"] else None, swap=case["swap"], q_out=torch.zeros(N, Hq, D, dtype=x.dtype, device="cuda"),
                k_out=torch.zeros(N, H, D, dtype=x.dtype, device="cuda"))


def _prepare_append(case, g, gd):
    B, n, Hq, H, D, page = case["requests"], case["new"], case["heads"], case["kv_heads"], case["dim"], case["page"]
    new = _spread(n, B, g)
    rank = torch.randperm(B, generator=g)
    blocks = torch.randint(0, max((case["far"] - n) // BLOCK, 1), (B,), generator=g)
    start = torch.where(rank % 3 == 0, 0, blocks * BLOCK + rank * 7 % BLOCK)      # what each session holds already
    first = torch.zeros(B + 1, dtype=torch.int64)
    first[1:] = torch.cumsum(new, 0)
    live, N = int(first[-1]), int(first[-1]) + B // 8                  # the slot map is padded behind the last token
    off = start % page                                                 # each session's pages from the one it is in
    held = (off + new + page - 1) // page
    base = torch.cumsum(held, 0) - held
    n_pages = int(held.sum()) + 2
    ids = torch.randperm(n_pages, generator=g)
    b = torch.searchsorted(first[1:], torch.arange(live), right=True)
    t = torch.arange(live) - first[b]
    slots, pos = torch.full((N,), -1), torch.full((N,), -1)
    place = off[b] + t
    slots[:live] = ids[base[b] + place // page] * page + place % page
    pos[:live] = start[b] + t
    inside = torch.arange(BLOCK) < (off % BLOCK)[:, None]              # rows that the first block of a run already holds
    older = ids[base + off // page] * page + off % page // BLOCK * BLOCK
    older = (older[:, None] + torch.arange(BLOCK))[inside]
    x = _rows_of_model(N, Hq + 2 * H, D, case["dtype"], gd)
    back = torch.cat([older, slots[:live]]).to(torch.int32).cuda()
    cache = torch.empty(n_pages, H, page * 2 * D + page // 2, dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 25) // (page * H * D))
    for p in range(0, n_pages, step):
        m = min(step, n_pages - p)
        kv = torch.randn(2, m * page, H, D, generator=gd, device="cuda")
        cache[p:p + m] = _records(kv[0], kv[1], page)
    wq, wk = _norm_weights(case, gd)
    out = torch.bfloat16 if case["dtype"] == "f32" else x.dtype
    return dict(kind="append", page=page, q=x[:, :Hq], k=x[:, Hq:Hq + H], v=x[:, Hq + H:], slots=slots.to(torch.int32).cuda(),
                pos=pos.to(torch.int32).cuda(), inv_freq=_inv_freq(case), wq=wq, wk=wk, eps=1e-6 if case["norm"] else None,
                swap=case["swap"], older=older.numel(), back=back, cache=cache,
                q_out=torch.zeros(N, Hq, D, dtype=x.dtype, device="cuda"),
                k_back=torch.zeros(back.numel(), H, D, dtype=out, device="cuda"),
                v_back=torch.zeros(back.numel(), H, D, dtype=out, device="cuda"))


def _lengths(case, g):
    """(new tokens, tokens held with them) of each request, on the host: spread evenly up to what the case allows, in an
    order and with offsets of the seed's; the first as long as allowed, and one empty where there are many."""
    B, q, n = case["requests"], case["new"], case["length"]
    news = _spread(q, B, g) if q > 8 else torch.full((B,), q)
    lens = _spread(n, B, g)
    lens[1:] -= torch.randint(0, n // (4 * B) + 1, (B - 1,), generator=g)
    lens = torch.maximum(lens, news)
    if B > 8:
        lens[B // 2] = 0      # a session that holds nothing yet: its queries see no key
    return news, lens


def _prepare_attend(case, g, gd):
    B, Hq, H, D, page = case["requests"], case["heads"], case["kv_heads"], case["dim"], case["page"]
    news, lens = _lengths(case, g)
    held = _pages(lens, page)
    total = int(held.sum())
    n_pages = total + 2
    ids = torch.randperm(n_pages, generator=g)
    table = torch.zeros(B, _pages(case["length"], page) + 1, dtype=torch.int64)
    table[torch.arange(table.shape[1]) < held[:, None]] = ids[:total]
    cache = torch.zeros(n_pages, H, page * 2 * D + page // 2, dtype=torch.uint8, device="cuda")
    size = torch.exp(0.7 * torch.randn(2, 1, H, D, generator=gd, device="cuda"))      # channels of uneven size
    step = max(1, (1 << 25) // (page * H * D))
    for p in range(0, n_pages, step):
        n = min(step, n_pages - p)
        kv = torch.randn(2, n * page, H, D, generator=gd, device="cuda") * size
        cache[p:p + n] = _records(kv[0], kv[1], page)
    first = torch.zeros(B + 1, dtype=torch.int64)
    first[1:] = torch.cumsum(news, 0)
    N = int(first[-1])
    q = torch.randn(N, Hq + 2 * H, D, generator=gd, device="cuda").to(DTYPES[case["dtype"]])[:, :Hq]
    out = torch.zeros(N, Hq, D, dtype=q.dtype, device="cuda")
    return dict(kind="attend", page=page, window=case["window"], scale=1.0 / math.sqrt(D), q=q, cache=cache, max_new=case["new"],
                max_len=case["length"], table=table.to(torch.int32).cuda(), lens=lens.to(torch.int32).cuda(),
                first=first.to(torch.int32).cuda(), out=out, lse=torch.zeros(N, Hq, device="cuda"))


def _prepare_verify(case, g, gd):
    B, n, V = case["requests"], case["new"], case["vocab"]
    new = _spread(n, B, g)                                             # the last token and the drafted ones behind it
    first = torch.zeros(B + 1, dtype=torch.int64)
    first[1:] = torch.cumsum(new, 0)
    N = int(first[-1])
    x = torch.randn(N, V + case["pad"], generator=gd, device="cuda") * 2.0
    top = torch.randint(0, V, (N, 12), generator=gd, device="cuda")    # what the model has in mind, over a broad tail
    x.scatter_add_(1, top, 6.0 * torch.rand(N, 12, generator=gd, device="cuda") + 3.0)
    t = 0.5 + 0.8 * torch.rand(2, B, generator=g)
    row = torch.arange(B)
    if B > 8:
        t[0] = torch.where(row % 16 == 7, 0.0, t[0])                   # greedy sessions
    t = t.float().cuda()
    rows = torch.searchsorted(first[1:].cuda(), torch.arange(N, device="cuda"), right=True)
    y = x[:, :V] + 1.0 * torch.randn(N, V, generator=gd, device="cuda")        # the smaller model thinks nearly the same
    y[torch.rand(y.shape, generator=gd, device="cuda") < 0.02] = -math.inf
    x[torch.rand(x.shape, generator=gd, device="cuda") < 0.03] = -math.inf     # tokens that the caller bars
    x, y = x.to(DTYPES[case["dtype"]])[:, :V], y.to(DTYPES[case["dtype"]])
    noise = -torch.log(-torch.log(torch.rand(N, V, generator=gd, device="cuda").clamp(1e-20, 1 - 1e-7)))
    guess = (y.float() / t[1][rows][:, None] + noise).argmax(-1)       # drawn from the draft's own probabilities
    if not case["draft"]:
        guess = torch.where(torch.rand(N, generator=gd, device="cuda") < 0.7, x.float().argmax(-1), guess)
    tokens = torch.cat([guess.new_zeros(1), guess[:-1]])               # what went into the model: row r's draft is tokens[r + 1]
    i32 = dict(dtype=torch.int32, device="cuda")
    lens = torch.randint(n, 5000, (B,), generator=g) + new
    return dict(kind="verify", logits=x, tokens=tokens.to(torch.int32), first=first.to(torch.int32).cuda(),
                draft=y if case["draft"] else None, temperature=t[0].contiguous(), draft_temperature=t[1].contiguous(),
                u=torch.rand(N, generator=gd, device="cuda"), u_draw=torch.rand(B, generator=gd, device="cuda"),
                lens=lens.to(torch.int32).cuda(), max_new=n, out=torch.zeros(N, **i32), accepted=torch.zeros(B, **i32),
                lens_out=torch.zeros(B, **i32), prob=torch.zeros(N, device="cuda"))


# ---- one pass ----

_loaded = []


def _lm():
    if not _loaded:
        import __graft_entry__
        __graft_entry__.load_package()
        from parakeet_amd import lm
        _loaded.append(lm)
    return _loaded[0]


def run(state):
    s = state
    if not own:
        return globals()["_plain_" + s["kind"]](s)
    lm = _lm()
    if s["kind"] == "rope":
        lm.qk_rope(s["q"], s["q_out"], s["pos"], s["inv_freq"], k=s["k"], k_out=s["k_out"], eps=s["eps"], q_weight=s["wq"],
                   k_weight=s["wk"], interleaved=s["swap"])
        return {"q": s["q_out"], "k": s["k_out"]}
    if s["kind"] == "append":
        lm.kv8_append(s["k"], s["v"], s["slots"], s["cache"], s["page"], pos=s["pos"], inv_freq=s["inv_freq"], eps=s["eps"],
                      k_weight=s["wk"], q=s["q"], q_out=s["q_out"], q_weight=s["wq"], interleaved=s["swap"])
        lm.kv8_load(s["cache"], s["back"], s["k_back"], s["v_back"], s["page"])
        return {"q": s["q_out"], "k": s["k_back"], "v": s["v_back"]}
    if s["kind"] == "attend":
        lm.kv8_attend(s["q"], s["cache"], s["table"], s["lens"], s["out"], s["page"], first=s["first"], max_new=s["max_new"],
                      max_len=s["max_len"], scale=s["scale"], window=s["window"], lse=s["lse"])
        return {"out": s["out"], "lse": s["lse"]}
    lm.verify(s["logits"], s["tokens"], s["first"], s["u"], s["u_draw"], s["out"], s["accepted"], max_new=s["max_new"],
              draft=s["draft"], temperature=s["temperature"], draft_temperature=s["draft_temperature"], lens=s["lens"],
              lens_out=s["lens_out"], prob=s["prob"])
    return {"out": s["out"], "accepted": s["accepted"], "lens_out": s["lens_out"], "prob": s["prob"]}


def _rotated(x, w, s):
    """Rows x [N, heads, D] normed (where the state has an eps) and rotated by their positions, in 32 bits."""
    y = x.float()
    if s["eps"] is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + s["eps"]) * w
    angle = s["pos"].double()[:, None] * s["inv_freq"].double()        # 32 bits lose the angles of far positions
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    rot = 2 * s["inv_freq"].numel()
    head, rest = y[..., :rot], y[..., rot:]
    a, b = (head[..., 0::2], head[..., 1::2]) if s["swap"] else (head[..., :rot // 2], head[..., rot // 2:])
    c, d = a * cos - b * sin, a * sin + b * cos
    head = torch.stack([c, d], -1).flatten(-2) if s["swap"] else torch.cat([c, d], -1)
    return torch.cat([head, rest], -1)


def _plain_rope(s):
    live = (s["pos"] >= 0)[:, None, None]
    return {"q": torch.where(live, _rotated(s["q"], s["wq"], s).to(s["q"].dtype), s["q_out"]),
            "k": torch.where(live, _rotated(s["k"], s["wk"], s).to(s["k"].dtype), s["k_out"])}


def _pow2(e):
    """2^e of whole numbers -126 .. 127."""
    return (e.int() + 127 << 23).view(torch.float32)


def _exponent(top):
    """The smallest e with top <= 448 2^e."""
    m, e = torch.frexp(top)
    return torch.where(top == 0, E_MIN, (e - 9 + (m > 0.875).to(e.dtype)).clamp(E_MIN, E_MAX))


def _codes(x, e):
    """Values as bytes under the scale 2^e."""
    y = (x * _pow2(-e)).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)
    return torch.where(torch.isfinite(x), y, 0x7F)


def _values(code, scale):
    return code.view(torch.float8_e4m3fn).float() * scale.abs()


def _top(x):
    return torch.where(torch.isfinite(x), x.abs(), 0.0).amax(-1)


def _records(k, v, page):
    """Whole pages of rows k, v [n page, H, D] as the cache holds them: [n, H, bytes]."""
    H, D = k.shape[1:]
    n, parts, scales = k.shape[0] // page, [], []
    for x in (k, v):
        x = x.float().view(n, page // BLOCK, BLOCK, H, D)
        e = _exponent(_top(x).amax(2))                                 # [n, blocks, H]
        parts.append(_codes(x, e[:, :, None, :, None]).view(n, page, H, D))
        bad = (~torch.isfinite(x)).any(-1).any(2)
        scales.append(torch.where(bad, -_pow2(e), _pow2(e)))
    kc = parts[0].permute(0, 2, 1, 3).reshape(n, H, -1)
    vc = parts[1].view(n, page // 8, 8, H, 32, D // 32).permute(0, 3, 1, 4, 2, 5).reshape(n, H, -1)
    sc = torch.stack(scales + [torch.zeros_like(scales[0])] * 2, -1).transpose(1, 2).reshape(n, H, -1).contiguous()
    return torch.cat([kc, vc, sc.view(torch.uint8)], -1)


def _scales(cache, page, D):
    """The scales as f32 [pages, H, blocks, 4]."""
    return cache[..., 2 * page * D:].contiguous().view(torch.float32).unflatten(-1, (page // BLOCK, 4))


def _code_places(off, page, D):
    """Byte places [rows, D] of K and of V codes at these offsets of their pages."""
    d, per = torch.arange(D, device=off.device), D // 32
    return (off[:, None] * D + d,
            page * D + ((off[:, None] // 8 * 32 + d // per) * 8 + off[:, None] % 8) * per + d % per)


def _plain_append(s):
    """Blocks by their number, page id * blocks of a page + block; the last, past the cache, takes the padding."""
    page, cache, slots = s["page"], s["cache"], s["slots"].long()
    N, H, D = s["k"].shape
    n_pages, per = cache.shape[0], page // BLOCK
    rows = (_rotated(s["k"], s["wk"], s), s["v"].float())
    q = torch.where((s["pos"] >= 0)[:, None, None], _rotated(s["q"], s["wq"], s).to(s["q"].dtype), s["q_out"])
    live, block = slots >= 0, torch.where(slots >= 0, slots // BLOCK, n_pages * per)
    start = torch.full((n_pages * per + 1,), BLOCK, device=cache.device).scatter_reduce(0, block, slots % BLOCK, "amin")
    scales = _scales(cache, page, D)
    older = s["back"][:s["older"]].long()
    at = older // BLOCK
    h = torch.arange(H, device=cache.device)[None, :, None]
    back, found = s["back"].long(), []
    for i, x in enumerate(rows):
        top = torch.zeros(n_pages * per + 1, H, device=cache.device).scatter_reduce(
            0, block[:, None].expand(N, H), _top(x), "amax")
        bad = torch.zeros(n_pages * per + 1, H, device=cache.device).scatter_reduce(
            0, block[:, None].expand(N, H), (~torch.isfinite(x)).any(-1).float(), "amax") > 0
        e, before = _exponent(top)[:-1], scales[..., i].transpose(1, 2).reshape(-1, H).clone()     # [blocks, H]
        old_e = torch.frexp(before.abs())[1] - 1
        kept = (start[:-1] > 0) & (start[:-1] < BLOCK)
        e = torch.where(kept[:, None], torch.maximum(e, old_e), e)
        sign = torch.where(bad[:-1] | (kept[:, None] & (before < 0)), -1.0, 1.0)
        after = torch.where((start[:-1] < BLOCK)[:, None], sign * _pow2(e), before)
        scales[..., i] = after.view(n_pages, per, H).transpose(1, 2)
        place = _code_places(older % page, page, D)[i][:, None].expand(-1, H, D)
        page_of = (older // page)[:, None, None]
        held = _values(cache[page_of, h, place], before[at][..., None])                    # rows held already, rounded anew
        cache[page_of, h, place] = _codes(held, e[at][..., None])
        place = _code_places(slots[live] % page, page, D)[i][:, None].expand(-1, H, D)
        cache[(slots[live] // page)[:, None, None], h, place] = _codes(x[live], e[block[live]][..., None])
        place = _code_places(back % page, page, D)[i][:, None].expand(-1, H, D)            # and back
        found.append(_values(cache[(back // page)[:, None, None], h, place], after[back // BLOCK][..., None]).to(s["k_back"].dtype))
    cache[..., 2 * page * D:] = scales.flatten(-2).contiguous().view(torch.uint8)
    return {"q": q, "k": found[0], "v": found[1]}


def _rows(records, page, D):
    """The values k, v [..., H, page, D] that records [..., H, bytes] stand for."""
    sc = _scales(records, page, D)
    kc = records[..., :page * D].contiguous().unflatten(-1, (page // BLOCK, BLOCK, D))
    vc = records[..., page * D:2 * page * D].contiguous().unflatten(-1, (page // 8, 32, 8, D // 32)).transpose(-3, -2)
    vc = vc.flatten(-4).unflatten(-1, (page // BLOCK, BLOCK, D))
    return (_values(kc, sc[..., 0, None, None]).flatten(-3, -2), _values(vc, sc[..., 1, None, None]).flatten(-3, -2))


def _plain_attend(s):
    """softmax(scale q K^T) V over the keys that query i of request b sees: its own place p = lens - new + i and those
    before it, the last `window` of them where a window is set.  A query that sees none gives zeros, lse -inf."""
    q, table, lens, page, D = s["q"], s["table"].long(), s["lens"].long(), s["page"], s["q"].shape[-1]
    B, Hq, H = table.shape[0], q.shape[1], s["cache"].shape[1]
    used = -(-s["max_len"] // page)
    k, v = _rows(s["cache"][table[:, :used]].transpose(1, 2), page, D)            # [B, H, pages, page, D]
    k, v = k.flatten(2, 3), v.flatten(2, 3)
    L = k.shape[2]
    first = s["first"].long()
    new = first[1:] - first[:-1]
    i = torch.arange(s["max_new"], device=q.device)
    row = (first[:-1, None] + i).clamp(max=q.shape[0] - 1)                        # [B, max_new]
    p = lens[:, None] - new[:, None] + i
    j = torch.arange(L, device=q.device)
    see = (j <= p[..., None]) & (i < new[:, None])[..., None]
    if s["window"]:
        see &= j > p[..., None] - s["window"]
    see = see[:, None, None]                                                      # [B, 1, 1, max_new, L]
    qq = q[row].float().unflatten(2, (H, Hq // H)).permute(0, 2, 3, 1, 4)         # [B, H, G, max_new, D]
    z = torch.matmul(qq.flatten(2, 3), k.transpose(2, 3)).unflatten(2, (Hq // H, -1)) * s["scale"]
    z = z.masked_fill(~see, -math.inf)
    top = z.amax(-1, keepdim=True)
    e = torch.exp(z - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e.flatten(2, 3), v).unflatten(2, (Hq // H, -1)) / torch.where(total == 0, 1.0, total)
    lse = (top + torch.log(total)).squeeze(-1)
    live = i < new[:, None]
    out = torch.zeros(q.shape[0] + 1, Hq, D, device=q.device)
    place = torch.where(live, row, q.shape[0]).flatten()
    out[place] = o.permute(0, 3, 1, 2, 4).flatten(2, 3).flatten(0, 1)
    back = torch.zeros(q.shape[0] + 1, Hq, device=q.device)
    back[place] = lse.permute(0, 3, 1, 2).flatten(2, 3).flatten(0, 1)
    return {"out": out[:-1].to(q.dtype), "lse": back[:-1]}


def _share(total, part):
    """floor(total part / 2^31) of whole numbers."""
    return (total >> 31) * part + (((total & (2 ** 31 - 1)) * part) >> 31)


def _weights(logits, t):
    """round(2^30 exp((x - max) / T)) as whole numbers, so that no sum depends on its order; T <= 0: the first largest alone."""
    x = logits.float()
    x = torch.where(torch.isnan(x), -math.inf, x)
    greedy = ~(t > 0)
    inv = torch.where(greedy, 1.0, 1.0 / t).clamp(max=3e38)
    top = x.amax(-1, keepdim=True)
    z = torch.where(x == top, 0.0, (x - top) * inv[:, None])
    w = torch.where(x == -math.inf, 0, torch.round(torch.exp(z) * 2.0 ** 30).long())
    i = torch.arange(x.shape[1], device=x.device)
    alone = i == torch.where(x == top, i, x.shape[1]).amin(-1, keepdim=True)
    return torch.where(greedy[:, None] & ~alone, 0, w)


def _plain_verify(s):
    """Row r of request b has the target's logits behind token r; its draft is tokens[r + 1], the last row has none.  With
    weights w of the target and v of the draft (as pk_sample has them), p = w / sum w and q = v / sum v, or 1 at the draft where
    no draft logits are given: the draft is accepted while u q < p.  The token behind the accepted ones is drawn, by rising index,
    from max(p - q, 0) in steps of 2^-52, or p without its draft; from w behind the last draft, and where that leaves nothing."""
    x, first = s["logits"], s["first"].long()
    N, V = x.shape
    B, dev = first.numel() - 1, x.device
    row = torch.arange(N, device=dev)
    b = torch.searchsorted(first[1:], row, right=True)
    w = _weights(x, s["temperature"][b])
    W = w.sum(-1)
    iW = torch.where(W > 0, 1.0 / W.clamp(min=1).double(), 0.0)
    d = torch.cat([s["tokens"][1:], s["tokens"].new_zeros(1)]).long()
    last = row == first[1:][b] - 1
    d = torch.where(last | (d < 0) | (d >= V), V, d)                   # none
    at = d.clamp(max=V - 1)[:, None]
    p = torch.where(d < V, w.gather(1, at)[:, 0].double() * iW, 0.0)
    u = (s["u"].clamp(0, 1) * 2.0 ** 31).long().clamp(max=2 ** 31 - 1).double() * 2.0 ** -31
    q = torch.ones_like(p)
    if s["draft"] is not None:
        v = _weights(s["draft"], s["draft_temperature"][b])
        total = v.sum(-1)
        iV = torch.where(total > 0, 1.0 / total.clamp(min=1).double(), 0.0)
        q = v.gather(1, at)[:, 0].double() * iV
    ok = (u * q < p) & (d < V)
    before = torch.where(ok, N, row).flip(0).cummin(0).values.flip(0)  # the next row that is not accepted
    stop = before[first[:-1].clamp(max=N - 1)]
    accepted = stop - first[:-1]
    wr, dr = w[stop], d[stop]
    i = torch.arange(V, device=dev)
    left = torch.where(i == dr[:, None], 0, wr)
    if s["draft"] is not None:
        far = torch.clamp(wr.double() * iW[stop][:, None] - v[stop].double() * iV[stop][:, None], min=0.0)
        left = torch.where((dr < V)[:, None], (far * 2.0 ** 52).long(), wr)
    left = torch.where(left.sum(-1, keepdim=True) > 0, left, wr)
    mass = left.sum(-1)
    draw = (s["u_draw"].clamp(0, 1) * 2.0 ** 31).long().clamp(max=2 ** 31 - 1)
    over = torch.cumsum(left, -1) > _share(mass, draw)[:, None]
    token = torch.where(over, i, V).amin(-1)
    token = torch.where(mass > 0, token, -1)
    out = torch.where(row < stop[b], d, torch.where(row == stop[b], token[b], -1))
    prob = torch.where(out >= 0, w.gather(1, out.clamp(min=0)[:, None])[:, 0].double() * iW, 0.0)
    i32 = lambda t: t.to(torch.int32)  # noqa: E731
    return {"out": i32(out), "accepted": i32(accepted), "lens_out": i32(s["lens"] - (first[1:] - first[:-1] - 1 - accepted)),
            "prob": prob.float()}


# ---- what a pass cannot do without ----

def work(case):
    c = case
    if c["kind"] == "rope":
        live = c["tokens"] - (c["tokens"] // 8 if c["tokens"] > 8 else 0)
        return {"bytes": 2.0 * live * (c["heads"] + c["kv_heads"]) * c["dim"] * SIZEOF[c["dtype"]] + 4.0 * c["tokens"], "flops": 0}
    if c["kind"] == "append":
        B, n = c["requests"], c["new"]
        live = sum(max(1, n * r // B) for r in range(1, B + 1))
        older = sum(r * 7 % BLOCK for r in range(B) if r % 3)
        values, size = live * c["dim"], SIZEOF[c["dtype"]]
        return {"bytes": values * c["heads"] * 2 * size + values * 2 * c["kv_heads"] * (size + 1)
                + (live + older) * c["dim"] * 2 * c["kv_heads"] * 3 + 12.0 * live, "flops": 0}
    if c["kind"] == "attend":
        news, lens = _lengths(c, torch.Generator().manual_seed(1))
        rows, place = int(news.sum()), lens - news     # of a query's place p, its keys: min(p + 1, window)
        low = place.clamp(min=0)
        W = c["window"] or c["length"]
        upto = lambda n: torch.where(n <= W, n * (n + 1) // 2, W * (W + 1) // 2 + (n - W) * W)  # noqa: E731
        pairs = int((upto(lens) - upto(low)).clamp(min=0).sum())
        seen = int(torch.minimum(lens, W - 1 + lens - low).sum())
        return {"bytes": seen * c["kv_heads"] * (c["dim"] * 2 + 0.25) + rows * c["heads"] * (c["dim"] * 4.0 + 4),
                "flops": 4.0 * c["dim"] * c["heads"] * pairs}
    rows = sum(max(1, c["new"] * r // c["requests"]) for r in range(1, c["requests"] + 1))
    drafted = rows - c["requests"] if c["draft"] else 0
    return {"bytes": (rows + drafted) * c["vocab"] * SIZEOF[c["dtype"]] + 16.0 * rows, "flops": 0}


# ---- the same from the definitions, in 64 bits ----

def exact(case, seed):
    return globals()["_exact_" + case["kind"]](case, prepare(case, seed))


def _exact_rows(x, weight, pos, inv_freq, eps, swap):
    """Rows [N, heads, D]: the norm, then one turned pair of channels after the other."""
    y = x.double()
    if eps is not None:
        y = y * torch.rsqrt(y.square().sum(-1, keepdim=True) / y.shape[-1] + eps) * weight.double()
    half = inv_freq.numel()
    turned = y.clone()
    for j in range(half):
        one, two = (2 * j, 2 * j + 1) if swap else (j, half + j)
        z = torch.polar(torch.ones_like(pos, dtype=torch.float64), pos.double() * float(inv_freq[j]))[:, None]
        z = torch.complex(y[..., one], y[..., two]) * z
        turned[..., one], turned[..., two] = z.real, z.imag
    return turned


def _exact_rope(case, s):
    found = {}
    for name in ("q", "k"):
        y = _exact_rows(s[name], s["w" + name], s["pos"], s["inv_freq"], s["eps"], s["swap"])
        found[name] = y * (s["pos"] >= 0)[:, None, None]
    return found


def _exact_round(y):
    """To the nearest 8-bit value, ties to the even code: from the list of all of them."""
    codes = torch.arange(127, device=y.device)
    level = torch.where(codes < 8, codes * 2.0 ** -9, (8 + codes % 8).double() * torch.exp2((codes // 8 - 10).double()))
    a = y.abs().clamp(max=448.0)
    up = torch.searchsorted(level, a).clamp(1, 126)
    low = up - 1
    middle = (level[low] + level[up]) / 2
    code = torch.where((a > middle) | ((a == middle) & (up % 2 == 0)), up, low)
    return torch.where(y < 0, -1.0, 1.0) * level[code]


def _exact_append(case, s):
    page, D, H = case["page"], case["dim"], case["kv_heads"]
    per = page // BLOCK
    q = _exact_rows(s["q"], s["wq"], s["pos"], s["inv_freq"], s["eps"], s["swap"]) * (s["pos"] >= 0)[:, None, None]
    live = s["slots"] >= 0
    slots, back = s["slots"][live].long(), s["back"].long()
    n = s["cache"].shape[0] * per
    runs = torch.full((n,), BLOCK, device="cuda").scatter_reduce(0, slots // BLOCK, slots % BLOCK, "amin")
    found = {"q": q}
    for i, name in enumerate(("k", "v")):
        x = s[name][live].double()
        if name == "k":
            x = _exact_rows(s["k"][live], s["wk"], s["pos"][live], s["inv_freq"], s["eps"], s["swap"])
        top = torch.zeros(n, H, dtype=torch.float64, device="cuda").scatter_reduce(
            0, (slots // BLOCK)[:, None].expand(-1, H), x.abs().amax(-1), "amax")
        e = torch.ceil(torch.log2(torch.where(top > 0, top, 1e-300) / 448.0)).clamp(E_MIN, E_MAX)
        e = torch.where(top > 448.0 * torch.exp2(e), e + 1, torch.where(top <= 448.0 * torch.exp2(e - 1), e - 1, e))
        e = e.clamp(E_MIN, E_MAX)
        held = s["cache"][..., 2 * page * D:].reshape(-1, H, per, 16)[..., 4 * i:4 * i + 4].contiguous().view(torch.float32)[..., 0]
        before = held.transpose(1, 2).reshape(n, H).double().abs()
        e = torch.where(((runs > 0) & (runs < BLOCK))[:, None], torch.maximum(e, torch.log2(before).round()), e)
        old = back[:s["older"]]
        d = torch.arange(D, device="cuda")
        off = old % page
        width = D // 32
        place = off[:, None] * D + d if name == "k" else (
            page * D + off[:, None] // 8 * (8 * D) + d // width * (8 * width) + off[:, None] % 8 * width + d % width)
        code = s["cache"][(old // page)[:, None, None], torch.arange(H, device="cuda")[:, None], place[:, None]].int()
        value = torch.where(code % 128 < 8, (code % 128) * 2.0 ** -9,
                            (8 + code % 8).double() * torch.exp2((code % 128 // 8 - 10).double())) * torch.where(code > 127, -1.0, 1.0)
        value = value * before[old // BLOCK][..., None]
        scale = torch.exp2(e)
        both = torch.cat([value, x]) / scale[back // BLOCK][..., None]
        found[name] = _exact_round(both) * scale[back // BLOCK][..., None]
    return found


def _exact_attend(case, s):
    D, page = case["dim"], case["page"]
    B, Hq, H = case["requests"], case["heads"], case["kv_heads"]
    first, lens, table = s["first"].tolist(), s["lens"].tolist(), s["table"].long()
    codes = torch.arange(128, device="cuda")
    level = torch.where(codes < 8, codes * 2.0 ** -9, (8 + codes % 8).double() * torch.exp2((codes // 8 - 10).double()))
    level = torch.cat([level, -level])
    q = s["q"].double()
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    d = torch.arange(D, device="cuda")
    width = D // 32
    for b in range(B):
        n, new = lens[b], first[b + 1] - first[b]
        if n == 0:
            continue
        t = torch.arange(n, device="cuda")
        pages, off = table[b, t // page], t % page
        places = (off[:, None] * D + d,
                  page * D + off[:, None] // 8 * (8 * D) + d // width * (8 * width) + off[:, None] % 8 * width + d % width)
        for h in range(H):
            rec = s["cache"][:, h]
            scale = rec[:, 2 * page * D:].contiguous().view(torch.float32).view(-1, page // BLOCK, 4).double()
            k, v = (level[rec[pages[:, None], at].long()] * scale[pages, off // BLOCK, i, None] for i, at in enumerate(places))
            for i0 in range(0, new, 512):
                i1 = min(new, i0 + 512)
                p = n - new + torch.arange(i0, i1, device="cuda")
                see = t <= p[:, None]
                if case["window"]:
                    see &= t > p[:, None] - case["window"]
                for hq in range(h * (Hq // H), (h + 1) * (Hq // H)):
                    r = slice(first[b] + i0, first[b] + i1)
                    z = (q[r, hq] @ k.T * s["scale"]).masked_fill(~see, -math.inf)
                    lse[r, hq] = torch.logsumexp(z, -1)
                    out[r, hq] = torch.softmax(z, -1) @ v
    return {"out": out, "lse": lse}


def _exact_verify(case, s):
    """The probabilities of the tokens that come out, request by request; which ones these are is whole numbers."""
    x, y, u, first = s["logits"], s["draft"], s["u"].tolist(), s["first"].tolist()
    tokens, t, td = s["tokens"].tolist(), s["temperature"].tolist(), s["draft_temperature"].tolist()
    prob = torch.zeros(x.shape[0], dtype=torch.float64, device="cuda")
    for b in range(case["requests"]):
        for r in range(first[b], first[b + 1]):
            z = x[r].double()
            p = torch.softmax(z / t[b], -1) if t[b] > 0 else torch.nn.functional.one_hot(z.argmax(), z.numel()).double()
            left = p
            if r + 1 < first[b + 1]:
                d = tokens[r + 1]
                q = torch.zeros_like(p)
                q[d] = 1.0
                if y is not None:
                    q = torch.softmax(y[r].double() / td[b], -1)
                if u[r] * float(q[d]) < float(p[d]):
                    prob[r] = p[d]
                    continue
                left = (p - q).clamp(min=0.0)
                if y is None:
                    left = p * (q == 0)
            run_ = torch.cumsum(left, 0)
            at = min(int(torch.searchsorted(run_, float(s["u_draw"][b]) * run_[-1], right=True)), int(left.nonzero().max()))
            prob[r] = p[at]
            break
    return {"out": None, "accepted": None, "lens_out": None, "prob": prob}

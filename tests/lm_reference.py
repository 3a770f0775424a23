"""The language-model serving operators (include/parakeet_lm.h) in plain numpy, in 64 bits and whole numbers,
written from their definitions."""
import numpy as np

LEVELS = np.array([0, .5, 1, 1.5, 2, 3, 4, 6])
VALUES = np.concatenate([LEVELS, -LEVELS])
UNIT = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}     # unit roundoff


def to_dtype(x, dtype):
    """f64 -> the array a caller would hold (bf16: its 16-bit patterns, rounded to nearest even)."""
    if dtype == "f32":
        return np.asarray(x, np.float32)
    if dtype == "f16":
        return np.asarray(x, np.float16)
    b = np.asarray(x, np.float32).view(np.uint32)
    r = ((b + 0x7FFF + (b >> 16 & 1)) >> 16).astype(np.uint16)
    return np.where((b & 0x7FFFFFFF) > 0x7F800000, np.uint16(0x7FC0), r)


def to_f64(x, dtype):
    if dtype == "bf16":
        return (x.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return np.asarray(x, np.float64)


# ---- the cache ----

def quantise(x):
    """Rows [..., D] f64 -> codes [..., D] (0 .. 15), scale bytes [..., D/32]."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    top = np.abs(b).max(-1)
    bad = ~np.isfinite(b).all(-1)
    top = np.where(bad, 1.0, top)
    e = np.where(top > 0, np.frexp(np.where(top > 0, top, 1.0))[1] - 3, -120)     # top in [4, 8) 2^e
    e = np.clip(np.where(top > 7 * 2.0 ** e, e + 1, e), -120, 125)
    y = np.abs(np.where(bad[..., None], 0.0, b)) / 2.0 ** e[..., None]
    far = np.abs(y[..., None] - LEVELS)
    near = far.min(-1, keepdims=True)
    ties = far == near                        # one or two neighbours: the even code of two
    code = np.where(ties[..., 0::2].any(-1), 2 * ties[..., 0::2].argmax(-1), 2 * ties[..., 1::2].argmax(-1) + 1)
    code = code + 8 * np.signbit(b)
    return np.where(bad[..., None], 0, code).reshape(x.shape).astype(np.uint8), np.where(bad, 255, e + 127).astype(np.uint8)


def value(codes, scales):
    s = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    return VALUES[codes] * np.repeat(s, 32, -1)


def record_bytes(page, D):
    return page * (D + D // 16)


def put_row(rec, off, page, D, k, v):
    """A token's (codes, scales) of K and of V into a record (in place), byte by byte from the layout's description."""
    (kc, ks), (vc, vs) = k, v
    kpart = rec[:page * D // 2].reshape(page, D // 2)
    vpart = rec[page * D // 2:page * D].reshape(page // 8, 16, 8, D // 32)
    kscale = rec[page * D:page * D + page * D // 32].reshape(page, D // 32)
    vscale = rec[page * D + page * D // 32:].reshape(D // 32, page)
    kpart[off] = kc[0::2] | kc[1::2] << 4
    pairs = vc.reshape(16, D // 16)
    vpart[off // 8, :, off % 8] = pairs[:, 0::2] | pairs[:, 1::2] << 4
    kscale[off] = ks
    vscale[:, off] = vs


def get_row(rec, off, page, D):
    """K and V values of a token."""
    def nibbles(b):
        return np.stack([b & 15, b >> 4], -1).reshape(*b.shape[:-1], -1)

    kc = nibbles(rec[:page * D // 2].reshape(page, D // 2)[off])
    vc = nibbles(rec[page * D // 2:page * D].reshape(page // 8, 16, 8, D // 32)[off // 8, :, off % 8]).reshape(-1)
    return (value(kc, rec[page * D:page * D + page * D // 32].reshape(page, D // 32)[off]),
            value(vc, rec[page * D + page * D // 32:].reshape(D // 32, page)[:, off]))


def store(cache, page, D, k, v, slots):
    """k, v [n, H, D] f64 into cache [n_pages, H, bytes] (in place)."""
    (kc, ks), (vc, vs) = quantise(k), quantise(v)
    for i, slot in enumerate(slots):
        if 0 <= slot < cache.shape[0] * page:
            for h in range(cache.shape[1]):
                put_row(cache[slot // page, h], slot % page, page, D, (kc[i, h], ks[i, h]), (vc[i, h], vs[i, h]))


# ---- attention ----

def attend(q, cache, table, lens, first, page, scale, window, dtype):
    """(out, lse, tolerance of out, tolerance of lse) in f64.

    Tolerances, of a query row with probabilities p over keys k, values v:
      a score is off by at most ds = |scale| (2^-20 max|q| sum|k| + 2^-21 sum|q k|): the query is split to about
      2^-21 of its largest value, sums are f32;
      out is rounded to its type (unit), p to bf16 (f16 results: to twice its bits), and sums of p v are f32:
      unit |out| + (2^-8 or 2^-15 + 2 ds + 2^-17) sum p |v|;
      probabilities below 2^-126, f32's least normal number, count as none: 2^-126 sum |v|.
    """
    N, Hq, D = q.shape
    H = cache.shape[1]
    out, lse = np.zeros(q.shape), np.full((N, Hq), -np.inf)
    tol, ltol = np.zeros(q.shape), np.zeros((N, Hq))
    up = 2.0 ** -8 if dtype == "bf16" else 2.0 ** -15
    for b in range(len(lens)):
        n, new = int(lens[b]), int(first[b + 1] - first[b])
        if n <= 0:
            continue
        for h in range(H):
            rows = [get_row(cache[table[b, t // page], h], t % page, page, D) if 0 <= table[b, t // page] < cache.shape[0] else None
                    for t in range(n)]
            fine = np.array([r is not None for r in rows])
            k = np.array([r[0] if r else np.zeros(D) for r in rows])
            v = np.array([r[1] if r else np.zeros(D) for r in rows])
            for i in range(new):
                p = n - new + i
                lo = max(0, p + 1 - window) if window else 0
                at = np.arange(lo, p + 1)
                at = at[fine[at]] if len(at) else at
                if not len(at):
                    continue
                for hq in range(h * (Hq // H), (h + 1) * (Hq // H)):
                    x = q[first[b] + i, hq]
                    z = k[at] @ x * scale
                    m = z.max()
                    e = np.exp(z - m)
                    w = e / e.sum()
                    ds = abs(scale) * (2.0 ** -20 * np.abs(x).max() * np.abs(k[at]).sum(1)
                                       + 2.0 ** -21 * (np.abs(k[at]) @ np.abs(x))).max()
                    out[first[b] + i, hq] = w @ v[at]
                    lse[first[b] + i, hq] = m + np.log(e.sum())
                    tol[first[b] + i, hq] = (UNIT[dtype] * np.abs(w @ v[at]) + (up + 2 * ds + 2.0 ** -17) * (w @ np.abs(v[at]))
                                             + 2.0 ** -126 * np.abs(v[at]).sum(0)
                                             + (2.0 ** -24 if dtype == "f16" else 0))
                    ltol[first[b] + i, hq] = ds + 2.0 ** -19 + 2.0 ** -22 * abs(m)
    return out, lse, tol, ltol


# ---- the page plan ----

def plan(old, new, table, ring, state, page, cap):
    table, ring = table.copy(), ring.copy()
    B, width = table.shape
    n = len(ring)
    head, count = state[0] % n, min(max(state[1], 0), n)
    out = dict(lens=np.array(old), ok=np.zeros(B, np.int32), first=np.zeros(B + 1, np.int32),
               slots=np.full(cap, -1, np.int32), pos=np.full(cap, -1, np.int32))
    lacked = freed = used = t = 0
    for b in range(B):
        o, m = int(old[b]), int(new[b])
        out["first"][b] = t
        if not (0 <= o <= width * page and 0 <= m <= width * page):
            continue
        had, want = -(-o // page), -(-m // page)
        need = max(want - had, 0)
        lacked += need
        if need == 0 or lacked <= count:
            out["ok"][b], out["lens"][b] = 1, m
            for i in range(need):
                table[b, had + i] = ring[(head + lacked - need + i) % n]
                used = lacked
            for j in range(want, had):
                if count + freed < n:
                    ring[(head + count + freed) % n] = table[b, j]
                freed += 1
        for p in range(o, m):
            if out["ok"][b] and t < cap:
                out["slots"][t], out["pos"][t] = table[b, p // page] * page + p % page, p
            t += 1
    out["first"][B] = t
    out["state_out"] = np.array([(head + used) % n, min(count - used + freed, n)], np.int32)
    return dict(out, table=table, ring=ring)


# ---- sampling ----

def sample_bounds(x, u, temperature, top_k, top_p, min_p):
    """What a right pk_sample may answer for one row: dict(tokens, kept=(lo, hi), prob={token: (lo, hi)}).

    Weights are f32 exponentials (relative error below 2^-21 of the f32 steps (x - max) / T and exp, |x - max| / T
    up to 22: 22 * 2^-23 + 2^-23) rounded to whole multiples of 2^-30 of the largest: a token's share is off by at
    most eps = 2^-18 of itself and 2^-30 of the largest weight.  u and top_p are taken to 2^-31.
    """
    x = np.where(np.isnan(x), -np.inf, x).astype(np.float64)
    V = len(x)
    top = x.max()
    if top == -np.inf:
        return dict(tokens={-1}, kept=(0, 0), prob={-1: (0.0, 0.0)})
    order = np.lexsort((np.arange(V), -x))
    if not temperature > 0:
        return dict(tokens={int(order[0])}, kept=(1, 1), prob={int(order[0]): (1.0, 1.0)})
    with np.errstate(invalid="ignore"):
        z = np.where(x == top, 0.0, (x - top) / temperature)
    w = np.where(x == -np.inf, 0.0, np.exp(z))
    eps, grain = 2.0 ** -18, 2.0 ** -30
    k = top_k if 0 < top_k < V else V
    ws = w[order].copy()
    ws[k:] = 0
    total = ws[:k].sum()
    slack = eps * total + k * grain                      # of any sum of weights
    before = np.cumsum(ws) - ws
    p = min(max(top_p, 0.0), 1.0)
    rank = np.arange(V)

    def count(sign):
        keep = (rank < k) & (before < p * total + sign * (2 * slack)) & (ws >= min(min_p, 1.0) * (1 - sign * eps) - sign * grain)
        if sign < 0:
            keep &= ws > grain                           # weights that may round to none
        else:
            keep &= ws > 0.25 * grain
        keep[0] = True
        return int(np.argmin(np.append(keep, False)))    # a prefix
    lo, hi = count(-1), count(+1)
    tokens, prob = set(), {}
    for n in {lo, hi} | (set(range(lo, hi)) if hi - lo < 50 else set()):
        kept = np.zeros(V)
        kept[order[:n]] = ws[:n]
        run = np.cumsum(kept)
        mass = run[-1]
        off = (eps * mass + n * grain) * 2 + 2.0 ** -30 * mass
        lo_t = np.searchsorted(run, u * mass - off, side="right")
        hi_t = min(np.searchsorted(run, u * mass + off, side="right"), V - 1)
        for t in range(lo_t, hi_t + 1):
            if kept[t] > 0:
                tokens.add(int(t))
                a, b_ = (kept[t] * (1 - eps) - grain) / (mass + off), (kept[t] * (1 + eps) + grain) / (mass - off)
                old = prob.get(int(t), (a, b_))
                prob[int(t)] = (min(a, old[0]), max(b_, old[1]))
    return dict(tokens=tokens, kept=(lo, hi), prob=prob)

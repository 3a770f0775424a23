"""The operators of a step with drafted tokens (include/parakeet_lm.h: pk_qk_rope, pk_kv8_*, pk_verify) in plain numpy, in 64
bits, written from their definitions."""
import numpy as np

from lm_reference import UNIT

# the 8-bit codes: sign, 4 exponent bits, 3 of fraction
_c = np.arange(128)
LEVELS = np.where(_c < 8, _c * 2.0 ** -9, (8 + _c % 8) * 2.0 ** (_c // 8 - 10.0))
LEVELS[127] = np.nan
VALUES = np.concatenate([LEVELS, -LEVELS])
E_MIN, E_MAX, BLOCK = -100, 119, 32


# ---- norms and rotation ----

def rope(x, pos, inv_freq, eps=None, weight=None, interleaved=False):
    """(rows, tolerance without the result's own rounding) of x [n, heads, D] f64.

    The norm's factor is an f32 sum of D squares, in 8 adds a lane and 5 across lanes, and three roundings more: off by at most
    2^-19 of itself.  An angle is f64 turns, its rest rounded to f32 (2^-26 turns) and its sine good to 4 units of 2^-24: 2^-21.
    Products and their sum round thrice more, 2^-22.  Values turned are at most |a| + |b|.
    """
    D = x.shape[-1]
    y = x.copy()
    if eps is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * (1.0 if weight is None else weight.astype(np.float64))
    tol = np.abs(y) * (0.0 if eps is None else 2.0 ** -19)
    if inv_freq is not None:
        half = len(inv_freq)
        t = pos.astype(np.float64)[:, None] * inv_freq.astype(np.float64)
        c, s = np.cos(t)[:, None], np.sin(t)[:, None]
        one, two = (np.arange(half) * 2, np.arange(half) * 2 + 1) if interleaved else (np.arange(half), half + np.arange(half))
        a, b = y[..., one], y[..., two]
        out, size = y.copy(), (np.abs(a) + np.abs(b)) * (2.0 ** -21 + 2.0 ** -22 + (0.0 if eps is None else 2.0 ** -19))
        out[..., one], out[..., two] = a * c - b * s, a * s + b * c
        tol[..., one], tol[..., two] = size, size
        y = out
    assert D == y.shape[-1]
    return y, tol


# ---- the cache ----

def round8(y):
    """To the nearest code (0 .. 127 and the sign's 128), ties to the even one; |y| <= 448."""
    a = np.abs(y)
    fine = np.isfinite(a)
    up = np.clip(np.searchsorted(LEVELS[:127], np.where(fine, a, 0.0)), 1, 126)
    low = up - 1
    mid = (LEVELS[low] + LEVELS[up]) / 2
    code = np.where((a > mid) | ((a == mid) & (up % 2 == 0)), up, low)
    return np.where(fine, code + 128 * np.signbit(y), 127).astype(np.uint8)


def exponent(top):
    """The smallest e with top <= 448 2^e."""
    if top == 0:
        return E_MIN
    e = int(np.frexp(top)[1]) - 9
    if top > 448.0 * 2.0 ** e:
        e += 1
    return min(max(e, E_MIN), E_MAX)


def record_bytes(page, D):
    return page * 2 * D + page // 2


def parts(rec, page, D):
    """Views of a record: K codes [page, D], V codes [page/8, 32, 8, D/32], scales [page/32, 4] f32."""
    return (rec[:page * D].reshape(page, D), rec[page * D:2 * page * D].reshape(page // 8, 32, 8, D // 32),
            rec[2 * page * D:].view(np.float32).reshape(page // BLOCK, 4))


def get_codes(rec, off, page, D):
    k, v, _ = parts(rec, page, D)
    return k[off], v[off // 8, :, off % 8].reshape(-1)


def get_row(rec, off, page, D):
    """K and V values of a token."""
    kc, vc = get_codes(rec, off, page, D)
    s = np.abs(parts(rec, page, D)[2][off // BLOCK].astype(np.float64))
    return VALUES[kc] * s[0], VALUES[vc] * s[1]


def put_rows(rec, off, page, D, k, v):
    """Rows k, v [n, D] behind the rows that the block of offset `off` holds already (in place)."""
    n, o0 = len(k), off % BLOCK
    assert o0 + n <= BLOCK
    kc, vc, scales = parts(rec, page, D)
    at = off // BLOCK * BLOCK
    for which, x in enumerate((k, v)):
        fine = np.isfinite(x)
        e = exponent(np.abs(np.where(fine, x, 0.0)).max())
        bad = not fine.all()
        codes = [kc, vc][which]
        if o0:
            before = float(scales[off // BLOCK, which])
            old = int(np.frexp(abs(before))[1]) - 1
            bad |= before < 0
            if e > old:
                for o in range(at, at + o0):
                    c = codes[o] if which == 0 else codes[o // 8, :, o % 8]
                    c[...] = round8(VALUES[c] * abs(before) / 2.0 ** e)
            e = max(e, old)
        y = np.where(fine, np.clip(np.where(fine, x, 0.0) / 2.0 ** e, -448, 448), np.nan)
        for i in range(n):
            c = codes[off + i] if which == 0 else codes[(off + i) // 8, :, (off + i) % 8]
            c[...] = round8(y[i]).reshape(c.shape)
        scales[off // BLOCK, which] = (-1.0 if bad else 1.0) * 2.0 ** e
    scales[off // BLOCK, 2:] = 0


def store(cache, page, D, k, v, slots):
    """k, v [n, H, D] f64 into cache [n_pages, H, bytes] (in place), run by run."""
    slots = [int(s) if 0 <= s < cache.shape[0] * page else -1 for s in slots]
    i = 0
    while i < len(slots):
        j = i + 1
        while j < len(slots) and slots[i] >= 0 and slots[j] == slots[j - 1] + 1 and slots[j] % BLOCK:
            j += 1
        if slots[i] >= 0:
            for h in range(cache.shape[1]):
                put_rows(cache[slots[i] // page, h], slots[i] % page, page, D, k[i:j, h], v[i:j, h])
        i = j


def same_codes(a, b):
    """Whether two codes' arrays are alike, NaNs of either sign and zeros of either sign too."""
    va, vb = VALUES[a], VALUES[b]
    return np.array_equal(va, vb, equal_nan=True)


# ---- attention ----

def attend(q, cache, table, lens, first, page, scale, window, dtype):
    """(out, lse, tolerance of out, tolerance of lse) in f64, as lm_reference.attend's, of attention over the 8-bit cache.

    Tolerances, of a query row with probabilities p over keys k, values v:
      a score is off by at most ds = |scale| (2^-20 max|q| sum|k| + 2^-21 sum|q k|): products are exact, sums are f32;
      out is rounded to its type (unit); p, f32 sums apart, to f16's 11 bits, 2^-11, down to 2^-28 of the largest p,
      and below that to 2^-39 of it: unit |out| + (2^-11 + 2 ds + 2^-17) sum p |v| + 2^-38 sum |v| max p;
      v, in f16 with the largest block's values at 2^8 .. 2^16, to 2^-25: 2^-32 of a value over half the block's largest code,
      2^-39 of the largest |v| that the request's tiles meet.
    """
    N, Hq, D = q.shape
    H = cache.shape[1]
    out, lse = np.zeros(q.shape), np.full((N, Hq), -np.inf)
    tol, ltol = np.zeros(q.shape), np.zeros((N, Hq))
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
            most = np.nanmax(np.abs(v), initial=0.0)
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
                    tol[first[b] + i, hq] = (UNIT[dtype] * np.abs(w @ v[at]) + (2.0 ** -11 + 2 * ds + 2.0 ** -17) * (w @ np.abs(v[at]))
                                             + 2.0 ** -38 * np.abs(v[at]).sum(0) * w.max() + 2.0 ** -39 * most
                                             + (2.0 ** -24 if dtype == "f16" else 0))
                    ltol[first[b] + i, hq] = ds + 2.0 ** -19 + 2.0 ** -22 * abs(m)
    return out, lse, tol, ltol


# ---- verification ----

def weights(x, t):
    """exp((x - max) / T) of a row, the first largest alone where T <= 0."""
    x = np.where(np.isnan(x), -np.inf, x).astype(np.float64)
    if x.max() == -np.inf:
        return np.zeros(len(x))
    if not t > 0:
        w = np.zeros(len(x))
        w[int(x.argmax())] = 1.0
        return w
    with np.errstate(over="ignore"):
        return np.exp(np.where(x == x.max(), 0.0, (x - x.max()) / t))


def verify_bounds(x, y, drafts, u, u_draw, t, td):
    """What a right pk_verify may answer for one request: set of (accepted, token), {(accepted, token): p of the token}.

    Weights are off by 2^-18 of themselves and 2^-30 of the largest (see lm_reference.sample_bounds), so that a share w of a
    total of V weights is off by 2^-17 w + 2^-30 (1 + V w).  u is taken to 2^-31.
    """
    V = x.shape[1]
    off = lambda p: 2.0 ** -17 * p + 2.0 ** -30 * (1 + V * p)  # noqa: E731
    answers, prob = set(), {}
    for j in range(len(drafts) + 1):
        w = weights(x[j], t)
        if w.sum() == 0:
            answers.add((j, -1))
            prob[j, -1] = 0.0
            return answers, prob
        p = w / w.sum()
        d = drafts[j] if j < len(drafts) else -1
        real = 0 <= d < V
        q = None
        may_go, may_stop = False, True
        if real:
            if y is None:
                q = np.zeros(V)
                q[d] = 1.0
            else:
                v = weights(y[j], td)
                q = v / v.sum() if v.sum() else v
            slack = off(p[d]) + u[j] * (off(q[d]) if y is not None else 0) + 2.0 ** -31
            may_go, may_stop = u[j] * q[d] < p[d] + slack, u[j] * q[d] >= p[d] - slack
            if p[d] == 0:
                may_go = False
        if may_stop:
            if not real:
                left, slack = p, V * 2.0 ** -30 + 2.0 ** -17
            elif y is None:
                left = np.where(np.arange(V) == d, 0.0, p)
                slack = V * 2.0 ** -30 + 2.0 ** -17
            else:
                left = np.maximum(p - q, 0.0)
                slack = 2 * (V * 2.0 ** -30 + 2.0 ** -17)
            run = np.cumsum(left)
            at = u_draw * run[-1]
            wide = 2 * slack + 2.0 ** -30
            may = (run >= at - wide) & (run - left <= at + wide) & (left + (off(p) + off(q) if y is not None and real else 0) * (p > 0) > 0)
            if run[-1] <= 2 * slack:                     # what is left may be nothing: then from the target
                may |= p > 0
            for k in np.flatnonzero(may):
                answers.add((j, int(k)))
                prob[j, int(k)] = p[k]
        if not may_go:
            break
    return answers, prob


__all__ = ["UNIT"]

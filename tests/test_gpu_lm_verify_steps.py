"""pk_verify's arithmetic bit for bit: what is left to draw from in single f64 steps, and a row cut either way."""
from fractions import Fraction

import numpy as np
import pytest

from test_gpu_lm_verify import call

pytestmark = pytest.mark.gpu

TOP = 1 << 30                                     # the weight of the largest logit


def weights_of(z):
    """The weights of logits z [n], -5.5 < z < -4.9, beside a largest of 0: whole numbers, from which drafts stand.

    p = w / (2^30 + w) lies between 2^-8 and 2^-7, where f32 holds u = k 2^-31; a draft stands while k 2^-31 < p, and a step of w is
    two of k.  Weights are off by 2^-19 of themselves and half a step, k by less than 70.
    """
    n = len(z)
    x = np.zeros((2 * n, 2), np.float32)
    x[::2, 1] = z
    e = np.exp(z.astype(float))
    low = (e / (1 + e) * 2.0 ** 31).astype(np.int64) - 70          # stands at low, not at high
    high = low + 140
    while (high - low > 1).any():
        mid = (low + high) // 2
        u = np.zeros(2 * n, np.float32)
        u[::2] = mid * 2.0 ** -31
        assert (u[::2].astype(float) * 2.0 ** 31 == mid).all()
        _, stood, _, _ = call(x, None, np.tile([0, 1], n), 2 * np.arange(n + 1), u, np.zeros(n), max_new=2)
        low, high = np.where(stood == 1, mid, low), np.where(stood == 1, high, mid)
    found = []
    for k in high:
        p = (k - 0.5) * 2.0 ** -31
        guess = round(TOP * p / (1 - p))
        fits = [w for w in range(guess - 2, guess + 3) if k - 1 < w * (1.0 / (TOP + w)) * 2.0 ** 31 <= k]
        assert len(fits) == 1, (k, fits)
        found.append(fits[0])
    return found


def steps_left(w, v, total, total_v, fused):
    """max(p - q, 0) in whole steps of 2^-52: p and q rounded ("no"), or one of them not."""
    ip, iq = 1.0 / total, 1.0 / total_v
    if fused == "no":
        d = w * ip - v * iq
    elif fused == "p":
        d = float(Fraction(w) * Fraction(ip) - Fraction(v * iq))
    else:
        d = float(Fraction(w * ip) - Fraction(v) * Fraction(iq))
    return int(d * 2.0 ** 52) if d > 0 else 0


def test_what_is_left_is_taken_in_single_steps():
    """Two tokens whose shares are a weight or two above their draft's leave some 2^23 steps, and a draw that falls on the border between
    them tells whether p or q went into the difference without its rounding."""
    g = np.random.default_rng(0)
    z = np.float32(g.uniform(-5.45, -4.95, 1024))
    z = np.stack([z, np.nextafter(z, np.float32(0))])
    w = np.array(weights_of(z.ravel())).reshape(2, -1)
    close = np.flatnonzero((w[1] - w[0] >= 1) & (w[1] - w[0] <= 2))
    assert len(close) > 100
    cases = []
    want = {"p": 20, "q": 20}
    for _ in range(200000):
        a, b, c = (int(i) for i in g.choice(close, 3, replace=False))
        total, total_v = TOP + int(w[1, a] + w[1, b] + w[0, c]), TOP + int(w[0, a] + w[0, b] + w[0, c])
        left = {f: [steps_left(int(w[1, i]), int(w[0, i]), total, total_v, f) for i in (a, b)] for f in ("no", "p", "q")}
        for f in ("p", "q"):
            if want[f] and left[f][0] != left["no"][0]:
                u = np.float32(left["no"][0] / sum(left["no"]))
                near = [u]
                for _ in range(3):
                    near += [np.nextafter(near[-1], np.float32(1))]
                for _ in range(3):
                    near.insert(0, np.nextafter(near[0], np.float32(0)))
                for u in near:
                    part = int(float(u) * 2.0 ** 31)
                    first = {k: (sum(n) * part >> 31) < n[0] for k, n in left.items()}
                    if first[f] != first["no"]:
                        cases.append((a, b, c, u, 1 if first["no"] else 2))
                        want[f] -= 1
                        break
        if not any(want.values()):
            break
    assert not any(want.values()), want
    n = len(cases)
    for V in (6, 9000, 16385, 17001):
        x, y = (np.full((2 * n, V), -np.inf, np.float32) for _ in range(2))
        x[:, 0] = y[:, 0] = 0
        for i, (a, b, c, _, _) in enumerate(cases):
            x[2 * i, 1], x[2 * i, 2], x[2 * i, 3] = z[1, a], z[1, b], z[0, c]
            y[2 * i, 1], y[2 * i, 2], y[2 * i, 3] = z[0, a], z[0, b], z[0, c]
        out, stood, _, _ = call(x, y, np.tile([0, 4], n), 2 * np.arange(n + 1), np.full(2 * n, 0.5), [k[3] for k in cases], max_new=2)
        assert not stood.any() and list(out[::2]) == [k[4] for k in cases], V


@pytest.mark.parametrize("drafted", [False, True])
@pytest.mark.parametrize("cut", [2048, 4096, 16384])
def test_a_row_cut_either_way_answers_alike(cut, drafted):
    """One barred token more brings a row to another kernel, or another number of threads."""
    g = np.random.default_rng(cut)
    news = [1 + i % 5 for i in range(40)]
    first = np.concatenate([[0], np.cumsum(news)])
    N, B = int(first[-1]), len(news)
    x = (g.standard_normal((N, cut + 1)) * 3).astype(np.float32)
    y = x + (g.standard_normal(x.shape) * 2.0 ** g.integers(-22, 1, (N, 1))).astype(np.float32)
    x[:, cut], y[:, cut] = -np.inf, -np.inf
    tokens = np.concatenate([[0], x.argmax(1)[:-1]])
    u, u_draw, t = g.random(N), g.random(B), 0.5 + g.random(B)
    got = [call(np.ascontiguousarray(x[:, :V]), np.ascontiguousarray(y[:, :V]) if drafted else None, tokens, first, u, u_draw, t=t, td=t, max_new=5)
           for V in (cut, cut + 1)]
    assert all(np.array_equal(a, b) for a, b in zip(*got))

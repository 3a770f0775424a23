"""The numpy statements of the serving operators against independent ones (CPU)."""
import numpy as np
import pytest

import lm_reference as R


def test_quantise_is_nearest_under_its_scale():
    g = np.random.default_rng(0)
    x = g.standard_normal((400, 64)) * np.exp(3 * g.standard_normal((400, 1)))
    x[0] = 0
    x[1, :32] = np.linspace(-7, 7, 32)
    c, s = R.quantise(x)
    v = R.value(c, s)
    top = np.abs(x.reshape(400, 2, 32)).max(-1)
    e = 2.0 ** (s.astype(float) - 127)
    ok = top > 0
    assert (top[ok] <= 7 * e[ok]).all() and (top[ok] > 3.5 * e[ok]).all()
    # nearest level, by trying all of them
    y = x.reshape(400, 2, 32) / e[..., None]
    best = np.abs(y[..., None] - R.VALUES).min(-1)
    assert np.allclose(np.abs(v.reshape(400, 2, 32) / e[..., None] - y), best, atol=1e-12)


@pytest.mark.parametrize("y,code", [(0.25, 0), (0.75, 2), (1.25, 2), (1.75, 4), (2.5, 4), (3.5, 6), (5.0, 6), (6.9, 7)])
def test_quantise_ties_go_to_the_even_code(y, code):
    x = np.zeros((1, 32))
    x[0, 0], x[0, 1] = 6.5, y
    x[0, 2] = -y
    c, s = R.quantise(x)
    assert s[0, 0] == 127 and c[0, 1] == code and c[0, 2] == code + 8


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_quantise_marks_blocks_that_are_not_finite(bad):
    x = np.ones((1, 64))
    x[0, 5] = bad
    c, s = R.quantise(x)
    v = R.value(c, s)
    assert np.isnan(v[0, :32]).all() and (v[0, 32:] == 1).all()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 64])
def test_rows_survive_their_record(D, page):
    g = np.random.default_rng(D + page)
    cache = g.integers(0, 256, (3, 2, R.record_bytes(page, D)), dtype=np.uint8)
    slots = g.permutation(3 * page)[:20]
    k, v = g.standard_normal((2, 20, 2, D))
    before = cache.copy()
    R.store(cache, page, D, k, v, slots)
    for i, s in enumerate(slots):
        for h in range(2):
            a, b = R.get_row(cache[s // page, h], s % page, page, D)
            assert np.array_equal(a, R.value(*R.quantise(k[i, h]))) and np.array_equal(b, R.value(*R.quantise(v[i, h])))
    R.store(before, page, D, k[::-1], v[::-1], slots[::-1])        # rows do not touch one another's bytes
    assert np.array_equal(before, cache)


def test_plan_conserves_pages():
    g = np.random.default_rng(5)
    B, width, page, n = 9, 6, 16, 40
    table = np.zeros((B, width), np.int32)
    ring, state, lens = np.arange(n, dtype=np.int32), np.array([7, n], np.int32), np.zeros(B, np.int32)
    for step in range(60):
        new = g.integers(0, width * page + 1, B).astype(np.int32)
        r = R.plan(lens, new, table, ring, state, page, 1000)
        lens, table, ring, state = r["lens"], r["table"], r["ring"], r["state_out"]
        held = [int(table[b, j]) for b in range(B) for j in range(-(-int(lens[b]) // page))]
        free = [int(ring[(state[0] + i) % n]) for i in range(state[1])]
        assert sorted(held + free) == list(range(n))
        assert ((r["ok"] == 1) == (lens == new)).all()


def test_sample_bounds_hold_the_definition():
    """A direct sampler in 64 bits falls inside the bounds, and they are narrow."""
    g = np.random.default_rng(3)
    for _ in range(200):
        V = int(g.integers(1, 60))
        x = g.standard_normal(V) * 3
        T, k, p, m, u = g.uniform(0.3, 2), int(g.integers(0, V + 2)), g.uniform(0.1, 1.0), g.uniform(0, 0.2), g.uniform()
        w = np.exp((x - x.max()) / T)
        order = np.argsort(-x, kind="stable")[:k if 0 < k < V else V]
        s = w[order]
        keep = (np.cumsum(s) - s < p * s.sum()) & (s >= m)
        keep[0] = True
        kept = np.zeros(V)
        kept[order[keep]] = s[keep]
        token = int(np.searchsorted(np.cumsum(kept), u * kept.sum(), side="right"))
        r = R.sample_bounds(x, u, T, k, p, m)
        assert token in r["tokens"] and r["kept"][0] <= keep.sum() <= r["kept"][1] and len(r["tokens"]) <= 2
        lo, hi = r["prob"][token]
        assert lo <= kept[token] / kept.sum() <= hi

"""pk_sample against sampling in 64 bits: the token, how many were kept and its share have to be ones that rounded
weights allow (lm_reference.sample_bounds); where the answer is a whole-number matter, exactly."""
import numpy as np
import pytest

import lm_reference as R

pytestmark = pytest.mark.gpu
f32 = np.float32


def run(x, u, temperature=None, top_k=None, top_p=None, min_p=None, dtype="f32", stride=None, stream=None):
    from parakeet_amd import hipmem, lm
    B, V = x.shape
    if stride:
        wide = np.full((B, stride), 30000.0, x.dtype) if dtype != "bf16" else np.full((B, stride), 0x4700, np.uint16)
        wide[:, :V] = x
        lg = hipmem.Tensor.from_numpy(wide, dtype).view((B, V), (stride, 1))
    else:
        lg = hipmem.Tensor.from_numpy(x, dtype)
    opt = lambda a, t: None if a is None else hipmem.Tensor.from_numpy(np.ascontiguousarray(a, t))  # noqa: E731
    token, prob, kept = hipmem.Tensor((B,), "i32"), hipmem.Tensor((B,), "f32"), hipmem.Tensor((B,), "i32")
    for t in (token, prob, kept):
        t.zero()
    lm.sample(lg, hipmem.Tensor.from_numpy(np.ascontiguousarray(u, f32)), token, temperature=opt(temperature, f32), top_k=opt(top_k, np.int32),
              top_p=opt(top_p, f32), min_p=opt(min_p, f32), prob=prob, kept=kept, stream=stream)
    hipmem.synchronize()
    return token.numpy(), prob.numpy(), kept.numpy()


def check(x, u, temperature, top_k, top_p, min_p, dtype="f32", stride=None):
    token, prob, kept = run(x, u, temperature, top_k, top_p, min_p, dtype, stride)
    xs = R.to_f64(x, dtype)
    for b in range(len(x)):
        r = R.sample_bounds(xs[b], float(f32(u[b])), float(f32(temperature[b])), int(top_k[b]), float(f32(top_p[b])), float(f32(min_p[b])))
        what = (b, token[b], prob[b], kept[b], r["kept"], sorted(r["tokens"])[:5])
        assert int(token[b]) in r["tokens"], what
        assert r["kept"][0] <= kept[b] <= r["kept"][1], what
        lo, hi = r["prob"][int(token[b])]
        assert lo * (1 - 2.0 ** -22) <= prob[b] <= hi * (1 + 2.0 ** -22), what
    return token, prob, kept


def settings(g, B):
    return (np.where(g.random(B) < 0.1, 0.0, g.uniform(0.2, 1.6, B)), np.where(g.random(B) < 0.4, 0, g.integers(1, 120, B)),
            np.where(g.random(B) < 0.4, 1.0, g.uniform(0.05, 1.0, B)), np.where(g.random(B) < 0.5, 0.0, g.uniform(0, 0.3, B)))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V", [1, 2, 31, 64, 65, 1000, 1027, 8193, 33000])
def test_mixed_settings(V, dtype):
    g = np.random.default_rng(V)
    B = 40 if V < 5000 else 12
    x = g.standard_normal((B, V)) * 2.5
    x[:, g.integers(0, V, 5)] += 6
    x[g.random(x.shape) < 0.05] = -np.inf
    x[0] = -np.inf
    x = R.to_dtype(x, dtype)
    u = g.random(B)
    u[:4] = [0.3, 0.0, np.nextafter(f32(1), f32(0)), 1e-7]
    check(x, u, *settings(g, B), dtype=dtype, stride=(None, V + 5)[V % 2])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_large_vocabularies(dtype):
    g = np.random.default_rng(9)
    for V, B in ((128001, 9), (262147, 3), (1048576, 2)):
        x = g.standard_normal((B, V)) * 2
        x[:, :10] += 7
        check(R.to_dtype(x, dtype), g.random(B), np.full(B, 0.9), np.arange(B) % 3 * 40, np.where(np.arange(B) % 2, 0.92, 1.0),
              np.zeros(B), dtype=dtype)
        check(R.to_dtype(x, dtype), g.random(B), np.full(B, 1.4), np.full(B, V // 3), np.full(B, 0.97), np.full(B, 1e-5), dtype=dtype)


def test_flat_rows_are_exact():
    """Equal logits: equal weights, so every answer is a whole-number one."""
    for V in (1, 7, 64, 1000, 4097, 70000):
        g = np.random.default_rng(V)
        B = 16
        x = np.full((B, V), -3.25, f32)
        u = g.random(B).astype(f32)
        token, prob, kept = run(x, u)
        t = (np.floor(u.astype(np.float64) * 2 ** 31).astype(object) * V * 2 ** 30) // 2 ** 31 // 2 ** 30
        assert np.array_equal(token, t.astype(np.int64)) and (kept == V).all() and (prob == f32(2 ** 30) / f32(V * 2 ** 30)).all()
        k = g.integers(1, V + 1, B)                              # the lowest indices win ties
        token, prob, kept = run(x, u, top_k=k)
        assert (kept == k).all() and (token < k).all()
        p = g.uniform(0.01, 1, B).astype(f32)
        token, prob, kept = run(x, u, top_p=p)
        need = (np.floor(p.astype(np.float64) * 2 ** 31).astype(object) * V * 2 ** 30) // 2 ** 31
        assert (kept == [max(1, -(-int(n) // 2 ** 30)) for n in need]).all() and (token < kept).all()
        token, _, kept = run(x, u, min_p=np.full(B, 1.0))
        assert (kept == V).all()


def test_ties_at_the_cut():
    """Two levels, many ties at the lower one: which of them are kept goes by index."""
    V = 5000
    g = np.random.default_rng(1)
    x = np.full((8, V), 1.0, f32)
    high = g.permutation(V)[:30]
    x[:, high] = 1.5
    x[:, g.permutation(V)[:100]] = -0.0
    x[4:, x[4] == 1.0] = 0.0          # zeros of both signs are one level
    token, prob, kept = run(x, np.linspace(0, 0.999, 8), top_k=np.full(8, 45))
    assert (kept == 45).all()
    for b in range(8):
        order = np.lexsort((np.arange(V), -x[b]))[:45]
        assert token[b] in order
    check(x, np.linspace(0, 0.999, 8), np.full(8, 0.7), np.full(8, 45), np.full(8, 0.8), np.zeros(8))
    check(x, np.linspace(0, 0.999, 8), np.full(8, 0.7), np.zeros(8, int), np.full(8, 0.5), np.zeros(8))


def test_greedy_takes_the_lowest_index():
    x = np.zeros((5, 300), f32)
    x[0, [17, 200]] = 4
    x[1] = -np.inf
    x[2, :] = np.nan
    x[3, :] = -1e30
    x[4, [5, 9]] = np.inf
    for T in (0.0, -1.0, np.nan):
        token, prob, kept = run(x, np.full(5, 0.9), temperature=np.full(5, T))
        assert token.tolist() == [17, -1, -1, 0, 5] and kept.tolist() == [1, 0, 0, 1, 1] and prob.tolist() == [1, 0, 0, 1, 1]
    token, _, kept = run(x, np.full(5, 0.9), temperature=np.full(5, 1e-30))       # as good as greedy, ties shared
    assert token.tolist() == [200, -1, -1, token[3], 9] and kept[0] == 2 and kept[4] == 2


def test_values_that_are_no_numbers():
    x = np.zeros((4, 100), f32)
    x[0, 40:] = np.nan
    x[1, 7] = np.inf
    x[2, :] = np.finfo(f32).min
    x[2, 3] = -np.inf
    x[3, :50] = -np.inf
    token, prob, kept = run(x, np.full(4, 0.999))
    assert kept.tolist() == [40, 1, 99, 50] and token.tolist() == [39, 7, 99, 99]
    for T in (np.inf, 1e30):
        token, prob, kept = run(x, np.full(4, 0.0), temperature=np.full(4, T))
        assert kept.tolist() == [40, 1, 99, 50] and token.tolist() == [0, 7, 0, 50]


def test_filters_at_their_ends():
    g = np.random.default_rng(2)
    x = (g.standard_normal((6, 500)) * 3).astype(f32)
    x[:, 123] = 20
    u = g.random(6)
    for kw in (dict(top_p=np.zeros(6)), dict(top_p=np.full(6, -1.0)), dict(top_p=np.full(6, 1e-12)), dict(top_k=np.ones(6)), dict(min_p=np.full(6, 1.0)),
               dict(min_p=np.full(6, 7.0))):
        token, prob, kept = run(x, u, **kw)
        assert (token == 123).all() and (kept == 1).all() and (prob == 1).all(), kw
    a = run(x, u)
    for kw in (dict(top_p=np.full(6, 1.0)), dict(top_p=np.full(6, 5.0)), dict(top_k=np.zeros(6)), dict(top_k=np.full(6, -3)), dict(top_k=np.full(6, 500)),
               dict(top_k=np.full(6, 10 ** 9)), dict(min_p=np.zeros(6)), dict(min_p=np.full(6, -2.0))):
        b = run(x, u, **kw)
        assert all(np.array_equal(p, q) for p, q in zip(a, b)), kw


def test_frequencies():
    """Even uniform numbers over one row: every token comes as often as its share says, to the count's rounding."""
    g = np.random.default_rng(7)
    V, B = 50, 4096
    x = (g.standard_normal(V) * 1.5).astype(f32)
    token, prob, _ = run(np.tile(x, (B, 1)), (np.arange(B) + 0.5) / B, temperature=np.full(B, 0.8))
    w = np.exp((x.astype(np.float64) - x.max()) / np.float64(f32(0.8)))
    w /= w.sum()
    assert (np.abs(np.bincount(token, minlength=V) - B * w) <= 1.001).all()
    assert np.allclose(prob, w[token], rtol=1e-5)
    assert (np.diff(token) >= 0).all()


@pytest.mark.parametrize("V", [300, 5000, 70000])
def test_few_of_many_equal_logits(V):
    """A small top_k inside more equal logits than any list holds; with fewer logits of any weight than top_k; beside
    logits so far below that they have no weight."""
    g = np.random.default_rng(V)
    B = 8
    x = np.full((B, V), -1.0, f32)
    x[4:, g.permutation(V)[:3]] = 0.25
    u = g.random(B)
    for k in (1, 2, 5, 60, 200, 256, 257):
        token, prob, kept = run(x, u, top_k=np.full(B, k))
        assert (kept == min(k, V)).all()
        for b in range(B):
            assert token[b] in np.lexsort((np.arange(V), -x[b]))[:k]
        check(x, u, np.full(B, 0.6), np.full(B, k), np.full(B, 0.8), np.zeros(B))
    x[:] = -50.0
    x[:, g.permutation(V)[:40]] = (g.standard_normal(40)).astype(f32)
    x[:, 7] = x.max() - 21.52          # as good as none
    token, prob, kept = check(x, u, np.full(B, 1.0), np.full(B, 100), np.full(B, 1.0), np.zeros(B))
    check(x, u, np.full(B, 1.0), np.full(B, 100), np.full(B, 0.7), np.full(B, 0.01))
    assert (x[np.arange(B), token] > -40).all()


def test_every_row_length_up_to_a_few_thousand():
    """Lengths around every number of tokens a thread takes."""
    g = np.random.default_rng(12)
    for V in sorted({64 * i + d for i in (1, 3, 4, 5, 15, 16, 17, 31, 32, 33, 47, 48, 49, 63, 64, 65, 128, 129, 193, 255, 256, 257) for d in (-1, 0, 1)}):
        x = (g.standard_normal((3, V)) * 3).astype(f32)
        check(x, g.random(3), np.full(3, 0.9), np.array([0, 5, 0]), np.array([0.9, 0.9, 1.0]), np.zeros(3))

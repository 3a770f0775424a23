"""pk_verify against what its definition allows (lm_step_reference.verify_bounds), exactly where weights are whole, and by its
distribution."""
import numpy as np
import pytest

import lm_reference as R
import lm_step_reference as S

pytestmark = pytest.mark.gpu


def call(x, y, tokens, first, u, u_draw, dtype="f32", t=None, td=None, lens=None, max_new=None, pad=0, fill=-9):
    from parakeet_amd import hipmem, lm
    put = hipmem.Tensor.from_numpy
    N, V = x.shape

    def rows(a):
        if a is None:
            return None
        wide = np.full((N, V + pad), 7, a.dtype)
        wide[:, :V] = a
        return put(wide, dtype).view((N, V), (V + pad, 1))
    B = len(first) - 1
    i32 = lambda n: put(np.full(n, fill, np.int32))  # noqa: E731
    out, accepted, lens_out, prob = i32(N), i32(B), i32(B), put(np.full(N, -9, np.float32))
    opt = lambda a, ty: None if a is None else put(np.asarray(a, ty))  # noqa: E731
    lm.verify(rows(x), put(np.asarray(tokens, np.int32)), put(np.asarray(first, np.int32)), put(np.asarray(u, np.float32)),
              put(np.asarray(u_draw, np.float32)), out, accepted, max_new=max_new, draft=rows(y), temperature=opt(t, np.float32),
              draft_temperature=opt(td, np.float32), lens=opt(lens, np.int32), lens_out=None if lens is None else lens_out, prob=prob)
    hipmem.synchronize()
    return out.numpy(), accepted.numpy(), lens_out.numpy(), prob.numpy()


def check(seed, V, news, dtype="f32", drafted=True, pad=0, temps=True, extra=0, spread=2.0):
    g = np.random.default_rng(seed)
    first = np.concatenate([[0], np.cumsum(news)])
    B, N = len(news), int(first[-1]) + extra
    x = g.standard_normal((N, V)) * spread
    x[np.arange(N), g.integers(0, V, N)] += 6
    y = x + g.standard_normal((N, V))
    x[g.random((N, V)) < 0.05] = -np.inf
    y[g.random((N, V)) < 0.03] = -np.inf
    with np.errstate(over="ignore"):
        x, y = R.to_dtype(x, dtype), R.to_dtype(y, dtype)
    t, td = (0.4 + g.random(B), 0.4 + g.random(B)) if temps else (None, None)
    if temps and B > 3:
        t[2], td[1] = 0.0, 0.0
    tt, ttd = (np.ones(B), np.ones(B)) if t is None else (t.astype(np.float32).astype(float), td.astype(np.float32).astype(float))
    tokens = np.zeros(N, int)
    xf, yf = R.to_f64(x, dtype), R.to_f64(y, dtype)
    for b in range(B):
        for r in range(first[b], first[b + 1] - 1):
            w = S.weights(yf[r], ttd[b])
            tokens[r + 1] = g.choice(V, p=w / w.sum())
    u, u_draw = g.random(N).astype(np.float32), g.random(B).astype(np.float32)
    lens = g.integers(20, 99, B)
    out, accepted, lens_out, prob = call(x, y if drafted else None, tokens, first, u, u_draw, dtype, t, td, lens, max(news), pad)
    for b in range(B):
        r = slice(first[b], first[b + 1])
        n = first[b + 1] - first[b]
        if n == 0:
            assert accepted[b] == 0 and lens_out[b] == lens[b]
            continue
        drafts = tokens[r][1:]
        answers, p = S.verify_bounds(xf[r], yf[r] if drafted else None, drafts, u[r].astype(float), float(u_draw[b]), tt[b], ttd[b])
        a = int(accepted[b])
        token = int(out[first[b] + a])
        assert (a, token) in answers, (b, a, token)
        assert np.array_equal(out[r][:a], drafts[:a]) and (out[r][a + 1:] == -1).all() and (prob[r][a + 1:] == 0).all()
        assert lens_out[b] == lens[b] - (n - 1 - a)
        for j in range(a):
            w = S.weights(xf[first[b] + j], tt[b])
            assert abs(prob[first[b] + j] - w[drafts[j]] / w.sum()) <= 2.0 ** -16 * prob[first[b] + j] + 2.0 ** -30 * (1 + V)
        assert abs(prob[first[b] + a] - p[a, token]) <= 2.0 ** -16 * p[a, token] + 2.0 ** -30 * (1 + V * p[a, token])
    assert (out[first[-1]:] == -9).all() and (prob[first[-1]:] == -9).all()             # rows of no request
    return accepted


@pytest.mark.parametrize("V", [1, 2, 63, 64, 65, 300, 1023, 1024, 1025, 2048, 2049, 4096, 4097, 8193, 16384, 16385, 32001, 70001])
@pytest.mark.parametrize("drafted", [False, True])
def test_vocabularies(V, drafted):
    check(V, V, [5, 1, 3, 2, 0, 4], drafted=drafted)
    check(V + 1, V, [1], drafted=drafted, pad=3)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("V", [50, 1027, 9000, 40000])
def test_types_strides_and_rows_of_no_request(dtype, V):
    for drafted in (False, True):
        check(V, V, [3, 2, 5, 1, 1, 2], dtype, drafted, pad=5, extra=3)
        check(V + 7, V, [2, 3], dtype, drafted, temps=False)


def test_many_requests():
    a = check(5, 130, [1 + i % 6 for i in range(600)])
    assert a.min() == 0 and a.max() >= 3
    check(6, 17000, [1 + i % 3 for i in range(90)])


def test_many_drafts():
    """Longer drafts than a wave has lanes, accepted whole and refused far in."""
    V, n = 40, 150
    for V in (40, 17000):
        x = np.zeros((2 * n, V), np.float32)
        x[:, 7] = 90.0                                  # all weight at one token
        x[n + 100, 7], x[n + 100, 9] = 0.0, 90.0
        tokens = np.full(2 * n, 7)
        out, acc, lens, prob = call(x, None, tokens, [0, n, 2 * n], np.full(2 * n, 0.5), [0.5, 0.5], lens=[500, 500], max_new=n)
        assert list(acc) == [n - 1, 100] and list(lens) == [500, 500 - 49]
        assert (out[:n] == 7).all() and (out[n:n + 100] == 7).all() and out[n + 100] == 9 and (out[n + 101:] == -1).all()
        assert (prob[:n] == 1).all() and (prob[n + 101:] == 0).all()


@pytest.mark.parametrize("V", [8, 20000])
def test_whole_weights(V):
    """Logits that are all alike or barred: shares are exact, and so are the answers at and beside every border."""
    x = np.full((2, V), -np.inf, np.float32)
    x[:, :8] = 1.5                                       # p = 1/8 each
    y = np.full((2, V), -np.inf, np.float32)
    y[:, 2:6] = -3.0                                     # q = 1/4 each: half of these drafts stand
    up = 2.0 ** -20
    for u, ok in ((0.0, 1), (0.5 - up, 1), (0.5, 0), (0.5 + up, 0)):
        out, acc, _, prob = call(x, y, [0, 4], [0, 2], [u, 0], [0.0])
        assert acc[0] == ok and out[0] == (4 if ok else 0) and prob[0] == 0.125
        assert out[1] == (0 if ok else -1)
    # refused: what is left is 1/8 each at 0, 1, 6, 7
    for u, token in ((0.0, 0), (0.25 - up, 0), (0.25, 1), (0.5, 6), (0.75 - up, 6), (0.75, 7), (1 - 2.0 ** -24, 7)):
        assert call(x, y, [0, 4], [0, 2], [0.9, 0], [u])[0][0] == token
    # drafts that were not drawn stand with p, and leave the others
    for u, ok in ((0.125 - up, 1), (0.125, 0)):
        out, acc, _, _ = call(x, None, [0, 4], [0, 2], [u, 0], [4 / 7 - up])
        assert acc[0] == ok and out[0] == (4 if ok else 3)
    assert call(x, None, [0, 4], [0, 2], [0.5, 0], [4 / 7 + up])[0][0] == 5
    # behind the last draft from the target
    assert call(x, y, [0, 4], [0, 2], [0, 0], [0.5])[0][1] == 4
    # a draft that the draft's own logits bar, and one that the target bars
    assert call(x, y, [0, 7], [0, 2], [0.99, 0], [0.5])[0][0] == 7
    y[0, 9 % V if V > 9 else 7] = -3.0
    if V > 9:
        out, acc, _, prob = call(x, y, [0, 9], [0, 2], [0.0, 0], [0.0])
        assert acc[0] == 0 and out[0] == 0 and prob[0] == 0.125
    # alike distributions: every draft stands but for u q = p, which no u below 1 gives
    assert call(x, x, [0, 3], [0, 2], [1 - 2.0 ** -24, 0], [0.0])[1][0] == 1
    # nothing is left where q has all that p has (a draft outside of both): from the target
    assert call(x, x, [0, V - 1], [0, 2], [0.5, 0], [0.5])[0][0] == 4 or V == 8


@pytest.mark.parametrize("V", [12, 17001])
def test_drafts_outside_the_vocabulary_and_barred_rows(V):
    x = np.zeros((4, V), np.float32)
    x[:, 3] = 50
    for bad in (-1, V, 2 ** 31 - 1, -2 ** 31):
        out, acc, _, prob = call(x, None, [0, 3, bad, 3], [0, 4], [0.5] * 4, [0.5])
        assert acc[0] == 1 and list(out) == [3, 3, -1, -1]
    x[1] = -np.inf
    for y in (None, np.zeros_like(x)):
        out, acc, _, prob = call(x, y, [0, 3, 3, 3], [0, 4], [1e-9] * 4, [0.5])
        assert acc[0] == 1 and list(out) == [3, -1, -1, -1] and prob[1] == 0
    x[1] = np.nan
    assert list(call(x, None, [0, 3, 3, 3], [0, 4], [0.5] * 4, [0.5])[0]) == [3, -1, -1, -1]
    x[1] = 0
    x[1, [2, 5]] = np.inf
    assert call(x, None, [0, 3, 5, 3], [0, 4], [0.25] * 4, [0.9])[1][0] == 3


def test_greedy_rows_take_the_first_largest():
    for V in (70, 20000):
        x = np.zeros((3, V), np.float32)
        x[:, [5, 60]] = 4
        for d, want in ((5, [5, 5, 5]), (60, [5, -1, -1])):
            for u in (0.0, 0.999):
                out, acc, _, prob = call(x, None, [0, d, d], [0, 3], [u] * 3, [0.99], t=[0.0])
                assert list(out) == want and acc[0] == (2 if d == 5 else 0) and prob[0] == 1


@pytest.mark.parametrize("V", [70, 20000, 70000])
def test_infinite_logits_count_as_the_largest_number(V):
    x = np.zeros((2, V), np.float32)
    x[:, 9], x[:, 12], x[:, V - 1] = np.inf, np.finfo(np.float32).max, np.inf
    assert list(call(x, None, [0, 9], [0, 2], [0.5] * 2, [0.99], t=[0.0])[0]) == [9, 9]
    x[:, 9], x[:, 12] = np.finfo(np.float32).max, np.inf
    assert list(call(x, None, [0, 9], [0, 2], [0.5] * 2, [0.99], t=[0.0])[0]) == [9, 9]
    assert list(call(x, None, [0, 12], [0, 2], [0.3] * 2, [0.4])[0]) == [12, 12]


def test_counts_cut_first_and_out_of_range_offsets():
    V = 30
    x = np.zeros((6, V), np.float32)
    x[:, 3] = 60
    out, acc, lens, _ = call(x, None, [0, 3, 3, 3, 3, 3], [0, 6], [0.5] * 6, [0.5], lens=[50], max_new=3)
    assert acc[0] == 2 and list(out) == [3, 3, 3, -9, -9, -9] and lens[0] == 50
    out, acc, _, _ = call(x, None, [0, 3, 3, 3, 3, 3], [-5, 2, 900, 4], [0.5] * 6, [0.5] * 3, max_new=9)
    assert list(acc) == [1, 3, 0] and (out == 3).all()


@pytest.mark.parametrize("drafted", [False, True])
def test_distribution(drafted):
    """60,000 drafts of one row: the first token out has the target's probabilities, within 6 standard deviations."""
    g = np.random.default_rng(8)
    V, B, turns = 9, 4096, 15
    x = (g.standard_normal(V) * 1.5).astype(np.float32)
    y = (g.standard_normal(V) * 1.5).astype(np.float32)
    p, q = (S.weights(a.astype(float), 1.0) for a in (x, y))
    p, q = p / p.sum(), q / q.sum()
    count = np.zeros(V)
    for _ in range(turns):
        drafts = g.choice(V, B, p=q) if drafted else np.full(B, 4)
        tokens = np.stack([np.zeros(B, int), drafts], 1).ravel()
        out, acc, _, _ = call(np.tile(x, (2 * B, 1)), np.tile(y, (2 * B, 1)) if drafted else None, tokens, 2 * np.arange(B + 1), g.random(2 * B),
                              g.random(B), max_new=2)
        count += np.bincount(out.reshape(B, 2)[:, 0], minlength=V)
    n = B * turns
    assert (np.abs(count / n - p) <= 6 * np.sqrt(p * (1 - p) / n)).all()


def test_calls_repeat_and_leave_their_workspace_ready():
    g = np.random.default_rng(9)
    for V in (700, 20000):
        x = g.standard_normal((40, V)).astype(np.float32) * 3
        first, tokens, u, d = np.arange(0, 41, 4), x.argmax(1), g.random(40) * 0.5, g.random(10)
        tokens = np.concatenate([[0], tokens[:-1]])
        a = call(x, None, tokens, first, u, d, max_new=4)
        for _ in range(3):
            b = call(x, None, tokens, first, u, d, max_new=4)
            assert all(np.array_equal(i, j) for i, j in zip(a, b))

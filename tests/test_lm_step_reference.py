"""The plain statements of tests/lm_step_reference.py against torch's 8-bit type and against a distribution."""
import numpy as np
import pytest

import lm_step_reference as S


def test_levels_and_rounding_are_the_types():
    torch = pytest.importorskip("torch")
    codes = torch.arange(256, dtype=torch.uint8)
    assert np.array_equal(codes.view(torch.float8_e4m3fn).double().numpy(), S.VALUES, equal_nan=True)
    g = np.random.default_rng(0)
    edges = np.concatenate([S.LEVELS[:127], (S.LEVELS[:126] + S.LEVELS[1:127]) / 2])
    y = np.concatenate([edges, -edges, edges * (1 + 2.0 ** -20), np.clip(g.standard_normal(5000) * 2.0 ** g.integers(-10, 8, 5000), -448, 448)])
    y = np.clip(y, -448, 448).astype(np.float32).astype(np.float64)
    want = torch.from_numpy(y.astype(np.float32)).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(S.round8(y), want)


def test_scale_is_the_smallest():
    for top in (1e-40, 2.0 ** -101, 0.3, 447.9, 448.0, 448.1, 1e38):
        e = S.exponent(top)
        assert top <= 448.0 * 2.0 ** e or e == S.E_MAX
        assert top > 448.0 * 2.0 ** (e - 1) or e == S.E_MIN
    assert S.exponent(0.0) == S.E_MIN


def test_rows_come_back():
    g = np.random.default_rng(1)
    page, D = 64, 64
    rec = g.integers(0, 256, S.record_bytes(page, D), dtype=np.uint8)
    k, v = g.standard_normal((2, 20, D))
    S.put_rows(rec, 32, page, D, k[:5], v[:5])
    S.put_rows(rec, 37, page, D, 40 * k[5:], 40 * v[5:])                  # the scale grows
    for i in range(20):
        a, b = S.get_row(rec, 32 + i, page, D)
        f = 1 if i < 5 else 40
        assert (np.abs(a - f * k[i]) <= 2.0 ** -4 * np.abs(f * k[i]) + 2.0 ** -9 * 1.0).all()
        assert (np.abs(b - f * v[i]) <= 2.0 ** -4 * np.abs(f * v[i]) + 2.0 ** -9 * 1.0).all()


def test_rotation_keeps_lengths_and_differences():
    g = np.random.default_rng(2)
    inv = (10000.0 ** (-np.arange(0, 64, 2) / 64)).astype(np.float32)
    x = g.standard_normal((2, 1, 64))
    for swap in (False, True):
        a, _ = S.rope(np.repeat(x[:1], 3, 0), np.array([5, 1005, 7]), inv, interleaved=swap)
        b, _ = S.rope(np.repeat(x[1:], 3, 0), np.array([2, 1002, 7]), inv, interleaved=swap)
        assert np.allclose((a * a).sum(-1), (x[0] * x[0]).sum())
        dots = (a * b).sum(-1)[:, 0]
        assert np.isclose(dots[0], dots[1]) and np.isclose(dots[2], (x[0] * x[1]).sum())


def test_verified_tokens_are_distributed_as_the_target():
    """Over a grid of both uniform numbers the first token out has the target's probabilities."""
    x = np.log(np.array([[0.5, 0.2, 0.2, 0.1], [0.25] * 4]))
    y = np.log(np.array([[0.1, 0.6, 0.1, 0.2], [0.25] * 4]))
    n, count = 40, np.zeros(4)
    for d, share in enumerate(np.exp(y[0])):
        for i in range(n):
            for k in range(n):
                u = np.array([(i + 0.5) / n, 0.0])
                p, q = np.exp(x[0]), np.exp(y[0])
                if u[0] * q[d] < p[d]:
                    count[d] += share / n / n
                else:
                    left = np.maximum(p - q, 0)
                    count[int(np.searchsorted(np.cumsum(left), (k + 0.5) / n * left.sum(), side="right"))] += share / n / n
                answers, _ = S.verify_bounds(x, y, [d], u, (k + 0.5) / n, 1.0, 1.0)
                assert len({a for a, _ in answers}) == 1
    assert np.allclose(count, np.exp(x[0]), atol=1.0 / n)

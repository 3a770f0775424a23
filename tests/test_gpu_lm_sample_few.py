"""A small top_k over fewer tokens of any weight than that, beside more than a thousand whose logits lie just so far below
the largest that their weights round to none (exp(-21.55) 2^30 < 1/2) while a count by logits still has them."""
import numpy as np
import pytest

import test_gpu_lm_sample as S

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V", [5000, 16385, 70000])
@pytest.mark.parametrize("band", [1100, 4500, None])
@pytest.mark.parametrize("spread", [0.0, 0.05])
def test_tokens_without_weight_take_no_place(V, band, spread):
    g = np.random.default_rng(V + (band or 0))
    B = 8
    order = g.permutation(V)
    live, low = order[:40], order[40:band and 40 + band]
    x = np.full((B, V), -60.0, np.float32)
    x[:, live] = 3 * g.random((B, 40))
    x[:, live[0]] = 4.0
    x[:, low] = 4.0 - 21.55 + spread * (g.random((B, len(low))) - 0.5)
    u = g.random(B)
    for top_k in (41, 100, 256, 257):
        for top_p in (1.0, 0.9, 0.3):
            for min_p in (0.0, 0.2):
                kw = dict(top_p=np.full(B, top_p), min_p=np.full(B, min_p))
                got = S.run(x, u, top_k=np.full(B, top_k), **kw)
                assert all(np.array_equal(a, b) for a, b in zip(got, S.run(x, u, **kw))), (top_k, top_p, min_p)
                if top_p == 1 and min_p == 0:
                    assert (got[2] == 40).all()
        S.check(x, u, np.ones(B), np.full(B, top_k), np.full(B, 0.7), np.zeros(B))

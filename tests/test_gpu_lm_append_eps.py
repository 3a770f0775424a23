"""pk_kv8_append with a norm whose eps is 0: rows beside the call's are no part of it, and a block is marked for its own NaNs alone."""
import numpy as np
import pytest

import lm_reference as R
import lm_step_reference as S

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("D,half,interleaved", [(64, 32, False), (128, 64, False), (256, 128, False), (128, 16, False), (128, 64, True), (128, 0, False)])
@pytest.mark.parametrize("n", [1, 5, 31])
def test_blocks_without_a_nan_are_not_marked(dtype, D, half, interleaved, n):
    from parakeet_amd import hipmem, lm
    g = np.random.default_rng(D + half + n)
    put = hipmem.Tensor.from_numpy
    H, page, start = 2, 64, 33                                # a block that holds one row, and one that holds none
    cache = np.zeros((2, H, S.record_bytes(page, D)), np.uint8)
    S.store(cache, page, D, *g.standard_normal((2, 1, H, D)), [start - 1])
    slots = np.concatenate([np.arange(start, start + n), [64]]).astype(np.int32)
    pos = np.concatenate([np.arange(n), [3]]).astype(np.int32)
    k, v = (R.to_dtype(g.standard_normal((n + 1, H, D)), dtype) for _ in range(2))
    inv = (10000.0 ** (-np.arange(half) / max(half, 1))).astype(np.float32) if half else None
    kw = dict(pos=put(pos), inv_freq=None if inv is None else put(inv), interleaved=interleaved)
    dev = put(cache)
    lm.kv8_append(put(k, dtype), put(v, dtype), put(slots), dev, page, eps=0.0, **kw)
    hipmem.synchronize()
    got = dev.numpy()
    want, tol = S.rope(R.to_f64(k, dtype), pos, inv, 0.0, None, interleaved)
    for i, s in enumerate(slots):
        for h in range(H):
            rec = got[s // page, h]
            scales = S.parts(rec, page, D)[2][s % page // 32]
            assert (scales[:2] > 0).all(), (s, h, scales)
            a = S.get_row(rec, s % page, page, D)[0]
            assert (np.abs(a - want[i, h]) <= 2.0 ** -4 * np.abs(want[i, h]) + 2.0 ** -10 * scales[0] + 2 * tol[i, h]).all()
    # a row of zeros has no norm: NaN, and its block's mark
    k = np.zeros((1, H, D), k.dtype)
    at = np.array([start + n if n < 31 else 65], np.int32)
    kw["pos"] = put(pos[:1])
    lm.kv8_append(put(k, dtype), put(v[:1], dtype), put(at), dev, page, eps=0.0, **kw)
    hipmem.synchronize()
    got = dev.numpy()
    for h in range(H):
        rec, off = got[at[0] // page, h], int(at[0]) % page
        scales = S.parts(rec, page, D)[2][off // 32]
        assert scales[0] < 0 < scales[1] and np.isnan(S.get_row(rec, off, page, D)[0]).all()

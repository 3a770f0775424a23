"""f16 rows near the type's end.  The cache holds what lies over 57,344 as 4 x 2^14 = 65,536, a step past f16's largest value;
an f16 result has 65,504 there, so that finite rows stay finite."""
import numpy as np
import pytest

import lm_reference as R
import test_gpu_lm_attend as A

pytestmark = pytest.mark.gpu
TOP = 65504.0


@pytest.mark.parametrize("D", [64, 128, 256])
def test_load(D):
    from parakeet_amd import hipmem, lm
    g = np.random.default_rng(D)
    n, page = 40, 16
    k = g.uniform(-1, 1, (n, 2, D)) * TOP
    k[0, 0, :8] = [57344, 57376, 58000, 65504, -57344, -57376, -58000, -65504]
    k[1, 1, 5] = np.nan
    k, v = R.to_dtype(k, "f16"), R.to_dtype(np.roll(k, 3, -1), "f16")
    cache = hipmem.Tensor.from_numpy(np.zeros((3, 2, R.record_bytes(page, D)), np.uint8))
    slots = hipmem.Tensor.from_numpy(np.arange(n, dtype=np.int32))
    lm.kv4_store(hipmem.Tensor.from_numpy(k), hipmem.Tensor.from_numpy(v), slots, cache, page)
    back = [hipmem.Tensor.from_numpy(np.zeros((n, 2, D), np.float16)) for _ in range(2)]
    lm.kv4_load(cache, slots, *back, page)
    hipmem.synchronize()
    for x, b in zip((k, v), back):
        want = np.clip(R.value(*R.quantise(R.to_f64(x, "f16"))), -TOP, TOP)
        assert (np.abs(want) == TOP).any() and np.array_equal(b.numpy(), want.astype(np.float16), equal_nan=True)


def test_load_of_values_that_f16_has_not():
    """Rows stored in f32 and read in f16: beyond 65,536 an infinity, as in any conversion."""
    from parakeet_amd import hipmem, lm
    D, page = 64, 16
    x = np.zeros((4, 1, D), np.float32)
    x[0, 0, 0], x[1, 0, 0], x[2, 0, 40], x[3, 0, 63] = 1e30, -98304, 65536, -65536
    cache = hipmem.Tensor.from_numpy(np.zeros((1, 1, R.record_bytes(page, D)), np.uint8))
    slots = hipmem.Tensor.from_numpy(np.arange(4, dtype=np.int32))
    xd = hipmem.Tensor.from_numpy(x)
    lm.kv4_store(xd, xd, slots, cache, page)
    back = [hipmem.Tensor.from_numpy(np.zeros((4, 1, D), np.float16)) for _ in range(2)]
    lm.kv4_load(cache, slots, *back, page)
    hipmem.synchronize()
    want = np.zeros((4, 1, D), np.float16)
    want[0, 0, 0], want[1, 0, 0], want[2, 0, 40], want[3, 0, 63] = np.inf, -np.inf, TOP, -TOP
    for b in back:
        assert np.array_equal(b.numpy(), want)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("many", [False, True])
def test_attention_over_such_rows(D, many):
    """Every value of V at f16's end, so every mean of them is 65,536 to the rounding of f32 sums, which f16 has as 65,504."""
    p = A.problem(D, D, 32, 4, 2, [100, 1, 40], [90, 1, 3], "f16")
    slots = [p["table"][b, t // 32] * 32 + t % 32 for b, n in enumerate(p["lens"]) for t in range(n)]
    k = np.random.default_rng(1).standard_normal((len(slots), 2, D))
    v = np.full((len(slots), 2, D), TOP)
    v[..., 1::2] *= -1
    R.store(p["cache"], 32, D, k, v, slots)
    out, lse = A.run(p, max_new=70000 if many else None)
    assert np.array_equal(out, np.broadcast_to(np.where(np.arange(D) % 2, -TOP, TOP), out.shape)) and np.isfinite(lse).all()

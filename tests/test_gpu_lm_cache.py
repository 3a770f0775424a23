"""pk_kv4_store / pk_kv4_load: the cache's bytes against the plain statement's, exactly, and the values they stand for."""
import numpy as np
import pytest

import lm_reference as R

pytestmark = pytest.mark.gpu


def rows(g, n, H, D, dtype):
    x = g.standard_normal((n, H, D)) * np.exp(2 * g.standard_normal((n, H, 1)))
    x[::5, :, :32] = 0
    x[1::7] *= 2.0 ** -20
    return R.to_dtype(x, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 32, 256])
def test_store_and_load(dtype, D, page):
    from parakeet_amd import hipmem, lm
    g = np.random.default_rng(D * page)
    for n, H in ((1, 1), (37, 3), (65, 8)):
        n_pages = -(-n // page) + 3
        k, v = rows(g, n, H, D, dtype), rows(g, n, H, D, dtype)
        slots = g.permutation(n_pages * page)[:n].astype(np.int32)
        if n > 10:
            slots[3], slots[7] = -1, n_pages * page           # padding and one past the end: skipped
        size = R.record_bytes(page, D)
        assert lm.kv4_shape(n_pages, H, D, page) == (n_pages, H, size)
        cache = g.integers(0, 256, (n_pages, H, size), dtype=np.uint8)
        dev = hipmem.Tensor.from_numpy(cache)
        kd, vd = (hipmem.Tensor.from_numpy(a, dtype) for a in (k, v))
        sd = hipmem.Tensor.from_numpy(slots)
        lm.kv4_store(kd, vd, sd, dev, page)
        back = [hipmem.Tensor.from_numpy(R.to_dtype(np.full((n, H, D), 9.0), dtype), dtype) for _ in range(2)]
        lm.kv4_load(dev, sd, back[0], back[1], page)
        hipmem.synchronize()
        R.store(cache, page, D, R.to_f64(k, dtype), R.to_f64(v, dtype), slots)
        got = dev.numpy()
        assert np.array_equal(got, cache)
        for which, b in enumerate(back):
            b = R.to_f64(b.numpy(), dtype)
            for i, s in enumerate(slots):
                for h in range(H):
                    want = R.get_row(cache[s // page, h], s % page, page, D)[which] if 0 <= s < n_pages * page else np.full(D, 9.0)
                    assert np.array_equal(b[i, h], R.to_f64(R.to_dtype(want, dtype), dtype))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_every_level_tie_and_scale(dtype):
    """Values at and beside every rounding border, blocks of every magnitude the type has, NaN and infinities."""
    from parakeet_amd import hipmem, lm
    D, page = 128, 16
    borders = np.array([0, .25, .5, .75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 7])
    near = np.concatenate([borders, borders * (1 - 2 ** -7), borders * (1 + 2 ** -7), -borders, -borders * (1 + 2 ** -7)])
    lo, hi = {"bf16": (-130, 125), "f16": (-22, 13), "f32": (-140, 125)}[dtype]
    x = []
    for e in range(lo, hi + 1):
        for first in (3.6, 5.0, 7.0, 7.0 * (1 + 2 ** -7)):
            b = np.resize(np.roll(near, e), D).copy()
            b[::32] = first
            x.append(np.clip(b, -first, first) * 2.0 ** e)
    x = np.array(x)
    x[3, 40], x[5, 0], x[6, 127] = np.nan, np.inf, -np.inf
    x[8] = 0
    with np.errstate(over="ignore"):
        x = R.to_dtype(x, dtype)[:, None]
    n = len(x)
    cache = hipmem.Tensor.from_numpy(np.zeros((-(-n // page), 1, R.record_bytes(page, D)), np.uint8))
    xd, sd = hipmem.Tensor.from_numpy(x, dtype), hipmem.Tensor.from_numpy(np.arange(n, dtype=np.int32))
    lm.kv4_store(xd, xd, sd, cache, page)
    back = [hipmem.Tensor(x.shape, "f32") for _ in range(2)]
    if dtype == "f32":
        lm.kv4_load(cache, sd, back[0], back[1], page)
    hipmem.synchronize()
    want = np.zeros((-(-n // page), 1, R.record_bytes(page, D)), np.uint8)
    R.store(want, page, D, R.to_f64(x, dtype), R.to_f64(x, dtype), range(n))
    got = cache.numpy()
    for i in range(n):
        for a, b in zip(R.get_row(got[i // page, 0], i % page, page, D), R.get_row(want[i // page, 0], i % page, page, D)):
            assert np.array_equal(a, b, equal_nan=True), i
    if dtype == "f32":
        for b in back:
            v = R.value(*R.quantise(R.to_f64(x, dtype)))
            with np.errstate(over="ignore"):
                assert np.array_equal(b.numpy(), v.astype(np.float32), equal_nan=True)


def test_strided_rows_unaligned_rows_and_a_cache_of_layers():
    """Rows cut out of a joint product, at addresses that allow no 16-byte access, into one layer of a cache of layers."""
    from parakeet_amd import hipmem, lm
    g = np.random.default_rng(2)
    D, H, page, n, layers, n_pages = 128, 2, 32, 45, 3, 4
    size = R.record_bytes(page, D)
    for shift in (0, 1):
        wide = R.to_dtype(g.standard_normal((n, 3 * H * D + 8)), "bf16")
        flat = hipmem.Tensor.from_numpy(wide.reshape(-1), "bf16")
        row = 3 * H * D + 8
        k = flat.view((n, H, D), (row, D, 1), H * D + shift)
        v = flat.view((n, H, D), (row, D, 1), 2 * H * D + shift)
        cache = np.zeros((n_pages, layers, H, size), np.uint8)
        dev = hipmem.Tensor.from_numpy(cache)
        one = dev.view((n_pages, H, size), (layers * H * size, size, 1), H * size)
        slots = g.permutation(n_pages * page)[:n].astype(np.int32)
        sd = hipmem.Tensor.from_numpy(slots)
        lm.kv4_store(k, v, sd, one, page)
        out = hipmem.Tensor((n, 2, H, D), "f32")
        lm.kv4_load(one, sd, out.view((n, H, D), (2 * H * D, D, 1)), out.view((n, H, D), (2 * H * D, D, 1), H * D), page)
        hipmem.synchronize()
        kn, vn = R.to_f64(k.numpy(), "bf16"), R.to_f64(v.numpy(), "bf16")
        R.store(cache[:, 1], page, D, kn, vn, slots)
        assert np.array_equal(dev.numpy(), cache)
        assert np.array_equal(out.numpy()[:, 0], R.value(*R.quantise(kn))) and np.array_equal(out.numpy()[:, 1], R.value(*R.quantise(vn)))


def test_no_rows():
    from parakeet_amd import hipmem, lm
    cache = hipmem.Tensor.from_numpy(np.full((2, 1, R.record_bytes(16, 64)), 7, np.uint8))
    k = hipmem.Tensor((0, 1, 64), "f16")
    lm.kv4_store(k, k, hipmem.Tensor((0,), "i32"), cache, 16)
    hipmem.synchronize()
    assert (cache.numpy() == 7).all()


def test_offsets_past_32_bits():
    """A cache of more than 4 GiB: the last page's rows come back, and no others change."""
    from parakeet_amd import hipmem, lm
    D, H, page = 256, 8, 256
    size = R.record_bytes(page, D)
    n_pages = (4 << 30) // (H * size) + 40
    cache = hipmem.Tensor((n_pages, H, size), "u8")
    cache.zero()
    g = np.random.default_rng(0)
    k, v = R.to_dtype(g.standard_normal((2, 4, H, D)), "bf16")
    slots = np.array([n_pages * page - 1, (n_pages - 30) * page + 3, 5, (n_pages - 1) * page], np.int32)
    sd = hipmem.Tensor.from_numpy(slots)
    lm.kv4_store(hipmem.Tensor.from_numpy(k, "bf16"), hipmem.Tensor.from_numpy(v, "bf16"), sd, cache, page)
    a, b = hipmem.Tensor((4, H, D), "f32"), hipmem.Tensor((4, H, D), "f32")
    lm.kv4_load(cache, sd, a, b, page)
    probe = hipmem.Tensor.from_numpy(np.array([6, n_pages * page - 2], np.int32))
    c, d = hipmem.Tensor((2, H, D), "f32"), hipmem.Tensor((2, H, D), "f32")
    lm.kv4_load(cache, probe, c, d, page)
    hipmem.synchronize()
    assert np.array_equal(a.numpy(), R.value(*R.quantise(R.to_f64(k, "bf16")))) and np.array_equal(b.numpy(), R.value(*R.quantise(R.to_f64(v, "bf16"))))
    assert (c.numpy() == 0).all() and (d.numpy() == 0).all()
    cache.buffer.free()

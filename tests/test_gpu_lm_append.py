"""pk_kv8_append / pk_kv8_load: the cache's bytes against the plain statement's, exactly where nothing is normed or turned, and the
values they stand for."""
import numpy as np
import pytest

import lm_reference as R
import lm_step_reference as S

pytestmark = pytest.mark.gpu


def rows(g, n, H, D, dtype):
    x = g.standard_normal((n, H, D)) * np.exp(1.5 * g.standard_normal((n, H, 1)))
    x[::5, :, :32] = 0
    x[1::7] *= 2.0 ** -12
    return R.to_dtype(x, dtype)


def place(g, lens, news, page, extra=2):
    """(slots of the new tokens, pages) of requests that hold lens tokens, pages in an order of their own; with older[b], slots
    of the tokens held already."""
    held = [-(-(a + b) // page) for a, b in zip(lens, news)]
    n_pages = sum(held) + extra
    ids = g.permutation(n_pages)
    at, new, older = 0, [], []
    for a, b, h in zip(lens, news, held):
        mine = ids[at:at + h]
        at += h
        older.append([int(mine[t // page] * page + t % page) for t in range(a)])
        new += [int(mine[t // page] * page + t % page) for t in range(a, a + b)]
    return np.array(new, np.int32), n_pages, older


def same_cache(got, want, page, D, slots_held):
    """Held rows' codes and their blocks' scales are alike."""
    H = got.shape[1]
    for s in slots_held:
        for h in range(H):
            a, b = got[s // page, h], want[s // page, h]
            off = s % page
            for x, y in zip(S.get_codes(a, off, page, D), S.get_codes(b, off, page, D)):
                assert S.same_codes(x, y), (s, h)
            assert np.array_equal(S.parts(a, page, D)[2][off // 32], S.parts(b, page, D)[2][off // 32]), (s, h)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("page", [32, 64, 256])
def test_append_and_load(dtype, D, page):
    """Prompts, then steps of one and of a few tokens behind them, the scale of a block growing on the way."""
    from parakeet_amd import hipmem, lm
    g = np.random.default_rng(D * page)
    put = hipmem.Tensor.from_numpy
    H, B = 3, 6
    lens = np.zeros(B, int)
    slots, n_pages, _ = place(g, lens, [130, 31, 32, 33, 1, 70], page)
    per = [slots[a:a + n] for a, n in zip(np.cumsum([0, 130, 31, 32, 33, 1]), [130, 31, 32, 33, 1, 70])]
    size = S.record_bytes(page, D)
    assert lm.kv8_shape(n_pages, H, D, page) == (n_pages, H, size)
    cache = g.integers(0, 256, (n_pages, H, size), dtype=np.uint8)
    dev, held = put(cache), []
    for step, news in enumerate(([70, 5, 32, 20, 0, 64], [1, 1, 0, 1, 1, 1], [5, 3, 0, 2, 0, 5], [54, 22, 0, 10, 0, 0])):
        new = np.concatenate([p[a:a + n] for p, a, n in zip(per, lens, news)]).astype(np.int32)
        lens = lens + news
        pad = np.concatenate([new, [-1, n_pages * page]]).astype(np.int32)           # padding and one past the end: skipped
        k, v = rows(g, len(pad), H, D, dtype), rows(g, len(pad), H, D, dtype)
        if step == 2:
            k = R.to_dtype(R.to_f64(k, dtype) * 37, dtype)
        lm.kv8_append(put(k, dtype), put(v, dtype), put(pad), dev, page)
        hipmem.synchronize()
        S.store(cache, page, D, R.to_f64(k, dtype), R.to_f64(v, dtype), pad)
        held += list(new)
        same_cache(dev.numpy(), cache, page, D, held)
    at = np.array(held + [-1, n_pages * page], np.int32)
    for out in ("bf16", "f16", "f32"):
        back = [put(R.to_dtype(np.full((len(at), H, D), 9.0), out), out) for _ in range(2)]
        lm.kv8_load(dev, put(at), back[0], back[1], page)
        hipmem.synchronize()
        for which, b in enumerate(back):
            b = R.to_f64(b.numpy(), out)
            assert (b[-2:] == 9.0).all()
            for i, s in enumerate(held):
                for h in range(H):
                    assert np.array_equal(b[i, h], R.to_f64(R.to_dtype(S.get_row(cache[s // page, h], s % page, page, D)[which], out), out))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_every_code_tie_and_scale(dtype):
    """Values at and beside every rounding border, blocks of every magnitude the type has, NaN and infinities."""
    from parakeet_amd import hipmem, lm
    D, page = 128, 32
    mids = (S.LEVELS[:126] + S.LEVELS[1:127]) / 2
    near = np.concatenate([S.LEVELS[:127], mids, -mids, mids * (1 + 2 ** -7), mids * (1 - 2 ** -7), -S.LEVELS[:127]])
    lo, hi = {"bf16": (-126, 127), "f16": (-14, 15), "f32": (-126, 127)}[dtype]
    blocks = []
    for e in range(lo, hi + 1, 3):
        for first in (1.0, 1.75, 1.75 * (1 + 2 ** -7)):
            b = np.resize(np.roll(near, 5 * e), page * D) / 256
            b = np.clip(b, -first, first)
            b[7] = first
            blocks.append((b * 2.0 ** e).reshape(page, D))
    x = np.array(blocks)
    x[3, 4, 40], x[5, 0, 0], x[6, 31, 127] = np.nan, np.inf, -np.inf
    x[8] = 0
    with np.errstate(over="ignore"):
        x = R.to_dtype(x.reshape(-1, 1, D), dtype)
    n = len(x)
    put = hipmem.Tensor.from_numpy
    want = np.zeros((n // page, 1, S.record_bytes(page, D)), np.uint8)
    dev, slots = put(want), np.arange(n, dtype=np.int32)
    lm.kv8_append(put(x, dtype), put(x, dtype), put(slots), dev, page)
    hipmem.synchronize()
    S.store(want, page, D, R.to_f64(x, dtype), R.to_f64(x, dtype), slots)
    same_cache(dev.numpy(), want, page, D, range(n))
    back = [hipmem.Tensor(x.shape, dtype) for _ in range(2)]
    lm.kv8_load(dev, put(slots), back[0], back[1], page)
    hipmem.synchronize()
    got, src = R.to_f64(back[0].numpy(), dtype), R.to_f64(x, dtype)
    assert (np.isfinite(got) == np.isfinite(src)).all()            # finite rows stay finite


def test_nan_marks_stay_until_the_block_begins_anew():
    from parakeet_amd import hipmem, lm
    D, page = 64, 32
    put = hipmem.Tensor.from_numpy
    g = np.random.default_rng(3)
    want = g.integers(0, 256, (2, 1, S.record_bytes(page, D)), dtype=np.uint8)
    dev = put(want)
    for first, n, bad in ((32, 5, True), (37, 3, False), (32, 2, False)):
        k, v = g.standard_normal((2, n, 1, D))
        if bad:
            v[2, 0, 9], k[1, 0, 3] = np.nan, np.inf
        slots = np.arange(first, first + n, dtype=np.int32)
        lm.kv8_append(put(k.astype(np.float32)), put(v.astype(np.float32)), put(slots), dev, page)
        hipmem.synchronize()
        S.store(want, page, D, k.astype(np.float32).astype(float), v.astype(np.float32).astype(float), slots)
        same_cache(dev.numpy(), want, page, D, range(32, first + n))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D,half,interleaved", [(64, 32, False), (128, 64, False), (128, 16, True), (256, 128, False), (256, 128, True), (128, 0, False)])
def test_norm_and_rotation_on_the_way(dtype, D, half, interleaved):
    """Each held key lies within its rounding of the turned one: half a step of its code, 2^-4 of itself or 2^-10 of the scale, both
    with the turned row's own tolerance; the scale is the smallest, up to that tolerance.  V is exact."""
    from parakeet_amd import hipmem, lm
    g = np.random.default_rng(D + half)
    put = hipmem.Tensor.from_numpy
    H, Hq, page = 2, 6, 64
    news = [75, 1, 5, 40, 0, 33]
    lens = [0, 31, 62, 17, 3, 64]
    slots, n_pages, older = place(g, lens, news, page)
    n = len(slots) + 3
    slots = np.concatenate([slots, [-1, -1, n_pages * page]]).astype(np.int32)
    pos = np.concatenate([np.arange(a, a + b) for a, b in zip(lens, news)] + [[-1, 7, 8]]).astype(np.int32)
    cache = np.zeros((n_pages, H, S.record_bytes(page, D)), np.uint8)
    for held in older:
        S.store(cache, page, D, *g.standard_normal((2, len(held), H, D)) * 0.5, held)
    x = rows(g, n, Hq + 2 * H, D, dtype)
    q, k, v = x[:, :Hq], x[:, Hq:Hq + H], x[:, Hq + H:]
    wq, wk = (1 + 0.2 * g.standard_normal((2, D))).astype(np.float32)
    inv = (10000.0 ** (-np.arange(half) / max(half, 1))).astype(np.float32) if half else None
    dev, xd = put(cache), put(x, dtype)
    cut = lambda a, h: xd.view((n, h, D), ((Hq + 2 * H) * D, D, 1), a * D)  # noqa: E731
    q_out = put(R.to_dtype(np.full((n, Hq, D), 9.0), dtype), dtype)
    lm.kv8_append(cut(Hq, H), cut(Hq + H, H), put(slots), dev, page, pos=put(pos), inv_freq=None if inv is None else put(inv), eps=1e-6,
                  k_weight=put(wk), q=cut(0, Hq), q_out=q_out, q_weight=put(wq), interleaved=interleaved)
    hipmem.synchronize()
    got = dev.numpy()
    want, tol = S.rope(R.to_f64(q, dtype), pos, inv, 1e-6, wq, interleaved)
    tol = tol + R.UNIT[dtype] * (np.abs(want) + tol) + 2.0 ** -25
    mine = R.to_f64(q_out.numpy(), dtype)
    assert (mine[pos < 0] == 9.0).all() and (np.abs(mine - want)[pos >= 0] <= tol[pos >= 0]).all()       # a query needs no slot
    kk, ktol = S.rope(R.to_f64(k, dtype), pos, inv, 1e-6, wk, interleaved)
    exact = cache.copy()
    S.store(exact, page, D, kk, R.to_f64(v, dtype), slots)
    for i, s in enumerate(slots[:-3]):
        for h in range(H):
            rec, ref, off = got[s // page, h], exact[s // page, h], s % page
            assert S.same_codes(S.get_codes(rec, off, page, D)[1], S.get_codes(ref, off, page, D)[1])
            sk, sv = S.parts(rec, page, D)[2][off // 32][:2], S.parts(ref, page, D)[2][off // 32][:2]
            assert sk[1] == sv[1] and (sk[0] == sv[0] or abs(np.log2(sk[0] / sv[0])) == 1)
            a = S.get_row(rec, off, page, D)[0]
            assert (np.abs(a - kk[i, h]) <= (2.0 ** -4) * np.abs(kk[i, h]) + 2.0 ** -10 * sk[0] + 2 * ktol[i, h]).all()
    differ = np.mean([S.get_codes(got[s // page, h], s % page, page, D)[0] != S.get_codes(exact[s // page, h], s % page, page, D)[0]
                      for s in slots[:-3] for h in range(H)])
    assert differ <= 2.0 ** -8                 # a tolerance of 2^-18 of a value against steps of 2^-3: 2^-14, blocks of another scale aside


def test_a_scale_counts_all_rows_of_a_run_over_two_workgroups():
    """Long runs at every offset: rows of a block that lie in two workgroups' parts of the call."""
    from parakeet_amd import hipmem, lm
    g = np.random.default_rng(9)
    put = hipmem.Tensor.from_numpy
    D, page, H = 64, 64, 1
    news = [3000, 2971, 1, 2, 3, 3100, 64, 4001, 4500, 6000]
    lens = [0, 13, 31, 5, 30, 33, 0, 1, 63, 32]
    slots, n_pages, older = place(g, lens, news, page)
    cache = np.zeros((n_pages, H, S.record_bytes(page, D)), np.uint8)
    for held in older:
        S.store(cache, page, D, *g.standard_normal((2, len(held), H, D)), held)
    dev = put(cache)
    k, v = g.standard_normal((2, len(slots), H, D)).astype(np.float32) * np.exp(2 * g.standard_normal((2, len(slots), 1, 1))).astype(np.float32)
    lm.kv8_append(put(k), put(v), put(slots), dev, page)
    hipmem.synchronize()
    S.store(cache, page, D, k.astype(float), v.astype(float), slots)
    got = dev.numpy()
    scales = [np.ascontiguousarray(c[..., 2 * page * D:]).view(np.float32).reshape(n_pages, page // 32, 4) for c in (got, cache)]
    blocks = np.unique(slots // 32)
    assert np.array_equal(scales[0].reshape(-1, 4)[blocks], scales[1].reshape(-1, 4)[blocks])
    same_cache(got, cache, page, D, np.concatenate([slots[::17], *[np.array(o[-31:], int) for o in older]]))


def test_offsets_past_32_bits_layers_and_unaligned_rows():
    from parakeet_amd import hipmem, lm
    D, H, page = 256, 8, 256
    size = S.record_bytes(page, D)
    n_pages = (4 << 30) // (H * size) + 40
    put = hipmem.Tensor.from_numpy
    big = hipmem.Tensor((n_pages, H, size), "u8")
    g = np.random.default_rng(10)
    slots = ((n_pages - 3) * page + np.arange(300)).astype(np.int32)
    flat = R.to_dtype(g.standard_normal(300 * (2 * H * D + 8) + 1), "bf16")
    fd = put(flat, "bf16")
    k, v = (fd.view((300, H, D), (2 * H * D + 8, D, 1), 1 + i * H * D) for i in range(2))
    lm.kv8_append(k, v, put(slots), big, page)
    layers = hipmem.Tensor((4, 3, H, size), "u8")
    layers.zero()
    one = layers.view((4, H, size), (3 * H * size, size, 1), H * size)
    low = (np.arange(300) + page).astype(np.int32)
    lm.kv8_append(k, v, put(low), one, page)
    back = [hipmem.Tensor((300, H, D), "bf16") for _ in range(4)]
    lm.kv8_load(big, put(slots), back[0], back[1], page)
    lm.kv8_load(one, put(low), back[2], back[3], page)
    hipmem.synchronize()
    want = np.zeros((4, H, size), np.uint8)
    S.store(want, page, D, R.to_f64(k.numpy(), "bf16"), R.to_f64(v.numpy(), "bf16"), low)
    for i in range(2):
        a, b = back[i].numpy(), back[2 + i].numpy()
        assert np.array_equal(a, b)
        for j in (0, 31, 32, 255, 256, 299):
            for h in (0, 7):
                w = S.get_row(want[low[j] // page, h], low[j] % page, page, D)[i]
                assert np.array_equal(R.to_f64(a[j, h], "bf16"), R.to_f64(R.to_dtype(w, "bf16"), "bf16"))
    rest = layers.numpy()
    assert not rest[:, 0].any() and not rest[:, 2].any() and not rest[0].any() and not rest[3].any()
    big.buffer.free()

"""pk_kv4_attend against attention in 64 bits over the values the cache stands for, within the tolerances that
lm_reference.attend derives."""
import numpy as np
import pytest

import lm_reference as R

pytestmark = pytest.mark.gpu


def problem(seed, D, page, Hq, H, lens, news, dtype, extra_pages=3, spread=1.0):
    g = np.random.default_rng(seed)
    lens, news = np.array(lens, np.int32), np.array(news, np.int32)
    B = len(lens)
    held = -(-np.maximum(lens, 0) // page)
    n_pages = int(held.sum()) + extra_pages
    ids = g.permutation(n_pages).astype(np.int32)
    width = max(int(held.max()), 1) + 2
    table = np.full((B, width), n_pages + 11, np.int32)          # entries past a length are never looked at
    at = 0
    for b in range(B):
        table[b, :held[b]] = ids[at:at + held[b]]
        at += held[b]
    cache = g.integers(0, 256, (n_pages, H, R.record_bytes(page, D)), dtype=np.uint8)     # what is not written is noise
    total = int(np.maximum(lens, 0).sum())
    k = g.standard_normal((total, H, D)) * np.exp(spread * g.standard_normal((1, H, D)))
    v = g.standard_normal((total, H, D)) * np.exp(spread * g.standard_normal((total, H, 1)))
    slots = [table[b, t // page] * page + t % page for b in range(B) for t in range(max(int(lens[b]), 0))]
    R.store(cache, page, D, k, v, slots)
    first = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
    q = R.to_dtype(g.standard_normal((int(first[-1]), Hq, D)), dtype)
    return dict(q=q, cache=cache, table=table, lens=lens, first=first, page=page, D=D, dtype=dtype, news=news)


def run(p, window=0, scale=None, first=True, max_len=None, max_new=None, stream=None, repeat=1):
    from parakeet_amd import hipmem, lm
    q = hipmem.Tensor.from_numpy(p["q"], p["dtype"])
    out = hipmem.Tensor.from_numpy(R.to_dtype(np.full(p["q"].shape, 77.0), p["dtype"]), p["dtype"])
    lse = hipmem.Tensor.from_numpy(np.full(p["q"].shape[:2], 77.0, np.float32))
    args = [q, hipmem.Tensor.from_numpy(p["cache"]), hipmem.Tensor.from_numpy(p["table"]), hipmem.Tensor.from_numpy(p["lens"]), out, p["page"]]
    for _ in range(repeat):
        lm.kv4_attend(*args, first=hipmem.Tensor.from_numpy(p["first"]) if first else None,
                      max_new=(max(int(p["news"].max()), 1) if first else 1) if max_new is None else max_new,
                      max_len=max(int(p["lens"].max()), 1) if max_len is None else max_len, window=window, scale=scale, lse=lse,
                      stream=stream)
    hipmem.synchronize()
    return R.to_f64(out.numpy(), p["dtype"]), lse.numpy().astype(np.float64)


def check(p, window=0, scale=None, **kw):
    scale_ = p["D"] ** -0.5 if scale is None else scale
    want, wlse, tol, ltol = R.attend(R.to_f64(p["q"], p["dtype"]), p["cache"], p["table"], p["lens"], p["first"], p["page"], scale_,
                                     window, p["dtype"])
    out, lse = run(p, window, scale, **kw)
    assert np.array_equal(np.isnan(out), np.isnan(want)) and np.array_equal(np.isnan(lse), np.isnan(wlse))
    assert np.array_equal(np.isneginf(lse), np.isneginf(wlse))
    far = np.abs(out - want) - tol
    assert np.nanmax(far, initial=-1) <= 0, (np.nanmax(far), np.unravel_index(np.nanargmax(far), far.shape))
    fine = np.isfinite(wlse)
    assert (np.abs(lse[fine] - wlse[fine]) <= ltol[fine]).all()
    return out, lse


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 32, 64, 256])
def test_single_tokens(dtype, D, page):
    lens = [1, 0, 2, 15, 16, 17, 31, 32, 33, 127, 128, 129, 255, 257, 300]
    check(problem(D + page, D, page, 4, 2, lens, [1] * len(lens), dtype), first=False)


@pytest.mark.parametrize("heads", [(1, 1), (3, 3), (8, 1), (12, 4), (32, 2), (20, 1)])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_head_layouts(heads, dtype):
    for D in (64, 128):
        check(problem(sum(heads), D, 32, *heads, [70, 1, 33], [1, 1, 1], dtype), first=False)
        check(problem(sum(heads) + 1, D, 32, *heads, [70, 5, 33], [3, 5, 1], dtype))


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_prompts(D, dtype):
    """Whole prompts, prompts behind held tokens, drafted tokens, a request that brings none, one whose tokens were not
    taken in (more queries than tokens held: the first see nothing)."""
    check(problem(D, D, 64, 4, 2, [130, 200, 65, 40, 3, 97], [130, 37, 5, 0, 9, 64], dtype))
    check(problem(D + 1, D, 16, 2, 2, [33, 17, 150], [33, 2, 149], dtype))


@pytest.mark.parametrize("window", [1, 7, 32, 100])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_windows(window, dtype):
    check(problem(window, 64, 32, 4, 2, [130, 200, 1, 0], [130, 5, 1, 1], dtype), window=window)
    check(problem(window, 128, 16, 4, 2, [300, 50], [1, 1], dtype), window=window, first=False)
    check(problem(window, 128, 64, 8, 1, [190], [130], dtype), window=window)


@pytest.mark.parametrize("D,page", [(64, 64), (128, 16), (256, 128)])
def test_long_axis_is_split_and_joined(D, page):
    check(problem(D, D, page, 4, 1, [9001, 700, 5, 0, 4097], [1, 1, 1, 1, 1], "bf16"), first=False)
    check(problem(D, D, page, 2, 1, [5000, 40], [3, 2], "f16"))
    check(problem(D, D, page, 2, 2, [2500], [70], "bf16"))


def test_splits_repeat_to_the_bit_and_leave_their_workspace_ready():
    p = problem(3, 128, 64, 8, 2, [6000, 3000, 1], [1, 1, 1], "bf16")
    a = run(p, first=False)
    for _ in range(3):
        b = run(p, first=False, repeat=2)
        assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


def test_scales_and_large_values():
    for scale in (0.0, 1.0, -0.3, 3.0):
        check(problem(7, 128, 32, 2, 1, [90, 40], [4, 40], "bf16"), scale=scale)
    p = problem(8, 128, 32, 2, 1, [90], [6], "bf16")
    q = R.to_f64(p["q"], "bf16")
    q[0] *= 2.0 ** 90                  # softmax of one key
    q[1] *= 2.0 ** -110
    q[2] = 0
    q[3, :, 1:] = 0                    # one channel alone
    q[4, :, 0] = 2.0 ** 12             # the others far below it
    p["q"] = R.to_dtype(q, "bf16")
    want, wlse, tol, ltol = R.attend(q, p["cache"], p["table"], p["lens"], p["first"], 32, 128 ** -0.5, 0, "bf16")
    out, lse = run(p)
    far = np.abs(out - want) - tol
    assert (far[1:] <= 0).all()
    z = np.sort(np.array([R.get_row(p["cache"][p["table"][0, t // 32], 0], t % 32, 32, 128)[0] for t in range(85)]) @ q[0].T, 0)
    assert (z[-1] - z[-2] > 1e20).all()            # the largest score stands alone, whatever the rounding
    best = np.array([R.get_row(p["cache"][p["table"][0, t // 32], 0], t % 32, 32, 128)[0] for t in range(85)]) @ q[0].T
    for h in range(2):
        t = int(best[:, h].argmax())
        v = R.get_row(p["cache"][p["table"][0, t // 32], 0], t % 32, 32, 128)[1]
        assert np.allclose(out[0, h], v, rtol=2.0 ** -7, atol=0)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("news", [(50, 60, 1), (25, 30, 1)])      # many query rows of a request, and few
def test_nan_reaches_only_those_that_see_it(dtype, D, news):
    """A NaN block of K makes the queries that see its key NaN, one of V its 32 channels; no other query or channel."""
    p = problem(11, D, 32, 4, 2, [100, 60, 33], news, dtype)
    page = 32

    def poison(b, t, h, part, block):
        rec = p["cache"][p["table"][b, t // page], h]
        off = t % page
        if part == "k":
            rec[page * D + off * (D // 32) + block] = 255
        else:
            rec[page * D + page * D // 32 + block * page + off] = 255
    poison(0, 77, 0, "v", D // 32 - 1)
    poison(0, 90, 1, "k", 0)
    poison(1, 0, 1, "v", 0)
    poison(1, 59, 0, "v", 1)
    poison(1, 40, 1, "v", D // 32 - 1)
    out, _ = check(p)
    assert np.isnan(out).any() and not np.isnan(out).all()
    p["cache"][p["table"][2, 1], 0, page * D + page * D // 32 + 1] = 255      # key 33 of request 2: not held
    check(p)
    check(p, window=9)
    p["q"] = p["q"].copy()
    bad = R.to_dtype(np.array([np.nan, np.inf, -np.inf]), dtype)
    second = news[0] + 10
    p["q"][1, 0, 5], p["q"][second, 1, 0], p["q"][second + 10, 2, D - 1] = bad
    out, lse = run(p)
    for i, h in ((1, 0), (second, 1), (second + 10, 2)):
        assert np.isnan(out[i, h]).all() and np.isnan(lse[i, h])
    assert not np.isnan(lse[2:news[0] // 4]).any()


def test_page_ids_out_of_range_are_skipped():
    p = problem(13, 128, 16, 4, 2, [100, 50], [1, 3], "bf16")
    p["table"][0, 2], p["table"][1, 0] = -1, len(p["cache"])
    check(p)
    p["table"][0, :7] = -5                     # nothing left to see
    out, lse = check(p)
    assert (out[0] == 0).all() and np.isneginf(lse[0]).all()
    for D, page in ((64, 16), (128, 32), (128, 64), (256, 16)):
        p = problem(14, D, page, 4, 2, [300, 90], [80, 90], "bf16")
        p["table"][0, 1], p["table"][0, 200 // page], p["table"][1, 0] = -1, 1 << 30, len(p["cache"])
        check(p)
        check(p, window=70)


def test_few_rows_and_many_rows_agree():
    """The last queries of a prompt in one call and in calls of their own: two kernels, one definition."""
    for dtype, D in (("bf16", 128), ("f16", 64)):
        p = problem(17, D, 64, 8, 2, [700], [90], dtype)
        a, la = check(p)
        few = dict(p, q=np.ascontiguousarray(p["q"][-5:]), first=np.array([0, 5], np.int32), news=np.array([5], np.int32))
        b, lb = check(few)
        assert np.allclose(a[-5:], b, atol=3 * R.UNIT[dtype] * np.abs(a[-5:]).max()) and np.allclose(la[-5:], lb, atol=1e-5)


def test_prompts_over_a_long_axis():
    check(problem(18, 128, 64, 16, 2, [4500, 130], [17, 130], "bf16"))
    check(problem(19, 64, 32, 8, 8, [3000], [129], "f16"), window=1500)


def test_lengths_are_cut_at_max_len_and_table():
    p = problem(14, 64, 16, 2, 1, [100, 50], [1, 1], "bf16")
    cut = dict(p, lens=np.array([64, 50], np.int32))
    a, b = run(p, first=False, max_len=64), run(cut, first=False, max_len=64)
    assert np.array_equal(a[0], b[0])
    q = dict(p, table=np.ascontiguousarray(p["table"][:, :4]))
    assert np.array_equal(run(q, first=False, max_len=1000)[0], b[0])


def test_strides_layers_and_unaligned_rows():
    from parakeet_amd import hipmem, lm
    p = problem(15, 128, 32, 4, 2, [70, 45], [2, 45], "bf16")
    want, wlse, tol, ltol = R.attend(R.to_f64(p["q"], "bf16"), p["cache"], p["table"], p["lens"], p["first"], 32, 128 ** -0.5, 0, "bf16")
    n, Hq, D = p["q"].shape
    for shift in (0, 1, 8):
        row = (Hq + 4) * D + 8
        flat = np.zeros(n * row + 16, np.uint16)
        at = np.arange(n)[:, None, None] * row + np.arange(Hq)[:, None] * D + np.arange(D) + shift
        flat[at] = p["q"]
        q = hipmem.Tensor.from_numpy(flat, "bf16").view((n, Hq, D), (row, D, 1), shift)
        big = hipmem.Tensor.from_numpy(np.full(n * row + 16, 0x4242, np.uint16), "bf16")
        out = big.view((n, Hq, D), (row, D, 1), shift)
        wide = np.full((2, 9), 5, np.int32)
        wide[:, :p["table"].shape[1]] = p["table"]
        table = hipmem.Tensor.from_numpy(wide).view(p["table"].shape, (9, 1))
        layers = np.zeros((len(p["cache"]), 3, *p["cache"].shape[1:]), np.uint8)
        layers[:, 2] = p["cache"]
        size = p["cache"].shape[2]
        cache = hipmem.Tensor.from_numpy(layers).view(p["cache"].shape, (3 * 2 * size, size, 1), 4 * size)
        lm.kv4_attend(q, cache, table, hipmem.Tensor.from_numpy(p["lens"]), out, 32, first=hipmem.Tensor.from_numpy(p["first"]),
                      max_new=45, max_len=70)
        hipmem.synchronize()
        got = R.to_f64(out.numpy(), "bf16")
        assert (np.abs(got - want) <= tol).all()
        rest = np.ones(n * row + 16, bool)
        rest[at] = False
        assert (big.numpy()[rest] == 0x4242).all()


def test_offsets_past_32_bits():
    """A cache of more than 4 GiB whose last pages are read."""
    from parakeet_amd import hipmem, lm
    D, H, page = 256, 8, 256
    size = R.record_bytes(page, D)
    n_pages = (4 << 30) // (H * size) + 40
    p = problem(16, D, page, 8, 8, [600], [1], "bf16", extra_pages=0)
    cache = hipmem.Tensor((n_pages, H, size), "u8")
    cache.zero()
    ids = np.array([n_pages - 1, 3, n_pages - 25], np.int32)
    slots = np.concatenate([ids[t // page:t // page + 1] * page + t % page for t in range(600)]).astype(np.int32)
    rows = np.array([[R.get_row(p["cache"][p["table"][0, t // page], h], t % page, page, D) for h in range(H)] for t in range(600)])
    k, v = (hipmem.Tensor.from_numpy(np.ascontiguousarray(rows[:, :, i], np.float32)) for i in range(2))
    lm.kv4_store(k, v, hipmem.Tensor.from_numpy(slots), cache, page)       # values the cache has: they go in unchanged
    out = hipmem.Tensor(p["q"].shape, "bf16")
    lm.kv4_attend(hipmem.Tensor.from_numpy(p["q"], "bf16"), cache, hipmem.Tensor.from_numpy(ids[None]),
                  hipmem.Tensor.from_numpy(p["lens"]), out, page, max_len=600)
    hipmem.synchronize()
    want, _, tol, _ = R.attend(R.to_f64(p["q"], "bf16"), p["cache"], p["table"], p["lens"], p["first"], page, D ** -0.5, 0, "bf16")
    assert (np.abs(R.to_f64(out.numpy(), "bf16") - want) <= tol).all()
    cache.buffer.free()

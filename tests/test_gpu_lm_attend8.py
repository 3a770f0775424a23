"""pk_kv8_attend on the cases of pk_kv4_attend, over caches of 8 bits, by both kernels, within the tolerances that
lm_step_reference.attend derives; NaNs, which lie at single values here, and offsets by cases of their own."""
import numpy as np
import pytest

import lm_reference as R
import lm_step_reference as S
import test_gpu_lm_attend as A

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, params=["few", "many"])
def over_8_bits(request, monkeypatch):
    """The other cache's functions are this one's; `many`: a bound of many new tokens, which brings every call to the kernel
    for prompts."""
    from parakeet_amd import lm
    for name in ("record_bytes", "store", "get_row", "attend"):
        monkeypatch.setattr(R, name, getattr(S, name))
    monkeypatch.setattr(lm, "kv4_attend", lm.kv8_attend)
    own = A.problem
    monkeypatch.setattr(A, "problem", lambda seed, D, page, *a, **k: own(seed, D, max(page, 32), *a, **k))
    if request.param == "many":
        run = A.run
        monkeypatch.setattr(A, "run", lambda p, window=0, scale=None, first=True, max_len=None, max_new=None, **kw:
                            run(p, window, scale, True, max_len, 70000 if max_new is None else max_new, **kw))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("page", [32, 64, 256])
def test_single_tokens(dtype, D, page):
    A.test_single_tokens(dtype, D, page)


@pytest.mark.parametrize("heads", [(1, 1), (3, 3), (8, 1), (12, 4), (32, 2), (20, 1)])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_head_layouts(heads, dtype):
    A.test_head_layouts(heads, dtype)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_prompts(D, dtype):
    A.test_prompts(D, dtype)
    A.check(A.problem(D + 2, D, 128, 4, 2, [130, 300, 65, 40, 3, 97, 1, 0, 64], [130, 37, 5, 0, 9, 64, 1, 1, 64], dtype))


@pytest.mark.parametrize("window", [1, 7, 32, 100])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_windows(window, dtype):
    A.test_windows(window, dtype)


@pytest.mark.parametrize("D,page", [(64, 64), (128, 32), (256, 128)])
def test_long_axes(D, page):
    A.test_long_axis_is_split_and_joined(D, page)


def test_splits_repeat_to_the_bit():
    A.test_splits_repeat_to_the_bit_and_leave_their_workspace_ready()


def test_scales_and_large_values():
    A.test_scales_and_large_values()


@pytest.mark.parametrize("scale", [0.0, 1e-20, -1e-30])
def test_keys_of_zeros_at_scales_near_zero(scale):
    """A block of zeros has the least scale, 2^-100: its product with the call's is none that f32 has."""
    p = A.problem(17, 64, 32, 4, 2, [150, 70], [60, 70], "bf16")
    for b, t in ((0, 96), (1, 32), (1, 64)):
        for h in range(2):
            k, _, scales = S.parts(p["cache"][p["table"][b, t // 32], h], 32, 64)
            k[:] = 0
            scales[0, 0] = 2.0 ** -100
    A.check(p, scale=scale)
    A.check(p, scale=scale, window=33)


def test_page_ids_out_of_range_are_skipped():
    p = A.problem(13, 128, 32, 4, 2, [100, 50], [1, 3], "bf16")
    p["table"][0, 2], p["table"][1, 0] = -1, len(p["cache"])
    A.check(p)
    p["table"][0, :7] = -5                     # nothing left to see
    out, lse = A.check(p)
    assert (out[0] == 0).all() and np.isneginf(lse[0]).all()
    for D, page in ((64, 32), (128, 32), (128, 64), (256, 64)):
        p = A.problem(14, D, page, 4, 2, [300, 90], [80, 90], "bf16")
        p["table"][0, 1], p["table"][0, 200 // page], p["table"][1, 0] = -1, 1 << 30, len(p["cache"])
        A.check(p)
        A.check(p, window=70)


def test_few_rows_and_many_rows_agree():
    A.test_few_rows_and_many_rows_agree()


def test_lengths_are_cut():
    p = A.problem(14, 64, 32, 2, 1, [100, 50], [1, 1], "bf16")
    cut = dict(p, lens=np.array([64, 50], np.int32))
    a, b = A.run(p, first=False, max_len=64), A.run(cut, first=False, max_len=64)
    assert np.array_equal(a[0], b[0])
    q = dict(p, table=np.ascontiguousarray(p["table"][:, :2]))
    assert np.array_equal(A.run(q, first=False, max_len=1000)[0], b[0])


def test_strides_layers_and_unaligned_rows():
    A.test_strides_layers_and_unaligned_rows()


def poison(p, b, t, h, part, channel, code=0x7F):
    page, D = p["page"], p["D"]
    rec = p["cache"][p["table"][b, t // page], h]
    S.get_codes(rec, 0, page, D)
    k, v, scales = S.parts(rec, page, D)
    off = t % page
    if part == "k":
        k[off, channel] = code
    else:
        v[off // 8, channel // (D // 32), off % 8, channel % (D // 32)] = code
    i = 0 if part == "k" else 1
    scales[off // 32, i] = -abs(scales[off // 32, i])


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("news", [(50, 60, 1), (25, 30, 1)])
def test_nan_reaches_only_those_that_see_it(dtype, D, news):
    """A NaN of K makes the queries that see its key NaN, one of V its channel; no other query or channel."""
    p = A.problem(11, D, 32, 4, 2, [100, 60, 33], news, dtype)
    poison(p, 0, 77, 0, "v", D - 1)
    poison(p, 0, 78, 0, "v", 0, 0xFF)
    poison(p, 0, 90, 1, "k", 0)
    poison(p, 1, 0, 1, "v", 0)
    poison(p, 1, 59, 0, "v", 40)
    for c in range(7, D, 9):
        poison(p, 1, 40 + c % 16, 1, "v", c)
    out, _ = A.check(p)
    assert np.isnan(out).any() and not np.isnan(out).all()
    A.check(p, window=9)
    page, D = p["page"], p["D"]
    for off in range(1, 32):                   # keys 33 .. of request 2: not held, whatever lies there
        rec = p["cache"][p["table"][2, 1], 0]
        S.parts(rec, page, D)[0][off], S.parts(rec, page, D)[1][off // 8, :, off % 8] = 0x7F, 0xFF
    A.check(p)
    A.check(p, window=9)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("D,page", [(64, 64), (128, 32), (128, 128), (256, 32)])
def test_nan_at_an_edge_of_some_waves(dtype, D, page):
    """128 tokens of one head a kv head: the first 64 keys are an edge for waves 0 and 1 of a prompt's workgroup alone."""
    p = A.problem(D, D, page, 2, 2, [128], [128], dtype)
    poison(p, 0, 10, 0, "v", 0)
    poison(p, 0, 63, 1, "v", D - 1)
    out, _ = A.check(p)
    assert np.isnan(out[10:, 0, 0]).all() and not np.isnan(out[:10]).any() and not np.isnan(out[:, 0, 1:]).any()
    p = A.problem(D, D, page, 1, 1, [428], [128], "bf16")
    poison(p, 0, 200, 0, "v", 3)
    poison(p, 0, 230, 0, "v", 4)
    out, _ = A.check(p, window=200)
    assert np.isnan(out).any(-1).all()


def test_offsets_past_32_bits():
    """A cache of more than 4 GiB whose last pages are read."""
    from parakeet_amd import hipmem, lm
    D, H, page = 256, 8, 256
    size = S.record_bytes(page, D)
    n_pages = (4 << 30) // (H * size) + 40
    cache = hipmem.Tensor((n_pages, H, size), "u8")
    cache.zero()
    p = A.problem(16, D, page, 8, 8, [600], [1], "bf16", extra_pages=0)
    ids = np.array([n_pages - 1, 3, n_pages - 25], np.int32)
    slots = np.concatenate([ids[t // page:t // page + 1] * page + t % page for t in range(600)]).astype(np.int32)
    kv = np.array([[S.get_row(p["cache"][p["table"][0, t // page], h], t % page, page, D) for h in range(H)] for t in range(600)])
    k, v = (hipmem.Tensor.from_numpy(np.ascontiguousarray(kv[:, :, i], np.float32)) for i in range(2))
    lm.kv8_append(k, v, hipmem.Tensor.from_numpy(slots), cache, page)      # values that a cache held: they go in unchanged
    out = hipmem.Tensor(p["q"].shape, "bf16")
    lm.kv8_attend(hipmem.Tensor.from_numpy(p["q"], "bf16"), cache, hipmem.Tensor.from_numpy(ids[None]),
                  hipmem.Tensor.from_numpy(p["lens"]), out, page, max_len=600)
    hipmem.synchronize()
    want, _, tol, _ = R.attend(R.to_f64(p["q"], "bf16"), p["cache"], p["table"], p["lens"], p["first"], page, D ** -0.5, 0, "bf16")
    assert (np.abs(R.to_f64(out.numpy(), "bf16") - want) <= tol).all()
    cache.buffer.free()

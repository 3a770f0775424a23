"""pk_qk_rope against norms and rotations in 64 bits, within the tolerances that lm_step_reference.rope derives."""
import numpy as np
import pytest

import lm_reference as R
import lm_step_reference as S

pytestmark = pytest.mark.gpu


def inv_freq(half, base=10000.0):
    return (base ** (-np.arange(half) / max(half, 1))).astype(np.float32)


def check(n, heads, kv_heads, D, dtype, half, norm=True, interleaved=False, weights=True, pos=None, inplace=False, seed=0, size=1.0):
    from parakeet_amd import hipmem, lm
    g = np.random.default_rng(seed)
    put = hipmem.Tensor.from_numpy
    x = [R.to_dtype(g.standard_normal((n, h, D)) * size * np.exp(g.standard_normal((1, h, D))), dtype) for h in (heads, kv_heads)]
    w = [(1 + 0.3 * g.standard_normal(D)).astype(np.float32) if weights else None for _ in range(2)]
    if pos is None:
        pos = g.integers(0, 200003, n)
    pos = np.array(pos, np.int32)
    inv = inv_freq(half) if half else None
    eps = 1e-6 if norm else None
    dev = [put(a, dtype) for a in x]
    out = dev if inplace else [put(R.to_dtype(np.full(a.shape, 9.0), dtype), dtype) for a in x]
    wd = [None if a is None else put(a) for a in w]
    lm.qk_rope(dev[0], out[0], put(pos), None if inv is None else put(inv), k=dev[1] if kv_heads else None, k_out=out[1] if kv_heads else None,
               eps=eps, q_weight=wd[0], k_weight=wd[1], interleaved=interleaved)
    hipmem.synchronize()
    for i in range(2 if kv_heads else 1):
        got = R.to_f64(out[i].numpy(), dtype)
        before = R.to_f64(x[i], dtype)
        want, tol = S.rope(before, pos, inv, eps, w[i], interleaved)
        tol = tol + R.UNIT[dtype] * (np.abs(want) + tol) + (2.0 ** -25 if dtype == "f16" else 2.0 ** -133)     # half a step of subnormal results
        dead = pos < 0
        assert (np.abs(got - want)[~dead] <= tol[~dead]).all(), np.max((np.abs(got - want) - tol)[~dead])
        assert np.array_equal(got[dead], before[dead] if inplace else np.full(before[dead].shape, 9.0))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("interleaved", [False, True])
def test_types_and_widths(dtype, D, interleaved):
    for n, heads, kv_heads in ((1, 1, 0), (1, 8, 8), (3, 5, 1), (37, 12, 3)):
        for half in (D // 2, D // 4, 8, 0):
            check(n, heads, kv_heads, D, dtype, half, interleaved=interleaved, seed=n + half)


def test_norm_and_weights_are_optional():
    for norm in (False, True):
        for weights in (False, True):
            check(9, 3, 2, 128, "f32", 64, norm=norm, weights=weights)


def test_far_positions():
    check(8, 2, 2, 128, "f32", 64, norm=False, pos=[0, 1, 131071, 200003, 2 ** 24 + 1, 2 ** 26 - 1, 2 ** 27 + 3, 5])


@pytest.mark.parametrize("D,half", [(64, 32), (128, 64), (256, 128), (128, 24), (256, 40)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_in_place_and_rows_left_out(D, half, interleaved):
    g = np.random.default_rng(5)
    pos = g.integers(0, 9000, 71)
    pos[::4] = -1
    pos[-9:] = -3
    check(71, 6, 2, D, "bf16", half, pos=pos, inplace=True, interleaved=interleaved)
    check(71, 6, 2, D, "bf16", half, pos=pos, interleaved=interleaved)


def test_many_rows():
    check(5000, 3, 1, 64, "bf16", 32)


@pytest.mark.parametrize("D,dtype", [(64, "f16"), (128, "bf16"), (128, "f32"), (256, "bf16")])
def test_padding_behind_many_rows(D, dtype):
    """Blocks of rows that begin in the padding, one that it begins in, a call of nothing else."""
    pos = np.random.default_rng(7).integers(0, 9000, 4103)
    pos[3300:] = -1
    check(4103, 2, 1, D, dtype, D // 2, pos=pos)
    check(4103, 2, 1, D, dtype, D // 2, pos=pos, inplace=True)
    check(45, 5, 2, D, dtype, D // 2, pos=np.full(45, -1))


def test_norms_of_small_and_large_rows():
    for size in (2.0 ** -40, 2.0 ** -12, 2.0 ** 40):
        check(5, 2, 1, 128, "f32", 64, size=size)
    check(3, 2, 1, 128, "bf16", 64, size=0.0)


def test_strides_and_unaligned_rows():
    from parakeet_amd import hipmem, lm
    g = np.random.default_rng(6)
    n, Hq, H, D, inv = 21, 4, 2, 64, inv_freq(32)
    pos = g.integers(0, 999, n).astype(np.int32)
    for shift in (0, 1, 8):
        row = (Hq + 2 * H) * D + 8
        flat = R.to_dtype(g.standard_normal(n * row + 16), "bf16")
        buf = hipmem.Tensor.from_numpy(flat, "bf16")
        q, k = buf.view((n, Hq, D), (row, D, 1), shift), buf.view((n, H, D), (row, D, 1), shift + Hq * D)
        out = hipmem.Tensor.from_numpy(np.full(n * row + 16, 0x4242, np.uint16), "bf16")
        qo = out.view((n, Hq, D), (row, D, 1), shift)
        ko = out.view((n, H, D), (row, D, 1), shift + Hq * D)
        put = hipmem.Tensor.from_numpy
        lm.qk_rope(q, qo, put(pos), put(inv), k=k, k_out=ko, eps=1e-5)
        hipmem.synchronize()
        for a, o in ((q, qo), (k, ko)):
            want, tol = S.rope(R.to_f64(a.numpy(), "bf16"), pos, inv, 1e-5)
            assert (np.abs(R.to_f64(o.numpy(), "bf16") - want) <= tol + R.UNIT["bf16"] * (np.abs(want) + tol)).all()
        mask = np.ones(n * row + 16, bool)
        at = np.arange(n)[:, None] * row + np.arange((Hq + H) * D) + shift
        mask[at] = False
        assert (out.numpy()[mask] == 0x4242).all()

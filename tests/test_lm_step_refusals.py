"""What the operators of a step with drafted tokens refuse, before any launch (no GPU needed), and that their mirror is the
header's."""
import ctypes
import os
import subprocess

import pytest

from test_lm_refusals import ROOT, Arr


def test_descriptors_match_the_header(pkg, tmp_path):
    from parakeet_amd import lm
    want = {"pk_qk_rope_desc": (lm._ROPE, "eps"), "pk_kv8_append_desc": (lm._APPEND, "eps"), "pk_verify_desc": (lm._VERIFY, "reserved")}
    src = tmp_path / "s.cpp"
    src.write_text('#include "parakeet_lm.h"\n#include <cstddef>\n#include <cstdio>\nint main() {\n' + "".join(
        f'std::printf("%zu %zu\\n", sizeof({d}), offsetof({d}, {last}));\n' for d, (_, last) in want.items()) + "}\n")
    subprocess.run(["g++", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "s")], check=True)
    lines = subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout.split("\n")
    for (d, (s, _)), line in zip(want.items(), lines):
        size, last = map(int, line.split())
        assert s.size == size and last + 4 <= size < last + 4 + 8, d
    assert ctypes.sizeof(ctypes.c_float) == 4


def refused(call, kw, err):
    from parakeet_amd import pk
    with pytest.raises((pk.PkError, ValueError, TypeError), match=err):
        call(**kw)


ROWS = (5, 4, 128)


@pytest.mark.parametrize("kw,err", [
    (dict(q=Arr((5, 4, 96), "bf16"), q_out=Arr((5, 4, 96), "bf16")), "head_dim 96"), (dict(q=Arr(ROWS, "i32"), q_out=Arr(ROWS, "i32")), "i32"),
    (dict(q_out=Arr(ROWS, "f16")), "q_out"), (dict(q_out=None), "q_out"), (dict(q_out=Arr((5, 3, 128), "bf16")), "q_out"),
    (dict(q_out=Arr(ROWS, "bf16", strides=(0, 128, 1))), "overlap"), (dict(q_out=Arr(ROWS, "bf16", strides=(512, 64, 1))), "overlap"),
    (dict(q=Arr(ROWS, "bf16", strides=(512, 1, 4))), "adjacent"), (dict(pos=None), "NULL positions"), (dict(pos=Arr((4,), "i32")), "pos"),
    (dict(pos=Arr((5,), "f32")), "pos"), (dict(inv_freq=Arr((65,), "f32")), "turned"), (dict(inv_freq=Arr((12,), "f32")), "turned"),
    (dict(inv_freq=Arr((64,), "f16")), "inv_freq"), (dict(inv_freq=Arr((72,), "f32")), "turned"), (dict(q=Arr(ROWS, "bf16", ptr=0)), "NULL"),
    (dict(q=Arr(ROWS, "bf16", ptr=4097)), "aligned"), (dict(q_weight=Arr((64,), "f32")), "q_weight"), (dict(q_weight=Arr((128,), "bf16")), "q_weight"),
    (dict(eps=-1e-6), "eps"), (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"),
    (dict(k=Arr((4, 2, 128), "bf16"), k_out=Arr((4, 2, 128), "bf16")), "k bf16"), (dict(k=Arr((5, 2, 128), "f16"), k_out=Arr((5, 2, 128), "f16")), "k f16"),
    (dict(k=Arr((5, 2, 128), "bf16")), "k_out"), (dict(k=Arr((5, 2, 128), "bf16"), k_out=Arr((5, 2, 128), "bf16"), k_weight=Arr((2,), "f32")), "k_weight"),
    (dict(q=Arr((5, 70000, 64), "bf16"), q_out=Arr((5, 70000, 64), "bf16")), "65535")])
def test_rope_refuses(pkg, kw, err):
    from parakeet_amd import lm
    a = dict(q=Arr(ROWS, "bf16"), q_out=Arr(ROWS, "bf16"), pos=Arr((5,), "i32"), inv_freq=Arr((64,), "f32"))
    a.update(kw)
    refused(lm.qk_rope, a, err)


def cache(n=4, heads=2, dim=128, page=32, **kw):
    return Arr((n, heads, page * 2 * dim + page // 2), "u8", **kw)


KV = (5, 2, 128)


@pytest.mark.parametrize("kw,err", [
    (dict(page=16, cache=cache(page=16)), "pages of 16"), (dict(page=24), "kv8_shape|pages of 24"), (dict(cache=cache(dim=96)), "rows of|head_dim"),
    (dict(page=0), "kv8_shape"), (dict(page=-32), "kv8_shape"), (dict(cache=cache(ptr=4104)), "aligned"), (dict(cache=cache(ptr=0)), "NULL"),
    (dict(cache=Arr((4, 2, 8208), "u8", strides=(8208, 8208, 1))), "page_stride"), (dict(cache=Arr((4, 2, 8208), "u8", strides=(16424, 8208, 1))), "page_stride"),
    (dict(cache=Arr((4, 2, 8208), "u8", strides=(32832, 16416, 1))), "adjacent"), (dict(cache=Arr((4, 2, 8208), "f32")), "uint8"),
    (dict(v=Arr(KV, "f16")), "bf16"), (dict(v=Arr((4, 2, 128), "bf16")), "v bf16"), (dict(k=Arr(KV, "i32"), v=Arr(KV, "i32")), "i32"),
    (dict(k=Arr(KV, "bf16", strides=(256, 1, 2))), "adjacent"), (dict(slots=Arr((4,), "i32")), "slots"), (dict(k=Arr(KV, "bf16", ptr=4097)), "aligned"),
    (dict(k=Arr(KV, "bf16", ptr=0)), "NULL"), (dict(cache=cache(n=70_000_000)), "32 bits")])
def test_append_and_load_refuse(pkg, kw, err):
    from parakeet_amd import lm
    a = dict(k=Arr(KV, "bf16"), v=Arr(KV, "bf16"), slots=Arr((5,), "i32"), cache=cache(), page=32)
    a.update(kw)
    refused(lm.kv8_append, a, err)
    refused(lm.kv8_load, a, err)


@pytest.mark.parametrize("kw,err", [
    (dict(inv_freq=Arr((64,), "f32")), "NULL positions"), (dict(pos=Arr((6,), "i32")), "pos"), (dict(inv_freq=Arr((60,), "f32"), pos=Arr((5,), "i32")), "turned"),
    (dict(eps=float("nan")), "eps"), (dict(k_weight=Arr((2,), "f32")), "k_weight"), (dict(q=Arr((5, 4, 128), "bf16")), "q_out"),
    (dict(q=Arr((5, 4, 64), "bf16"), q_out=Arr((5, 4, 64), "bf16")), "q bf16"), (dict(q=Arr((5, 4, 128), "f16"), q_out=Arr((5, 4, 128), "f16")), "q f16"),
    (dict(q=Arr((5, 4, 128), "bf16"), q_out=Arr((5, 4, 128), "bf16", strides=(0, 0, 1))), "overlap"),
    (dict(q=Arr((5, 4, 128), "bf16"), q_out=Arr((5, 4, 128), "bf16", ptr=0)), "NULL"),
    (dict(q=Arr((5, 4, 128), "bf16"), q_out=Arr((5, 4, 128), "bf16"), q_weight=Arr((129,), "f32")), "q_weight")])
def test_append_refuses(pkg, kw, err):
    from parakeet_amd import lm
    a = dict(k=Arr(KV, "bf16"), v=Arr(KV, "bf16"), slots=Arr((5,), "i32"), cache=cache(), page=32)
    a.update(kw)
    refused(lm.kv8_append, a, err)


@pytest.mark.parametrize("kw,err", [
    (dict(q=Arr((3, 4, 128), "f32"), out=Arr((3, 4, 128), "f32")), "dtype"), (dict(q=Arr((3, 3, 128), "bf16"), out=Arr((3, 3, 128), "bf16")), "heads"),
    (dict(q=Arr((3, 4, 64), "bf16"), out=Arr((3, 4, 64), "bf16")), "heads of 64"), (dict(out=Arr((3, 4, 128), "f16")), "out"),
    (dict(out=Arr((3, 4, 128), "bf16", strides=(0, 128, 1))), "overlap"), (dict(lens=Arr((2,), "i32")), "lens"), (dict(window=-1), "window"),
    (dict(max_new=2), "without first"), (dict(cache=cache(ptr=4104)), "aligned"), (dict(page=16, cache=cache(page=16)), "pages of 16"),
    (dict(q=Arr((3, 4, 128), "bf16", ptr=0)), "NULL"), (dict(scale=float("nan")), "scale"), (dict(max_len=2 ** 31 - 1), "32 bits"),
    (dict(max_len=2 ** 31 - 5000, workspace=Arr((4096,), "u8")), "workspace"), (dict(max_new=1 << 28, first=Arr((4,), "i32")), "in one call")])
def test_attend_refuses(pkg, kw, err):
    from parakeet_amd import lm
    a = dict(q=Arr((3, 4, 128), "bf16"), cache=cache(), table=Arr((3, 5), "i32"), lens=Arr((3,), "i32"), out=Arr((3, 4, 128), "bf16"), page=32,
             max_len=100)
    a.update(kw)
    refused(lm.kv8_attend, a, err)


@pytest.mark.parametrize("kw,err", [
    (dict(logits=Arr((7, 0), "f32")), "0 logits"), (dict(logits=Arr((7, 1048577), "f32")), "1048577 logits"), (dict(logits=Arr((7, 50), "i32")), "i32"),
    (dict(logits=Arr((7, 50), "f32", strides=(100, 2))), "adjacent"), (dict(logits=Arr((7, 50), "f32", ptr=4098)), "aligned"),
    (dict(logits=Arr((7, 50), "f32", ptr=0)), "NULL"), (dict(tokens=Arr((6,), "i32")), "tokens"), (dict(tokens=Arr((7,), "f32")), "tokens"),
    (dict(first=Arr((0,), "i32")), "first"), (dict(first=Arr((4, 1), "i32")), "first"), (dict(first=Arr((5,), "i32")), "u_draw"),
    (dict(u=Arr((6,), "f32")), "u"), (dict(u_draw=Arr((3,), "f16")), "u_draw"), (dict(out=Arr((8,), "i32")), "out"),
    (dict(out=Arr((7,), "i32", ptr=512)), "tokens are read"), (dict(accepted=Arr((4,), "i32")), "accepted"), (dict(draft=Arr((7, 50), "f16")), "draft"),
    (dict(draft=Arr((6, 50), "f32")), "draft"), (dict(draft=Arr((7, 50), "f32", strides=(100, 2))), "adjacent"), (dict(draft=Arr((7, 50), "f32", ptr=4098)), "aligned"),
    (dict(temperature=Arr((7,), "f32")), "temperature"), (dict(draft_temperature=Arr((3,), "i32")), "draft_temperature"),
    (dict(lens_out=Arr((3,), "i32")), "lens_out"), (dict(lens=Arr((3,), "i32"), lens_out=Arr((3,), "i32")), "lens_out"),
    (dict(prob=Arr((3,), "f32")), "prob"), (dict(max_new=-1), "max_new"), (dict(max_new=0), "max_new"), (dict(max_new=1 << 30), "in one call"),
    (dict(workspace=Arr((64,), "u8")), "workspace"), (dict(workspace=Arr((1 << 20,), "u8", ptr=4100)), "workspace"),
    (dict(first=Arr((4098,), "i32"), u_draw=Arr((4097,), "f32"), accepted=Arr((4097,), "i32")), "4097 requests")])
def test_verify_refuses(pkg, kw, err):
    from parakeet_amd import lm
    a = dict(logits=Arr((7, 50), "f32"), tokens=Arr((7,), "i32", ptr=512), first=Arr((4,), "i32"), u=Arr((7,), "f32"), u_draw=Arr((3,), "f32"),
             out=Arr((7,), "i32"), accepted=Arr((3,), "i32"), workspace=Arr((1 << 20,), "u8"))
    a.update(kw)
    refused(lm.verify, a, err)


def test_shapes(pkg):
    from parakeet_amd import lm
    assert lm.kv8_shape(7, 2, 128, 32) == (7, 2, 32 * 256 + 16)
    for bad in ((1, 1, 96, 32), (1, 1, 64, 16), (1, 1, 64, 20)):
        with pytest.raises(ValueError):
            lm.kv8_shape(*bad)


def test_rows_beyond_a_launch(pkg):
    from parakeet_amd import lm
    n = 2 ** 31 - 1
    k = Arr((n, 2, 256), "bf16")
    refused(lm.kv8_load, dict(cache=cache(dim=256), slots=Arr((n,), "i32"), k=k, v=k, page=32), "in one call")

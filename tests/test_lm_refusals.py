"""What the serving operators refuse, and how: the Python mirror's checks and the library's, all before any launch (no
GPU needed), and that the mirror's descriptors, constants and exports are the header's."""
import ctypes
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "parakeet_lm.h")


class Arr:
    """A device array that is nowhere: enough for calls that have to end before they touch it."""

    def __init__(self, shape, dtype, strides=None, ptr=4096):
        self.shape, self.dtype, self.ptr = tuple(shape), dtype, ptr
        if strides is None:
            strides, n = [], 1
            for k in reversed(self.shape):
                strides.insert(0, n)
                n *= k
        self.s = tuple(strides)

    def stride(self):
        return self.s

    def data_ptr(self):
        return self.ptr

    def is_contiguous(self):
        n = 1
        for k, s in zip(reversed(self.shape), reversed(self.s)):
            if k > 1 and s != n:
                return False
            n *= k
        return True

    def numel(self):
        n = 1
        for k in self.shape:
            n *= k
        return n


def test_exports_and_constants(pkg):
    from parakeet_amd import lm, pk
    text = open(HEADER).read()
    names = sorted(set(re.findall(r"PK_API\s+[\w\s\*]+?\b(pk_\w+)\s*\(", text)))
    assert sorted(lm.EXPORTED) == names
    lib = ctypes.CDLL(pk.LIB_PATH)
    assert all(hasattr(lib, n) for n in names)
    enum = dict(re.findall(r"PK_DTYPE_(\w+)\s*=\s*(\d+)", text))
    assert {k: getattr(lm, k) for k in enum} == {k: int(v) for k, v in enum.items()}
    define = dict(re.findall(r"#define PK_LM_(\w+) (\d+)", text))
    assert {k: getattr(lm, k) for k in define} == {k: int(v) for k, v in define.items()}


def test_descriptors_match_the_header(pkg, tmp_path):
    from parakeet_amd import lm
    want = {"pk_kv_plan_desc": (lm._PLAN, "n_tokens"), "pk_kv4_rows_desc": (lm._ROWS, "n_pages"), "pk_kv4_attend_desc": (lm._ATTEND, "scale"),
            "pk_sample_desc": (lm._SAMPLE, "reserved")}
    src = tmp_path / "s.cpp"
    src.write_text('#include "parakeet_lm.h"\n#include <cstddef>\n#include <cstdio>\nint main() {\n' + "".join(
        f'std::printf("%zu %zu\\n", sizeof({d}), offsetof({d}, {last}));\n' for d, (_, last) in want.items()) + "}\n")
    subprocess.run(["g++", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "s")], check=True)
    lines = subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout.split("\n")
    for (d, (s, _)), line in zip(want.items(), lines):
        size, last = map(int, line.split())
        assert s.size == size, d
        assert ctypes.sizeof(ctypes.c_int) == 4 and last + 4 <= size < last + 4 + 8, d


def plan_args(**kw):
    i = lambda *s: Arr(s, "i32", ptr=kw.pop("ptr", 4096))  # noqa: E731
    a = dict(old_len=Arr((3,), "i32", ptr=4096), new_len=Arr((3,), "i32", ptr=8192), table=i(3, 5), ring=i(9), state=Arr((2,), "i32", ptr=512), page=16,
             state_out=i(2), lens=Arr((3,), "i32", ptr=12288), ok=i(3), first=i(4), slots=i(7), pos=i(7))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,err", [
    (dict(page=48), "pages of 48"), (dict(page=8), "pages of 8"), (dict(old_len=Arr((2,), "i32")), "old_len"),
    (dict(first=Arr((3,), "i32")), "first"), (dict(slots=Arr((7,), "f32")), "slots"), (dict(pos=Arr((6,), "i32")), "pos"),
    (dict(state_out=Arr((2,), "i32", ptr=512)), "state_out"), (dict(lens=Arr((3,), "i32", ptr=4096)), "lens"),
    (dict(table=Arr((3, 5), "i32", strides=(4, 1))), "table rows"), (dict(table=Arr((3, 5), "i32", strides=(1, 3))), "table"),
    (dict(table=Arr((3, 50_000_000), "i32")), "32 bits"), (dict(ring=Arr((200_000_000,), "i32")), "32 bits"),
    (dict(ring=Arr((0,), "i32")), "0 pages"), (dict(lens=Arr((3,), "i32", strides=(2,))), "contiguous")])
def test_plan_refuses(pkg, kw, err):
    from parakeet_amd import lm, pk
    a = plan_args(**kw)
    with pytest.raises((pk.PkError, ValueError, TypeError), match=err):
        lm.kv_plan(a.pop("old_len"), a.pop("new_len"), a.pop("table"), a.pop("ring"), a.pop("state"), a.pop("page"), **a)


def test_plan_refuses_too_many_requests(pkg):
    from parakeet_amd import lm, pk
    n = lm.MAX_REQUESTS + 1
    i = lambda *s, p=4096: Arr(s, "i32", ptr=p)  # noqa: E731
    with pytest.raises(pk.PkError, match="requests"):
        lm.kv_plan(i(n), i(n), i(n, 2), i(5), i(2, p=512), 16, state_out=i(2), lens=i(n, p=8), ok=i(n), first=i(n + 1), slots=i(4))


def cache(n=4, heads=2, dim=128, page=32, **kw):
    return Arr((n, heads, page * (dim + dim // 16)), "u8", **kw)


@pytest.mark.parametrize("kw,err", [
    (dict(page=24), "kv4_shape|pages of 24"), (dict(cache=cache(dim=96)), "rows of|head_dim"), (dict(cache=cache(ptr=4104)), "aligned"),
    (dict(cache=Arr((4, 2, 4352), "u8", strides=(8712, 4352, 1))), "page_stride"), (dict(cache=Arr((4, 2, 4352), "u8", strides=(4352, 4352, 1))), "page_stride"),
    (dict(cache=Arr((4, 2, 4352), "u8", strides=(17408, 8704, 1))), "adjacent"), (dict(cache=Arr((4, 2, 4352), "f32")), "uint8"),
    (dict(v=Arr((5, 2, 128), "f16")), "bf16"), (dict(v=Arr((4, 2, 128), "bf16")), "v bf16"), (dict(k=Arr((5, 2, 128), "i32"), v=Arr((5, 2, 128), "i32")), "i32"),
    (dict(k=Arr((5, 2, 128), "bf16", strides=(256, 1, 2))), "adjacent"), (dict(slots=Arr((4,), "i32")), "slots"),
    (dict(k=Arr((5, 2, 128), "bf16", ptr=4097)), "aligned"), (dict(k=Arr((5, 2, 128), "bf16", ptr=0)), "NULL"),
    (dict(cache=cache(n=70_000_000)), "32 bits")])
def test_store_and_load_refuse(pkg, kw, err):
    from parakeet_amd import lm, pk
    a = dict(k=Arr((5, 2, 128), "bf16"), v=Arr((5, 2, 128), "bf16"), slots=Arr((5,), "i32"), cache=cache(), page=32)
    a.update(kw)
    with pytest.raises((pk.PkError, ValueError, TypeError), match=err):
        lm.kv4_store(a["k"], a["v"], a["slots"], a["cache"], a["page"])
    with pytest.raises((pk.PkError, ValueError, TypeError), match=err):
        lm.kv4_load(a["cache"], a["slots"], a["k"], a["v"], a["page"])


@pytest.mark.parametrize("kw,err", [
    (dict(q=Arr((3, 4, 128), "f32"), out=Arr((3, 4, 128), "f32")), "dtype"), (dict(q=Arr((3, 3, 128), "bf16"), out=Arr((3, 3, 128), "bf16")), "heads"),
    (dict(q=Arr((3, 4, 64), "bf16"), out=Arr((3, 4, 64), "bf16")), "heads of 64"), (dict(out=Arr((3, 4, 128), "f16")), "out"),
    (dict(out=Arr((3, 4, 128), "bf16", strides=(0, 128, 1))), "overlap"), (dict(lens=Arr((2,), "i32")), "lens"),
    (dict(first=Arr((3,), "i32")), "first"), (dict(lse=Arr((3, 4), "f16")), "lse"), (dict(lse=Arr((3, 2), "f32")), "lse"),
    (dict(window=-1), "window"), (dict(max_new=-1), "max_new"), (dict(max_len=-1), "max_len"), (dict(max_new=2), "without first"),
    (dict(q=Arr((4, 4, 128), "bf16"), out=Arr((4, 4, 128), "bf16")), "without first"), (dict(cache=cache(ptr=4104)), "aligned"),
    (dict(table=Arr((3, 5), "i32", strides=(3, 1))), "table rows"), (dict(q=Arr((3, 4, 128), "bf16", ptr=0)), "NULL"),
    (dict(max_len=2 ** 31 - 5000, workspace=Arr((4096,), "u8")), "workspace"), (dict(max_len=2 ** 31 - 1), "32 bits"), (dict(max_new=2 ** 30), "32 bits"),
    (dict(table=Arr((3, 2 ** 26), "i32")), "32 bits"), (dict(table=Arr((3, 0), "i32")), "width"),
    (dict(q=Arr((3, 4, 128), "bf16", strides=(1024, 1, 4))), "adjacent")])
def test_attend_refuses(pkg, kw, err):
    from parakeet_amd import lm, pk
    a = dict(q=Arr((3, 4, 128), "bf16"), cache=cache(), table=Arr((3, 5), "i32"), lens=Arr((3,), "i32"), out=Arr((3, 4, 128), "bf16"), page=32,
             max_len=100)
    a.update(kw)
    with pytest.raises((pk.PkError, ValueError, TypeError), match=err):
        lm.kv4_attend(a.pop("q"), a.pop("cache"), a.pop("table"), a.pop("lens"), a.pop("out"), a.pop("page"), **a)


@pytest.mark.parametrize("kw,err", [
    (dict(logits=Arr((3, 0), "f32")), "0 logits"), (dict(logits=Arr((3, 1048577), "f32")), "1048577 logits"), (dict(logits=Arr((3, 50), "i32")), "i32"),
    (dict(logits=Arr((3, 50), "f32", strides=(100, 2))), "adjacent"), (dict(logits=Arr((3, 50), "f32", ptr=4098)), "aligned"),
    (dict(u=Arr((2,), "f32")), "u"), (dict(u=Arr((3,), "f16")), "u"), (dict(top_k=Arr((3,), "f32")), "top_k"), (dict(top_p=Arr((3, 1), "f32")), "top_p"),
    (dict(token=Arr((3,), "f32")), "token"), (dict(token=Arr((3,), "i32", ptr=0)), "NULL"), (dict(kept=Arr((3,), "i32", strides=(2,))), "contiguous")])
def test_sample_refuses(pkg, kw, err):
    from parakeet_amd import lm, pk
    a = dict(logits=Arr((3, 50), "f32"), u=Arr((3,), "f32"), token=Arr((3,), "i32"))
    a.update(kw)
    with pytest.raises((pk.PkError, ValueError, TypeError), match=err):
        lm.sample(a.pop("logits"), a.pop("u"), a.pop("token"), **a)


def test_library_takes_no_missing_descriptor(pkg):
    from parakeet_amd import lm, pk
    lm._load()
    for name in lm.EXPORTED:
        assert lm._calls[name](None, None) == 3 and b"descriptor" in pk.lib().pk_last_error(), name


def test_kv4_shape(pkg):
    from parakeet_amd import lm
    assert lm.kv4_shape(7, 2, 128, 16) == (7, 2, 16 * 136)
    for bad in ((1, 1, 96, 16), (1, 1, 64, 20)):
        with pytest.raises(ValueError):
            lm.kv4_shape(*bad)

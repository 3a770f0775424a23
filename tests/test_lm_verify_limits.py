"""What pk_verify takes and refuses by its sizes and by where its arrays lie (no GPU needed)."""
import ctypes as C

import pytest

from test_lm_refusals import Arr
from test_lm_step_refusals import refused


def workspace(n, B, V, max_new, draft=True):
    """Bytes, None where the call is refused."""
    from parakeet_amd import lm, pk
    wanted = C.c_int64()
    try:
        lm._call("pk_verify_workspace", lm._VERIFY.pack(1 << 20, draft << 20, *[0] * 13, V, V, n, B, V, 0, max_new, 0), C.addressof(wanted))
    except pk.PkError as e:
        assert "in one call" in str(e)
        return None
    return wanted.value


@pytest.mark.parametrize("n,B,V", [(1280, 256, 1027), (810, 162, 128001), (320, 64, 128001), (20480, 4096, 8193), (20480, 4096, 128001)])
def test_the_bound_defaults_to_all_rows(pkg, n, B, V):
    """The sizes of a call go by the rows that there are, not by how many each request might have had."""
    assert 0 < workspace(n, B, V, n) <= 2 * workspace(n, B, V, 5)
    assert workspace(n, B, V, (2 ** 31 - 1) // B) and workspace(n, B, V, 2 ** 31 // B + 1) is None


@pytest.mark.parametrize("kw,err", [
    (dict(out=Arr((7,), "i32", ptr=4096 + 4)), "tokens are read"), (dict(out=Arr((7,), "i32", ptr=4096 - 24)), "tokens are read"),
    (dict(lens=Arr((3,), "i32", ptr=8192), lens_out=Arr((3,), "i32", ptr=8192 + 8)), "lens_out"),
    (dict(lens=Arr((3,), "i32", ptr=8192), lens_out=Arr((3,), "i32", ptr=8192 - 4)), "lens_out")])
def test_outputs_that_lie_over_what_is_read_are_refused(pkg, kw, err):
    from parakeet_amd import lm
    a = dict(logits=Arr((7, 50), "f32"), tokens=Arr((7,), "i32", ptr=4096), first=Arr((4,), "i32"), u=Arr((7,), "f32"), u_draw=Arr((3,), "f32"),
             out=Arr((7,), "i32", ptr=1 << 16), accepted=Arr((3,), "i32"), workspace=Arr((1 << 20,), "u8"))
    a.update(kw)
    refused(lm.verify, a, err)


def test_a_call_without_rows_is_asked_for_its_requests_arrays(pkg):
    from parakeet_amd import lm
    none = dict(logits=Arr((0, 50), "f32", ptr=0), tokens=Arr((0,), "i32", ptr=0), u=Arr((0,), "f32", ptr=0), out=Arr((0,), "i32", ptr=0))
    a = dict(none, first=Arr((4,), "i32"), u_draw=Arr((3,), "f32"), accepted=Arr((3,), "i32"), workspace=Arr((1 << 20,), "u8"))
    for name in ("first", "u_draw", "accepted"):
        refused(lm.verify, dict(a, **{name: Arr(a[name].shape, a[name].dtype, ptr=0)}), "NULL")

"""Arguments at the ends of what the serving operators take, refused before any launch (no GPU needed)."""
import pytest

from test_lm_refusals import Arr, cache


def attend(**kw):
    from parakeet_amd import lm
    a = dict(q=Arr((3, 4, 128), "bf16"), cache=cache(), table=Arr((3, 5), "i32"), lens=Arr((3,), "i32"), out=Arr((3, 4, 128), "bf16"), page=32,
             max_len=100)
    a.update(kw)
    return lm.kv4_attend(a.pop("q"), a.pop("cache"), a.pop("table"), a.pop("lens"), a.pop("out"), a.pop("page"), **a)


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), float("-inf"), 1e39])
def test_scales_that_are_no_numbers(pkg, scale):
    from parakeet_amd import pk
    with pytest.raises((pk.PkError, OverflowError), match="scale|float"):
        attend(scale=scale)

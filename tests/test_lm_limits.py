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


@pytest.mark.parametrize("dtype,dim", [("bf16", 128), ("f16", 256)])
def test_more_attention_than_a_launch_holds(pkg, dtype, dim):
    """A launch has fewer than 2^32 threads."""
    from parakeet_amd import pk
    q = Arr((3, 4, dim), dtype)
    with pytest.raises(pk.PkError, match="in one call"):
        attend(q=q, out=q, cache=cache(dim=dim), first=Arr((4,), "i32"), max_new=1 << 28)
    many = 1 << 24
    q = Arr((many, 4, dim), dtype)
    with pytest.raises(pk.PkError, match="in one call"):
        attend(q=q, out=q, cache=cache(dim=dim), table=Arr((many, 5), "i32"), lens=Arr((many,), "i32"))


def test_more_rows_than_a_launch_holds(pkg):
    from parakeet_amd import lm, pk
    for n, dim in (((1 << 29) + 1, 256), ((1 << 31) - 1, 128)):
        k = Arr((n, 2, dim), "bf16")
        for call in (lambda: lm.kv4_store(k, k, Arr((n,), "i32"), cache(dim=dim), 32), lambda: lm.kv4_load(cache(dim=dim), Arr((n,), "i32"), k, k, 32)):
            with pytest.raises(pk.PkError, match="in one call"):
                call()


@pytest.mark.parametrize("rows,vocab", [(1 << 24, 50), (1 << 22, 2049), (1 << 22, 16384)])
def test_more_samples_than_a_launch_holds(pkg, rows, vocab):
    from parakeet_amd import lm, pk
    with pytest.raises(pk.PkError, match="in one call"):
        lm.sample(Arr((rows, vocab), "f16"), Arr((rows,), "f32"), Arr((rows,), "i32"))

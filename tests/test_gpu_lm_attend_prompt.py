"""The attention kernel for prompts on the cases of the other one.  Which of the two a call gets follows from its upper
bounds alone, so a bound of many new tokens brings it to small cases; the results do not depend on it."""
import pytest

import test_gpu_lm_attend as A

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def bound_of_many(monkeypatch):
    own = A.run

    def run(p, window=0, scale=None, first=True, max_len=None, max_new=None, **kw):
        return own(p, window, scale, True, max_len, 70000 if max_new is None else max_new, **kw)
    monkeypatch.setattr(A, "run", run)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_prompts(D, dtype, page):
    A.check(A.problem(D + page, D, page, 4, 2, [130, 300, 65, 40, 3, 97, 1, 0, 64], [130, 37, 5, 0, 9, 64, 1, 1, 64], dtype))


@pytest.mark.parametrize("heads", [(1, 1), (3, 3), (8, 1), (12, 4), (32, 2), (20, 1)])
def test_head_layouts(heads):
    for D in (64, 128):
        A.check(A.problem(sum(heads), D, 64, *heads, [70, 45, 133], [3, 45, 17], "bf16"))


@pytest.mark.parametrize("window", [1, 7, 32, 100])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_windows(window, dtype):
    A.test_windows(window, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_nan_reaches_only_those_that_see_it(dtype, D):
    A.test_nan_reaches_only_those_that_see_it(dtype, D, (50, 60, 1))


def test_scales_and_large_values():
    A.test_scales_and_large_values()


def test_page_ids_out_of_range_are_skipped():
    A.test_page_ids_out_of_range_are_skipped()


def test_long_axes():
    A.test_prompts_over_a_long_axis()
    A.check(A.problem(20, 128, 128, 8, 2, [9001, 4097], [3, 300], "bf16"))


def test_both_kernels_agree():
    p = A.problem(17, 128, 64, 8, 2, [700, 90], [90, 7], "bf16")
    A.check(p)
    A.check(p, max_new=90)


def test_lengths_are_cut_at_max_len_and_table():
    A.test_lengths_are_cut_at_max_len_and_table()

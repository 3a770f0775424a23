"""NaN blocks of V in key tiles that only some waves of a prompt's workgroup see in part: a wave whose columns see the
whole tile has to get the NaN too."""
import numpy as np
import pytest

import test_gpu_lm_attend as A
from test_gpu_lm_attend_prompt import bound_of_many  # noqa: F401  (every call goes to the prompt kernel)

pytestmark = pytest.mark.gpu


def poison(p, key, head, block):
    page, D = p["page"], p["D"]
    p["cache"][p["table"][0, key // page], head, page * D + page * (D // 32) + block * page + key % page] = 255


def check(p, **kw):
    out, _ = A.check(p, **kw)
    return np.isnan(out).any(-1)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("D,page", [(64, 64), (128, 16), (128, 128), (256, 32)])
def test_fresh_prompt(dtype, D, page):
    """128 tokens of one head a kv head: the first 64 keys are an edge for waves 0 and 1 alone."""
    p = A.problem(D, D, page, 2, 2, [128], [128], dtype)
    poison(p, 10, 0, 0)
    poison(p, 63, 1, D // 32 - 1)
    nan = check(p)
    assert nan[10:, 0].all() and not nan[:10, 0].any() and nan[63:, 1].all() and not nan[:63, 1].any()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128])
def test_prompt_behind_held_tokens(dtype, D):
    """50 tokens held, two query heads a kv head: the first 64 keys are an edge for wave 0 alone."""
    p = A.problem(D + 1, D, 64, 2, 1, [114], [64], dtype)
    poison(p, 10, 0, 1)
    assert check(p).all()


@pytest.mark.parametrize("D,page", [(64, 16), (128, 64), (256, 64)])
def test_windows(D, page):
    """300 tokens held, a window of 200: keys 192 .. 255 are whole for waves 0 and 1, and cut by the windows of 2 and 3."""
    p = A.problem(D, D, page, 1, 1, [428], [128], "bf16")
    poison(p, 200, 0, 0)
    poison(p, 230, 0, 1)
    nan = check(p, window=200)
    assert nan.all()

"""pk_verify: NaN logits beside the largest ones."""
import numpy as np
import pytest

from test_gpu_lm_verify import call

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V", [70, 3001, 8193, 20000])
@pytest.mark.parametrize("most", [np.inf, np.finfo(np.float32).max])
def test_nan_beside_the_largest_number(V, most):
    """NaN counts as -inf also where +inf, or what it counts as, is in the row: greedy targets, and greedy drafts."""
    x = np.zeros((2, V), np.float32)
    x[:, 3], x[:, 9], x[:, V - 1] = np.nan, most, np.nan
    for d, want in ((9, [9, 9]), (3, [9, -1])):
        out, stood, _, prob = call(x, None, [0, d], [0, 2], [0.5] * 2, [0.99], t=[0.0])
        assert list(out) == want and stood[0] == (d == 9) and prob[0] == 1
    assert list(call(x, None, [0, 9], [0, 2], [0.5] * 2, [0.99])[0]) == [9, 9]
    even = np.zeros((2, V), np.float32)
    for d in (9, 3):        # q is 1 at 9: a draft of 9 is refused, what is left begins at 0; one of 3 was none that q would draw
        out, stood, _, _ = call(even, x, [0, d], [0, 2], [0.9] * 2, [0.0], td=[0.0])
        assert stood[0] == (d == 3) and out[0] == (3 if d == 3 else 0)

"""pk_verify without max_new, and calls whose requests bring rows of very different numbers: the same answers, whatever bound is given."""
import os
import subprocess
import sys

import numpy as np
import pytest

import lm_reference as R
from test_gpu_lm_verify import call

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,V,dtype,drafted", [(256, 1027, "f32", True), (256, 130, "f32", False), (1000, 64, "bf16", True), (162, 17000, "bf16", True),
                                               (64, 40003, "bf16", False)])
def test_the_bound_may_be_left_out(B, V, dtype, drafted):
    g = np.random.default_rng(V)
    x = g.standard_normal((5 * B, V)) * 3
    x, y = R.to_dtype(x, dtype), R.to_dtype(x + g.standard_normal(x.shape), dtype) if drafted else None
    tokens = np.concatenate([[0], R.to_f64(x, dtype).argmax(1)[:-1]])
    rest = tokens, 5 * np.arange(B + 1), g.random(5 * B), g.random(B), dtype
    a, b, c = (call(x, y, *rest, lens=np.full(B, 99), max_new=m) for m in (5, None, 9))
    for other in (b, c):
        assert all(np.array_equal(i, j) for i, j in zip(a, other))
    assert a[1].max() >= 1 and a[1].min() == 0


@pytest.mark.parametrize("V", [40, 5000, 17000])
def test_one_request_of_many_rows_among_short_ones(V):
    """The long one's rows, far more than the others have, stand up to one that refuses."""
    B, n, stop = 70, 701, 640
    news = np.ones(B, int)
    news[33], news[40], news[50] = n, 4, 0
    first = np.concatenate([[0], np.cumsum(news)])
    N, at = int(first[-1]), int(first[33])
    x = np.zeros((N, V), np.float32)
    x[:, 7] = 90.0
    x[at + stop, 7], x[at + stop, 9] = 0.0, 90.0
    for m in (None, n):
        for _ in range(2):
            out, acc, lens, prob = call(x, None, np.full(N, 7), first, np.full(N, 0.5), np.full(B, 0.5), lens=np.full(B, 999), max_new=m)
            want = np.full(N, 7)
            want[at + stop], want[at + stop + 1:at + n] = 9, -1
            assert np.array_equal(out, want) and np.array_equal(prob, (want >= 0).astype(np.float32))
            assert acc[33] == stop and acc[40] == 3 and acc.sum() == stop + 3
            assert lens[33] == 999 - (n - 1 - stop) and (np.delete(lens, 33) == 999).all()


def test_as_many_requests_as_a_call_takes():
    """4,096 requests of none to two rows of a vocabulary that is cut in chunks: each row finds its own."""
    B, V = 4096, 16400
    news = np.arange(B) * 7 % 3
    first = np.concatenate([[0], np.cumsum(news)])
    N = int(first[-1])
    token = np.arange(N) % V
    x = np.zeros((N, V), np.uint16)
    x[np.arange(N), token] = R.to_dtype(90.0, "bf16")
    tokens = np.concatenate([[0], token[:-1]])
    tokens[first[:-1][news == 2][::2] + 1] = V - 1                      # every other draft is refused
    for m in (None, 2):
        out, acc, lens, prob = call(x, None, tokens, first, np.full(N, 0.5), np.full(B, 0.5), "bf16", lens=np.full(B, 9), max_new=m)
        stood = np.zeros(B, int)
        stood[np.flatnonzero(news == 2)[1::2]] = 1
        want = token.copy()
        want[first[:-1][(news == 2) & (stood == 0)] + 1] = -1
        assert np.array_equal(acc, stood) and np.array_equal(out, want) and np.array_equal(lens, 9 - np.maximum(news - 1 - stood, 0))
        assert np.array_equal(prob, (want >= 0).astype(np.float32))


@pytest.mark.parametrize("V", [30, 17000])
def test_offsets_outside_the_rows_and_over_each_other(V):
    """Offsets are cut to the call's rows; requests over each other's rows leave theirs undefined, and the next call whole."""
    x = np.zeros((6, V), np.float32)
    x[:, 3] = 60
    out, acc, lens, _ = call(x, None, [0, 3, 3, 3, 3, 3], [0, 6], [0.5] * 6, [0.5], lens=[50], max_new=3)
    assert acc[0] == 2 and list(out) == [3, 3, 3, -9, -9, -9]
    for _ in range(2):
        out, acc, _, _ = call(x, None, [0, 3, 3, 3, 3, 3], [-5, 2, 900, 4], [0.5] * 6, [0.5] * 3, max_new=9)
        assert list(acc) == [1, 3, 0] and (out == 3).all()
        for first in ([0, 5, 2, 6], [4, 1, 6, 0], [-9, 99, -9, 99]):
            _, acc, _, _ = call(x, None, [0, 3, 3, 3, 3, 3], first, [0.5] * 6, [0.5] * 3, max_new=9)
            assert (0 <= acc).all() and (acc < 6).all()


TORCH_EMPTY = """
import sys
import torch
sys.path.insert(0, sys.argv[1])
import __graft_entry__ as graft
graft.load_package()
from parakeet_amd import lm
i32 = dict(dtype=torch.int32, device="cuda")
for V in (50, 17000):
    for more in (dict(), dict(max_new=5), dict(draft=torch.zeros(0, V, device="cuda"))):
        accepted, cut = torch.full((3,), -9, **i32), torch.full((3,), -9, **i32)
        lens = torch.tensor([5, 0, 77], **i32)
        lm.verify(torch.zeros(0, V, device="cuda"), torch.zeros(0, **i32), torch.zeros(4, **i32), torch.zeros(0, device="cuda"),
                  torch.zeros(3, device="cuda"), torch.zeros(0, **i32), accepted, lens=lens, lens_out=cut, **more)
        assert accepted.tolist() == [0, 0, 0] and cut.tolist() == [5, 0, 77], (V, accepted, cut)
print("ok empty")
"""


@pytest.mark.parametrize("V", [50, 17000])
def test_a_call_without_rows(V):
    """A step to which no request brings a token: nothing is accepted, lengths stay."""
    for m in (None, 0, 5):
        for y in (None, np.zeros((0, V), np.float32)):
            out, acc, lens, _ = call(np.zeros((0, V), np.float32), y, [], [0] * 4, [], [0.5] * 3, lens=[5, 0, 77], max_new=m)
            assert list(acc) == [0, 0, 0] and list(lens) == [5, 0, 77]


def test_a_call_without_rows_on_torch_tensors():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    p = subprocess.run([sys.executable, "-c", TORCH_EMPTY, root], capture_output=True, text=True, timeout=110)
    assert p.returncode == 0 and "ok empty" in p.stdout, p.stdout[-1000:] + p.stderr[-3000:]

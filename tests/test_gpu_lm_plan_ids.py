"""pk_kv_plan on tables and rings that hold ids which are no pages: a token on such a page has no slot, also where the id
times the page's size would wrap round to a slot of another page."""
import numpy as np
import pytest

import lm_reference as R
import test_gpu_lm_plan as P

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_ids_without_a_slot(page):
    width, n = 6, 40
    wrap = (1 << 32) // page                       # wrap * page = 0 in 32 bits
    bad = [wrap // 2, wrap // 2 - 1 + wrap // 2, -1, -wrap // 2, wrap // 4 * 2, -(1 << 31)]
    bad = np.array([b if b < 1 << 31 else b - (1 << 32) for b in bad], np.int64)
    last = (1 << 31) // page - 1                   # the largest id whose slots are 32-bit numbers
    g = np.random.default_rng(page)
    table = g.permutation(n).astype(np.int32)[:4 * width].reshape(4, width)
    old = np.array([page // 2, 3 * page, 0, page + 1], np.int32)
    new = np.array([page // 2 + 3, 3 * page + 1, 4 * page, page + 2], np.int32)
    table[0, 0], table[3, 1] = bad[0], last
    ring = np.arange(n, dtype=np.int32)
    ring[1:5] = bad[1:5]                           # request 1 takes ring[0], request 2 ring[1 .. 4]
    cap = int((new - old).sum()) + 3
    got = P.run(old, new, table, ring, np.array([0, n], np.int32), page, cap)
    want = R.plan(old.astype(np.int64), new.astype(np.int64), table.astype(np.int64), ring.astype(np.int64),
                  np.array([0, n]), page, 0)       # the plain form's table, positions and slots without wrapping:
    first, slots, pos = want["first"], np.full(cap, -1, np.int64), np.full(cap, -1, np.int64)
    for b in range(4):
        for i, q in enumerate(range(old[b], new[b])):
            at, pos[first[b] + i] = int(want["table"][b, q // page]), q
            slots[first[b] + i] = at * page + q % page if 0 <= at <= last else -1
    assert np.array_equal(got["slots"], slots) and np.array_equal(got["pos"], pos) and (slots >= 0).sum() == 2
    for k in ("table", "ring", "state_out", "lens", "ok", "first"):
        assert np.array_equal(got[k], want[k]), k

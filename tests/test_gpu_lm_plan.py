"""pk_kv_plan against the plain statement of it: page tables, slot maps, positions and the ring, exactly."""
import numpy as np
import pytest

import lm_reference as R

pytestmark = pytest.mark.gpu


def run(old, new, table, ring, state, page, cap, stride=None, pos=True, stream=None):
    from parakeet_amd import hipmem, lm
    i32 = lambda a: hipmem.Tensor.from_numpy(np.ascontiguousarray(a, np.int32))  # noqa: E731
    B, width = table.shape
    if stride:
        wide = np.full((B, stride), -7, np.int32)
        wide[:, :width] = table
        tab = i32(wide).view((B, width), (stride, 1))
    else:
        tab = i32(table)
    o = dict(ring=i32(ring), state_out=i32(np.full(2, -9)), lens=i32(np.full(B, -9)), ok=i32(np.full(B, -9)),
             first=i32(np.full(B + 1, -9)), slots=i32(np.full(cap, -9)), pos=i32(np.full(cap, -9)))
    lm.kv_plan(i32(old), i32(new), tab, o["ring"], i32(state), page, state_out=o["state_out"], lens=o["lens"], ok=o["ok"],
               first=o["first"], slots=o["slots"], pos=o["pos"] if pos else None, stream=stream)
    hipmem.synchronize()
    got = {k: v.numpy() for k, v in o.items()}
    got["table"] = tab.numpy()
    if not pos:
        del got["pos"]
    return got


def check(old, new, table, ring, state, page, cap, **kw):
    want = R.plan(old, new, table, ring, state, page, cap)
    got = run(old, new, table, ring, state, page, cap, **kw)
    for k, v in got.items():
        assert np.array_equal(v, want[k]), k
    return want


def start(g, B, width, page, free, n, full=1.0):
    """A random state: requests of random lengths, their pages dealt from n, `free` pages left in the ring."""
    old = g.integers(0, int(width * page * full) + 1, B).astype(np.int32)
    held = -(-old // page)
    while held.sum() > n - free:
        b = g.integers(B)
        old[b] //= 2
        held = -(-old // page)
    ids = g.permutation(n).astype(np.int32)
    table = np.full((B, width), 12345678, np.int32)
    at = 0
    for b in range(B):
        table[b, :held[b]] = ids[at:at + held[b]]
        at += held[b]
    head = int(g.integers(0, n))
    ring = np.full(n, 87654321, np.int32)
    for i in range(free):
        ring[(head + i) % n] = ids[at + i]
    return old, table, ring, np.array([head, free], np.int32)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("B", [1, 2, 63, 257])
def test_mixed_steps(B, page):
    g = np.random.default_rng(B * 1000 + page)
    width, n = 7, 3 * B + 20
    for step, free in enumerate((n // 3, 3, 0)):
        old, table, ring, state = start(g, B, width, page, free, n, 0.6)
        new = old.copy()
        kind = g.integers(0, 6, B)
        new[kind == 0] += 1
        new[kind == 1] = g.integers(0, width * page + 1, (kind == 1).sum())
        new[kind == 2] = 0
        new[kind == 3] = old[kind == 3] // 2
        new[kind == 4] = np.minimum(old[kind == 4] + page, width * page)
        new = np.minimum(new, width * page).astype(np.int32)
        total = int(np.maximum(new - old, 0).sum())
        check(old, new, table, ring, state, page, total + (0, 5, 33)[step], stride=(None, width + 3, None)[step])


def test_requests_out_of_range_and_a_short_slot_map():
    g = np.random.default_rng(8)
    old, table, ring, state = start(g, 6, 4, 16, 9, 30, 0.5)
    new = old + 3
    old[1], new[2], new[3], old[4] = -5, -1, 4 * 16 + 1, 4 * 16 + 1
    check(old, new.astype(np.int32), table, ring, state, 16, 2)


def test_not_enough_pages_serves_a_prefix_and_those_that_need_none():
    page, width = 16, 8
    old = np.array([16, 16, 16, 17, 40], np.int32)
    new = np.array([40, 100, 32, 18, 3], np.int32)
    table = np.arange(5 * width, dtype=np.int32).reshape(5, width)
    ring = np.arange(100, 160, dtype=np.int32)
    want = check(old, new, table, ring, np.array([57, 4], np.int32), page, 200)     # the ring's end wraps
    assert want["ok"].tolist() == [1, 0, 0, 1, 1] and want["state_out"].tolist() == [59, 4]


def test_ends_of_range():
    """No tokens, no slots, an empty ring, one request of the largest kind, the most requests of a call."""
    z = lambda *s: np.zeros(s, np.int32)  # noqa: E731
    check(z(3), z(3), z(3, 2), z(4), z(2), 16, 0)
    check(z(0), z(0), z(0, 2), z(4), z(2), 16, 5)
    g = np.random.default_rng(1)
    check(z(1), np.array([200003], np.int32), z(1, 1600), g.permutation(1600).astype(np.int32), np.array([1500, 1600], np.int32), 128, 200003)
    B = 4096
    old, table, ring, state = start(g, B, 3, 16, 5000, 20000)
    check(old, np.minimum(old + 1, 48).astype(np.int32), table, ring, state, 16, B + 1)


def test_same_call_again_gives_the_same():
    from parakeet_amd import hipmem, lm
    i32 = lambda a: hipmem.Tensor.from_numpy(np.ascontiguousarray(a, np.int32))  # noqa: E731
    g = np.random.default_rng(4)
    old, table, ring, state = start(g, 50, 6, 16, 60, 200, 0.5)
    new = g.integers(0, 97, 50).astype(np.int32)
    total = int(np.maximum(new - old, 0).sum())
    want = R.plan(old, new, table, ring, state, 16, total)
    t, r = i32(table), i32(ring)
    a = [i32(old), i32(new), t, r, i32(state)]
    o = {k: i32(np.zeros_like(want[k])) for k in ("state_out", "lens", "ok", "first", "slots", "pos")}
    for _ in range(3):
        lm.kv_plan(*a, 16, **o)
    hipmem.synchronize()
    for k, v in dict(o, table=t, ring=r).items():
        assert np.array_equal(v.numpy(), want[k]), k

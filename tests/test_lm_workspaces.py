"""Which workspace a call on hipmem tensors gets (no GPU needed: the device's state and its memory are stood in for)."""
import pytest


class Memory:
    def __init__(self, shape, dtype, contiguous=True):
        self.shape, self.dtype, self.zeroed, self.contiguous = shape, dtype, False, contiguous

    def zero(self):
        self.zeroed = True

    def numel(self):
        return self.shape[0]

    def data_ptr(self):
        return id(self)

    def is_contiguous(self):
        return self.contiguous


@pytest.fixture
def state(pkg, monkeypatch):
    from parakeet_amd import hipmem, lm
    s = dict(device=0, capturing=False, waits=0)
    monkeypatch.setattr(lm, "_workspaces", {})
    monkeypatch.setattr(hipmem, "Tensor", Memory)
    monkeypatch.setattr(hipmem, "device", lambda: s["device"], raising=False)
    monkeypatch.setattr(hipmem, "capturing", lambda stream: s["capturing"], raising=False)
    monkeypatch.setattr(hipmem, "synchronize", lambda: s.update(waits=s["waits"] + 1))
    return s


def test_each_device_and_stream_has_its_own(state):
    from parakeet_amd import lm
    a = lm._workspace("attend", None, 100, None)
    assert lm._workspace("attend", None, 5000, None) == a and a[1] >= 5000 and state["waits"] == 1
    state["device"] = 1
    b = lm._workspace("attend", None, 100, None)
    assert b[0] != a[0]
    assert lm._workspace("attend", 8, 100, None)[0] not in (a[0], b[0]) and lm._workspace("sample", None, 100, None)[0] not in (a[0], b[0])
    state["device"] = 0
    assert lm._workspace("attend", None, 100, None) == a
    assert all(w.zeroed for kept in lm._workspaces.values() for w in kept)


def test_none_is_made_during_a_capture(state):
    from parakeet_amd import lm
    kept = lm._workspace("attend", 8, 100, None)
    state["capturing"] = True
    assert lm._workspace("attend", 8, 100, None) == kept
    for stream, wanted in ((16, 100), (8, 1 << 22)):
        with pytest.raises(RuntimeError, match="workspace="):
            lm._workspace("attend", stream, wanted, None)
    own = Memory((1 << 22,), "u8")
    assert lm._workspace("attend", 16, 1 << 22, own) == (own.data_ptr(), 1 << 22) and lm._workspace("attend", 16, 0, None) == (0, 0)


@pytest.mark.parametrize("given", [Memory((64,), "f32"), Memory((64,), "u8", contiguous=False)])
def test_a_given_one_is_contiguous_bytes(state, given):
    from parakeet_amd import lm
    with pytest.raises(TypeError, match="uint8"):
        lm._workspace("attend", None, 10, given)

"""ops.PagedCache's own bookkeeping on the CPU, its device arrays counted and not made."""
import numpy as np
import pytest

from helpers import ops


class Counted:
    """A device array that is only an address and a size."""
    live = {}

    def __init__(self, shape, dtype, zero=False):
        self.shape, self.zero = shape, zero
        self.nbytes = int(np.prod(shape)) * np.dtype(dtype).itemsize
        self.ptr = 4096 + len(Counted.live)
        Counted.live[self] = self.nbytes

    @classmethod
    def from_host(cls, a):
        return cls(a.shape, a.dtype)

    def free(self):
        Counted.live.pop(self, None)


@pytest.fixture
def counted(monkeypatch):
    Counted.live = {}
    monkeypatch.setattr(ops, "DeviceArray", Counted)
    monkeypatch.setattr(ops, "sync", lambda: None)
    return Counted.live


def test_one_workspace(counted):
    """Calls of many sizes hold the largest's workspace and no other, zero-filled."""
    c = ops.PagedCache(4, 2, 40, 32, 8)
    before = sum(counted.values())
    f, sizes = ops.lib().oxb_attn_prefill_paged_ws_bytes, []
    for n in (1, 300, 40, 700, 512, 1100, 9):
        need = f(n, 4, 8, 2, 128)
        sizes.append(need)
        ptr, have = c._workspace(need)
        assert have == max(sizes) and c._ws.ptr == ptr and c._ws.zero
        assert sum(counted.values()) - before == max(sizes)
    with pytest.raises(ValueError):
        c._workspace(0)

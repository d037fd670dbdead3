"""ops.PagedCache's own bookkeeping on the CPU, its device arrays counted and not made, and
refusals of calls larger than a launch, and workspaces over all batches."""
import ctypes as C

import numpy as np
import pytest

from helpers import ops, pkg


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


def test_shapes_are_checked_before_anything_is_allocated(counted):
    for batch, table_pages in ((0, 8), (-1, 8), (4097, 8), (4, 0), (4, -3), (4, (1 << 19) + 1)):
        with pytest.raises(ValueError):
            ops.PagedCache(batch, 2, 40, 32, table_pages)
    with pytest.raises(ops.NativeError):
        ops.PagedCache(4, 2, 40, 33, 8)
    assert not counted
    ops.PagedCache(4096, 2, 40, 32, 8), ops.PagedCache(1, 2, 40, 32, 1 << 19)
    header = open(ops.__file__.replace("0xbitnet_amd/ops.py", "include/oxbitnet_ops.h")).read()
    for name, value in (("UNIT 32", ops.PAGED_UNIT), ("MAX_SEQ (1 << 24)", ops.PAGED_MAX_SEQ),
                        ("MAX_BATCH 4096", ops.PAGED_MAX_BATCH), ("MAX_PREFILL 128", ops.PAGED_MAX_PREFILL)):
        assert f"#define OXB_PAGED_{name}\n" in header and value == eval(name.split(" ", 1)[1])


def test_calls_larger_than_a_launch():
    """2^32 threads or more are refused before any device call."""
    L, P = ops.lib(), C.c_void_p(4096)
    last = pkg._native.last_error
    for n in ((1 << 29) - 31, (1 << 30) - 1, 2 ** 31 - 1):
        assert L.oxb_paged_append(P, 4, 32, 1, 128, P, P, 128, 128, None, P, n, None) == -1
        assert f"{n} tokens" in last()
    for w in (1, 1 << 10):      # uncut or cut
        assert L.oxb_attn_decode_paged(P, 0, P, 4, 32, P, w, P, 4096, 4096, 4096, 128, P, P, 1 << 40, None) == -1
        assert "batch 4096 of 4096 kv heads" in last()


def test_workspace_grows_with_the_batch():
    """Up to the most sequences that a call takes, every size there is."""
    f = ops.lib().oxb_attn_prefill_paged_ws_bytes
    for H, hkv in ((20, 5), (8, 8), (32, 2), (7, 1), (640, 640)):
        for n in (1, 33, 129, 1000, 4096, 33000, 100000):
            last = 1
            for b in (1, 2, 64, 65, 127, 128):
                assert f(n, b, H, hkv, 128) >= last
                last = f(n, b, H, hkv, 128)
            assert f(n, 129, H, hkv, 128) == 0
        sizes = [f(n, 128, H, hkv, 128) for n in (1, 2, 500, 8000, 33000, 500000, 4000000)]
        assert sizes[0] > 0 and sizes == sorted(sizes) and sizes[-1] == sizes[-2]

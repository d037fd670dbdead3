"""Logit rules on the GPU: lists as long as their counts allow."""
import numpy as np
import pytest

from helpers import ops
import kv8_reference as ref
from test_gpu_kv8 import bits, rng_of

pytestmark = pytest.mark.gpu


def test_rules_at_the_end_of_the_longest_lists():
    """Rows whose ids are the last of 2^31 - 1 (8 GB each of ids and values): a thread's
    next places lie past what 31 bits hold."""
    L, rng = ops.lib(), rng_of("longest")
    V, n = 9000, 2 ** 31 - 1
    lens_h, lens_b = [5000, 37], [700, 3]
    x = rng.standard_normal((2, V)).astype(np.float32)
    pen = np.array([[1.3, 0.2, 0.4], [0.8, 0.5, 0.125]], np.float32)
    hist = [rng.integers(0, V, m).astype(np.int32) for m in lens_h]
    ids = [rng.integers(0, V, m).astype(np.int32) for m in lens_b]
    val = [rng.standard_normal(m).astype(np.float32) for m in lens_b]

    def at_end(parts, dtype):
        a = ops.DeviceArray((n,), dtype)
        flat = np.concatenate(parts)
        ops.check(L.oxb_memcpy_h2d(a.offset(4 * (n - flat.size)), flat.ctypes.data, flat.nbytes, None))
        off = n - np.cumsum([flat.size, *[-p.size for p in parts]])
        return a, ops.DeviceArray.from_host(off.astype(np.int32))

    dh, ho = at_end(hist, np.int32)
    di, bo = at_end(ids, np.int32)
    dv, _ = at_end(val, np.float32)
    dx, dp = ops.DeviceArray.from_host(x), ops.DeviceArray.from_host(pen)
    out = ops.DeviceArray((2, V), np.float32)
    assert ho.download()[-1] == n and bo.download()[-1] == n
    ops.check(L.oxb_logits_rules(dx.ptr, V, 2, V, dp.ptr, dh.ptr, ho.ptr, n, di.ptr, dv.ptr, bo.ptr, n, None, 0,
                                 out.ptr, V, None))
    ops.sync()
    want = ref.rules(x, pen, [h.tolist() for h in hist], [list(zip(i.tolist(), v.tolist())) for i, v in zip(ids, val)],
                     None)
    assert np.array_equal(bits(out.download()), bits(want))


@pytest.mark.parametrize("off", [[0, -1, 20], [-5, -2, -1], [20, 10, 0], [-2 ** 31, 2 ** 31 - 1, 5]])
def test_rules_with_offsets_outside_the_lists(off):
    """Ranges are kept inside the lists; one that ends before it begins is empty."""
    L, rng = ops.lib(), rng_of("offsets", off)
    V, m = 300, 20
    x = rng.standard_normal((2, V)).astype(np.float32)
    pen = np.array([[1.3, 0.2, 0.4]] * 2, np.float32)
    ids, val = rng.integers(0, V, m).astype(np.int32), rng.standard_normal(m).astype(np.float32)
    dx, dp, di, dv, do = (ops.DeviceArray.from_host(a) for a in (x, pen, ids, val, np.array(off, np.int32)))
    out = ops.DeviceArray((2, V), np.float32)
    ops.check(L.oxb_logits_rules(dx.ptr, V, 2, V, dp.ptr, di.ptr, do.ptr, m, di.ptr, dv.ptr, do.ptr, m, None, 0,
                                 out.ptr, V, None))
    ops.sync()
    o = np.clip(off, 0, m)
    r = [slice(o[i], max(o[i], o[i + 1])) for i in (0, 1)]
    want = ref.rules(x, pen, [ids[s].tolist() for s in r], [list(zip(ids[s].tolist(), val[s].tolist())) for s in r], None)
    assert np.array_equal(bits(out.download()), bits(want))

"""The 8-bit cache's calls at the ends of their documented ranges on the GPU."""
import numpy as np
import pytest

from helpers import ops
import kv8_reference as ref
from test_gpu_kv8 import FMTS, HD, bits, filled, held, new_cache, rng_of, rows

pytestmark = pytest.mark.gpu


def test_decode_more_rows_than_arrival_counters():
    """300 sequences of 5 KV heads: rows past 1024 have one run each, whatever their length."""
    B, H, hkv = 300, 10, 5
    rng = rng_of("rows")
    lens = [(37 * z) % 400 for z in range(B)]
    c, K, V = filled(rng, lens, hkv, 400, 0)
    q = rng.standard_normal((B, H * HD)).astype(np.float32)
    got = c.attn_decode(q, [n - 1 for n in lens], True)
    w = c.weights()
    for z in range(0, B, 13):
        want, tol, ww, wtol = ref.attend_rows(q[z:z + 1], K[z], V[z], hkv, lens[z] - 1)
        ref.check_rows(got[z:z + 1], want, tol + 1e-37, z)
        nb = (lens[z] + 31) // 32
        ref.check_rows(w[z, :, :nb], ww[:, :nb], wtol[:, :nb], z)


@pytest.mark.parametrize("n,pos0", [(5, 300), (1, 0), (40, 500)])
def test_prefill_more_kv_heads_than_resident_workgroups(n, pos0):
    """600 KV heads: nothing is cut, and nothing runs beside its pair."""
    hkv, fmt = 600, n % 2
    rng = rng_of("heads", n, pos0)
    c, K, V = filled(rng, [pos0 + n], hkv, pos0 + n, fmt)
    q = rng.standard_normal((n, hkv * HD)).astype(np.float32)
    got = c.attn_prefill(q, pos0, add_weights=True).reshape(n, hkv, HD)
    w = c.weights()[0]
    for h in (0, 1, 255, 256, 511, 512, 599):
        want, tol, ww, wtol = ref.attend_rows(q.reshape(n, hkv, HD)[:, h], K[0][h:h + 1], V[0][h:h + 1], 1, pos0)
        ref.check_rows(got[:, h], want, tol, h)
        ref.check_rows(w[h:h + 1], ww, wtol, h)


@pytest.mark.parametrize("fmt", FMTS)
def test_append_begins_an_earlier_block_again(fmt):
    """From a block's start any earlier rows may be replaced: scale, weight and what is
    appended behind are as if nothing had stood there."""
    rng = rng_of("again", fmt)
    k, v = rows(rng, 1, 2, 150)
    k2, v2 = rows(rng, 1, 2, 70)
    c = new_cache(1, 2, 160, fmt)
    c.append(k, v, [0])
    c.attn_decode(rng.standard_normal((1, 4 * HD)).astype(np.float32), [149], True)
    assert (c.weights()[0, :, :5] > 0).all()
    c.append(k2[:, :, :10], v2[:, :, :10], [64])
    assert (c.weights()[0, :, [0, 1]] > 0).all() and not c.weights()[0, :, 2].any()
    c.append(k2[:, :, 10:], v2[:, :, 10:], [74])
    gk, gv = c.read([0], 134)
    for got, x, y in ((gk, k, k2), (gv, v, v2)):
        assert np.array_equal(bits(got[0]), bits(held(np.concatenate([x[0, :, :64], y[0]], 1), 134, fmt)))
    assert not c.weights()[0, :, 2:5].any()


def test_append_rows_at_their_position_of_a_batch():
    """src_at_pos with strides between sequences and heads wider than the rows, counts
    and positions per sequence."""
    L, rng = ops.lib(), rng_of("batch at")
    B, hkv, ms, pad = 3, 2, 96, 128
    k, v = rows(rng, B, hkv + 1, pad)
    dk, dv = (ops.DeviceArray.from_host(x.view(np.uint16)) for x in (k, v))
    c = new_cache(B, hkv, ms, 1)
    first, second = np.array([33, 0, 90], np.int32), np.array([20, 96, 6], np.int32)
    for pos, cnt, n in ((np.zeros(3, np.int32), first, 90), (first, second, 96)):
        dp, dc = ops.DeviceArray.from_host(pos), ops.DeviceArray.from_host(cnt)
        ops.check(L.oxb_kv8_append(c.data.ptr, c.stride, 1, B, hkv, HD, ms, dk.ptr, dv.ptr, (hkv + 1) * pad * HD,
                                   pad * HD, 1, dp.ptr, 1, 0, n, dc.ptr, None))
        ops.sync()
    lens = (first + second).tolist()
    gk, gv = c.read([0] * B, ms, lens)
    for z, n in enumerate(lens):
        assert np.array_equal(bits(gk[z, :, :n]), bits(held(k[z, :hkv], n, 1)))
        assert np.array_equal(bits(gv[z, :, :n]), bits(held(v[z, :hkv], n, 1)))

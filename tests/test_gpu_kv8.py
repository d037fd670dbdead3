"""The 8-bit KV cache (append, read, attention, eviction) on the GPU against numpy in
64 bits.  Caches start filled with 0xff: NaN codes, scales, weights and rows
wherever nothing has been written."""
import ctypes as C
import zlib

import numpy as np
import pytest

from helpers import ops, synth, ternary
import kv8_reference as ref

pytestmark = pytest.mark.gpu
HD = 128
FMTS = [ops.KV8_INT8, ops.KV8_E4M3]


def rng_of(*key):
    return np.random.default_rng(zlib.crc32(repr(key).encode()))


def new_cache(batch, hkv, max_seq, fmt):
    c = ops.Kv8Cache(batch, hkv, max_seq, fmt)
    c.data.upload(np.full(c.data.shape, 0xff, np.uint8))
    return c


def rows(rng, batch, hkv, n, scale=1.0):
    k = rng.standard_normal((batch, hkv, n, HD)) * np.exp(0.4 * rng.standard_normal((batch, hkv, 1, HD)))
    return (k * scale).astype(np.float16), (rng.standard_normal((batch, hkv, n, HD)) * scale).astype(np.float16)


def held(x, n, fmt):
    """The values of a sequence's first n rows [Hkv][..][128]."""
    return np.stack([ref.values(h[:n], fmt) for h in x])


def filled(rng, lens, hkv, max_seq, fmt, scale=1.0):
    """A cache with lens[z] rows, and the values it holds."""
    c = new_cache(len(lens), hkv, max_seq, fmt)
    n = max(1, max(lens))
    k, v = rows(rng, len(lens), hkv, n, scale)
    c.append(k, v, [0] * len(lens), lens)
    return c, [held(k[z], m, fmt) for z, m in enumerate(lens)], [held(v[z], m, fmt) for z, m in enumerate(lens)]


def bits(a):
    return np.ascontiguousarray(a).view(np.uint32)


# ---------------------------------------------------------------------------
# append and read
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("hkv,n,max_seq", [(1, 1, 1), (2, 1, 64), (3, 31, 31), (1, 32, 40), (2, 33, 100),
                                           (5, 150, 150), (1, 700, 1000)])
def test_append_read_values(fmt, hkv, n, max_seq):
    """Values are code * scale with the correctly rounded code: equal to the bit."""
    rng = rng_of("append", fmt, hkv, n)
    lens = [n, max(1, n // 2), 0, 1]
    c = new_cache(4, hkv, max_seq, fmt)
    k, v = rows(rng, 4, hkv, n)
    k[0, 0, :, 3] *= 30                   # a loud channel sets the scale
    v[1, -1] *= np.float16(1e-6)          # f16 denormals
    c.append(k, v, [0] * 4, lens)
    gk, gv = c.read([0] * 4, n, lens)
    for z, m in enumerate(lens):
        assert np.array_equal(bits(gk[z, :, :m]), bits(held(k[z], m, fmt))), z
        assert np.array_equal(bits(gv[z, :, :m]), bits(held(v[z], m, fmt))), z
        assert not gk[z, :, m:].any() and not gv[z, :, m:].any()


@pytest.mark.parametrize("fmt", FMTS)
def test_append_does_not_depend_on_the_split(fmt):
    rng = rng_of("split", fmt)
    k, v = rows(rng, 2, 2, 131)
    whole = new_cache(2, 2, 160, fmt)
    whole.append(k, v, [0, 0], [131, 97])
    want = whole.read([0, 0], 131, [131, 97])
    for sizes in ([1] * 131, [31, 1, 32, 33, 34], [64, 67], [5, 60, 1, 65], [30, 70, 31]):
        c = new_cache(2, 2, 160, fmt)
        at = 0
        for s in sizes:
            cnt = [s, max(0, min(s, 97 - at))]
            c.append(k[:, :, at:at + s], v[:, :, at:at + s], [at, at], cnt)
            at += s
        got = c.read([0, 0], 131, [131, 97])
        assert all(np.array_equal(bits(a), bits(b)) for a, b in zip(got, want)), sizes


def test_append_rewinds_within_a_block():
    """Rows of the last block may be taken back: the scale is that of the rows left."""
    for fmt in FMTS:
        rng = rng_of("rewind", fmt)
        k, v = rows(rng, 1, 1, 60)
        k[0, 0, 50] *= 20                                   # its scale goes with it
        c = new_cache(1, 1, 96, fmt)
        c.append(k[:, :, :55], v[:, :, :55], [0])
        c.append(k[:, :, 55:], v[:, :, 55:], [40])          # rows 40.. replaced by five others
        k2, v2 = (np.concatenate([x[:, :, :40], x[:, :, 55:]], 2) for x in (k, v))
        gk, gv = c.read([0], 45)
        assert np.array_equal(bits(gk[0]), bits(held(k2[0], 45, fmt)))
        assert np.array_equal(bits(gv[0]), bits(held(v2[0], 45, fmt)))


def test_append_drops_what_does_not_fit():
    rng = rng_of("drop")
    k, v = rows(rng, 3, 2, 40)
    c = new_cache(3, 2, 70, 0)
    before = c.data.download()
    c.append(k, v, [32, -1, 70])                            # 38 rows fit; none; none
    gk, gv = c.read([32, 0, 0], 40)
    assert np.array_equal(bits(gk[0, :, :38]), bits(held(k[0], 38, 0)))
    assert np.array_equal(bits(gv[0, :, :38]), bits(held(v[0], 38, 0)))
    assert not gk[0, :, 38:].any() and not gv[0, :, 38:].any()
    after = c.data.download()
    assert np.array_equal(after[1:], before[1:])            # sequences that got nothing: untouched


def test_append_takes_rows_at_their_position():
    """src_at_pos: rows stand at their position in a f16 cache [Hkv][max_seq][128], as
    the q|k|v projections leave them."""
    L, rng = ops.lib(), rng_of("at")
    k, v = rows(rng, 1, 3, 100)
    dk, dv = (ops.DeviceArray.from_host(x.view(np.uint16)) for x in (k, v))
    c = new_cache(1, 3, 100, 1)
    at = ops.DeviceArray.from_host(np.array([0, 37], np.int32))
    for i, (p, n) in enumerate(((0, 37), (37, 63))):
        ops.check(L.oxb_kv8_append(c.data.ptr, c.stride, 1, 1, 3, HD, 100, dk.ptr, dv.ptr, 0, 100 * HD, 1,
                                   at.offset(4 * i) if i else None, 0, 0, n, None, None))
    ops.sync()
    gk, gv = c.read([0], 100)
    assert np.array_equal(bits(gk[0]), bits(held(k[0], 100, 1)))
    assert np.array_equal(bits(gv[0]), bits(held(v[0], 100, 1)))


@pytest.mark.parametrize("fmt", FMTS)
def test_append_special_rows(fmt):
    """Zero blocks, f16's largest and smallest values, Inf and NaN (that tensor's block
    is NaN, its neighbours are not)."""
    rng = rng_of("special", fmt)
    k, v = rows(rng, 1, 2, 128)
    k[0, 0, :32] = 0
    k[0, 0, 32:64] = 65504
    k[0, 1, :32] = np.float16(6e-8)
    k[0, 1, 70, 5] = np.inf
    v[0, 0, 100, 0] = np.nan
    c = new_cache(1, 2, 128, fmt)
    c.append(k, v, [0])
    gk, gv = c.read([0], 128)
    for got, x in ((gk, k), (gv, v)):
        want = held(x[0], 128, fmt)
        assert np.array_equal(np.isnan(got[0]), np.isnan(want))
        fine = ~np.isnan(want)
        assert np.array_equal(got[0][fine], want[fine])
    assert np.isnan(gk[0, 1, 64:96]).all() and not np.isnan(gk[0, 1, 96:]).any()


def test_read_ranges():
    rng = rng_of("read")
    c, K, V = filled(rng, [90, 40], 2, 96, 0)
    for pos, n, lim in (([5, 5], 60, None), ([-10, 30], 20, [90, 40]), ([80, 0], 50, None), ([96, -40], 33, None)):
        gk, gv = c.read(pos, n, lim)
        for z in range(2):
            top = min(96, lim[z]) if lim else 96
            for i in range(n):
                p = pos[z] + i
                if 0 <= p < min(top, K[z].shape[1]):
                    assert np.array_equal(gk[z, :, i], K[z][:, p]) and np.array_equal(gv[z, :, i], V[z][:, p])
                elif p < 0 or p >= top:
                    assert not gk[z, :, i].any() and not gv[z, :, i].any()


# ---------------------------------------------------------------------------
# decode attention
# ---------------------------------------------------------------------------
def check_rows(got, want, tol, what=""):
    bad = np.abs(got.astype(np.float64) - want) > tol
    assert not bad.any(), (what, int(bad.sum()), float((np.abs(got - want) / tol).max()))


def rel(got, want):
    n = np.linalg.norm(want)
    return np.linalg.norm(got - want) / n if n else np.linalg.norm(got)


DECODE = [  # H, Hkv, lengths, max_seq
    (4, 4, [1], 1),
    (20, 5, [1, 2, 31, 32, 33], 64),
    (6, 2, [64, 65, 0, 127, 129], 131),
    (32, 2, [100, 7], 128),              # 16 heads a KV head: two groups
    (9, 1, [300, 257], 301),             # nine: a full group and one more
    (20, 5, [1000], 4096),
    (8, 8, [500, 0, 1, 33, 320, 499, 64, 2], 512),
]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("H,hkv,lens,max_seq", DECODE)
def test_decode_matches_reference(fmt, H, hkv, lens, max_seq):
    rng = rng_of("decode", fmt, H, hkv, lens)
    c, K, V = filled(rng, lens, hkv, max_seq, fmt)
    q = rng.standard_normal((len(lens), H * HD)).astype(np.float32)
    pos = [n - 1 for n in lens]
    got = c.attn_decode(q, pos)
    assert np.array_equal(bits(got), bits(c.attn_decode(q, pos)))       # the same every time
    for z, n in enumerate(lens):
        if n == 0:
            assert not got[z].any()
            continue
        want, tol, _, _ = ref.attend_rows(q[z:z + 1], K[z], V[z], hkv, n - 1)
        check_rows(got[z:z + 1], want, tol, z)
        bound = max(ref.rms_bound(q[z, h * HD:(h + 1) * HD], K[z][h // (H // hkv)]) for h in range(H))
        assert rel(got[z], want[0]) <= bound, (z, rel(got[z], want[0]), bound)


@pytest.mark.parametrize("fmt", FMTS)
def test_decode_long_many_splits(fmt):
    rng = rng_of("long", fmt)
    n = 20011
    c, K, V = filled(rng, [n, 3], 1, n + 20, fmt)
    q = rng.standard_normal((2, 4 * HD)).astype(np.float32) * 2
    got = c.attn_decode(q, [n - 1, 2])
    assert np.array_equal(bits(c.attn_decode(q, [n - 1, 2], True)), bits(got))
    for z, m in enumerate((n, 3)):
        want, tol, w, wtol = ref.attend_rows(q[z:z + 1], K[z], V[z], 1, m - 1)
        check_rows(got[z:z + 1], want, tol, z)
        check_rows(c.weights()[z, :, :(m + 31) // 32], w[:, :(m + 31) // 32], wtol[:, :(m + 31) // 32], z)


@pytest.mark.parametrize("batch,H,hkv", [(13, 10, 5), (12, 10, 5), (3, 64, 32), (40, 5, 5)])
def test_decode_rows_of_many_lengths(batch, H, hkv):
    """Around 64 rows (sequence and KV head) the runs' least length changes: sequences
    of one run, of several and of none side by side, with their weights."""
    fmt = batch % 2
    rng = rng_of("lengths", batch, H)
    lens = [0, 1, 127, 128, 129, 255, 256, 257, 300, 511, 512, 513, 700]
    lens = (lens * 4)[:batch] if batch > 3 else [513, 0, 257]
    c, K, V = filled(rng, lens, hkv, 700, fmt)
    q = rng.standard_normal((batch, H * HD)).astype(np.float32)
    got = c.attn_decode(q, [n - 1 for n in lens], True)
    for z, n in enumerate(lens):
        if n == 0:
            assert not got[z].any()
            continue
        want, tol, w, wtol = ref.attend_rows(q[z:z + 1], K[z], V[z], hkv, n - 1)
        check_rows(got[z:z + 1], want, tol, z)
        nb = (n + 31) // 32
        check_rows(c.weights()[z, :, :nb], w[:, :nb], wtol[:, :nb], z)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("qscale", [1e-30, 1e-3, 40.0, 3e4])
def test_decode_scales_of_q(fmt, qscale):
    """q rows far from 1: even weights, and one position taking all the weight."""
    rng = rng_of("q", fmt, qscale)
    c, K, V = filled(rng, [77], 2, 96, fmt)
    q = (rng.standard_normal((1, 4 * HD)) * qscale).astype(np.float32)
    want, tol, _, _ = ref.attend_rows(q, K[0], V[0], 2, 76)
    # past 1 the bound on a weight is no bound at all: then only sane values are asked for
    got = c.attn_decode(q, [76])
    assert np.isfinite(got).all() and np.abs(got).max() <= np.abs(V[0]).max() * 1.0001
    check_rows(got, want, tol)


@pytest.mark.parametrize("qscale", [1e-42, 1e-36, 1e-30, 40.0, 3e4])
def test_prefill_scales_of_q(qscale):
    """As above, rows of subnormal numbers and of zeros among them."""
    for fmt in FMTS:
        rng = rng_of("qp", fmt, qscale)
        c, K, V = filled(rng, [300], 2, 300, fmt)
        q = (rng.standard_normal((150, 8 * HD)) * qscale).astype(np.float32)
        q[7] = 0
        q[60] = np.float32(1e-45)
        q[100, :HD] = 1.5
        want, tol, w, wtol = ref.attend_rows(q, K[0], V[0], 2, 150)
        tol = tol + max(ref.parts_floor(v) for v in V[0])
        got = c.attn_prefill(q, 150, add_weights=True)
        assert np.isfinite(got).all() and np.abs(got).max() <= np.abs(V[0]).max() * 1.0001
        check_rows(got, want, tol)
        check_rows(c.weights()[0, :, :10], w[:, :10], wtol[:, :10])


def test_decode_values_of_very_different_blocks():
    """A block of large values that no weight goes to leaves the small ones exact."""
    for fmt in FMTS:
        rng = rng_of("blocks", fmt)
        k, v = rows(rng, 1, 1, 200)
        q = rng.standard_normal((1, HD)).astype(np.float32) * 3
        k[0, 0, 64:96] = (-0.4 * q[0]).astype(np.float16)     # pushed away from q
        v[0, 0, 64:96] = 6e4
        v[0, 0, :64] *= np.float16(1e-3)
        v[0, 0, 96:] *= np.float16(1e-3)
        c = new_cache(1, 1, 256, fmt)
        c.append(k, v, [0])
        want, tol, _, _ = ref.attend_rows(q, held(k[0], 200, fmt), held(v[0], 200, fmt), 1, 199)
        check_rows(c.attn_decode(q, [199]), want, tol, "decode")
        qq = np.repeat(q, 3, 0)
        got = c.attn_prefill(qq, 197)
        want, tol, _, _ = ref.attend_rows(qq, held(k[0], 200, fmt), held(v[0], 200, fmt), 1, 197)
        check_rows(got, want, tol, "prefill")


def test_nan_and_inf_stay_where_they_are():
    rng = rng_of("nan")
    for fmt in FMTS:
        c, K, V = filled(rng, [50, 50, 50], 2, 64, fmt)
        k, v = rows(rng, 3, 2, 1)
        k[0, 1, 0, 7] = np.inf                     # sequence 0, KV head 1: block 1's K
        v[2, 0, 0, 9] = np.nan                     # sequence 2, KV head 0: block 1's V
        c.append(k, v, [50, 50, 50])
        q = rng.standard_normal((3, 4 * HD)).astype(np.float32)
        q[1, 2 * HD + 5] = np.nan                  # sequence 1, query head 2
        got = c.attn_decode(q, [50, 50, 50]).reshape(3, 4, HD)
        nan = np.isnan(got).all(-1)
        assert nan.tolist() == [[False, False, True, True], [False, False, True, False],
                                [True, True, False, False]]
        assert np.isfinite(got[~nan]).all()
        gp = c.attn_prefill(np.repeat(q[1:2], 3, 0), 48, slot=1).reshape(3, 4, HD)
        assert np.isnan(gp[:, 2]).all() and np.isfinite(gp[:, [0, 1, 3]]).all()
        # rows that see block 0 alone (positions 30, 31) stay finite beside those that see block 1
        for z, heads in ((0, [2, 3]), (2, [0, 1])):
            gp = c.attn_prefill(np.repeat(q[z:z + 1], 4, 0), 30, slot=z).reshape(4, 4, HD)
            want, tol, _, _ = ref.attend_rows(np.repeat(q[z:z + 1], 2, 0), K[z], V[z], 2, 30)
            check_rows(gp[:2].reshape(2, -1), want, tol)
            assert np.isnan(gp[2:, heads]).all()
            assert np.isfinite(gp[2:, [h for h in range(4) if h not in heads]]).all()


# ---------------------------------------------------------------------------
# prefill attention
# ---------------------------------------------------------------------------
PREFILL = [  # H, Hkv, n, pos0, max_seq
    (4, 4, 1, 0, 1), (20, 5, 1, 63, 64), (20, 5, 31, 0, 40), (20, 5, 33, 31, 64), (6, 2, 43, 20, 64),
    (32, 2, 20, 64, 100), (8, 8, 130, 1, 131), (9, 1, 15, 300, 320), (4, 1, 101, 0, 128),
    (4, 1, 70, 1000, 1100), (20, 5, 3, 2000, 2048),
]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("H,hkv,n,pos0,max_seq", PREFILL)
def test_prefill_matches_reference(fmt, H, hkv, n, pos0, max_seq):
    rng = rng_of("prefill", fmt, H, hkv, n, pos0)
    c, K, V = filled(rng, [0, pos0 + n], hkv, max_seq, fmt)
    q = rng.standard_normal((n, H * HD)).astype(np.float32)
    got = c.attn_prefill(q, pos0, slot=1)
    assert np.array_equal(bits(got), bits(c.attn_prefill(q, pos0, slot=1)))
    want, tol, _, _ = ref.attend_rows(q, K[1], V[1], hkv, pos0)
    check_rows(got, want, tol)
    bound = max(ref.rms_bound(q[i, h * HD:(h + 1) * HD], K[1][h // (H // hkv)])
                for i in range(n) for h in range(H))
    assert rel(got, want) <= bound


@pytest.mark.parametrize("H,hkv,n,pos0", [
    (8, 1, 2500, 700),       # row tiles cut into runs of different number
    (16, 1, 4200, 0),        # more row tiles than a plan orders
    (20, 5, 700, 3000)])
def test_prefill_long(H, hkv, n, pos0):
    """Long prompts, some of their rows against the reference."""
    fmt = n % 2
    rng = rng_of("long prefill", H, n)
    c, K, V = filled(rng, [pos0 + n], hkv, pos0 + n, fmt)
    q = rng.standard_normal((n, H * HD)).astype(np.float32)
    got = c.attn_prefill(q, pos0)
    for i in sorted({0, 1, 31, 32, n // 3, n // 2, n - 33, n - 1} | set(rng.integers(0, n, 8).tolist())):
        want, tol, _, _ = ref.attend_rows(q[i:i + 1], K[0], V[0], hkv, pos0 + i)
        check_rows(got[i:i + 1], want, tol, i)


@pytest.mark.parametrize("H,hkv,n,pos0", [(8, 1, 600, 200), (4, 2, 900, 0)])
def test_prefill_weights_long(H, hkv, n, pos0):
    """Weights over many rows (split over workgroups) against all rows' own."""
    rng = rng_of("long weights", H, n)
    c, K, V = filled(rng, [pos0 + n], hkv, pos0 + n, 0)
    q = rng.standard_normal((n, H * HD)).astype(np.float32)
    c.attn_prefill(q, pos0, add_weights=True)
    _, _, want, tol = ref.attend_rows(q, K[0], V[0], hkv, pos0)
    check_rows(c.weights()[0], want, tol)


def test_prefill_weights_in_several_launches():
    """Rows times blocks past what a launch's sums may take: outputs of rows on both
    sides of where the call is cut, weights against those of three calls, and each
    row's weights add up to 1."""
    rng = rng_of("cut")
    H, n, pos0 = 8, 600, 261000       # 8200 blocks: 8 heads' sums of 511 tokens fill 256 MB
    total = pos0 + n
    c, K, V = filled(rng, [total], 1, total, 0)
    q = rng.standard_normal((n, H * HD)).astype(np.float32)
    got = c.attn_prefill(q, pos0, add_weights=True)
    w = c.weights()[0].astype(np.float64)
    for i in (0, 299, 300, 511, n - 1):
        want, tol, _, _ = ref.attend_rows(q[i:i + 1], K[0], V[0], 1, pos0 + i)
        check_rows(got[i:i + 1], want, tol, i)
    for i in range(0, n, 200):
        c.attn_prefill(q[i:i + 200], pos0 + i, add_weights=True)
    parts = c.weights()[0] - w
    # attend()'s bound on a weight, S by Cauchy-Schwarz; the sums as in attend_rows,
    # and the two subtracted ones' roundings
    S = np.linalg.norm(q.reshape(-1, HD), axis=1).max() * np.linalg.norm(K[0][0], axis=1).max() / np.sqrt(HD)
    rel_w = 2 * (140 * ref.U * S + 8 * ref.U) + (total / 32 + 64 + 4 + n * H + 64) * ref.U
    check_rows(parts, w, 3 * rel_w * w + 1e-37)
    assert abs(w.sum() - n * H) <= rel_w * n * H


def test_prefill_leaves_rows_behind_the_last():
    rng = rng_of("behind")
    L = ops.lib()
    c, K, V = filled(rng, [45], 2, 64, 0)
    q = ops.DeviceArray.from_host(rng.standard_normal((45, 8 * HD)).astype(np.float32))
    out = ops.DeviceArray.from_host(np.full((64, 8 * HD), 7.0, np.float32))
    n = L.oxb_attn_prefill_kv8_ws_bytes(40, 5, 8, 2, HD, 0)
    ws = ops.DeviceArray((max(n, 16),), np.uint8, zero=True)
    before = c.data.download()
    ops.check(L.oxb_attn_prefill_kv8(q.ptr, c.data.ptr, 0, 40, 5, 8, 2, HD, 64, 0, out.ptr, ws.ptr, n, None))
    ops.sync()
    assert (out.download()[40:] == 7.0).all() and (out.download()[:40] != 7.0).all()
    assert np.array_equal(c.data.download(), before)       # without weights the cache is only read


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("H,hkv,n,pos0,max_seq", [(4, 2, 40, 0, 64), (20, 5, 9, 130, 160), (9, 1, 70, 33, 128),
                                                  (16, 2, 3, 600, 640)])
def test_weights_accumulate(fmt, H, hkv, n, pos0, max_seq):
    """Prefill's and decode's weights add up over calls; begun blocks start at 0."""
    rng = rng_of("weights", fmt, H, n, pos0)
    c, K, V = filled(rng, [pos0 + n, pos0 + n], hkv, max_seq, fmt)
    w = c.weights()
    nb = (pos0 + n + 31) // 32
    assert not w[:, :, :nb].any() and np.isnan(w[:, :, nb:]).all()
    q = rng.standard_normal((n, H * HD)).astype(np.float32)
    plain = c.attn_prefill(q, pos0, slot=1)
    assert np.array_equal(bits(c.attn_prefill(q, pos0, slot=1, add_weights=True)), bits(plain))
    _, _, want, tol = ref.attend_rows(q, K[1], V[1], hkv, pos0)
    check_rows(c.weights()[1, :, :nb], want, tol)
    assert not c.weights()[0, :, :nb].any()
    qd = rng.standard_normal((2, H * HD)).astype(np.float32)
    pos = [pos0 + n - 1, pos0 // 2]
    for times in (1, 2):
        c.attn_decode(qd, pos, add_weights=True)
        for z in range(2):
            _, _, w1, t1 = ref.attend_rows(qd[z:z + 1], K[z], V[z], hkv, pos[z])
            base, tb = (want, tol) if z else (0, 0)
            check_rows(c.weights()[z, :, :nb], base + times * w1, tb + times * t1 + 4 * ref.U * (base + times * w1))
    assert np.isnan(c.weights()[:, :, nb:]).all()


# ---------------------------------------------------------------------------
# eviction
# ---------------------------------------------------------------------------
def set_weights(c, w):
    nb = w.shape[-1]
    al = lambda b: (b + 255) // 256 * 256  # noqa: E731
    at = al(c.Hkv * nb * 8192) + al(c.Hkv * nb * 8)
    d = c.data.download()
    d[:, at:at + c.Hkv * nb * 4] = np.ascontiguousarray(w, np.float32).view(np.uint8).reshape(c.batch, -1)
    c.data.upload(d)


EVICT = [  # lengths, max_seq, budget, sink, recent
    ([320, 100, 0, 1], 320, 5, 1, 1),
    ([311, 65, 64, 33], 330, 3, 1, 2),
    ([1000, 999, 128], 1000, 4, 0, 4),          # only the recent ones stay
    ([640], 640, 1, 0, 1),
    ([9000, 4001], 9001, 100, 2, 3),            # more blocks than a workgroup's threads
    ([320], 320, 10, 1, 1), ([320], 320, 50, 1, 1),   # nothing to drop
]


@pytest.mark.parametrize("inplace", [True, False])
@pytest.mark.parametrize("lens,max_seq,budget,sink,recent", EVICT)
@pytest.mark.parametrize("how", ["spread", "ties", "nan"])
def test_evict_keeps_the_heaviest_blocks(inplace, lens, max_seq, budget, sink, recent, how):
    rng = rng_of("evict", lens, budget, how)
    hkv, fmt, B = 2, 1, len(lens)
    c, K, V = filled(rng, lens, hkv, max_seq, fmt)
    nb = (max_seq + 31) // 32
    w = rng.random((B, hkv, nb)).astype(np.float32)
    if how == "ties":
        w = np.floor(w * 3).astype(np.float32)
        w[:, :, ::5] *= -0.0
    if how == "nan":
        w[rng.random(w.shape) < 0.4] = np.nan
        w[:, :, 1::7] = np.inf
        w[:, :, 2::7] = -1.0
    set_weights(c, w)
    dst = None
    if not inplace:
        dst = new_cache(B, hkv, max(budget * 32, 1) if budget * 32 < max_seq else max_seq, fmt)
    new = c.evict(lens, budget, sink, recent, dst)
    d = dst or c
    got_w = d.weights()
    for z, n in enumerate(lens):
        nblk = (n + 31) // 32
        assert new[z] == n - 32 * max(0, nblk - budget)
        for h in range(hkv):
            keep = ref.kept_blocks(w[z, h], nblk, budget, sink, recent)
            at = np.concatenate([np.arange(32 * b, min(32 * b + 32, n)) for b in keep] or [np.zeros(0, int)]).astype(int)
            assert len(at) == new[z]
            if len(at):
                gk, gv = d.read([0] * B, len(at))
                assert np.array_equal(bits(gk[z, h]), bits(K[z][h, at]))
                assert np.array_equal(bits(gv[z, h]), bits(V[z][h, at]))
            assert np.array_equal(bits(got_w[z, h, :len(keep)]), bits(w[z, h, keep]))


def test_evict_with_room_for_all():
    """A budget past every block, sink and recent past the sequence's: nothing changes."""
    rng = rng_of("room")
    lens, ms = [100, 33, 0], 100
    c = new_cache(3, 2, ms, ops.KV8_INT8)
    k, v = (rng.standard_normal((3, 2, ms, HD)).astype(np.float16) for _ in "kv")
    c.append(k, v, [0] * 3, lens)
    want, wt = c.read([0] * 3, ms, lens), c.weights()
    assert c.evict(lens, (1 << 31) - 1, 40, 1 << 30).tolist() == lens
    for a, b in zip(c.read([0] * 3, ms, lens), want):
        assert np.array_equal(a, b)
    for z, n in enumerate(lens):
        assert np.array_equal(c.weights()[z][:, :(n + 31) // 32], wt[z][:, :(n + 31) // 32])


@pytest.mark.parametrize("inplace", [True, False])
def test_evict_then_append_and_attend(inplace):
    """The unfinished block goes on growing after a cut: rows, scales, attention."""
    for fmt in FMTS:
        rng = rng_of("grow", fmt, inplace)
        lens, hkv, H = [203, 170], 2, 8
        c = new_cache(2, hkv, 300, fmt)
        k, v = rows(rng, 2, hkv, 203)
        c.append(k, v, [0, 0], lens)
        w = rng.random((2, hkv, 10)).astype(np.float32)
        set_weights(c, w)
        d = c if inplace else new_cache(2, hkv, 200, fmt)
        new = c.evict(lens, 4, 1, 1, None if inplace else d)
        k2, v2 = rows(rng, 2, hkv, 50)
        d.append(k2[:, :, :9], v2[:, :, :9], new)
        d.append(k2[:, :, 9:], v2[:, :, 9:], new + 9)
        q = rng.standard_normal((2, H * HD)).astype(np.float32)
        got = d.attn_decode(q, new + 49)
        for z, n in enumerate(lens):
            nblk = (n + 31) // 32
            rk, rv = [], []
            for h in range(hkv):
                keep = ref.kept_blocks(w[z, h], nblk, 4, 1, 1)
                at = np.concatenate([np.arange(32 * b, min(32 * b + 32, n)) for b in keep])
                rk.append(ref.values(np.concatenate([k[z, h, at], k2[z, h]]), fmt))
                rv.append(ref.values(np.concatenate([v[z, h, at], v2[z, h]]), fmt))
            gk, gv = d.read([0, 0], int(new[z]) + 50)
            assert np.array_equal(bits(gk[z]), bits(np.stack(rk))) and np.array_equal(bits(gv[z]), bits(np.stack(rv)))
            want, tol, _, _ = ref.attend_rows(q[z:z + 1], np.stack(rk), np.stack(rv), hkv, int(new[z]) + 49)
            check_rows(got[z:z + 1], want, tol)


# ---------------------------------------------------------------------------
# together, and captured
# ---------------------------------------------------------------------------
def test_a_serving_run():
    """A prompt, decode steps, a cut, more steps and ruled draws: cache, attention and
    tokens against the reference at every step."""
    for fmt in FMTS:
        rng = rng_of("serve", fmt)
        hkv, H, B, V = 2, 8, 2, 1000
        c = new_cache(B, hkv, 192, fmt)
        lens = np.array([100, 61], np.int32)
        k, v = rows(rng, B, hkv, 100)
        c.append(k, v, [0, 0], lens)
        kept = [[[k[z, h, :n], v[z, h, :n]] for h in range(hkv)] for z, n in enumerate(lens)]
        w = [[np.zeros(0)] * hkv for _ in range(B)]
        wt = [[np.zeros(0)] * hkv for _ in range(B)]

        def grow(a, n):
            return np.concatenate([a, np.zeros(n - len(a))])

        def add(z, ww, tt):
            for h in range(hkv):
                w[z][h] = grow(w[z][h], ww.shape[1]) + ww[h]
                wt[z][h] = grow(wt[z][h], ww.shape[1]) + tt[h] + 4 * ref.U * w[z][h]

        def vals(z):
            return (np.stack([ref.values(kept[z][h][i], fmt) for h in range(hkv)]) for i in (0, 1))

        for z in range(B):
            q = rng.standard_normal((lens[z], H * HD)).astype(np.float32)
            got = c.attn_prefill(q, 0, z, True)
            want, tol, ww, tt = ref.attend_rows(q, *vals(z), hkv, 0)
            check_rows(got, want, tol)
            add(z, ww, tt)
        hist = [[], []]
        for step in range(40):
            nk, nv = rows(rng, B, hkv, 1)
            c.append(nk, nv, lens)
            for z in range(B):
                for h in range(hkv):
                    kept[z][h] = [np.concatenate([kept[z][h][i], x[z, h]]) for i, x in enumerate((nk, nv))]
            q = rng.standard_normal((B, H * HD)).astype(np.float32)
            got = c.attn_decode(q, lens, True)
            for z in range(B):
                want, tol, ww, tt = ref.attend_rows(q[z:z + 1], *vals(z), hkv, int(lens[z]))
                check_rows(got[z:z + 1], want, tol, (step, z))
                add(z, ww, tt)
            lens = lens + 1
            logits = rng.standard_normal((B, V)).astype(np.float32)
            pen = np.array([[1.2, 0.1, 0.2]] * B, np.float32)
            mask = rng.integers(0, 2 ** 32, (B, (V + 31) // 32), dtype=np.uint32)
            ruled = ops.logits_rules(logits, pen, hist, None, mask)
            assert np.array_equal(bits(ruled), bits(ref.rules(logits, pen, hist, None, mask)))
            for z in range(B):
                hist[z].append(int(ruled[z].argmax()))
            if step == 15:
                got_w = c.weights()
                for z in range(B):
                    for h in range(hkv):
                        m = len(w[z][h])
                        check_rows(got_w[z, h, :m], w[z][h], wt[z][h] + 1e-30)
                new = c.evict(lens, 3, 1, 1)
                for z in range(B):
                    nblk = (lens[z] + 31) // 32
                    for h in range(hkv):
                        keep = ref.kept_blocks(got_w[z, h], nblk, 3, 1, 1)
                        at = np.concatenate([np.arange(32 * b, min(32 * b + 32, lens[z])) for b in keep])
                        kept[z][h] = [x[at] for x in kept[z][h]]
                        w[z][h], wt[z][h] = w[z][h][keep], wt[z][h][keep]
                lens = new
        got_w = c.weights()
        for z in range(B):
            for h in range(hkv):
                m = len(w[z][h])
                check_rows(got_w[z, h, :m], w[z][h], wt[z][h] + 1e-30)


def test_behind_the_projections():
    """As a layer uses them: the q|k|v projections leave rotated f16 rows in a scratch
    cache, the append takes them at their position, attention follows; after a cut
    the tokens' own positions go on through a rope table shifted by the dropped
    rows."""
    L = ops.lib()
    for fmt in FMTS:
        rng = rng_of("layer", fmt)
        D, H, hkv, ms, n = 512, 8, 2, 256, 150
        Dq, Dkv = H * HD, hkv * HD
        N = Dq + 2 * Dkv
        Wt = ops.upload_ternary(synth.i2s_pack(ternary(rng, N, D)), D)
        g = ops.DeviceArray.from_host(rng.uniform(0.5, 1.5, D).astype(np.float32))
        wsc = ops.DeviceArray.from_host(rng.uniform(0.01, 0.02, N).astype(np.float32))
        table = np.empty((ms, HD // 2, 2), np.float32)
        ops.check(L.oxb_rope_table(table.ctypes.data, ms, HD, 500000.0))
        rope = ops.DeviceArray.from_host(table)
        kc, vc, k2, v2 = (ops.DeviceArray((hkv, ms, HD), np.uint16, zero=True) for _ in range(4))
        c = new_cache(1, hkv, ms, fmt)
        # the prompt
        x = ops.DeviceArray.from_host(rng.standard_normal((n, D)).astype(np.float32))
        pad = (n + 63) // 64 * 64
        Xt, sc, sm = (ops.DeviceArray((pad * D,), np.int8, zero=True), ops.DeviceArray((pad,), np.float32),
                      ops.DeviceArray((pad,), np.int32))
        q = ops.DeviceArray((n, Dq), np.float32)
        ops.quantize_rows_tiled(x, g, 1e-5, n, D, Xt, sc, sm)
        ops.check(L.oxb_gemm_qkv(Wt.ptr, Xt.ptr, sc.ptr, sm.ptr, wsc.ptr, Dq, Dkv, HD, D, n, 0, q.ptr, kc.ptr,
                                 vc.ptr, ms, rope.ptr, None))
        ops.check(L.oxb_kv8_append(c.data.ptr, c.stride, fmt, 1, hkv, HD, ms, kc.ptr, vc.ptr, 0, ms * HD, 1, None, 0,
                                   0, n, None, None))
        ops.sync()
        k, v = ([h[:n] for h in a.download().view(np.float16)] for a in (kc, vc))
        got = c.attn_prefill(q.download(), 0, add_weights=True)
        K, V = (np.stack([ref.values(h, fmt) for h in a]) for a in (k, v))
        want, tol, _, _ = ref.attend_rows(q.download(), K, V, hkv, 0)
        check_rows(got, want, tol)
        # a token a step; a cut before the fourth
        pos, dropped = n, 0
        dp, dt = ops.DeviceArray((1,), np.int32), ops.DeviceArray((1,), np.int32)
        q1, q2 = ops.DeviceArray((Dq,), np.float32), ops.DeviceArray((Dq,), np.float32)
        for step in range(8):
            if step == 3:
                w = c.weights()[0]
                new = int(c.evict([pos], 3, 1, 1)[0])
                for h in range(hkv):
                    keep = ref.kept_blocks(w[h], (pos + 31) // 32, 3, 1, 1)
                    at = np.concatenate([np.arange(32 * b, min(32 * b + 32, pos)) for b in keep])
                    k[h], v[h] = k[h][at], v[h][at]
                dropped, pos = pos - new, new
                assert dropped == 64
            x1 = ops.DeviceArray.from_host(rng.standard_normal(D).astype(np.float32))
            dp.upload(np.array([pos], np.int32))
            dt.upload(np.array([pos + dropped], np.int32))
            for qq, kk, vv, tab, p in ((q1, kc, vc, rope.offset(dropped * HD * 4), dp), (q2, k2, v2, rope.ptr, dt)):
                ops.check(L.oxb_bitlinear_qkv(Wt.ptr, x1.ptr, g.ptr, 1e-5, wsc.ptr, Dq, Dkv, HD, D, qq.ptr, kk.ptr,
                                              vv.ptr, ms, tab, p.ptr, None))
            ops.check(L.oxb_kv8_append(c.data.ptr, c.stride, fmt, 1, hkv, HD, ms, kc.ptr, vc.ptr, 0, ms * HD, 1,
                                       dp.ptr, 0, 0, 1, None, None))
            ops.sync()
            assert np.array_equal(bits(q1.download()), bits(q2.download()))
            ka, va = (a.download().view(np.float16)[:, pos] for a in (kc, vc))
            assert np.array_equal(ka.view(np.uint16), k2.download()[:, pos + dropped])
            k, v = ([np.concatenate([h, r[None]]) for h, r in zip(a, b)] for a, b in ((k, ka), (v, va)))
            qh = q1.download()[None]
            got = c.attn_decode(qh, [pos], True)
            K, V = (np.stack([ref.values(h, fmt) for h in a]) for a in (k, v))
            want, tol, _, _ = ref.attend_rows(qh, K, V, hkv, pos)
            check_rows(got, want, tol, step)
            pos += 1


def test_captured_step_replays():
    """Append and decode attention in one graph, replayed with new rows and positions
    and eager work between the replays, on a stream of its own."""
    L, rng = ops.lib(), rng_of("graph")
    hkv, H, B, ms, fmt = 2, 8, 3, 256, 0
    st = L.oxb_stream_create()
    c, e = new_cache(B, hkv, ms, fmt), new_cache(B, hkv, ms, fmt)
    k0, v0 = rows(rng, B, hkv, 120)
    lens = np.array([120, 31, 0], np.int32)
    for x in (c, e):
        x.append(k0, v0, [0] * B, lens)
    dk, dv = (ops.DeviceArray((B, hkv, 1, HD), np.uint16) for _ in "kv")
    dq, out = (ops.DeviceArray((B, H * HD), np.float32) for _ in "qo")
    dp = ops.DeviceArray((B,), np.int32)
    n = L.oxb_attn_decode_kv8_ws_bytes(B, H, hkv, HD, ms)
    ws = ops.DeviceArray((n,), np.uint8, zero=True)
    ops.sync()
    ops.check(L.oxb_stream_begin_capture(st))
    ops.check(L.oxb_kv8_append(c.data.ptr, c.stride, fmt, B, hkv, HD, ms, dk.ptr, dv.ptr, hkv * HD, HD, 0,
                               dp.ptr, 1, 0, 1, None, st))
    ops.check(L.oxb_attn_decode_kv8(dq.ptr, c.data.ptr, c.stride, fmt, dp.ptr, 1, B, H, hkv, HD, ms, 1,
                                    out.ptr, ws.ptr, n, st))
    g = L.oxb_stream_end_capture(st)
    assert g
    for step in range(6):
        k, v = rows(rng, B, hkv, 1)
        q = rng.standard_normal((B, H * HD)).astype(np.float32)
        dk.upload(k.view(np.uint16))
        dv.upload(v.view(np.uint16))
        dq.upload(q)
        dp.upload(lens)
        ops.check(L.oxb_graph_launch(g, st))
        ops.check(L.oxb_stream_sync(st))
        e.append(k, v, lens)
        want = e.attn_decode(q, lens, True)
        assert np.array_equal(bits(out.download()), bits(want)), step
        lens = lens + 1
    m = [(int(x) + 31) // 32 for x in lens]
    for z in range(B):
        assert np.array_equal(bits(c.weights()[z, :, :m[z]]), bits(e.weights()[z, :, :m[z]]))
    ops.check(L.oxb_graph_destroy(g))
    ops.check(L.oxb_stream_destroy(st))


def test_captured_prefill_evict_and_rules():
    """A prompt's attention in several runs with weights, a cut into another cache and
    logit rules in one graph, replayed with new inputs and eager work between."""
    L, rng = ops.lib(), rng_of("graph2")
    hkv, H, n, pos0, fmt, V = 2, 8, 150, 900, 1, 5003
    total = n + pos0
    st = L.oxb_stream_create()
    c, K, Vv = filled(rng, [total], hkv, total, fmt)
    e, d, ed = new_cache(1, hkv, total, fmt), new_cache(1, hkv, 10 * 32, fmt), new_cache(1, hkv, 10 * 32, fmt)
    start = c.data.download()
    dq, out = (ops.DeviceArray((n, H * HD), np.float32) for _ in "qo")
    dl, dn = ops.DeviceArray.from_host(np.array([total], np.int32)), ops.DeviceArray((1,), np.int32)
    lg, ro = ops.DeviceArray((2, V), np.float32), ops.DeviceArray((2, V), np.float32)
    pen = ops.DeviceArray.from_host(np.array([[1.2, 0.1, 0.3], [1, 0, 0.5]], np.float32))
    hist, hoff = ops.DeviceArray((64,), np.int32), ops.DeviceArray.from_host(np.array([0, 40, 64], np.int32))
    wsn = L.oxb_attn_prefill_kv8_ws_bytes(n, pos0, H, hkv, HD, 1)
    evn = L.oxb_kv8_evict_ws_bytes(1, hkv, total, 10)
    ws, ew = ops.DeviceArray((wsn,), np.uint8, zero=True), ops.DeviceArray((evn,), np.uint8)
    ops.sync()
    ops.check(L.oxb_stream_begin_capture(st))
    ops.check(L.oxb_attn_prefill_kv8(dq.ptr, c.data.ptr, fmt, n, pos0, H, hkv, HD, total, 1, out.ptr, ws.ptr, wsn, st))
    ops.check(L.oxb_kv8_evict(c.data.ptr, c.stride, total, d.data.ptr, d.stride, 320, dl.ptr, 1, dn.ptr, 1, 1, hkv, HD,
                              10, 1, 2, ew.ptr, evn, st))
    ops.check(L.oxb_logits_rules(lg.ptr, V, 2, V, pen.ptr, hist.ptr, hoff.ptr, 64, None, None, None, 0, None, 0,
                                 ro.ptr, V, st))
    g = L.oxb_stream_end_capture(st)
    assert g
    for step in range(4):
        q = rng.standard_normal((n, H * HD)).astype(np.float32)
        x, ids = rng.standard_normal((2, V)).astype(np.float32), rng.integers(0, 50, 64).astype(np.int32)
        for a, b in ((c.data, start), (e.data, start), (dq, q), (lg, x), (hist, ids)):
            a.upload(b)
        ops.check(L.oxb_graph_launch(g, st))
        ops.check(L.oxb_stream_sync(st))
        assert np.array_equal(bits(out.download()), bits(e.attn_prefill(q, pos0, add_weights=True))), step
        assert np.array_equal(bits(c.weights()), bits(e.weights()))
        assert dn.download()[0] == e.evict([total], 10, 1, 2, ed)[0]
        for a, b in zip(d.read([0], 320, dn.download()), ed.read([0], 320, dn.download())):
            assert np.array_equal(bits(a), bits(b)), step
        want = ops.logits_rules(x, [[1.2, 0.1, 0.3], [1, 0, 0.5]], [ids[:40], ids[40:]])
        assert np.array_equal(bits(ro.download()), bits(want)), step
    ops.check(L.oxb_graph_destroy(g))
    ops.check(L.oxb_stream_destroy(st))


def test_offsets_past_32_bits():
    """A cache of which the last head's blocks and the second sequence lie past 4 GB."""
    hkv, ms, B, n = 17, 1 << 20, 2, 70
    rng = rng_of("4 GB")
    c = ops.Kv8Cache(B, hkv, ms, 1)
    assert c.stride > 1 << 32 and 16 * (ms // 32) * 8192 >= 1 << 32
    k, v = rows(rng, B, hkv, n)
    c.append(k, v, [0, 0])
    gk, gv = c.read([0, 0], n)
    K, V = [held(x, n, 1) for x in k], [held(x, n, 1) for x in v]
    for z in range(B):
        assert np.array_equal(bits(gk[z]), bits(K[z])) and np.array_equal(bits(gv[z]), bits(V[z]))
    q = rng.standard_normal((B, 2 * hkv * HD)).astype(np.float32)
    got = c.attn_decode(q, [n - 1, n - 2], True)
    qp = rng.standard_normal((5, 2 * hkv * HD)).astype(np.float32)
    gp = c.attn_prefill(qp, n - 5, slot=1, add_weights=True)
    for z in range(B):
        want, tol, _, _ = ref.attend_rows(q[z:z + 1], K[z], V[z], hkv, n - 1 - z)
        check_rows(got[z:z + 1], want, tol, z)
    want, tol, _, _ = ref.attend_rows(qp, K[1], V[1], hkv, n - 5)
    check_rows(gp, want, tol)
    new = c.evict([n, n], 2, 1, 1)
    assert new.tolist() == [n - 32] * 2
    gk, gv = c.read([0, 0], n - 32)
    at = np.r_[0:32, 64:n]
    for z in range(B):
        assert np.array_equal(bits(gk[z]), bits(K[z][:, at])) and np.array_equal(bits(gv[z]), bits(V[z][:, at]))


def test_one_workspace_for_calls_of_any_shape():
    """Decode and prefill calls of different shapes in turn on one workspace: each as
    on one of its own."""
    L, rng = ops.lib(), rng_of("ws")
    shapes = [(1, 8, 2, 3000), (3, 20, 5, 200), (1, 4, 4, 40), (2, 16, 1, 1500)]
    need = 0
    for b, H, hkv, n in shapes:
        need = max(need, L.oxb_attn_decode_kv8_ws_bytes(b, H, hkv, HD, n),
                   L.oxb_attn_prefill_kv8_ws_bytes(70, n - 70 if n > 70 else 0, H, hkv, HD, 1))
    ws = ops.DeviceArray((need,), np.uint8, zero=True)
    made = []
    for b, H, hkv, n in shapes:
        c, _, _ = filled(rng, [n] * b, hkv, n, 0)
        m = min(70, n)
        made.append((b, H, hkv, n, m, c, rng.standard_normal((b, H * HD)).astype(np.float32),
                     rng.standard_normal((m, H * HD)).astype(np.float32)))
    for _ in range(2):
        for b, H, hkv, n, m, c, q, qp in made:
            dq, dqp = ops.DeviceArray.from_host(q), ops.DeviceArray.from_host(qp)
            out, outp = ops.DeviceArray(q.shape, np.float32), ops.DeviceArray(qp.shape, np.float32)
            pos = ops.DeviceArray.from_host(np.full(b, n - 1, np.int32))
            ops.check(L.oxb_attn_decode_kv8(dq.ptr, c.data.ptr, c.stride, 0, pos.ptr, 1, b, H, hkv, HD, n, 0,
                                            out.ptr, ws.ptr, need, None))
            ops.check(L.oxb_attn_prefill_kv8(dqp.ptr, c.data.ptr, 0, m, n - m, H, hkv, HD, n, 1, outp.ptr,
                                             ws.ptr, need, None))
            ops.sync()
            assert np.array_equal(bits(out.download()), bits(c.attn_decode(q, [n - 1] * b)))
            assert np.array_equal(bits(outp.download()), bits(c.attn_prefill(qp, n - m)))


def test_two_streams_at_once():
    """Two sequences of calls on streams, caches and workspaces of their own, queued
    without waiting for either."""
    L, rng = ops.lib(), rng_of("streams")
    hkv, H, B, ms, steps = 2, 8, 2, 512, 12
    side = []
    for i in range(2):
        c, e = new_cache(B, hkv, ms, i), new_cache(B, hkv, ms, i)
        k, v = rows(rng, B, hkv, 300 + steps)
        for x in (c, e):
            x.append(k[:, :, :300], v[:, :, :300], [0, 0], [300, 180])
        q = rng.standard_normal((steps, B, H * HD)).astype(np.float32)
        pos = np.array([[300 + s, 180 + s] for s in range(steps)], np.int32)
        n = L.oxb_attn_decode_kv8_ws_bytes(B, H, hkv, HD, ms)
        side.append(dict(c=c, e=e, k=k, v=v, q=q, pos=pos, n=n, st=L.oxb_stream_create(),
                         ws=ops.DeviceArray((n,), np.uint8, zero=True), dq=ops.DeviceArray.from_host(q),
                         dk=ops.DeviceArray.from_host(k.view(np.uint16)), dv=ops.DeviceArray.from_host(v.view(np.uint16)),
                         dp=ops.DeviceArray.from_host(pos), out=ops.DeviceArray(q.shape, np.float32)))
    ops.sync()
    row = HD * 2
    for s in range(steps):
        for d in side:
            c, n_src = d["c"], (300 + steps) * HD
            ops.check(L.oxb_kv8_append(c.data.ptr, c.stride, c.fmt, B, hkv, HD, ms, d["dk"].offset((300 + s) * row),
                                       d["dv"].offset((300 + s) * row), hkv * n_src, n_src, 0, d["dp"].offset(8 * s), 1, 0,
                                       1, None, d["st"]))
            ops.check(L.oxb_attn_decode_kv8(d["dq"].offset(4 * s * B * H * HD), c.data.ptr, c.stride, c.fmt,
                                            d["dp"].offset(8 * s), 1, B, H, hkv, HD, ms, 1,
                                            d["out"].offset(4 * s * B * H * HD), d["ws"].ptr, d["n"], d["st"]))
    for d in side:
        ops.check(L.oxb_stream_sync(d["st"]))
    for d in side:
        got = d["out"].download()
        for s in range(steps):
            d["e"].append(d["k"][:, :, 300 + s:301 + s], d["v"][:, :, 300 + s:301 + s], d["pos"][s])
            assert np.array_equal(bits(got[s]), bits(d["e"].attn_decode(d["q"][s], d["pos"][s], True))), s
        assert np.array_equal(bits(d["c"].weights()[:, :, :6]), bits(d["e"].weights()[:, :, :6]))
        ops.check(L.oxb_stream_destroy(d["st"]))


# ---------------------------------------------------------------------------
# logit rules
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("V", [1, 31, 33, 4095, 4096, 4097, 50257, 128256])
def test_rules_match_reference(V):
    rng = rng_of("rules", V)
    n = 3
    x = (rng.standard_normal((n, V)) * 4).astype(np.float32)
    x[0, 0] = -np.inf
    x[1, V // 2] = np.nan
    x[2, V - 1] = np.inf
    hist = [rng.integers(0, V, 300).tolist() + [-1, V, 2 ** 31 - 1, -2 ** 31], [], [V - 1] * 70 + [0]]
    bias = [[(V - 1, 2.5), (0, -1.0), (V - 1, -3.0), (-5, 9.0), (V, 9.0)], [(V // 2, -np.inf)], []]
    pen = np.array([[1.3, 0.2, 0.4], [2.0, 1.0, 1.0], [0.7, 0.0, 0.125]], np.float32)
    mask = rng.integers(0, 2 ** 32, (n, (V + 31) // 32 + 2), dtype=np.uint32)
    for p in (None, pen):
        for h in (None, hist):
            for b in (None, bias):
                for m in (None, mask, mask[1], np.zeros_like(mask)):
                    got, want = ops.logits_rules(x, p, h, b, m), ref.rules(x, p, h, b, m)
                    assert np.array_equal(np.isnan(got), np.isnan(want))
                    f = ~np.isnan(want)
                    assert np.array_equal(got[f], want[f])


def test_rules_in_place_and_strides():
    """Rows apart, in place and with a mask wider than the vocabulary; what lies between
    the rows stays."""
    L, rng = ops.lib(), rng_of("inplace")
    n, V, st = 4, 5001, 5013
    x = rng.standard_normal((n, st)).astype(np.float32)
    hist = [rng.integers(0, V, 50).tolist() for _ in range(n)]
    pen = np.tile(np.array([1.5, 0.25, 0.5], np.float32), (n, 1))
    mask = rng.integers(0, 2 ** 32, (n, 200), dtype=np.uint32)
    want = ref.rules(x[:, :V], pen, hist, None, mask)
    dx, dp, dm = (ops.DeviceArray.from_host(a) for a in (x, pen, mask))
    flat = np.concatenate(hist).astype(np.int32)
    # offsets that run past the lists are kept inside them
    off = np.array([0, 50, 100, 150, 10 ** 9], np.int32)
    dh, do = ops.DeviceArray.from_host(flat), ops.DeviceArray.from_host(off)
    ops.check(L.oxb_logits_rules(dx.ptr, st, n, V, dp.ptr, dh.ptr, do.ptr, flat.size, None, None, None, 0,
                                 dm.ptr, 200, dx.ptr, st, None))
    ops.sync()
    got = dx.download()
    assert np.array_equal(bits(got[:, :V]), bits(want)) and np.array_equal(bits(got[:, V:]), bits(x[:, V:]))


def test_rules_then_draw():
    """Ruled logits go on to the device sampler: a greedy draw takes the best allowed id."""
    L, rng = ops.lib(), rng_of("draw")
    V = 128256
    x = rng.standard_normal((1, V)).astype(np.float32)
    mask = rng.integers(0, 2 ** 32, (1, (V + 31) // 32), dtype=np.uint32)
    ruled = ops.logits_rules(x, None, None, [[(17, 50.0)]], mask)
    want = int(ref.rules(x, None, None, [[(17, 50.0)]], mask)[0].argmax())
    b = L.oxb_sample_ws_bytes(V)
    lg, ws = ops.DeviceArray.from_host(ruled), ops.DeviceArray((b,), np.uint8)
    u, tok = ops.DeviceArray.from_host(np.array([0.5], np.float32)), ops.DeviceArray((1,), np.int32)
    ops.check(L.oxb_sample_device(lg.ptr, V, 1.0, 1, 1.0, None, 0, u.ptr, tok.ptr, ws.ptr, b, None))
    ops.sync()
    assert int(tok.download()[0]) == want

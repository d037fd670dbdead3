"""Paths of the paged attention that sizes choose: lists of uncut tiles, last tiles cut, groups of
more than eight heads, batches of more sequences than workgroups that are resident;
each value by its bound and all rows by their norm."""
import numpy as np
import pytest

import paged_reference as ref
from helpers import ops
from test_gpu_paged import HD, bits, expect, filled, packed, rng_of

pytestmark = pytest.mark.gpu
SLOTS = 512           # resident workgroups: two on each of 256 CUs
DTYPES = [np.float32, np.float16]


def tiles(new, G):
    return sum(-(-n * G // 128) for n in new)


def check(got, q, K, V, hkv, first, f16, parts, what):
    want, tol = expect(q, K, V, hkv, first, f16, parts)
    ref.check_rows(got, want, tol, what)
    ref.close_in_norm(got, want, q.reshape(-1, HD)[:200], K[:, 0], len(K), f16)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,hkv,spec,page", [
    (64, 8, [(1500, 0), (400, 1200)], 128),             # 119 for 64
    (32, 4, [(900, 0), (0, 70), (1300, 60), (11, 400)], 64),    # 139 for 128
    (16, 1, [(4100, 0)], 64),                           # 513 for 512
])
def test_uncut_lists(dtype, H, hkv, spec, page):
    rng = rng_of("uncut", H, hkv, page)
    new, lens, cu = packed(spec)
    G, f16 = H // hkv, dtype == np.float16
    assert ops.device_info()["cus"] == 256 and tiles(new, G) > SLOTS // hkv
    c, K, V = filled(rng, lens, hkv, page)
    q = rng.standard_normal((int(cu[-1]), H * HD)).astype(dtype)
    got = c.attn_prefill(q, cu)
    for z, m in enumerate(new):
        rows = [cu[z] + i for i in {0, 1, 31, 32, 127, m // 2, m - 2, m - 1} if 0 <= i < m]
        for r in rows:
            check(got[r:r + 1], q[r:r + 1], K[z], V[z], hkv, lens[z] - m + r - cu[z], f16, 1 if f16 else 2, (z, r))
        for h in (0, G - 1, H - 1):
            at, rows = slice(h * HD, (h + 1) * HD), np.arange(0, m, 9)
            if len(rows):
                want, tol = ref.attend(q[cu[z] + rows][:, at], K[z][:, h // G], V[z][:, h // G],
                                       lens[z] - m + 1 + rows, f16, 1 if f16 else 2)
                ref.check_rows(got[cu[z] + rows][:, at], want, tol, (z, h))
    assert np.array_equal(bits(got), bits(c.attn_prefill(q, cu)))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,past", [(1056, 3000), (1500, 2000), (1030, 2500)])
def test_tiles_past_a_round(dtype, n, past):
    """66, 94 and 65 tiles for 64 workgroups of a KV head, nearly equal: the last ones cut."""
    rng = rng_of("past a round", n, past)
    hkv, H, f16 = 8, 64, dtype == np.float16
    assert 0 < tiles([n], 8) % (SLOTS // hkv) and tiles([n], 8) > SLOTS // hkv
    c, K, V = filled(rng, [past + n], hkv, 64)
    q = rng.standard_normal((n, H * HD)).astype(dtype)
    got = c.attn_prefill(q, [0, n])
    for i in [0, n // 2, n - 20, n - 1]:
        check(got[i:i + 1], q[i:i + 1], K[0], V[0], hkv, past + i, f16, 1 if f16 else 2, i)
    for h in (0, 63):
        at = slice(h * HD, (h + 1) * HD)
        want, tol = ref.attend(q[::4, at], K[0][:, h // 8], V[0][:, h // 8], past + 1 + np.arange(n)[::4], f16,
                               1 if f16 else 2)
        ref.check_rows(got[::4, at], want, tol, h)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,hkv", [(9, 1), (32, 2), (17, 1), (75, 3)])
def test_groups_of_more_than_eight_heads(dtype, H, hkv):
    rng = rng_of("groups", H, hkv)
    spec = [(3, 2000), (1, 0), (40, 90), (1, 650)]
    new, lens, cu = packed(spec)
    f16 = dtype == np.float16
    c, K, V = filled(rng, lens, hkv, 64)
    q = rng.standard_normal((int(cu[-1]), H * HD)).astype(dtype)
    got, dec = c.attn_prefill(q, cu), c.attn_decode(q[:4])
    for z, m in enumerate(new):
        at = slice(cu[z], cu[z + 1])
        check(got[at], q[at], K[z], V[z], hkv, lens[z] - m, f16, 1 if f16 else 2, z)
        check(dec[z:z + 1], q[z:z + 1], K[z], V[z], hkv, lens[z] - 1, f16, 2, z)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,H,hkv,every", [(301, 6, 3, 60), (1025, 2, 1, 41), (1025, 32, 2, 300), (4096, 2, 1, 97)])
def test_decode_of_many_sequences(dtype, B, H, hkv, every):
    """More sequences than lanes and than resident workgroups: short ones, idle ones, and
    some in each stretch of 64 whose runs meet in the workspace."""
    rng = rng_of("many", B, H, hkv)
    lens = [int(x) for x in rng.integers(0, 70, B)]
    for z in range(B - 1, -1, -every):
        lens[z] = int(rng.integers(1500, 6000))
    c, K, V = filled(rng, lens, hkv, 32, table_pages=200)
    q = rng.standard_normal((B, H * HD)).astype(dtype)
    got, f16 = c.attn_decode(q), dtype == np.float16
    for z, n in enumerate(lens):
        if n:
            check(got[z:z + 1], q[z:z + 1], K[z], V[z], hkv, n - 1, f16, 2, z)
        else:
            assert not got[z].any()
    assert np.array_equal(bits(got), bits(c.attn_decode(q)))

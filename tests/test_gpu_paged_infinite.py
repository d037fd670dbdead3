"""Attention over the paged cache with scores of -Inf, from K elements of -Inf: a softmax
gives such a position weight 0, and NaN where a row sees nothing else.  Where the low
part of q is 0 or against the high one's sign the score itself is NaN, and so are all
rows that see it."""
import numpy as np
import pytest

import paged_reference as ref
from test_gpu_paged import HD, bits, expect, filled, packed, rng_of

pytestmark = pytest.mark.gpu
DIM = 9

# q's element that meets the -Inf: exact in one f16 part, or with a low part of either sign
Q = [(np.float16, 1.0), (np.float32, 1.0), (np.float32, 1.0 + 2.0 ** -13), (np.float32, 1.0 - 2.0 ** -13)]


def lowered(c, K, V, page, dead):
    """K with -Inf at DIM of the last KV head in the positions of `dead` (by sequence)."""
    t, out = c.table.download(), []
    for z, k in enumerate(K):
        k = k.copy()
        k[dead[z], -1, DIM] = -np.inf
        if len(k):
            c.append(k, V[z], ref.slots_of(t[z], len(k), page))
        out.append(k)
    return out


def check(got, q, K, V, dead, hkv, first, parts, what):
    """Rows at positions first.. : the heads of the last KV head as a softmax without the
    dead positions, or NaN where a row sees one; the other heads' as ever."""
    f16, n = q.dtype == np.float16, len(K)
    own = got.shape[1] - got.shape[1] // hkv
    want, tol = expect(q, np.where(np.isinf(K), 0, K).astype(np.float16), V, hkv, first, f16, parts)
    ref.check_rows(got[:, :own], want[:, :own], tol[:, :own], what)
    live = np.setdiff1d(np.arange(n), dead)
    for i in range(len(q)):
        seen = np.arange(min(first + 1 + i, n))
        some, hit = np.isin(seen, live).sum(), np.isin(seen, dead).any()
        row = got[i, own:]
        if not len(seen):
            assert not row.any(), (what, i)
        elif not some:
            assert np.isnan(row).all(), (what, i, row[:4])
        elif not (hit and np.isnan(row).all()):
            want, tol = expect(q[i:i + 1, own:], K[live][:, -1:], V[live][:, -1:], 1, some - 1, f16, parts)
            ref.check_rows(got[i:i + 1, own:], want, tol, (what, i))


@pytest.mark.parametrize("dtype,at", Q)
def test_decode(dtype, at):
    """A sequence of one position, of several, of runs that meet in the workspace; all of
    it -Inf, its beginning, its end, one run of it."""
    rng = rng_of("decode inf", at)
    H, hkv, page = 4, 2, 32
    lens = [1, 40, 100, 3000, 3000, 2500, 0, 64, 33]
    dead = [np.arange(1), np.arange(40), np.arange(70), np.arange(3000), np.arange(1000), np.arange(1900, 2500),
            np.arange(0), np.array([63]), np.arange(32)]
    c, K, V = filled(rng, lens, hkv, page)
    q = rng.standard_normal((len(lens), H * HD)).astype(dtype)
    q[:, DIM::HD] = at
    K = lowered(c, K, V, page, dead)
    got = c.attn_decode(q)
    for z, n in enumerate(lens):
        check(got[z:z + 1], q[z:z + 1], K[z], V[z], dead[z], hkv, n - 1, 2, z)
    assert np.array_equal(bits(got), bits(c.attn_decode(q)))


@pytest.mark.parametrize("dtype,at", Q)
@pytest.mark.parametrize("spec,dead", [
    ([(50, 0)], [range(1)]),                                        # the first token of a prompt
    ([(50, 0), (1, 0), (9, 20)], [range(33), range(1), range(29)]),
    ([(5, 2000), (70, 100)], [range(2005), range(10, 90)]),         # cut tiles
    ([(4, 3000), (3, 1500)], [range(1000), range(1200, 1503)]),
    ([(3, 0)] * 70 + [(150, 0)], [range(2)] * 70 + [range(65)]),    # more sequences than lanes
])
def test_prefill(dtype, at, spec, dead):
    rng = rng_of("prefill inf", at, spec)
    H, hkv, page = 4, 2, 32
    new, lens, cu = packed(spec)
    dead = [np.array(d) for d in dead]
    c, K, V = filled(rng, lens, hkv, page)
    q = rng.standard_normal((int(cu[-1]), H * HD)).astype(dtype)
    q[:, DIM::HD] = at
    K = lowered(c, K, V, page, dead)
    got = c.attn_prefill(q, cu)
    for z, m in enumerate(new):
        at_z = slice(cu[z], cu[z + 1])
        check(got[at_z], q[at_z], K[z], V[z], dead[z], hkv, lens[z] - m, 1 if dtype == np.float16 else 2, z)


def test_f16_prefill_has_weight_zero_beside_finite_scores():
    """With one part of q the score is -Inf for certain: rows that see a finite one are
    finite, on the path that hides positions and on the one that does not."""
    rng = rng_of("weight 0")
    n = 200
    c, K, V = filled(rng, [n], 1, 32)
    q = rng.standard_normal((n, 2 * HD)).astype(np.float16)
    q[:, DIM::HD] = 1
    lowered(c, K, V, 32, [np.arange(32, 64)])
    assert np.isfinite(c.attn_prefill(q, [0, n])).all()

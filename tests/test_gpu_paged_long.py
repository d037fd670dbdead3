"""Packed prefill of more row tiles than one list of runs takes: the call's launches,
each over a window of its tokens, against numpy in 64 bits."""
import numpy as np
import pytest

import paged_reference as ref
from helpers import ops
from test_gpu_paged import HD, bits, expect, filled, packed, rng_of

pytestmark = pytest.mark.gpu

CALLS = [  # H, Hkv, (new, past) of each sequence, page; row tiles
    (16, 1, [(9000, 300)], 64),                                       # 1125: a window's last tiles cut
    (8, 2, [(20000, 0), (0, 9), (13100, 70), (1, 4000)], 128),        # 1036: a window ends inside a sequence
    (32, 2, [(75, 40)] * 120, 32),                                    # 1125, 1200 with short ones
    (4, 1, [(3, 50), (36000, 0), (5, 1000)], 64),                     # 1126
]


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("H,hkv,spec,page", CALLS)
def test_more_tiles_than_a_list(dtype, H, hkv, spec, page):
    rng = rng_of("long list", H, hkv, len(spec), page)
    new, lens, cu = packed(spec)
    n, G, f16 = int(cu[-1]), H // hkv, dtype == np.float16
    assert n * G // 128 > 1024
    c, K, V = filled(rng, lens, hkv, page)
    q = rng.standard_normal((n + 5, H * HD)).astype(dtype)
    before = rng.standard_normal(q.shape).astype(dtype)
    got = c.attn_prefill(q, cu, before)
    assert np.array_equal(bits(got[n:]), bits(before[n:]))
    # every token is written; some of each sequence and around the windows' ends whole
    parts = 2 if n * G // 128 < 2000 else 3
    edges = [n * i // parts + d for i in range(1, parts) for d in range(-40, 41, 8)]
    for z, m in enumerate(new):
        at = np.unique([i for i in [0, 1, m // 3, m // 2, m - 1, *(e - cu[z] for e in edges)] if 0 <= i < m])
        for i in at.astype(int):
            r = cu[z] + i
            want, tol = expect(q[r:r + 1], K[z], V[z], hkv, lens[z] - m + i, f16, 1 if f16 else 2)
            ref.check_rows(got[r:r + 1], want, tol, (z, i))
        head = int(rng.integers(H))
        cols, rows = slice(head * HD, (head + 1) * HD), np.arange(0, m, max(20, m // 500))
        if len(rows):
            want, tol = ref.attend(q[cu[z] + rows][:, cols], K[z][:, head // G], V[z][:, head // G],
                                   lens[z] - m + 1 + rows, f16, 1 if f16 else 2)
            ref.check_rows(got[cu[z] + rows][:, cols], want, tol, (z, head))
    assert (bits(got[:n]) != bits(before[:n])).any(-1).all()


def test_in_place_and_captured():
    """The launches of one call in a graph, out in place of q: the eager call's bits on
    every replay."""
    L, rng = ops.lib(), rng_of("long graph")
    H, hkv, page, spec = 16, 1, 64, [(4000, 0), (4600, 90)]
    new, lens, cu = packed(spec)
    n = int(cu[-1])
    c, _, _ = filled(rng, lens, hkv, page)
    dc = ops.DeviceArray.from_host(cu)
    dq = ops.DeviceArray((n, H * HD), np.float32)
    need = L.oxb_attn_prefill_paged_ws_bytes(n, 2, H, hkv, HD)
    ws = ops.DeviceArray((need,), np.uint8)
    st = L.oxb_stream_create()
    ops.check(L.oxb_stream_begin_capture(st))
    ops.check(L.oxb_attn_prefill_paged(dq.ptr, 0, c.pool.ptr, c.n_pages, page, c.table.ptr, c.table.shape[1], dc.ptr,
                                       c.len.ptr, n, 2, H, hkv, HD, dq.ptr, ws.ptr, need, st))
    g = L.oxb_stream_end_capture(st)
    assert g
    for _ in range(3):
        q = rng.standard_normal((n, H * HD)).astype(np.float32)
        dq.upload(q)
        ops.check(L.oxb_graph_launch(g, st))
        ops.check(L.oxb_stream_sync(st))
        assert np.array_equal(bits(dq.download()), bits(c.attn_prefill(q, cu)))
    ops.check(L.oxb_graph_destroy(g))
    ops.check(L.oxb_stream_destroy(st))

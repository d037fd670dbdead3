"""The paged cache's entry points on the CPU: argument checks come before any device
call, sizes, and the reference's own bookkeeping."""
import ctypes as C

import numpy as np
import pytest

from helpers import ops, pkg
import paged_reference as ref

nat = pkg._native
P = C.c_void_p(4096)      # never dereferenced: every call below fails its checks first
BAD = C.c_void_p(4104)


def L():
    return nat.lib()


def test_sizes():
    """512 bytes a position and KV head."""
    assert L().oxb_paged_bytes(1, 32, 1, 128) == 32 * 512
    assert L().oxb_paged_bytes(1000, 256, 5, 128) == 1000 * 256 * 5 * 512
    assert L().oxb_paged_bytes(1 << 19, 4096, 8, 128) == 0          # 2^31 slots
    assert L().oxb_paged_bytes((1 << 19) - 1, 4096, 8, 128) > 1 << 42
    for args in ((0, 32, 1, 128), (1, 16, 1, 128), (1, 48, 1, 128), (1, 8192, 1, 128), (1, 0, 1, 128),
                 (1, -32, 1, 128), (1, 32, 0, 128), (1, 32, 1, 64)):
        assert L().oxb_paged_bytes(*args) == 0, args


def refused(call, cases):
    for kw, msg in cases:
        assert call(**kw) == -1, kw
        assert msg in nat.last_error(), (kw, nat.last_error())


def test_update_refusals():
    def up(page=32, batch=2, ln=P, d=P, t=P, w=4, f=P, cap=8, nf=P, lo=P, nfo=P, cu=P, g=None, s=None, p=None, n=4):
        return L().oxb_paged_update(page, batch, ln, d, t, w, f, cap, nf, lo, nfo, cu, g, s, p, n, None)
    refused(up, [(dict(page=16), "page size 16"), (dict(page=33), "page size 33"), (dict(page=8192), "page size 8192"),
                 (dict(page=0), "page size 0"), (dict(page=-2 ** 31), "page size"), (dict(batch=0), "batch 0"),
                 (dict(batch=4097), "batch 4097"), (dict(t=None), "block table"), (dict(w=0), "0 pages"),
                 (dict(w=(1 << 19) + 1), "pages a sequence"), (dict(ln=None), "NULL"), (dict(d=None), "NULL"),
                 (dict(f=None), "NULL"), (dict(nf=None), "NULL"), (dict(lo=None), "NULL"), (dict(nfo=None), "NULL"),
                 (dict(cu=None), "NULL"), (dict(cap=0), "free list of 0"), (dict(cap=1 << 30), "free list"),
                 (dict(n=-1), "-1 tokens"), (dict(n=1 << 30), "tokens")])


def test_append_refusals():
    def ap(pool=P, np_=4, page=32, hkv=1, hd=128, k=P, v=P, ts=128, hs=128, sp=None, s=P, n=1):
        return L().oxb_paged_append(pool, np_, page, hkv, hd, k, v, ts, hs, sp, s, n, None)
    refused(ap, [(dict(pool=None), "pool is NULL"), (dict(pool=BAD), "256-byte"), (dict(np_=0), "0 pages"),
                 (dict(np_=1 << 26), "pages of 32"), (dict(page=24), "page size 24"), (dict(hkv=0), "kv heads 0"),
                 (dict(hkv=4097), "kv heads"), (dict(hd=64), "head_dim 64"), (dict(k=None), "NULL"),
                 (dict(v=None), "NULL"), (dict(s=None), "NULL"), (dict(k=BAD), "aligned"), (dict(v=BAD), "aligned"),
                 (dict(ts=129), "strides 129"), (dict(hs=4), "strides"), (dict(n=-1), "-1 tokens")])
    assert ap(n=0, k=None) == 0          # nothing to do


def test_attention_refusals():
    need = L().oxb_attn_decode_paged_ws_bytes(2, 4, 1, 128)
    assert need > 0

    def dec(q=P, t=0, pool=P, np_=4, page=32, tab=P, w=2, ln=P, b=2, H=4, hkv=1, hd=128, out=P, ws=P, wsb=1 << 40):
        return L().oxb_attn_decode_paged(q, t, pool, np_, page, tab, w, ln, b, H, hkv, hd, out, ws, wsb, None)
    common = [(dict(q=None), "q or out"), (dict(out=None), "q or out"), (dict(q=BAD), "aligned"),
              (dict(out=BAD), "aligned"), (dict(t=2), "type 2"), (dict(t=-1), "type -1"), (dict(pool=None), "pool"),
              (dict(pool=BAD), "pool"), (dict(np_=0), "0 pages"), (dict(page=31), "page size 31"),
              (dict(tab=None), "block table"), (dict(w=0), "0 pages"), (dict(ln=None), "len is NULL"),
              (dict(b=0), "batch 0"), (dict(b=4097), "batch 4097"), (dict(H=5, hkv=2), "heads 5"),
              (dict(H=0), "heads 0"), (dict(H=65536), "65536 heads"), (dict(hkv=0), "kv heads 0"),
              (dict(hd=64), "head_dim 64"), (dict(ws=None), "workspace"), (dict(ws=C.c_void_p(4096 + 64)), "workspace")]
    refused(dec, common + [(dict(wsb=need - 1), "workspace")])
    need = L().oxb_attn_prefill_paged_ws_bytes(8, 2, 4, 1, 128)
    assert need > 0

    def pre(q=P, t=0, pool=P, np_=4, page=32, tab=P, w=2, cu=P, ln=P, n=8, b=2, H=4, hkv=1, hd=128, out=P, ws=P,
            wsb=1 << 40):
        return L().oxb_attn_prefill_paged(q, t, pool, np_, page, tab, w, cu, ln, n, b, H, hkv, hd, out, ws, wsb, None)
    common[12] = (dict(ln=None), "cu or len")
    refused(pre, common + [(dict(wsb=need - 1), "workspace"), (dict(cu=None), "cu or len"), (dict(n=0), "0 tokens"),
                           (dict(n=-3), "-3 tokens"), (dict(n=1 << 29), "tokens"),
                           (dict(n=(1 << 27) + 1, H=1), "tokens"),
                           (dict(n=1 << 20, H=4096, hkv=4096), "4096 heads")])
    for args in ((0, 4, 1, 128), (1, 5, 2, 128), (1, 4, 1, 64), (4097, 4, 1, 128), (1, 4, 0, 128)):
        assert L().oxb_attn_decode_paged_ws_bytes(*args) == 0
        assert L().oxb_attn_prefill_paged_ws_bytes(1, *args) == 0
    assert L().oxb_attn_prefill_paged_ws_bytes(0, 1, 4, 1, 128) == 0


def test_sequences_of_a_prefill_call():
    """128 at most; decode takes 4096."""
    f, need = L().oxb_attn_prefill_paged_ws_bytes, L().oxb_attn_prefill_paged_ws_bytes(4096, 128, 4, 2, 128)
    assert need > 0 and f(4096, 129, 4, 2, 128) == 0 and f(4096, 4096, 4, 2, 128) == 0
    assert L().oxb_attn_decode_paged_ws_bytes(4096, 4, 2, 128) > 0
    refused(lambda b: L().oxb_attn_prefill_paged(P, 0, P, 4, 32, P, 2, P, P, 4096, b, 4, 2, 128, P, P, 1 << 40, None),
            [(dict(b=129), "batch 129"), (dict(b=4096), "batch 4096")])


def test_workspace_grows_with_the_call():
    """One workspace of the largest call serves every smaller one; decode's depends on
    the group alone."""
    f = L().oxb_attn_prefill_paged_ws_bytes
    for H, hkv in ((20, 5), (8, 8), (32, 2), (7, 1), (640, 640)):
        last = 0
        for n in (1, 2, 7, 31, 32, 33, 100, 128, 129, 1000, 4096, 100000):
            for b in (1, 2, 64, 4096):
                assert f(n, b, H, hkv, 128) >= f(n, max(1, b // 2), H, hkv, 128)
            assert f(n, 64, H, hkv, 128) >= last
            last = f(n, 64, H, hkv, 128)
    d = L().oxb_attn_decode_paged_ws_bytes
    assert d(1, 20, 5, 128) == d(4096, 20, 5, 128) == d(3, 4, 1, 128)


def test_python_refusals():
    c = ops.PagedCache.__new__(ops.PagedCache)
    c.batch, c.Hkv, c.hd, c.n_pages, c.page_size = 2, 2, 128, 4, 32
    for call in (lambda: c.step([1]), lambda: c.append(np.zeros((2, 2, 128)), np.zeros((1, 2, 128)), [0, 1]),
                 lambda: c.append(np.zeros((2, 2, 64)), np.zeros((2, 2, 64)), [0, 1]),
                 lambda: c.attn_decode(np.zeros((2, 4 * 128))), lambda: c.attn_decode(np.zeros((2, 300), np.float32)),
                 lambda: c.attn_decode(np.zeros((3, 512), np.float32)),
                 lambda: c.attn_prefill(np.zeros((3, 512), np.float32), [0, 3])):
        with pytest.raises(ValueError):
            call()


def test_reference_bookkeeping():
    """By hand: pages of 32, three sequences; the second gives two pages back, the
    first takes the last of them, the third the other one and one of the list."""
    table = [[5, -1, -1], [7, 8, 9], [-1, -1, -1]]
    after, t, free, n, cu, granted, slots, pos = ref.update(32, [31, 70, 0], [2, -60, 40], table, [3, 4, 0, 0], 2, 44)
    assert after == [33, 10, 40] and granted == [2, 0, 40] and cu == [0, 2, 2, 42]
    assert t.tolist() == [[5, 9, -1], [7, 8, 9], [8, 4, -1]]
    assert n == 1 and free.tolist() == [3, 4, 0, 0]
    assert slots[:3].tolist() == [5 * 32 + 31, 9 * 32, 8 * 32] and pos[:3].tolist() == [31, 32, 0]
    assert slots[41] == 4 * 32 + 7 and slots[42:].tolist() == [-1, -1]
    # one page for two: the first that does not fit, and none after it that needs one
    after, t, free, n, cu, granted, _, _ = ref.update(32, [32, 32, 31], [33, 1, 1], [[1, 0, 0], [2, 0, 0], [3, 0, 0]],
                                                      [6], 1, 40)
    assert after == [32, 32, 32] and granted == [0, 0, 1] and n == 1 and cu == [0, 33, 34, 35]


def test_reference_layout():
    """The header's formula for a pool's elements, and every element once."""
    page, hkv, n = 64, 2, 3
    seen = np.zeros(n * page * hkv * 256, np.int64)
    for s in range(n * page):
        for h in range(hkv):
            for e in ref.elements(page, hkv, h, s):
                seen[e] += 1
    assert (seen == 1).all()
    k, v = ref.elements(64, 2, 1, 2 * 64 + 37)
    base = ((2 * 2 + 1) * 2 + 1) * 8192
    assert k[9] == base + (1 * 32 + 5) * 8 + 1 and v[9] == base + 4096 + (0 * 128 + 9) * 8 + 5

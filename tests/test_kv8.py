"""The 8-bit KV cache's entry points and the logit rules on the CPU: argument checks
come before any device call, sizes, and the reference's own arithmetic."""
import ctypes as C
from fractions import Fraction

import numpy as np
import pytest

from helpers import ops, pkg
import kv8_reference as ref

nat = pkg._native
P = C.c_void_p(4096)      # never dereferenced: every call below fails its checks first


def L():
    return nat.lib()


def err():
    return nat.last_error()


def test_sizes():
    """codes 8192 B a block and head, 8 B scales, 4 B weight, 16 KB tail a head; each
    part 256-byte aligned."""
    assert L().oxb_kv8_bytes(1, 128, 1) == 8192 + 256 + 256 + 16384
    assert L().oxb_kv8_bytes(5, 128, 4096) == 5 * 128 * 8192 + 5 * 128 * 8 + 5 * 128 * 4 + 5 * 16384
    assert L().oxb_kv8_bytes(5, 64, 4096) == 0 and L().oxb_kv8_bytes(0, 128, 4096) == 0
    assert L().oxb_kv8_bytes(1, 128, (1 << 24) + 1) == 0
    big = L().oxb_kv8_bytes(8, 128, 1 << 24)
    assert big > (1 << 32)          # sizes past 32 bits come whole


def _append(cache=P, stride=0, fmt=0, batch=1, hkv=1, hd=128, ms=64, k=P, v=P, ss=0, hs=128, pos=None,
            ps=0, pos0=0, n=1):
    return L().oxb_kv8_append(cache, stride, fmt, batch, hkv, hd, ms, k, v, ss, hs, 0, pos, ps, pos0, n,
                              None, None)


@pytest.mark.parametrize("kw,msg", [
    (dict(cache=None), "cache is NULL"),
    (dict(cache=C.c_void_p(4096 + 16)), "256-byte aligned"),
    (dict(fmt=2), "format 2"),
    (dict(fmt=-1), "format -1"),
    (dict(hd=64), "head_dim 64"),
    (dict(batch=0), "batch 0"),
    (dict(batch=65536), "batch 65536"),
    (dict(hkv=0), "kv heads 0"),
    (dict(ms=0), "max_seq 0"),
    (dict(ms=(1 << 24) + 1), "max_seq"),
    (dict(batch=2, stride=256), "cache stride 256"),
    (dict(batch=2, stride=1000001), "cache stride 1000001"),
    (dict(k=None), "k or v is NULL"),
    (dict(v=C.c_void_p(4104)), "16-byte aligned"),
    (dict(hs=129), "16-byte aligned"),
    (dict(n=0), "0 rows"),
    (dict(n=65), "65 rows"),
    (dict(pos0=64), "rows 64..64 of 64"),
    (dict(pos0=-1), "rows -1..-1 of 64"),
    (dict(pos=P, ps=-1), "pos stride -1"),
])
def test_append_refusals(kw, msg):
    assert _append(**kw) == -1
    assert msg in err()


def test_read_refusals():
    def read(k=P, v=P, n=1, ps=0, ls=0):
        return L().oxb_kv8_read(P, 0, 0, 1, 1, 128, 64, None, ps, 0, n, None, ls, k, v, None)
    for kw, msg in ((dict(k=None), "NULL"), (dict(v=C.c_void_p(4100)), "aligned"), (dict(n=0), "0 rows"),
                    (dict(ps=-1), "stride"), (dict(ls=-2), "stride")):
        assert read(**kw) == -1 and msg in err(), kw


def test_attention_refusals():
    def dec(q=P, cache=P, stride=0, fmt=0, pos=P, ps=1, batch=1, H=4, hkv=1, hd=128, ms=64, out=P, ws=P,
            wsb=1 << 30):
        return L().oxb_attn_decode_kv8(q, cache, stride, fmt, pos, ps, batch, H, hkv, hd, ms, 0, out, ws,
                                       wsb, None)
    need = L().oxb_attn_decode_kv8_ws_bytes(1, 4, 1, 128, 64)
    assert need > 0
    for kw, msg in ((dict(q=None), "q or out"), (dict(out=C.c_void_p(4100)), "aligned"),
                    (dict(pos=None), "pos is NULL"), (dict(ps=-1), "stride -1"),
                    (dict(H=5, hkv=2), "heads 5"), (dict(H=0), "heads 0"), (dict(hd=96), "head_dim 96"),
                    (dict(fmt=7), "format 7"), (dict(ms=0), "max_seq 0"), (dict(ws=None), "workspace"),
                    (dict(wsb=need - 1), "workspace"), (dict(ws=C.c_void_p(4096 + 64)), "workspace")):
        assert dec(**kw) == -1 and msg in err(), kw

    def pre(q=P, cache=P, fmt=0, n=8, pos0=0, H=4, hkv=1, hd=128, ms=64, w=1, out=P, ws=P, wsb=1 << 30):
        return L().oxb_attn_prefill_kv8(q, cache, fmt, n, pos0, H, hkv, hd, ms, w, out, ws, wsb, None)
    need = L().oxb_attn_prefill_kv8_ws_bytes(8, 0, 4, 1, 128, 1)
    assert need > 0
    for kw, msg in ((dict(q=None), "q or out"), (dict(n=0), "bad range"), (dict(pos0=57), "bad range"),
                    (dict(pos0=-1), "bad range"), (dict(n=65), "bad range"), (dict(H=6, hkv=4), "heads 6"),
                    (dict(hd=64), "head_dim 64"), (dict(ws=None), "workspace"),
                    (dict(wsb=need - 1), "workspace"), (dict(cache=None), "cache is NULL")):
        assert pre(**kw) == -1 and msg in err(), kw
    assert L().oxb_attn_decode_kv8_ws_bytes(1, 5, 2, 128, 64) == 0
    assert L().oxb_attn_prefill_kv8_ws_bytes(0, 0, 4, 1, 128, 0) == 0


def test_evict_refusals():
    far = C.c_void_p(1 << 40)

    def ev(cache=P, stride=0, ms=1024, dst=far, ds=0, dms=256, ln=P, ls=1, lo=P, los=1, batch=1, hkv=1,
           hd=128, budget=8, sink=1, recent=1, ws=P, wsb=1 << 20):
        return L().oxb_kv8_evict(cache, stride, ms, dst, ds, dms, ln, ls, lo, los, batch, hkv, hd, budget,
                                 sink, recent, ws, wsb, None)
    seq = L().oxb_kv8_bytes(1, 128, 1024)
    for kw, msg in ((dict(cache=None), "cache is NULL"), (dict(dst=None), "cache is NULL"),
                    (dict(ln=None), "len or len_out"), (dict(lo=None), "len or len_out"),
                    (dict(ls=-1), "length stride"), (dict(batch=2, stride=seq, ds=seq, los=0), "length stride"),
                    (dict(budget=0), "budget of 0"), (dict(recent=0), "budget of 8"),
                    (dict(sink=-1), "budget of 8"), (dict(sink=8), "budget of 8"),
                    (dict(sink=2 ** 31 - 1), "budget of 8"), (dict(recent=2 ** 31 - 1), "budget of 8"),
                    (dict(dms=255), "255 positions"), (dict(dst=P), "keeps its max_seq"),
                    (dict(dst=C.c_void_p(4096 + 256)), "overlaps"), (dict(ws=None), "workspace"),
                    (dict(wsb=16), "workspace"), (dict(hd=64), "head_dim 64")):
        assert ev(**kw) == -1 and msg in err(), kw
    assert L().oxb_kv8_evict_ws_bytes(1, 1, 1024, 0) == 0


def test_rules_refusals():
    def rl(lg=P, st=100, n=2, V=100, pen=P, h=P, ho=P, nh=4, bi=P, b=P, bo=P, nb=4, m=P, ms=4,
           out=C.c_void_p(1 << 40), os=100):
        return L().oxb_logits_rules(lg, st, n, V, pen, h, ho, nh, bi, b, bo, nb, m, ms, out, os, None)
    for kw, msg in ((dict(lg=None), "logits or out"), (dict(out=None), "logits or out"), (dict(n=0), "0 rows"),
                    (dict(V=0), "vocabulary 0"), (dict(st=99), "row strides 99"), (dict(os=99), "and 99"),
                    (dict(nh=-1), "history of -1"), (dict(h=None), "history of 4"), (dict(ho=None), "history of 4"),
                    (dict(nb=-1), "-1 biases"), (dict(b=None), "4 biases"), (dict(bo=None), "4 biases"),
                    (dict(ms=3), "mask rows of 3"), (dict(out=C.c_void_p(4100)), "overlaps"),
                    (dict(out=P, os=200), "overlaps")):
        assert rl(**kw) == -1 and msg in err(), kw


def test_reference_codes_are_correctly_rounded():
    """The quotient 127 x / a in f64 and in f32 rounds to the code of the exact
    rational: ties are met exactly, nothing else falls on one."""
    rng = np.random.default_rng(5)
    x = (rng.standard_normal(400) * 3).astype(np.float16)
    for a in (np.float16(127 / 64), np.float16(3.3), np.float16(11.0)):
        x = np.clip(x, -a, a).astype(np.float16)
        for top in (127, 448):
            r32 = np.float32(x) * np.float32(top) / np.float32(a)
            r64 = x.astype(np.float64) * top / np.float64(a)
            for v, p, q in zip(x.tolist(), r32, r64):
                exact = Fraction(v) * top / Fraction(float(a))
                if top == 127:
                    assert round(exact) == np.rint(p) == np.rint(q)
                else:
                    assert float(ref.e4m3_round(float(p))) == float(ref.e4m3_round(q))


def test_reference_e4m3():
    codes = [m / 8 * 2.0 ** -6 for m in range(8)]
    codes += [(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8)][:-1]
    codes = np.array(codes)
    assert codes.max() == 448 and np.array_equal(ref.e4m3_round(codes), codes)
    rng = np.random.default_rng(1)
    x = np.concatenate([rng.uniform(0, 448, 300), rng.uniform(0, 0.05, 300), (codes[1:] + codes[:-1]) / 2])
    for v, r in zip(x, ref.e4m3_round(x)):
        d = np.abs(codes - v)
        near = np.flatnonzero(d == d.min())
        assert r == codes[near[near % 2 == 0][0] if len(near) > 1 else near[0]]


def test_evict_workspace_is_of_the_cache_at_most():
    """A budget past the cache's blocks keeps all of them and asks for no more memory."""
    b = L().oxb_kv8_evict_ws_bytes
    assert b(3, 5, 100, 4) == 256 + 256
    assert b(3, 5, 100, (1 << 31) - 1) == b(3, 5, 100, 4)


def test_prefill_workspace_with_weights_stays_bounded():
    """8 bytes per row and block, 256 MB at most (and the parts of two launches' rows
    at a time beside them)."""
    b = L().oxb_attn_prefill_kv8_ws_bytes
    assert b(101, 0, 20, 5, 128, 1) - b(101, 0, 20, 5, 128, 0) == (20 * 101 * 4 + 255) // 256 * 256 + 5 * 4 * 512 * 8
    for n, pos0, H, hkv in ((8192, 0, 20, 5), (100000, 0, 20, 5), (600, 261000, 8, 1), (1, (1 << 24) - 1, 64, 1)):
        assert b(n, pos0, H, hkv, 128, 1) <= b(n, pos0, H, hkv, 128, 0) + (600 << 20), (n, pos0)


def test_python_arguments_of_other_shapes_are_refused():
    """Before anything is uploaded: the kernels take the arrays' sizes on trust."""
    c = ops.Kv8Cache.__new__(ops.Kv8Cache)
    c.batch, c.Hkv, c.max_seq, c.fmt, c.hd, c.stride = 2, 2, 64, ops.KV8_INT8, 128, 0
    d = ops.Kv8Cache.__new__(ops.Kv8Cache)
    d.batch, d.Hkv, d.max_seq, d.fmt, d.hd, d.stride = 2, 2, 64, ops.KV8_E4M3, 128, 0
    kv = np.zeros((2, 2, 3, 128), np.float16)
    q = np.zeros((2, 512), np.float32)
    x = np.zeros((2, 70), np.float32)
    for call in (lambda: c.append(kv[:1], kv, [0, 0]), lambda: c.append(kv, kv[:, :, :2], [0, 0]),
                 lambda: c.append(kv[..., :64], kv[..., :64], [0, 0]), lambda: c.append(kv, kv, [0]),
                 lambda: c.append(kv, kv, [0, 0], [1]), lambda: c.read([0], 3), lambda: c.read([0, 0], 3, [4]),
                 lambda: c.attn_decode(q, [5]), lambda: c.attn_decode(q[:, :200], [5, 5]),
                 lambda: c.attn_decode(q[:, :384], [5, 5]), lambda: c.attn_prefill(q, 0, slot=2),
                 lambda: c.attn_prefill(q[:, :100], 0), lambda: c.evict([1], 2), lambda: c.evict([1, 1], 2, dst=d),
                 lambda: ops.logits_rules(x, history=[[1]]), lambda: ops.logits_rules(x, bias=[[(1, 0.5)]]),
                 lambda: ops.logits_rules(x, mask=np.zeros((2, 2), np.uint32)),
                 lambda: ops.logits_rules(x, mask=np.zeros((1, 3), np.uint32)),
                 lambda: ops.logits_rules(x, penalties=np.ones((1, 3)))):
        with pytest.raises(ValueError):
            call()

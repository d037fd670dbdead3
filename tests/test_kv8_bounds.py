"""Bounds of the 8-bit cache's tests and workspaces, on the CPU."""
import numpy as np
import pytest

from helpers import pkg
import kv8_reference as ref

HEADS = [(20, 5), (32, 8), (8, 1), (4, 4), (32, 2), (9, 1), (64, 64), (1, 1), (2400, 600)]


def L():
    return pkg._native.lib()


def test_check_rows_takes_no_nan():
    """A NaN compares false either way: it has to count as outside its bound."""
    want, tol = np.ones((2, 3)), np.full((2, 3), 1e-3)
    ref.check_rows(want.astype(np.float32), want, tol)
    ref.check_rows(want + 1e-3 * 0.99, want, tol)
    for at in ((0, 0), (1, 2)):
        for i in range(3):
            a = [want.astype(np.float32), want.copy(), tol.copy()]
            a[i][at] = np.nan
            with pytest.raises(AssertionError):
                ref.check_rows(*a)
    with pytest.raises(AssertionError):
        ref.check_rows(want + 2e-3, want, tol)
    with pytest.raises(AssertionError):
        ref.check_rows(np.full((2, 3), np.inf), want, tol)


def prefill_need(n, pos0, H, hkv, weights, cus=256):
    """What one call of the prefill attention lays out: per launch (all tokens; with
    weights as many as keep 8 bytes per row and block under 256 MB) the parts of row
    tiles of 128 rows in even runs of the least length, 8 blocks or more, whose runs are
    at most two per CU; the rows' sums and the blocks' sums of weights."""
    G, al, blk = H // hkv, lambda b: -(-b // 256) * 256, lambda t: -(-t // 32)
    step = n
    if weights:
        most = max(1, (256 << 20) // (8 * H * blk(pos0 + n)))
        step = -(-n // -(-n // most))
    worst = 0
    for i in range(0, n, step):
        m, p = min(step, n - i), pos0 + i
        rows, most, slots = m * G, blk(p + m), min(2 * cus // hkv, 512)
        rt = -(-rows // 128)
        seen = [blk(p + (min((r + 1) * 128, rows) - 1) // G + 1) for r in range(rt)]
        per = most
        if rt <= slots and most > 8:
            per = next(x for x in range(8, most + 1) if x == most or sum(-(-b // x) for b in seen) <= slots)
        splits, at = -(-most // per), 4096
        if splits > 1:
            at += al(splits * hkv * rows * 8) + al(splits * hkv * rows * 512)
        if weights:
            at += al(hkv * rows * 4) + al(hkv * most * rt * 128 * 8)
        worst = max(worst, at)
    return worst


@pytest.mark.parametrize("weights", [0, 1])
@pytest.mark.parametrize("H,hkv", HEADS)
def test_prefill_workspace_of_the_largest_call_serves_all(H, hkv, weights):
    """Sized for n tokens behind pos0, it holds what any call of fewer tokens that ends
    no later lays out: a shorter prompt or a later chunk is never refused."""
    size = L().oxb_attn_prefill_kv8_ws_bytes
    rng = np.random.default_rng(H * 64 + hkv)
    for n, pos0 in ((1024, 0), (2048, 0), (3300, 0), (101, 20000), (512, 3584), (700, 30000), (6000, 100)):
        big = size(n, pos0, H, hkv, 128, weights)
        small = [(n, pos0), (1, 0), (1, n + pos0 - 1), (n, 0), (min(n, 101), n + pos0 - min(n, 101))]
        for _ in range(10):
            m = int(np.exp(rng.uniform(0, np.log(n))))
            small.append((m, int(rng.integers(0, n + pos0 - m + 1))))
        for m, p in small:
            assert size(m, p, H, hkv, 128, weights) <= big, (n, pos0, m, p)
            assert prefill_need(m, p, H, hkv, weights) <= size(m, p, H, hkv, 128, weights), (m, p)
            assert size(m, p, H, hkv, 128, 0) <= big


def decode_need(batch, H, hkv, max_seq, cus=256):
    """What a decode call lays out: two workgroups per CU over the rows (sequence and KV
    head) as runs, each of four blocks or more; past 1024 rows no cuts."""
    nb, rows, al = -(-max_seq // 32), batch * hkv, lambda b: -(-b // 256) * 256
    splits = 1 if rows > 1024 else max(1, min(2 * cus // rows, -(-nb // 4)))
    return 4096 + al(batch * H * splits * 8) + al(batch * H * splits * 512) + al(batch * H * nb * 8)


@pytest.mark.parametrize("H,hkv", HEADS)
def test_decode_workspace_of_the_largest_batch_serves_all(H, hkv):
    """52 sequences of 5 KV heads have one run each, 51 have two: a workspace for the
    larger batch and longer cache holds the smaller ones'."""
    size = L().oxb_attn_decode_kv8_ws_bytes
    for batch, max_seq in ((1, 1), (52, 2304), (64, 4096), (33, 700), (205, 130), (300, 40), (1025, 500)):
        big = size(batch, H, hkv, 128, max_seq)
        for b in sorted({1, 2, 3, 51, 52, 102, batch // 2 + 1, batch - 1, batch}):
            for ms in {1, 33, 129, 700, max_seq - 1, max_seq}:
                if 1 <= b <= batch and 1 <= ms <= max_seq:
                    n = size(b, H, hkv, 128, ms)
                    assert decode_need(b, H, hkv, ms) <= n <= big, (batch, max_seq, b, ms)

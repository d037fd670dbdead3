"""The 8-bit cache, its attention, eviction and the logit rules in numpy, 64 bits
(kept values and scales as the cache defines them)."""
import numpy as np

BLOCK, HD = 32, 128
INT8, E4M3 = 0, 1
U = 2.0 ** -24      # half a step of f32


def e4m3_round(x):
    """Nearest e4m3 number (ties to even) of |x| <= 448: 3 mantissa bits, steps of
    2^-9 below 2^-6."""
    x = np.asarray(x, np.float64)
    e = np.maximum(np.frexp(np.abs(x))[1] - 1, -6)
    step = np.ldexp(1.0, e - 3)
    return np.rint(x / step) * step


def quantize(x, fmt):
    """One block's rows [r][128] f16: values code * scale as f32."""
    if not np.all(np.isfinite(x)):
        return np.full(x.shape, np.nan, np.float32)
    top = 127.0 if fmt == INT8 else 448.0
    a = np.float64(np.abs(x).max()) if x.size else 0.0
    if a == 0:
        return np.zeros(x.shape, np.float32)
    r = x.astype(np.float64) * top / a
    code = np.rint(r) + 0.0 if fmt == INT8 else e4m3_round(r)   # (a whole number has no -0)
    return code.astype(np.float32) * (np.float32(a) / np.float32(top))


def values(rows, fmt):
    """Rows [n][128] of one head: what the cache stands for."""
    return np.concatenate([quantize(rows[i:i + BLOCK], fmt) for i in range(0, len(rows), BLOCK)]
                          or [np.zeros((0, HD), np.float32)])


def attend(q, k, v):
    """One query head q [128] over k, v [n][128]: (out, p, bound on an output's
    error, relative bound on a weight's).

    With u = 2^-24 and S = max_t sum_d |q_d K_td| / sqrt(128): a score is off by
    at most 2^-22 S for q's two f16 parts, 128 u S for the f32 sum, and 4 u S for
    the factors; its power of two by that and 4 u (the exponent's rounding is
    relative to it: another 2 u |x| log2(e), |x| <= S); numerator and
    denominator both: twice.  The sums over n positions add (n / 32 + 64) u and
    p's two parts 2^-22."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    s = k @ q / np.sqrt(HD)
    p = np.exp(s - s.max())
    p /= p.sum()
    S = (np.abs(k) @ np.abs(q)).max() / np.sqrt(HD)
    rel = 2 * ((4 + 128 + 4 + 4) * U * S + 8 * U) + (len(k) / BLOCK + 64) * U + 4 * U
    return p @ v, p, rel * (p @ np.abs(v)) + 1e-37, rel


def parts_floor(v):
    """What attend()'s bound leaves out where a position that takes nearly all of the
    weight has the value 0 in some dim, so that weights far below 2^-22 make up
    the whole output there: the two f16 parts of x = 2^6 2^(s - m2) vs hold it to
    2^-25 (f16's smallest step is 2^-24), so an output's numerator is off by at
    most n 2^-25 top (top: the largest code).  The denominator is at least 2^6
    2^(s_max - m2), and m2 <= s_max + e, 2^e <= 2 vs_max: the output is off by at
    most n 2^-25 top 2 vs_max 2^-6 = n 2^-30 max|v|."""
    return len(v) * 2.0 ** -30 * float(np.abs(v).max(initial=0))


def rms_bound(q, k):
    """A bound on the outputs' relative error in the 2-norm: roundings of a score's
    128 products fall either way, so they add as sqrt(128) u, with q's split
    (4 u) 16 u S; S as the mean over positions, and 16 u for the rest; doubled
    for numerator and denominator."""
    S = (np.abs(k.astype(np.float64)) @ np.abs(q.astype(np.float64))).mean() / np.sqrt(HD)
    return 2 * 16 * U * (S + 1)


def check_rows(got, want, tol, what=""):
    """Every value within its bound; a NaN on any side is within none."""
    ok = np.abs(np.asarray(got, np.float64) - want) <= tol
    assert ok.all(), (what, int((~ok).sum()), float(np.max(np.abs(got - want) / tol)))


def attend_rows(q, K, V, Hkv, first):
    """Queries q [n][H*128] at positions first.. over one sequence's K, V
    [Hkv][S][128]: out, error bounds, block weights [Hkv][blocks], their bounds."""
    n, H = q.shape[0], q.shape[1] // HD
    G = H // Hkv
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    nb = (K.shape[1] + BLOCK - 1) // BLOCK
    w, wtol = np.zeros((Hkv, nb)), np.zeros((Hkv, nb))
    for i in range(n):
        m = first + i + 1
        if m <= 0:
            continue
        for h in range(H):
            g, at = h // G, slice(h * HD, (h + 1) * HD)
            out[i, at], p, tol[i, at], rel = attend(q[i, at], K[g, :m], V[g, :m])
            for b in range((m + BLOCK - 1) // BLOCK):
                t = p[b * BLOCK:(b + 1) * BLOCK].sum()
                w[g, b] += t
                wtol[g, b] += rel * t
    # n * G terms added in f32
    return out, tol, w, wtol + (n * G + 64) * U * w + 1e-37


def kept_blocks(w, nblk, budget, sink, recent):
    if nblk <= budget:
        return list(range(nblk))
    must = set(range(sink)) | set(range(nblk - recent, nblk))
    rest = [b for b in range(nblk) if b not in must]
    rest.sort(key=lambda b: (-w[b] if w[b] == w[b] else np.inf, b))
    return sorted(must | set(rest[:budget - sink - recent]))


def rules(logits, pen, history, bias, mask):
    """oxb_logits_rules with each step rounded to f32."""
    x = np.array(logits, np.float32)
    n, V = x.shape
    for r in range(n):
        if pen is not None and history is not None:
            rep, f, p = (np.float32(t) for t in pen[r])
            ids = [i for i in history[r] if 0 <= i < V]
            for i in set(ids):
                y = x[r, i]
                y = y / rep if y > 0 else y * rep
                x[r, i] = y - (f * np.float32(ids.count(i)) + p)
        for i, b in dict(bias[r]).items() if bias is not None else ():
            if 0 <= i < V:
                x[r, i] += np.float32(b)
        if mask is not None:
            m = mask[r] if mask.ndim == 2 else mask
            bit = np.arange(V)
            x[r, (m[bit // 32] >> (bit % 32).astype(np.uint32)) & 1 == 0] = -np.inf
    return x

"""The paged cache in numpy: its bookkeeping one sequence after the other, its layout,
and attention in 64 bits with bounds on the kernels' errors."""
import numpy as np

HD, UNIT = 128, 32
U = 2.0 ** -24       # half a step of f32
H16 = 2.0 ** -11     # half a step of f16


def pages(n, page):
    return -(-n // page)


def update(page, length, delta, table, free, n_free, n_max):
    """oxb_paged_update with a list as the stack: new lengths, table, free list, its
    count, cu, granted, slots, pos (table and free: copies)."""
    table, free = np.array(table), np.array(free)
    B, W = table.shape
    cap = W * page
    held = [min(max(int(n), 0), cap) for n in length]
    after = list(held)
    n_free = min(max(int(n_free), 0), len(free))
    given = []                      # pages given back, in order
    for z, d in enumerate(delta):
        if d < 0:
            after[z] = max(held[z] + int(d), 0)
            given += [int(table[z, b]) for b in range(pages(after[z], page), pages(held[z], page))]
    stack = [int(x) for x in free[:n_free]] + given
    room, cu, granted = len(stack), [0], [0] * B
    slots, pos = np.full(n_max, -1, np.int32), np.full(n_max, -1, np.int32)
    want = 0                        # pages wanted so far, granted or not
    for z, d in enumerate(int(d) for d in delta):
        first = cu[-1] if len(cu) == 1 or cu[-1] < n_max else n_max
        total = sum(max(int(x), 0) for x in delta[:z + 1])
        cu.append(min(total, n_max))
        if d <= 0 or held[z] + d > cap or total > n_max:
            continue
        need = pages(held[z] + d, page) - pages(held[z], page)
        want += need
        if need and want > room:
            continue
        for b in range(pages(held[z], page), pages(held[z] + d, page)):
            table[z, b] = stack.pop()
        granted[z], after[z] = d, held[z] + d
        for i in range(d):
            p = held[z] + i
            pos[first + i] = p
            slot = int(table[z, p // page]) * page + p % page
            slots[first + i] = slot if 0 <= table[z, p // page] and slot < 2 ** 31 else -1
    left = min(len(stack), len(free))       # ids past the list's end are lost
    free[n_free:left] = stack[n_free:left]
    return after, table, free, left, cu, granted, slots, pos


def elements(page, hkv, head, slot):
    """Element indices of the K and V rows of a slot in the pool, [128] each."""
    d = np.arange(HD)
    base = (int(slot) // page * hkv + head) * page * 2 * HD + int(slot) % page // UNIT * (2 * UNIT * HD)
    t = int(slot) % UNIT
    return base + (d // 8 * UNIT + t) * 8 + d % 8, base + UNIT * HD + (t // 8 * HD + d) * 8 + t % 8


def slots_of(row, n, page):
    """Slots of positions 0 .. n-1 of a sequence with this row of the block table."""
    p = np.arange(n)
    return np.asarray(row)[p // page].astype(np.int64) * page + p % page


def place(pool, page, hkv, slots, k, v):
    """Rows k, v [n][Hkv][128] into a pool (a flat f16 array)."""
    for i, s in enumerate(slots):
        if s >= 0:
            for h in range(hkv):
                ke, ve = elements(page, hkv, h, s)
                pool[ke], pool[ve] = k[i, h], v[i, h]


def attend(q, k, v, seen, f16=False, parts=2):
    """Query rows q [R][128] of one head over k, v [n][128], row i over the first
    seen[i] positions: out [R][128], a bound on each output's error.

    With u = 2^-24 and S = max_t sum_d |q_d K_td| / sqrt(128) over the row's
    positions: a score is off by at most 2^-22 S = 4 u S for q's two f16 parts, 256 u S
    for the f32 sum of the two parts' 256 products (half a step each, in any order),
    and 4 u S for its factor; its power of two by that and by 4 u, the exponent's own
    rounding by 2 u S; numerator and denominator both: twice.  The sums over n
    positions round once a product of a part at most: (parts n) u in the numerator, n u
    in the denominator, 64 u for the joins.  p' in two parts 2^-22, in one
    H16 = 2^-11 of each weight.  Weights far below the largest: p' is held to 2^-25
    (f16's smallest step is 2^-24), at least 2^6 for the largest weight (l >= 2^6), so
    n 2^-31 max|V|.  An f16 output is rounded once more, H16 and 2^-25."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    n = len(k)
    hide = np.arange(n)[None] >= np.asarray(seen)[:, None]
    s = np.where(hide, -np.inf, q @ k.T / np.sqrt(HD))
    size = np.where(hide, 0.0, np.abs(q) @ np.abs(k).T / np.sqrt(HD))
    some = np.asarray(seen) > 0
    top = np.where(some, s.max(-1, initial=-np.inf), 0.0)
    p = np.exp(s - top[:, None])
    p = np.where(some[:, None], p / np.maximum(p.sum(-1, keepdims=True), 1e-300), 0.0)
    S = size.max(-1, initial=0.0)[:, None]
    av = np.abs(v)
    floor = np.where(hide[:, :, None], 0.0, av[None]).max((1, 2), initial=0.0)[:, None] * n * 2.0 ** -31 \
        if n * len(q) < 4e6 else np.full((len(q), 1), av.max(initial=0.0) * n * 2.0 ** -31)
    rel = 2 * ((4 + 256 + 4 + 2) * U * S + 8 * U) + ((parts + 1) * n + 64) * U
    rel = rel + (4 * U if parts == 2 else H16)
    out = p @ v
    tol = rel * (p @ av) + floor + 1e-37
    if f16:
        tol = tol + H16 * np.abs(out) + tol * H16 + 2.0 ** -25
    return out, tol


def close_in_norm(got, want, q, k, n, f16=False):
    """A tighter check of all rows together: roundings fall either way, so those of a
    score's 256 products add as 16 u S, with q's split and the factors 24 u S, S as the
    mean over positions; those of the sums over n positions as sqrt(3 n) u; numerator
    and denominator: doubled.  f16: the weights' and the output's roundings are
    H16 each at most."""
    S = (np.abs(np.asarray(k, np.float64)) @ np.abs(np.asarray(q, np.float64)).T).mean() / np.sqrt(HD)
    tol = 2 * (24 * U * (S + 1) + np.sqrt(3 * n) * U) + (3 * H16 if f16 else 0.0)
    err = np.linalg.norm(np.asarray(got, np.float64) - want) / np.linalg.norm(want)
    assert err <= tol, (err, tol)


def check_rows(got, want, tol, what=""):
    """Every value within its bound; a NaN on any side is within none."""
    ok = np.abs(np.asarray(got, np.float64) - want) <= tol
    assert ok.all(), (what, int((~ok).sum()), float(np.max(np.abs(got - want) / tol)))

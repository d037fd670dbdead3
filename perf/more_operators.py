"""The operators of a server whose sequences share one pool of cache pages, as cases
that can be timed: the step's bookkeeping on the device (block tables, slot maps, the
free list), the append of new rows through the slots, the attention of one new token
per sequence over its pages, and causal attention of packed prompts.

Kinds of case:

  update   lengths and wanted growth of each sequence in, pages taken and given back,
           block tables, slots and positions of the step's tokens out
  append   K/V rows of packed tokens into the pages that the slots name
  decode   attention of one token per sequence, ragged lengths, an idle sequence
  prefill  causal attention of packed sequences of different lengths, each behind
           the tokens that it holds already

`run` computes the plain torch form, or with `own` calls the C ABI
(include/oxbitnet_ops.h).  Both take the pool in the layout that header documents.
Head counts, vocabulary and lengths: the synthetic 2B configuration (20 query / 5 KV
heads of 128, 4096 positions), and longer contexts.
"""
import importlib
import math

import torch

own = False

H, HKV, HD = 20, 5, 128
UNIT = 32                        # positions of a layout unit: 4096 K elements, then 4096 V
HEADS = [(20, 5), (20, 5), (8, 8), (32, 8), (16, 2), (15, 5), (32, 2)]
TYPES = {"f32": 0, "f16": 1}     # of q and the output; the pages are f16
TORCH = {"f32": torch.float32, "f16": torch.float16}
DEV = "cuda"


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    heads = {"H": H, "HKV": HKV}
    return [
        # the bookkeeping of each decode step of a batch, some of whose chats end
        {"name": "update_step", "kind": "update", "batch": 64, "page": 32, "longest": 4096, "grow": 1},
        # a burst of prompts, chunks of prompts and ends of chats
        {"name": "update_prompts", "kind": "update", "batch": 48, "page": 64, "longest": 16384, "grow": 4096},
        # the new rows of a decode step, per layer
        {"name": "append_step", "kind": "append", "batch": 64, "n": 1, "past": 2000, "page": 32, **heads},
        # eight prompts packed
        {"name": "append_prompts", "kind": "append", "batch": 8, "n": 4095, "past": 0, "page": 64, **heads},
        # one chat at a long context
        {"name": "decode_1", "kind": "decode", "type": "f32", "batch": 1, "longest": 2304, "page": 32, **heads},
        # a serving batch of chats of very different lengths
        {"name": "decode_64", "kind": "decode", "type": "f32", "batch": 64, "longest": 4096, "page": 32, **heads},
        # a few sequences over whole books, an odd length
        {"name": "decode_4_long", "kind": "decode", "type": "f16", "batch": 4, "longest": 100001, "page": 256, **heads},
        # a chat's first turn, of odd length
        {"name": "prefill_101", "kind": "prefill", "type": "f32", "batch": 1, "n": 101, "past": 0, "page": 32, **heads},
        # prompts of different lengths packed into one call
        {"name": "prefill_packed", "kind": "prefill", "type": "f32", "batch": 12, "n": 4096, "past": 0, "page": 64,
         **heads},
        # the same for a caller of f16 activations
        {"name": "prefill_packed_f16", "kind": "prefill", "type": "f16", "batch": 12, "n": 4096, "past": 0, "page": 64,
         **heads},
        # drafts of a few tokens verified for a batch
        {"name": "prefill_drafts", "kind": "prefill", "type": "f32", "batch": 24, "n": 5, "past": 4000, "page": 32,
         **heads},
        # a question behind a long document, beside a few short ones
        {"name": "prefill_turn", "kind": "prefill", "type": "f16", "batch": 3, "n": 333, "past": 30011, "page": 128,
         **heads},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["update", "append", "decode", "decode", "prefill", "prefill"])
    h, hkv = rng.choice(HEADS)
    c = {"kind": kind, "page": rng.choice([32, 64, 128, 256])}
    if kind == "update":
        b = _log_int(rng, 1, 256)
        return {**c, "batch": b, "longest": _log_int(rng, 32, 16384),
                "grow": rng.choice([1, _log_int(rng, 1, max(1, 100000 // b))])}
    c.update({"H": h, "HKV": hkv})
    if kind == "append":
        n = rng.choice([1, _log_int(rng, 1, 4096)])
        return {**c, "batch": max(1, min(_log_int(rng, 1, 64), 20000 // n)), "n": n,
                "past": _log_int(rng, 1, 4000) - 1}
    c["type"] = rng.choice(["f32", "f16"])
    if kind == "decode":
        b = _log_int(rng, 1, 64)
        return {**c, "batch": b, "longest": _log_int(rng, 1, min(100000, 1300000 // (b * hkv)))}
    c.update({"batch": _log_int(rng, 1, 32), "n": _log_int(rng, 1, 4096),
              "past": rng.choice([0, _log_int(rng, 1, 30000)])})
    # at most the scores of the listed packed prompts, and the positions of the listed long ones
    while _scores(c) > MOST_SCORES or sum(_lengths(c)[1]) * hkv > 1000000:
        if c["past"] > c["n"]:
            c["past"] = c["past"] * 3 // 4
        else:
            c["batch"] = max(1, c["batch"] * 3 // 4)
            c["n"] = c["n"] * 7 // 8 if c["batch"] == 1 else c["n"]
    return c


# ---------------------------------------------------------------------------
# lengths: of a batch's sequences, the first is the longest and the others spread
# down to an eighth of it; from eight sequences on the fourth is idle
# ---------------------------------------------------------------------------
def _spread(batch, top, shift=0.0):
    u = [(0.618034 * i + shift) % 1.0 if i else 0.0 for i in range(batch)]
    out = [max(1, int(round(top * 8.0 ** -x))) if top else 0 for x in u]
    if batch >= 8:
        out[3] = 0
    return out


def _pages(n, page):
    return (n + page - 1) // page


def _lengths(case):
    """Tokens of the call and cached tokens with them, of each sequence."""
    kind = case["kind"]
    if kind == "decode":
        held = _spread(case["batch"], case["longest"])
        return [1] * case["batch"], held
    if kind == "append" and case["n"] == 1:
        new = [1] * case["batch"]
    else:
        new = _spread(case["batch"], case["n"])
    past = _spread(case["batch"], case["past"], 0.37)
    return new, [p + n for p, n in zip(past, new)]


def _pairs(case):
    """(token, visible position) pairs."""
    new, held = _lengths(case)
    if case["kind"] == "decode":
        return sum(held)
    return sum(m * (n - m) + m * (m + 1) // 2 for n, m in zip(held, new))


def _scores(case):
    return _pairs(case) * case["H"]


MOST_SCORES = 600 * 10 ** 6


# ---------------------------------------------------------------------------
# the pool's layout: [page][KV head][unit of 32 positions][K 4096, V 4096]
# ---------------------------------------------------------------------------
def _k_view(pool, hkv, page):
    """[page][head][unit][dim / 8][32 positions][8 dims]"""
    return pool.view(-1, hkv, page // UNIT, 2, 4096)[:, :, :, 0].unflatten(-1, (HD // 8, UNIT, 8))


def _v_view(pool, hkv, page):
    """[page][head][unit][position / 8][128 dims][8 positions]"""
    return pool.view(-1, hkv, page // UNIT, 2, 4096)[:, :, :, 1].unflatten(-1, (UNIT // 8, HD, 8))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 6151 + 11)
    return g


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device=DEV)


def _table(g, held, page, n_pages):
    """A block table over a random order of the pages; unused entries hold no page."""
    width = max(1, max(_pages(n, page) for n in held))
    order = torch.randperm(n_pages, generator=g, device=DEV).int()
    table = torch.full((len(held), width), -1, dtype=torch.int32, device=DEV)
    at = 0
    for z, n in enumerate(held):
        m = _pages(n, page)
        table[z, :m] = order[at:at + m]
        at += m
    return table


def _pool(g, held, table, case, n_pages):
    """K rows as RoPE leaves them (some channels of a head larger than others) and V
    rows; what no sequence holds is stale: any bytes, infinities and NaN among them."""
    hkv, page = case["HKV"], case["page"]
    pool = torch.empty(n_pages, hkv * page * 2 * HD, dtype=torch.float16, device=DEV)
    pool.view(-1).copy_(torch.randint(-32768, 32768, (pool.numel(),), generator=g, device=DEV,
                                      dtype=torch.int16).view(torch.float16))
    kv, vv = _k_view(pool, hkv, page), _v_view(pool, hkv, page)
    channel = torch.exp(0.4 * _normal(g, hkv, HD // 8, 8))
    for z, n in enumerate(held):
        if not n:
            continue
        at = table[z, :_pages(n, page)].long()
        live = (torch.arange(len(at) * page, device=DEV) < n).view(len(at), 1, page // UNIT, UNIT)
        k = _normal(g, len(at), *kv.shape[1:]) * channel[None, :, None, :, None]
        kv[at] = torch.where(live[:, :, :, None, :, None], k.half(), kv[at])
        v = _normal(g, len(at), *vv.shape[1:]).half()
        vv[at] = torch.where(live.unflatten(-1, (UNIT // 8, 1, 8)), v, vv[at])
    return pool


def _inputs(case, seed):
    g, kind, page, b = _gen(seed), case["kind"], case["page"], case["batch"]
    if kind == "update":
        top, grow = case["longest"], case["grow"]
        held = _spread(b, top)
        # most grow, some wait, some take back a draft, every seventh ends
        want = [1] * b if grow == 1 else _spread(b, grow, 0.5)
        delta = [-held[z] if z % 7 == 6 else -min(5, held[z]) if z % 11 == 5 else 0 if z % 13 == 8 else want[z]
                 for z in range(b)]
        n_pages = sum(_pages(n, page) for n in held) + sum(_pages(max(d, 0), page) for d in delta) + b
        width = _pages(top + grow, page) + 1
        table = torch.full((b, width), -1, dtype=torch.int32, device=DEV)
        order = torch.randperm(n_pages, generator=g, device=DEV).int()
        at = 0
        for z, n in enumerate(held):
            m = _pages(n, page)
            table[z, :m] = order[at:at + m]
            at += m
        free = torch.full((n_pages,), -1, dtype=torch.int32, device=DEV)
        free[:n_pages - at] = order[at:]
        total = sum(max(d, 0) for d in delta)
        return {"len": _ints(held), "delta": _ints(delta), "table": table, "free": free,
                "n_free": _ints([n_pages - at]), "n_max": (total + 63) // 64 * 64}
    new, held = _lengths(case)
    n_pages = sum(_pages(n, page) for n in held) + 3
    table = _table(g, held, page, n_pages)
    i = {"new": new, "held": held, "table": table, "n_pages": n_pages, "len": _ints(held)}
    hkv, h = case["HKV"], case["H"]
    if kind == "append":
        n = sum(new)
        i["n_max"] = (n + 63) // 64 * 64
        i["k"], i["v"] = (_normal(g, i["n_max"], hkv, HD).half() for _ in "kv")
        slots, pos = [], []
        for z in range(b):
            p = torch.arange(held[z] - new[z], held[z], device=DEV)
            slots.append(table[z].long()[p // page] * page + p % page)
        i["slots"] = torch.cat([*slots, torch.full((i["n_max"] - n,), -1, device=DEV)]).int()
        # (one page more, for the plain form's rows that no slot names)
        i["pool"] = _normal(g, n_pages + 1, hkv * page * 2 * HD).half()
        return i
    i["pool"] = _pool(g, held, table, case, n_pages)
    t = TORCH[case["type"]]
    if kind == "decode":
        i["q"] = _normal(g, b, h * HD).to(t)
        return i
    n = sum(new)
    i["n_max"] = (n + 63) // 64 * 64
    i["q"] = _normal(g, i["n_max"], h * HD).to(t)
    i["cu"] = _ints([0] + torch.tensor(new).cumsum(0).tolist())
    return i


# ---------------------------------------------------------------------------
# prepare and run
# ---------------------------------------------------------------------------
def _bind(name, *args):
    """A C ABI call with its arguments as a C program holds them."""
    native = importlib.import_module("0xbitnet_amd._native")
    fn = getattr(native.lib(), name)
    args = (*args, torch.cuda.current_stream().cuda_stream)
    vals = [a.data_ptr() if isinstance(a, torch.Tensor) else a for a in args]
    return name, fn, [t(x) for t, x in zip(fn.argtypes, vals)], native


def _workspace(s, name, *args):
    n = getattr(importlib.import_module("0xbitnet_amd._native").lib(), name)(*args)
    s["ws"] = torch.zeros(max(n, 16), dtype=torch.uint8, device=DEV)
    return s["ws"], n


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    kind, page, b = case["kind"], case["page"], case["batch"]
    if kind == "update":
        n = s["n_max"]
        s["out"] = {"len": torch.zeros_like(s["len"]), "n_free": torch.zeros_like(s["n_free"]),
                    "cu": _ints([0] * (b + 1)), "granted": torch.zeros_like(s["len"]),
                    "slots": _ints([0] * max(n, 1))[:n], "pos": _ints([0] * max(n, 1))[:n],
                    "table": s["table"], "free": s["free"]}
        if own:
            o = s["out"]
            s["call"] = _bind("oxb_paged_update", page, b, s["len"], s["delta"], s["table"],
                              s["table"].shape[1], s["free"], s["free"].numel(), s["n_free"], o["len"],
                              o["n_free"], o["cu"], o["granted"], o["slots"], o["pos"], n)
    elif kind == "append":
        hkv = case["HKV"]
        s["out"] = s["pool"][:s["n_pages"]]
        if own:
            s["call"] = _bind("oxb_paged_append", s["pool"], s["n_pages"], page, hkv, HD, s["k"], s["v"],
                              hkv * HD, HD, None, s["slots"], s["n_max"])
    else:
        h, hkv, t = case["H"], case["HKV"], TYPES[case["type"]]
        s["out"] = torch.zeros_like(s["q"])
        head = (s["q"], t, s["pool"], s["n_pages"], page, s["table"], s["table"].shape[1])
        if own and kind == "decode":
            ws = _workspace(s, "oxb_attn_decode_paged_ws_bytes", b, h, hkv, HD)
            s["call"] = _bind("oxb_attn_decode_paged", *head, s["len"], b, h, hkv, HD, s["out"], *ws)
        elif own:
            ws = _workspace(s, "oxb_attn_prefill_paged_ws_bytes", s["n_max"], b, h, hkv, HD)
            s["call"] = _bind("oxb_attn_prefill_paged", *head, s["cu"], s["len"], s["n_max"], b, h, hkv, HD,
                              s["out"], *ws)
    torch.cuda.synchronize()
    return s


def run(s):
    if own:
        name, fn, vals, native = s["call"]
        if fn(*vals):
            raise native.NativeError(f"{name}: {native.last_error()}")
        return s["out"]
    return {"update": _plain_update, "append": _plain_append, "decode": _plain_decode,
            "prefill": _plain_prefill}[s["case"]["kind"]](s, s["case"])


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _plain_update(s, case):
    page, o, table, free = case["page"], s["out"], s["table"], s["free"]
    b, width = table.shape
    n_max, cap = s["n_max"], free.numel()
    held = s["len"].long().clamp(0, width * page)
    delta, n_free = s["delta"].long(), s["n_free"].long()
    pages = lambda n: torch.div(n + page - 1, page, rounding_mode="floor")  # noqa: E731
    end = delta.clamp(min=0).cumsum(0)
    fits = (delta > 0) & (held + delta <= width * page) & (end <= n_max)
    short = torch.where(delta < 0, (held + delta).clamp(min=0), held)
    # pages given back, in the sequences' order
    blk = torch.arange(width, device=DEV)
    gone = (blk >= pages(short)[:, None]) & (blk < pages(held)[:, None])
    given = gone.sum()
    at = torch.where(gone.view(-1), gone.view(-1).cumsum(0) - 1, b * width)
    back = torch.zeros(b * width + 1, dtype=torch.int32, device=DEV).scatter_(0, at, table.reshape(-1))
    # pages taken: those given back first, the last first, then the list from its end
    need = torch.where(fits, pages(held + delta) - pages(held), 0)
    upto = need.cumsum(0)
    granted = fits & ((need == 0) | (upto <= n_free + given))
    taken = torch.where(granted, need, 0).sum()
    rank = torch.arange(b * width, device=DEV)
    took = torch.where(rank < given, back[(given - 1 - rank).clamp(min=0)],
                       free[(n_free - 1 - (rank - given)).clamp(0, cap - 1)])
    first = pages(held)[:, None]
    mine = granted[:, None] & (blk >= first) & (blk < first + need[:, None])
    r = ((upto - need)[:, None] + blk - first).clamp(0, b * width - 1)
    table.copy_(torch.where(mine, took[r], table))
    left = torch.arange(cap, device=DEV)
    free.copy_(torch.where((left >= n_free) & (left < n_free + given - taken),
                           back[(left - n_free).clamp(0, b * width - 1)], free))
    o["n_free"].copy_(n_free + given - taken)
    o["granted"].copy_(torch.where(granted, delta, 0))
    o["len"].copy_(torch.where(granted, held + delta, short))
    o["cu"][1:].copy_(end.clamp(max=n_max))
    t = torch.arange(n_max, device=DEV)
    z = torch.searchsorted(end, t, right=True)
    live = z < b
    z = z.clamp(max=b - 1)
    p = held[z] + t - (end - delta.clamp(min=0))[z]
    live = live & granted[z]
    p = torch.where(live, p, 0)
    at = table[z, torch.div(p, page, rounding_mode="floor")].long() * page + p % page
    o["slots"].copy_(torch.where(live, at, -1))
    o["pos"].copy_(torch.where(live, p, -1))
    return o


def _plain_append(s, case):
    page, hkv, n = case["page"], case["HKV"], s["n_max"]
    slot = s["slots"].long()
    slot = torch.where(slot >= 0, slot, s["n_pages"] * page)
    p, at = torch.div(slot, page, rounding_mode="floor"), slot % page
    unit, at = torch.div(at, UNIT, rounding_mode="floor"), at % UNIT
    _k_view(s["pool"], hkv, page)[p, :, unit, :, at] = s["k"].view(n, hkv, HD // 8, 8)
    _v_view(s["pool"], hkv, page)[p, :, unit, torch.div(at, 8, rounding_mode="floor"), :, at % 8] = s["v"]
    return s["out"]


def _rows(s, case, z):
    """Sequence z's K and V as f32 [Hkv][positions][128]."""
    hkv, page, n = case["HKV"], case["page"], s["held"][z]
    at = s["table"][z, :_pages(n, page)].long()
    k = _k_view(s["pool"], hkv, page)[at].permute(1, 0, 2, 4, 3, 5).reshape(hkv, -1, HD)
    v = _v_view(s["pool"], hkv, page)[at].permute(1, 0, 2, 3, 5, 4).reshape(hkv, -1, HD)
    return k[:, :n].float(), v[:, :n].float()


def _attend(s, case, z, q):
    """Rows q of sequence z, its newest tokens, over its positions."""
    h, hkv = case["H"], case["HKV"]
    k, v = _rows(s, case, z)
    n, held = q.shape[0], k.shape[1]
    q = q.float().view(n, hkv, h // hkv, HD).transpose(0, 1).reshape(hkv, -1, HD)
    x = torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.sqrt(HD)
    if n > 1:
        last = torch.arange(held - n, held, device=DEV).repeat_interleave(h // hkv)
        x = x.masked_fill(torch.arange(held, device=DEV)[None] > last[:, None], -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    o = torch.matmul(p / p.sum(-1, keepdim=True), v)
    return o.view(hkv, n, h // hkv, HD).transpose(0, 1).reshape(n, h * HD)


def _plain_decode(s, case):
    for z, n in enumerate(s["held"]):
        if n:
            s["out"][z:z + 1] = _attend(s, case, z, s["q"][z:z + 1])
        else:
            s["out"][z].zero_()
    return s["out"]


def _plain_prefill(s, case):
    at = 0
    for z, n in enumerate(s["new"]):
        if n:
            s["out"][at:at + n] = _attend(s, case, z, s["q"][at:at + n])
        at += n
    return s["out"]


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    kind, page = case["kind"], case["page"]
    if kind == "update":
        b, grow = case["batch"], case["grow"]
        total = sum([1] * b if grow == 1 else _spread(b, grow, 0.5))
        # a word in and three out a sequence, a slot and a position a token, a page's entry in and out
        return {"bytes": 4.0 * (6 * b + 2 * total + 2 * (total // page + b)), "flops": 4.0 * (b + total)}
    new, held = _lengths(case)
    hkv = case["HKV"]
    if kind == "append":
        return {"bytes": sum(new) * (hkv * HD * 2.0 * 4 + 4), "flops": 1.0 * sum(new) * hkv * HD}
    h, size = case["H"], 2.0 if case["type"] == "f16" else 4.0
    held = [n if m else 0 for n, m in zip(held, new)]
    return {"bytes": sum(held) * hkv * HD * 4.0 + sum(_pages(n, page) for n in held) * 4.0 +
            2 * size * sum(new) * h * HD, "flops": 4.0 * _scores(case) * HD}


# ---------------------------------------------------------------------------
# the same results in 64 bits
# ---------------------------------------------------------------------------
def _element(i, case, z, which, positions):
    """K (0) or V (1) rows of sequence z at the given positions, element by element
    from the layout's offsets: [positions][Hkv][128]."""
    hkv, page = case["HKV"], case["page"]
    t = torch.as_tensor(positions, device=DEV).view(-1, 1, 1)
    head = torch.arange(hkv, device=DEV).view(1, -1, 1)
    d = torch.arange(HD, device=DEV).view(1, 1, -1)
    base = (i["table"][z].long()[t // page] * hkv + head) * page * 2 * HD + (t % page) // UNIT * (2 * UNIT * HD)
    t = t % UNIT
    inside = (d // 8 * UNIT + t) * 8 + d % 8 if which == 0 else UNIT * HD + (t // 8 * HD + d) * 8 + t % 8
    return i["pool"].view(-1)[base + inside].double()


def exact(case, seed):
    kind = case["kind"]
    if kind == "update":
        return None
    i = _inputs(case, seed)
    h, hkv = case["H"], case["HKV"]
    if kind == "append":
        flat, page = i["pool"].double().view(-1), case["page"]
        n = sum(i["new"])
        t, d = i["slots"][:n].long().view(-1, 1, 1), torch.arange(HD, device=DEV).view(1, 1, -1)
        head = torch.arange(hkv, device=DEV).view(1, -1, 1)
        base = (t // page * hkv + head) * page * 2 * HD + (t % page) // UNIT * (2 * UNIT * HD)
        t = t % UNIT
        flat[base + (d // 8 * UNIT + t) * 8 + d % 8] = i["k"][:n].double()
        flat[base + UNIT * HD + (t // 8 * HD + d) * 8 + t % 8] = i["v"][:n].double()
        return flat.view(i["pool"].shape)[:i["n_pages"]]
    out, at = torch.zeros(i["q"].shape, dtype=torch.float64, device=DEV), 0
    for z, (n, held) in enumerate(zip(i["new"], i["held"])):
        if held and n:
            k, v = (_element(i, case, z, w, range(held)) for w in (0, 1))
            q = i["q"][at:at + n].double().view(n, h, HD)
            first = held - n
            for j in range(h):
                kv = j // (h // hkv)
                x = (q[:, j] @ k[:, kv].t().contiguous()) / math.sqrt(HD)
                late = torch.arange(held, device=DEV)[None] > first + torch.arange(n, device=DEV)[:, None]
                o = torch.softmax(x.masked_fill_(late, -math.inf), -1) @ v[:, kv].contiguous()
                out[at:at + n, j * HD:(j + 1) * HD] = o
        at += n
    return out

"""The operators of a long-running serving batch, as cases that can be timed: the
8-bit KV cache with the attention that reads it, eviction from that cache by
accumulated attention weight, and the rules on each sequence's logits.

Kinds of case:

  append   new K/V rows into the 8-bit cache of a batch (one row as in a decode
           step, more as in a prompt), then the touched blocks read back
  decode   attention of one decode step over the cache, ragged lengths, with or
           without accumulating each block's attention weight
  prefill  causal attention of n prompt tokens behind pos0 cached ones
  evict    the cache cut to a budget of blocks into another cache, read back
  rules    penalties, biases and a grammar mask on a batch's logits

`run` computes the plain torch form, or with `own` calls the C ABI
(include/oxbitnet_ops.h).  Both take the cache in the layout that header
documents; the plain form takes its values out of the bytes within the pass.
Head counts, vocabulary and lengths: the synthetic 2B configuration (20 query /
5 KV heads of 128, vocabulary 128256, 4096 positions), and longer caches.
"""
import importlib
import math

import torch

own = False

H, HKV, HD, V = 20, 5, 128, 128256
BLOCK = 32                       # positions of a block: one K and one V scale per head
FMT = {"int8": 0, "e4m3": 1}
TOP = {"int8": 127.0, "e4m3": 448.0}
HEADS = [(20, 5), (20, 5), (8, 8), (32, 8), (16, 2), (15, 5), (32, 2)]
DEV = "cuda"


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # each decode step of one chat, per layer: one row, its block quantized again
        {"name": "append_1", "kind": "append", "fmt": "int8", "batch": 1, "n": 1, "past": 1000,
         "H": H, "HKV": HKV},
        # four prompts of different lengths entering the cache
        {"name": "append_prompts", "kind": "append", "fmt": "e4m3", "batch": 4, "n": 2048,
         "past": 0, "H": H, "HKV": HKV},
        # one chat at long context
        {"name": "decode_1", "kind": "decode", "fmt": "int8", "batch": 1, "longest": 2304,
         "weights": False, "H": H, "HKV": HKV},
        # a serving batch of chats of different lengths that will be cut to a budget
        {"name": "decode_32_weights", "kind": "decode", "fmt": "int8", "batch": 32,
         "longest": 2304, "weights": True, "H": H, "HKV": HKV},
        # a few sequences over whole books, an odd length
        {"name": "decode_4_long", "kind": "decode", "fmt": "e4m3", "batch": 4, "longest": 100001,
         "weights": False, "H": H, "HKV": HKV},
        # a chat's first turn, of odd length
        {"name": "prefill_101", "kind": "prefill", "fmt": "int8", "n": 101, "pos0": 0,
         "weights": False, "H": H, "HKV": HKV},
        # a long document
        {"name": "prefill_2048", "kind": "prefill", "fmt": "int8", "n": 2048, "pos0": 0,
         "weights": False, "H": H, "HKV": HKV},
        # a question behind a long context, its weights kept for eviction
        {"name": "prefill_turn_weights", "kind": "prefill", "fmt": "e4m3", "n": 333,
         "pos0": 20011, "weights": True, "H": H, "HKV": HKV},
        # a full cache of one chat cut to half
        {"name": "evict_1", "kind": "evict", "fmt": "int8", "batch": 1, "longest": 4096,
         "budget": 64, "H": H, "HKV": HKV},
        # a batch at once, ragged
        {"name": "evict_32", "kind": "evict", "fmt": "int8", "batch": 32, "longest": 2304,
         "budget": 32, "H": H, "HKV": HKV},
        # the next token of one chat: the default window of 64 tokens
        {"name": "rules_1", "kind": "rules", "rows": 1, "V": V, "history": 64, "bias": 16},
        # a batch with long histories, each row with a mask of its own
        {"name": "rules_32", "kind": "rules", "rows": 32, "V": V, "history": 4096, "bias": 300},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "decode", "decode", "prefill", "prefill", "evict", "rules"])
    h, hkv = rng.choice(HEADS)
    c = {"kind": kind, "fmt": rng.choice(["int8", "e4m3"]), "H": h, "HKV": hkv}
    if kind == "append":
        n = rng.choice([1, _log_int(rng, 1, 2048)])
        b = _log_int(rng, 1, 32)
        return {**c, "batch": max(1, min(b, 16384 // n)), "n": n, "past": _log_int(rng, 1, 4000) - 1}
    if kind == "decode":
        b = _log_int(rng, 1, 64)
        top = _log_int(rng, 1, min(100000, 1600000 // (b * hkv)))
        return {**c, "batch": b, "longest": top, "weights": rng.random() < 0.5}
    if kind == "prefill":
        n = _log_int(rng, 1, 2048)
        pos0 = rng.choice([0, _log_int(rng, 1, 20000)])
        # at most the keys of the listed turn over all heads
        pos0 = max(0, min(pos0, 130000000 // (n * h) - n))
        return {**c, "n": n, "pos0": pos0, "weights": rng.random() < 0.3}
    if kind == "evict":
        b = _log_int(rng, 1, 32)
        top = _log_int(rng, 40, min(32768, 370000 // (b * hkv)))
        return {**c, "batch": b, "longest": top, "budget": _log_int(rng, 4, max(5, top // 32))}
    return {"kind": kind, "rows": _log_int(rng, 1, 32), "V": rng.choice([V, 32003, 50257]),
            "history": _log_int(rng, 1, 4096), "bias": _log_int(rng, 1, 300)}


# ---------------------------------------------------------------------------
# the cache's layout (one sequence: codes, scales, weights, tails, each part
# 256-byte aligned)
# ---------------------------------------------------------------------------
def _blocks(n):
    return (n + BLOCK - 1) // BLOCK


def _parts(hkv, max_seq):
    """Byte offsets of scales, weights and tails, and the bytes of one sequence."""
    nb, at = _blocks(max_seq), lambda b: (b + 255) // 256 * 256
    scales = at(hkv * nb * 2 * BLOCK * HD)
    weights = scales + at(hkv * nb * 8)
    tails = weights + at(hkv * nb * 4)
    return scales, weights, tails, tails + at(hkv * 2 * BLOCK * HD * 2)


def _token_order():
    """The token that byte p of a V row (one dim, 32 positions) holds."""
    p = torch.arange(BLOCK, device=DEV)
    return 16 * (p // 8 % 2) + 8 * (p // 4 % 2) + 4 * (p // 16) + p % 4


def _byte_order():
    """The byte of a V row that holds token t."""
    return torch.argsort(_token_order())


def _views(cache, hkv, max_seq):
    """K codes [B][Hkv][nb][32][128], V codes [B][Hkv][nb][128][32], scales
    [B][Hkv][nb][2], weights [B][Hkv][nb], tails [B][Hkv][2][32][128] of a cache."""
    b, nb = cache.shape[0], _blocks(max_seq)
    scales, weights, tails, _ = _parts(hkv, max_seq)
    codes = cache[:, :hkv * nb * 8192].view(b, hkv, nb, 2, 4096)
    return (codes[:, :, :, 0].view(b, hkv, nb, BLOCK, HD), codes[:, :, :, 1].view(b, hkv, nb, HD, BLOCK),
            cache[:, scales:scales + hkv * nb * 8].view(torch.float32).view(b, hkv, nb, 2),
            cache[:, weights:weights + hkv * nb * 4].view(torch.float32).view(b, hkv, nb),
            cache[:, tails:tails + hkv * 16384].view(torch.float16).view(b, hkv, 2, BLOCK, HD))


def _to_bytes(codes, fmt):
    """int8 codes are held as code + 128, e4m3 codes as they are."""
    if fmt == "int8":
        return (codes + 128.0).to(torch.uint8)
    return codes.to(torch.float8_e4m3fn).view(torch.uint8)


def _from_bytes(b, fmt):
    return b.float() - 128.0 if fmt == "int8" else b.view(torch.float8_e4m3fn).float()


def _quantize(x, fmt):
    """Blocks [..., 32, 128]: codes and f32 scales."""
    a = x.float().abs().amax((-1, -2), keepdim=True)
    r = x.float() * TOP[fmt] / torch.where(a > 0, a, 1.0)
    codes = torch.round(r) if fmt == "int8" else r.to(torch.float8_e4m3fn).float()
    # (a tensor: a division by a number would be a product with its rounded reciprocal)
    return codes, a / torch.full_like(a, TOP[fmt])


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 7919 + 29)
    return g


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device=DEV)


def _uniform(g, *shape):
    return torch.rand(shape, generator=g, device=DEV)


def _lengths(batch, top, seed):
    """The longest, the others down to a half of it."""
    g = torch.Generator()
    g.manual_seed(int(seed))
    r = torch.randint((top + 1) // 2, top + 1, (batch,), generator=g)
    r[0] = top
    return r.tolist()


def _keys(g, b, hkv, n):
    """K rows as RoPE leaves them: some channels of a head larger than others."""
    return (_normal(g, b, hkv, n, HD) * torch.exp(0.4 * _normal(g, b, hkv, 1, HD))).half()


def _cache(g, b, hkv, max_seq, lengths, fmt):
    """A cache holding `lengths` positions, stale bytes behind them."""
    nb = _blocks(max_seq)
    cache = torch.randint(0, 256, (b, _parts(hkv, max_seq)[3]), generator=g, device=DEV, dtype=torch.uint8)
    kc, vc, sc, w, tail = _views(cache, hkv, max_seq)
    sc.copy_(0.01 * _uniform(g, b, hkv, nb, 2))
    w.copy_(_uniform(g, b, hkv, nb) ** 8)     # few blocks carry most of the weight
    order = _token_order()
    for z, n in enumerate(lengths):
        m = _blocks(n)
        k, v = _keys(g, 1, hkv, m * BLOCK)[0], _normal(g, hkv, m * BLOCK, HD).half()
        k[:, n:], v[:, n:] = 0, 0
        k, v = k.view(hkv, m, BLOCK, HD), v.view(hkv, m, BLOCK, HD)
        (ck, sk), (cv, sv) = _quantize(k, fmt), _quantize(v, fmt)
        kc[z, :, :m] = _to_bytes(ck, fmt)
        vc[z, :, :m] = _to_bytes(cv, fmt)[:, :, order].transpose(-1, -2)
        sc[z, :, :m, 0], sc[z, :, :m, 1] = sk[..., 0, 0], sv[..., 0, 0]
        if n % BLOCK:
            tail[z, :, 0, :n % BLOCK], tail[z, :, 1, :n % BLOCK] = k[:, -1, :n % BLOCK], v[:, -1, :n % BLOCK]
    return cache


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _inputs(case, seed):
    g, kind = _gen(seed), case["kind"]
    if kind == "append":
        b, n, hkv, past = case["batch"], case["n"], case["HKV"], case["past"]
        pos = _lengths(b, past, seed)
        counts = _lengths(b, n, int(seed) + 1)
        max_seq = _blocks(past + n) * BLOCK
        return {"cache": _cache(g, b, hkv, max_seq, pos, case["fmt"]), "max_seq": max_seq,
                "k": _keys(g, b, hkv, n), "v": _normal(g, b, hkv, n, HD).half(), "pos": _ints(pos),
                "counts": _ints(counts), "start": _ints([p // BLOCK * BLOCK for p in pos]),
                "len": _ints([p + c for p, c in zip(pos, counts)]),
                "rows": _blocks(n + BLOCK - 1) * BLOCK}
    if kind == "decode":
        b, top, hkv = case["batch"], case["longest"], case["HKV"]
        lengths = _lengths(b, top, seed)
        return {"cache": _cache(g, b, hkv, top, lengths, case["fmt"]), "max_seq": top,
                "q": _normal(g, b, case["H"], HD), "pos": _ints([n - 1 for n in lengths])}
    if kind == "prefill":
        n, pos0, hkv = case["n"], case["pos0"], case["HKV"]
        return {"cache": _cache(g, 1, hkv, pos0 + n, [pos0 + n], case["fmt"]), "max_seq": pos0 + n,
                "q": _normal(g, n, case["H"], HD)}
    if kind == "evict":
        b, top, hkv = case["batch"], case["longest"], case["HKV"]
        lengths = _lengths(b, top, seed)
        return {"cache": _cache(g, b, hkv, top, lengths, case["fmt"]), "max_seq": top,
                "len": _ints(lengths)}
    rows, v = case["rows"], case["V"]
    hist, bias = _lengths(rows, case["history"], seed), _lengths(rows, case["bias"], int(seed) + 1)
    off = lambda n: _ints([0] + torch.tensor(n).cumsum(0).tolist())  # noqa: E731
    # a text repeats its tokens: ids drawn towards the low end; some biases forbid
    ids = lambda n: (v * _uniform(g, n) ** 4).int().clamp(max=v - 1)  # noqa: E731
    nb = sum(bias)
    value = torch.where(_uniform(g, nb) < 0.1, -math.inf, 4 * _normal(g, nb))
    pen = torch.stack([1.0 + 0.3 * _uniform(g, rows), 0.5 * _uniform(g, rows), 0.5 * _uniform(g, rows)], 1)
    words = (v + 31) // 32
    mask = torch.randint(-2 ** 31, 2 ** 31, (rows, words), generator=g, device=DEV, dtype=torch.int32)
    return {"logits": 4 * _normal(g, rows, v), "hist": ids(sum(hist)), "hist_off": off(hist),
            "bias_ids": ids(nb), "bias": value, "bias_off": off(bias), "pen": pen.contiguous(),
            "mask": mask, "n_hist": sum(hist), "n_bias": nb, "words": words}


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


def _lib():
    return importlib.import_module("0xbitnet_amd._native").lib()


def prepare(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    s["case"] = case
    if kind == "rules":
        s["out"] = torch.empty_like(s["logits"])
        if own:
            s["calls"] = [_bind("oxb_logits_rules", s["logits"], case["V"], case["rows"], case["V"],
                                s["pen"], s["hist"], s["hist_off"], s["n_hist"], s["bias_ids"],
                                s["bias"], s["bias_off"], s["n_bias"], s["mask"], s["words"],
                                s["out"], case["V"])]
        torch.cuda.synchronize()
        return s
    h, hkv, ms, fmt = case["H"], case["HKV"], s["max_seq"], FMT[case["fmt"]]
    c, stride = s["cache"], s["cache"].shape[1]
    b = c.shape[0]
    if kind == "append":
        n, rows = case["n"], s["rows"]
        s["out"] = {x: torch.empty(b, hkv, rows, HD, device=DEV) for x in "kv"}
        if own:
            s["calls"] = [_bind("oxb_kv8_append", c, stride, fmt, b, hkv, HD, ms, s["k"], s["v"],
                                hkv * n * HD, n * HD, 0, s["pos"], 1, 0, n, s["counts"]),
                          _bind("oxb_kv8_read", c, stride, fmt, b, hkv, HD, ms, s["start"], 1, 0, rows,
                                s["len"], 1, s["out"]["k"], s["out"]["v"])]
            # an append that leaves the block it began in leaves another tail: a pass
            # that appends at the same place again brings the first one back
            off = s["pos"] - s["start"]
            if ((off > 0) & (off + s["counts"] > BLOCK)).any():
                tail = _views(c, hkv, ms)[4]
                s["tail"] = (tail, tail.clone())
    elif kind == "decode":
        s["out"] = {"out": torch.empty(b, h * HD, device=DEV)}
        if own:
            n = _lib().oxb_attn_decode_kv8_ws_bytes(b, h, hkv, HD, ms)
            s["ws"] = torch.zeros(max(n, 16), dtype=torch.uint8, device=DEV)
            s["calls"] = [_bind("oxb_attn_decode_kv8", s["q"], c, stride, fmt, s["pos"], 1, b, h, hkv,
                                HD, ms, int(case["weights"]), s["out"]["out"], s["ws"], n)]
    elif kind == "prefill":
        n, pos0 = case["n"], case["pos0"]
        s["out"] = {"out": torch.empty(n, h * HD, device=DEV)}
        if own:
            wsb = _lib().oxb_attn_prefill_kv8_ws_bytes(n, pos0, h, hkv, HD, int(case["weights"]))
            s["ws"] = torch.zeros(max(wsb, 16), dtype=torch.uint8, device=DEV)
            s["calls"] = [_bind("oxb_attn_prefill_kv8", s["q"], c, fmt, n, pos0, h, hkv, HD, ms,
                                int(case["weights"]), s["out"]["out"], s["ws"], wsb)]
    else:
        # the budget holds the first block and the two newest ones whatever their weight
        m = case["budget"]
        s["dst"] = torch.zeros(b, _parts(hkv, m * BLOCK)[3], dtype=torch.uint8, device=DEV)
        s["out"] = {"k": torch.empty(b, hkv, m * BLOCK, HD, device=DEV),
                    "v": torch.empty(b, hkv, m * BLOCK, HD, device=DEV),
                    "weights": _views(s["dst"], hkv, m * BLOCK)[3], "len": torch.zeros_like(s["len"])}
        if own:
            n = _lib().oxb_kv8_evict_ws_bytes(b, hkv, ms, m)
            s["ws"] = torch.zeros(max(n, 16), dtype=torch.uint8, device=DEV)
            s["calls"] = [_bind("oxb_kv8_evict", c, stride, ms, s["dst"], s["dst"].shape[1], m * BLOCK,
                                s["len"], 1, s["out"]["len"], 1, b, hkv, HD, m, 1, 2, s["ws"], n),
                          _bind("oxb_kv8_read", s["dst"], s["dst"].shape[1], fmt, b, hkv, HD, m * BLOCK,
                                None, 0, 0, m * BLOCK, s["out"]["len"], 1, s["out"]["k"],
                                s["out"]["v"])]
    if kind in ("decode", "prefill") and case["weights"]:
        s["out"]["weights"] = _views(c, hkv, ms)[3]
    torch.cuda.synchronize()
    return s


def run(s):
    if own:
        if "tail" in s:
            s["tail"][0].copy_(s["tail"][1])
        for name, fn, vals, native in s["calls"]:
            if fn(*vals):
                raise native.NativeError(f"{name}: {native.last_error()}")
        return s["out"]
    return {"append": _plain_append, "decode": _plain_decode, "prefill": _plain_prefill,
            "evict": _plain_evict, "rules": _plain_rules}[s["case"]["kind"]](s, s["case"])


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _values(cache, hkv, max_seq, fmt):
    """K and V of every block, f32 [B][Hkv][nb * 32][128]."""
    kc, vc, sc, _, _ = _views(cache, hkv, max_seq)
    b, nb = cache.shape[0], sc.shape[2]
    k = _from_bytes(kc.contiguous(), fmt) * sc[..., 0, None, None]
    v = _from_bytes(vc.contiguous(), fmt)[..., _byte_order()].transpose(-1, -2) * sc[..., 1, None, None]
    return k.view(b, hkv, nb * BLOCK, HD), v.reshape(b, hkv, nb * BLOCK, HD)


def _plain_append(s, case):
    b, hkv, n, rows, fmt = case["batch"], case["HKV"], case["n"], s["rows"], case["fmt"]
    tail = _views(s["cache"], hkv, s["max_seq"])[4]
    r = torch.arange(rows, device=DEV)
    off = (s["pos"] - s["start"])[:, None]
    old, new = r < off, (r >= off) & (r - off < s["counts"][:, None])
    at = (r - off).clamp(0, n - 1).long()[:, None, :, None].expand(b, hkv, rows, HD)
    out = {}
    for i, name in enumerate("kv"):
        x = torch.where(new[:, None, :, None], s[name].gather(2, at), 0.0).float()
        x[:, :, :BLOCK] += torch.where(old[:, None, :BLOCK, None], tail[:, :, i], 0.0).float()
        codes, scale = _quantize(x.view(b, hkv, rows // BLOCK, BLOCK, HD), fmt)
        out[name] = (codes * scale).view(b, hkv, rows, HD)
    return out


def _softmax(scores, hide):
    scores = scores.masked_fill(hide, -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    return p / p.sum(-1, keepdim=True)


def _add_weights(cache, hkv, max_seq, p):
    """p summed over queries and heads [B][Hkv][S] into each block's weight."""
    w = _views(cache, hkv, max_seq)[3]
    w += p.view(*w.shape, BLOCK).sum(-1)
    return w


def _plain_decode(s, case):
    b, h, hkv, ms = case["batch"], case["H"], case["HKV"], s["max_seq"]
    k, v = _values(s["cache"], hkv, ms, case["fmt"])
    hide = torch.arange(k.shape[2], device=DEV)[None] > s["pos"][:, None]
    # stale positions: their bytes may stand for anything
    k, v = (torch.where(hide[:, None, :, None], 0.0, x) for x in (k, v))
    q = s["q"].view(b, hkv, h // hkv, HD)
    p = _softmax(torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.sqrt(HD), hide[:, None, None])
    out = {"out": torch.matmul(p, v).view(b, h * HD)}
    if case["weights"]:
        out["weights"] = _add_weights(s["cache"], hkv, ms, p.sum(2))
    return out


def _plain_prefill(s, case):
    n, pos0, h, hkv, ms = case["n"], case["pos0"], case["H"], case["HKV"], s["max_seq"]
    k, v = _values(s["cache"], hkv, ms, case["fmt"])
    at = torch.arange(k.shape[2], device=DEV)
    v = torch.where(at[:, None] < ms, v[0], 0.0)
    k = torch.where(at[:, None] < ms, k[0], 0.0)
    q = s["q"].view(n, hkv, h // hkv, HD).permute(1, 2, 0, 3).reshape(hkv, -1, HD)
    hide = at[None] > torch.arange(pos0, pos0 + n, device=DEV).repeat(h // hkv)[:, None]
    p = _softmax(torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.sqrt(HD), hide)
    out = torch.matmul(p, v).view(hkv, h // hkv, n, HD).permute(2, 0, 1, 3).reshape(n, h * HD)
    out = {"out": out}
    if case["weights"]:
        out["weights"] = _add_weights(s["cache"], hkv, ms, p.sum(1)[None])
    return out


def _kept(w, nblk, budget):
    """[B][Hkv][budget] indices of the kept blocks in order (nb past the last one)."""
    nb = w.shape[-1]
    at = torch.arange(nb, device=DEV)
    nblk = nblk[:, None, None]
    must = ((at < 1) | (at >= nblk - 2)) & (at < nblk)
    key = torch.where(must, math.inf, torch.where(at < nblk, w, -math.inf))
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    m = min(budget, nb)
    kept = torch.full((*w.shape[:2], budget), nb, device=DEV)
    kept[..., :m] = order[..., :m]
    short = torch.arange(budget, device=DEV) >= torch.clamp(nblk, max=budget)
    return torch.where(short, nb, kept).sort(-1).values


def _plain_evict(s, case):
    b, hkv, ms, m, fmt = case["batch"], case["HKV"], s["max_seq"], case["budget"], case["fmt"]
    kc, vc, sc, w, _ = _views(s["cache"], hkv, ms)
    nblk = torch.div(s["len"] + BLOCK - 1, BLOCK, rounding_mode="floor")
    new = s["len"] - BLOCK * torch.clamp(nblk - m, min=0).to(torch.int32)
    kept = _kept(w, nblk, m)
    there = kept < w.shape[-1]
    at = kept.clamp(max=w.shape[-1] - 1)
    take = lambda x: x.gather(2, at.view(*at.shape, *[1] * (x.dim() - 3)).expand(*at.shape, *x.shape[3:]))  # noqa: E731
    scale = take(sc)
    live = (torch.arange(m * BLOCK, device=DEV) < new[:, None])[:, None, :, None]
    k = _from_bytes(take(kc), fmt) * scale[..., 0, None, None]
    v = _from_bytes(take(vc), fmt)[..., _byte_order()].transpose(-1, -2) * scale[..., 1, None, None]
    return {"k": torch.where(live, k.view(b, hkv, m * BLOCK, HD), 0.0),
            "v": torch.where(live, v.reshape(b, hkv, m * BLOCK, HD), 0.0),
            "weights": torch.where(there, take(w), 0.0), "len": new}


def _rows_of(off, n):
    return torch.repeat_interleave(torch.arange(off.numel() - 1, device=DEV), (off[1:] - off[:-1]).long(),
                                   output_size=n)


def _plain_rules(s, case):
    rows, v = case["rows"], case["V"]
    x = s["logits"]
    flat = torch.zeros(rows * v, dtype=torch.int32, device=DEV)
    at = _rows_of(s["hist_off"], s["n_hist"]) * v + s["hist"].long()
    count = flat.scatter_add(0, at, torch.ones_like(at, dtype=torch.int32)).view(rows, v).float()
    r, f, p = (c[:, None] for c in s["pen"].unbind(1))
    x = torch.where(count > 0, torch.where(x > 0, x / r, x * r) - (f * count + p), x)
    at = _rows_of(s["bias_off"], s["n_bias"]) * v + s["bias_ids"].long()
    last = torch.full((rows * v,), -1, device=DEV).scatter_reduce(
        0, at, torch.arange(s["n_bias"], device=DEV), "amax").view(rows, v)
    x = x + torch.where(last >= 0, s["bias"][last.clamp(min=0)], 0.0)
    bit = torch.arange(v, device=DEV)
    allowed = (s["mask"][:, bit // 32] >> (bit % 32).int()) & 1
    return torch.where(allowed > 0, x, -math.inf)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "rules":
        rows, v = case["rows"], case["V"]
        return {"bytes": rows * (8.0 * v + v / 8 + 0.75 * (4 * case["history"] + 8 * case["bias"])),
                "flops": 4.0 * rows * v}
    h, hkv = case["H"], case["HKV"]
    # a batch's lengths are three quarters of the longest in the mean
    mean = lambda b, top: top + (b - 1) * 0.75 * top  # noqa: E731
    if kind == "append":
        # rows in, codes out, and the values of the returned rows
        rows = mean(case["batch"], case["n"])
        back = case["batch"] * _blocks(case["n"] + BLOCK - 1) * BLOCK
        return {"bytes": hkv * HD * 2.0 * (rows * 2 + rows + back * 4), "flops": 4.0 * rows * hkv * HD}
    if kind == "decode":
        n = mean(case["batch"], case["longest"])
        return {"bytes": n * hkv * (2.0 * HD + 8 / BLOCK) + 8.0 * case["batch"] * h * HD +
                (8.0 * n * hkv / BLOCK if case["weights"] else 0), "flops": 4.0 * n * h * HD}
    if kind == "prefill":
        n, p = case["n"], case["pos0"]
        pairs = n * p + n * (n + 1) // 2
        return {"bytes": (p + n) * hkv * (2.0 * HD + 8 / BLOCK) + 8.0 * n * h * HD,
                "flops": 4.0 * pairs * h * HD}
    n = min(mean(case["batch"], case["longest"]), case["batch"] * case["budget"] * BLOCK)
    back = case["batch"] * case["budget"] * BLOCK
    return {"bytes": hkv * (n * 2.0 * HD * 2 + back * HD * 8.0 + mean(case["batch"], case["longest"]) / 8),
            "flops": 2.0 * n * hkv * HD}


# ---------------------------------------------------------------------------
# the same results in 64 bits
# ---------------------------------------------------------------------------
def _power(e):
    """2 to whole exponents, from a table (the device's power function rounds)."""
    table = torch.tensor([2.0 ** k for k in range(-32, 33)], dtype=torch.float64, device=DEV)
    return table[e.long() + 32]


def _held64(i, case):
    """K and V that the cache's bytes stand for, [B][Hkv][positions][128]."""
    fmt, hkv, nb = case["fmt"], case["HKV"], _blocks(i["max_seq"])
    c, b = i["cache"], i["cache"].shape[0]
    raw = c[:, :hkv * nb * 8192].reshape(b, hkv, nb, 2, 4096)
    code = torch.arange(256, device=DEV, dtype=torch.float64) - 128
    if fmt == "e4m3":   # sign, 4 exponent bits (bias 7), 3 mantissa bits
        u = torch.arange(256, device=DEV)
        e, m = u >> 3 & 15, (u & 7).double()
        code = torch.where(e > 0, (1 + m / 8) * _power(e - 7), m / 8 * 2.0 ** -6)
        code = torch.where(u > 127, -code, code)
    val = code[raw.long()]
    at = _parts(hkv, i["max_seq"])[0]
    scale = c[:, at:at + hkv * nb * 8].contiguous().view(torch.float32).view(b, hkv, nb, 2).double()
    k = val[:, :, :, 0].reshape(b, hkv, nb, BLOCK, HD) * scale[..., 0, None, None]
    v = torch.empty_like(k)
    rows = val[:, :, :, 1].reshape(b, hkv, nb, HD, BLOCK) * scale[..., 1, None, None]
    for p in range(BLOCK):
        t = 16 * (p >> 3 & 1) + 8 * (p >> 2 & 1) + 4 * (p >> 4) + (p & 3)
        v[:, :, :, t] = rows[..., p]
    return k.view(b, hkv, -1, HD), v.view(b, hkv, -1, HD)


def _attend64(q, k, v, first):
    """Queries q [n][G][128] at positions first.. over k, v [S][128]: outputs, and
    each position's weight summed over queries and heads."""
    n, g, _ = q.shape
    s = torch.einsum("ngd,sd->ngs", q.double(), k) / math.sqrt(HD)
    late = torch.arange(k.shape[0], device=DEV)[None, None] > first + torch.arange(n, device=DEV)[:, None, None]
    p = torch.softmax(s.masked_fill_(late, -math.inf), -1)
    return torch.einsum("ngs,sd->ngd", p, v), p.sum((0, 1))


def exact(case, seed):
    i, kind = _inputs(case, seed), case["kind"]
    if kind == "rules":
        x = i["logits"].double()
        ho, bo = i["hist_off"].tolist(), i["bias_off"].tolist()
        for r in range(case["rows"]):
            n = torch.bincount(i["hist"][ho[r]:ho[r + 1]], minlength=case["V"]).double()
            rep, f, p = i["pen"][r].double()
            y = torch.where(x[r] > 0, x[r] / rep, x[r] * rep) - f * n - p
            x[r] = torch.where(n > 0, y, x[r])
            add = dict(zip(i["bias_ids"][bo[r]:bo[r + 1]].tolist(), i["bias"][bo[r]:bo[r + 1]].tolist()))
            x[r, torch.tensor(list(add), device=DEV)] += torch.tensor(list(add.values()), device=DEV,
                                                                      dtype=torch.float64)
        bits = torch.stack([i["mask"] >> j & 1 for j in range(32)], -1).view(case["rows"], -1)
        return x.masked_fill(bits[:, :case["V"]] == 0, -math.inf)
    hkv, h = case["HKV"], case["H"]
    if kind == "append":
        b, rows = case["batch"], i["rows"]
        tails = i["cache"][:, _parts(hkv, i["max_seq"])[2]:].contiguous().view(torch.float16)
        tails = tails[:, :hkv * 2 * BLOCK * HD].view(b, hkv, 2, BLOCK, HD)
        out = {}
        for which, name in enumerate("kv"):
            x = torch.zeros(b, hkv, rows, HD, dtype=torch.float64, device=DEV)
            for z in range(b):
                off, m = int(i["pos"][z] - i["start"][z]), int(i["counts"][z])
                x[z, :, :off] = tails[z, :, which, :off].double()
                x[z, :, off:off + m] = i[name][z, :, :m].double()
            x = x.view(b, hkv, -1, BLOCK * HD)
            a = x.abs().amax(-1, keepdim=True)
            r = torch.where(a > 0, x * TOP[case["fmt"]] / a, 0.0)
            if case["fmt"] == "int8":
                r = torch.round(r)
            else:   # 3 mantissa bits, steps of 2^-9 below 2^-6
                step = _power(torch.frexp(r.abs().clamp(min=2.0 ** -6)).exponent - 4)
                r = torch.round(r / step) * step
            out[name] = (r * a / TOP[case["fmt"]]).view(b, hkv, rows, HD)
        return out
    k, v = _held64(i, case)
    if kind in ("decode", "prefill"):
        group, outs = h // hkv, []
        w = torch.zeros(*k.shape[:3], dtype=torch.float64, device=DEV)
        for z in range(k.shape[0]):
            q = i["q"][z:z + 1] if kind == "decode" else i["q"]
            first = int(i["pos"][z]) if kind == "decode" else case["pos0"]
            n, heads = first + q.shape[0], []
            for j in range(hkv):
                o, p = _attend64(q[:, j * group:(j + 1) * group], k[z, j, :n], v[z, j, :n], first)
                heads.append(o)
                w[z, j, :n] = p
            outs.append(torch.cat(heads, 1).view(q.shape[0], h * HD))
        out = {"out": torch.cat(outs)}
        if case["weights"]:
            at, nb = _parts(hkv, i["max_seq"])[1], _blocks(i["max_seq"])
            held = i["cache"][:, at:at + hkv * nb * 4].contiguous().view(torch.float32).view(-1, hkv, nb)
            out["weights"] = held.double() + w.view(*w.shape[:2], nb, BLOCK).sum(-1)
        return out
    m, nb = case["budget"], _blocks(i["max_seq"])
    at = _parts(hkv, i["max_seq"])[1]
    w = i["cache"][:, at:at + hkv * nb * 4].contiguous().view(torch.float32).view(-1, hkv, nb)
    k, v = k.view(*w.shape, BLOCK, HD), v.view(*w.shape, BLOCK, HD)
    out = {"k": k.new_zeros(*w.shape[:2], m, BLOCK, HD), "v": k.new_zeros(*w.shape[:2], m, BLOCK, HD),
           "weights": k.new_zeros(*w.shape[:2], m), "len": None}
    held = w.tolist()
    for z, n in enumerate(i["len"].tolist()):
        nblk = _blocks(n)
        for j in range(hkv):
            keep = list(range(nblk))
            if nblk > m:
                must = {0, nblk - 2, nblk - 1}
                rest = sorted((-held[z][j][t], t) for t in keep if t not in must)
                keep = sorted(must | {t for _, t in rest[:m - 3]})
            at = torch.tensor(keep, device=DEV)
            for name, x in (("k", k), ("v", v), ("weights", w)):
                out[name][z, j, :len(keep)] = x[z, j, at].double()
        # the newest block's positions behind the last one hold nothing
        new = n - BLOCK * max(0, nblk - m)
        for name in "kv":
            out[name][z].view(hkv, m * BLOCK, HD)[:, new:] = 0
    for name in "kv":
        out[name] = out[name].view(*w.shape[:2], m * BLOCK, HD)
    return out

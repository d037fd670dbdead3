"""numpy-level access to the hot-path kernels through the C ABI.

Device memory is owned by DeviceArray (hipMalloc'd by liboxbitnet); every op
launches the HIP kernel on the library's stream and returns host numpy
arrays.  Used by the parity tests and the benchmark.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from ._native import check, lib, NativeError

STATE_POS, STATE_TOKEN, STATE_NGEN, STATE_LM_COUNTER, STATE_HIST_CAP = 0, 1, 2, 3, 4
STATE_INTS = 8


class DeviceArray:
    """A device allocation with a dtype/shape view for uploads and downloads."""

    def __init__(self, shape, dtype, zero: bool = False):
        self.shape = tuple(np.atleast_1d(shape)) if not isinstance(shape, tuple) else shape
        self.dtype = np.dtype(dtype)
        self.nbytes = int(np.prod(self.shape)) * self.dtype.itemsize
        self.ptr = lib().oxb_device_malloc(max(self.nbytes, 16))
        if not self.ptr:
            raise NativeError("oxb_device_malloc failed")
        if zero:
            check(lib().oxb_memset_d(self.ptr, 0, max(self.nbytes, 16), None), "memset")
            sync()

    @classmethod
    def from_host(cls, a: np.ndarray) -> "DeviceArray":
        a = np.ascontiguousarray(a)
        d = cls(a.shape, a.dtype)
        d.upload(a)
        return d

    def upload(self, a: np.ndarray) -> None:
        a = np.ascontiguousarray(a, dtype=self.dtype)
        assert a.nbytes <= self.nbytes, (a.nbytes, self.nbytes)
        check(lib().oxb_memcpy_h2d(self.ptr, a.ctypes.data, a.nbytes, None), "h2d")

    def download(self, shape=None, dtype=None) -> np.ndarray:
        dt = np.dtype(dtype) if dtype is not None else self.dtype
        shp = shape if shape is not None else self.shape
        out = np.empty(shp, dt)
        assert out.nbytes <= self.nbytes
        check(lib().oxb_memcpy_d2h(out.ctypes.data, self.ptr, out.nbytes, None), "d2h")
        return out

    def offset(self, nbytes: int) -> int:
        return self.ptr + nbytes

    def free(self) -> None:
        if self.ptr:
            lib().oxb_device_free(self.ptr)
            self.ptr = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


def sync() -> None:
    check(lib().oxb_device_sync(), "device sync")


def device_info() -> dict:
    name = C.create_string_buffer(256)
    cus, clk = C.c_int(), C.c_int()
    mem = C.c_size_t()
    check(lib().oxb_device_info(name, 256, C.byref(cus), C.byref(clk), C.byref(mem)), "device info")
    return {"name": name.value.decode(), "cus": cus.value, "clock_khz": clk.value,
            "hbm_bytes": mem.value}


def _p(x):
    if x is None:
        return None
    return x.ptr if isinstance(x, DeviceArray) else x


# ---- layouts -----------------------------------------------------------------
def repack_tiled(W_natural: DeviceArray, N: int, K: int) -> DeviceArray:
    out = DeviceArray((N * K // 4,), np.uint8)
    check(lib().oxb_repack_i2s_tiled(W_natural.ptr, out.ptr, N, K, None), "repack")
    sync()
    return out


def upload_ternary(W_natural: np.ndarray, K: int) -> DeviceArray:
    """Natural I2_S rows [N][K/4] (host) -> tiled device matrix."""
    N = W_natural.shape[0]
    nat = DeviceArray.from_host(np.ascontiguousarray(W_natural, np.uint8).reshape(-1))
    t = repack_tiled(nat, N, K)
    nat.free()
    return t


# ---- kernels -----------------------------------------------------------------
def gemv_i8(Wt: DeviceArray, xq: np.ndarray, xscale: float, wscale: np.ndarray, N: int, K: int):
    """Int8 GEMV: returns (acc int32 [N], y f32 [N])."""
    xq = np.ascontiguousarray(xq, np.int8)
    dx = DeviceArray.from_host(xq)
    ds = DeviceArray.from_host(np.array([xscale], np.float32))
    dsum = DeviceArray.from_host(np.array([int(xq.astype(np.int64).sum())], np.int32))
    dw = DeviceArray.from_host(np.ascontiguousarray(wscale, np.float32))
    y = DeviceArray((N,), np.float32)
    acc = DeviceArray((N,), np.int32)
    check(lib().oxb_gemv_i8(Wt.ptr, dx.ptr, ds.ptr, dsum.ptr, dw.ptr, N, K, y.ptr, acc.ptr, None),
          "gemv_i8")
    sync()
    return acc.download(), y.download()


def bitlinear_gemv(Wt, x: np.ndarray, gamma, eps: float, wscale: np.ndarray, N: int, K: int,
                   residual: np.ndarray | None = None):
    """One-token BitLinear: returns (acc, y, xq, xscale)."""
    dx = DeviceArray.from_host(np.ascontiguousarray(x, np.float32))
    dg = DeviceArray.from_host(np.ascontiguousarray(gamma, np.float32)) if gamma is not None else None
    dw = DeviceArray.from_host(np.ascontiguousarray(wscale, np.float32))
    y = DeviceArray.from_host(np.ascontiguousarray(residual, np.float32)) if residual is not None \
        else DeviceArray((N,), np.float32)
    acc = DeviceArray((N,), np.int32)
    xq = DeviceArray((K,), np.int8)
    xs = DeviceArray((1,), np.float32)
    check(lib().oxb_bitlinear_gemv(Wt.ptr, dx.ptr, _p(dg), eps, dw.ptr, N, K, y.ptr,
                                   1 if residual is not None else 0, acc.ptr, xq.ptr, xs.ptr, None),
          "bitlinear_gemv")
    sync()
    return acc.download(), y.download(), xq.download(), float(xs.download()[0])


def bitlinear_gateup(Wt, x, gamma, eps, wscale, N2, K):
    dx = DeviceArray.from_host(np.ascontiguousarray(x, np.float32))
    dg = DeviceArray.from_host(np.ascontiguousarray(gamma, np.float32)) if gamma is not None else None
    dw = DeviceArray.from_host(np.ascontiguousarray(wscale, np.float32))
    h = DeviceArray((N2 // 2,), np.float32)
    check(lib().oxb_bitlinear_gateup(Wt.ptr, dx.ptr, _p(dg), eps, dw.ptr, N2, K, h.ptr, None),
          "bitlinear_gateup")
    sync()
    return h.download()


def norm_quant_rows(x: np.ndarray, gamma, eps: float):
    x = np.ascontiguousarray(np.atleast_2d(x), np.float32)
    n, D = x.shape
    dx = DeviceArray.from_host(x)
    dg = DeviceArray.from_host(np.ascontiguousarray(gamma, np.float32)) if gamma is not None else None
    q = DeviceArray((n, D), np.int8)
    s = DeviceArray((n,), np.float32)
    sm = DeviceArray((n,), np.int32)
    check(lib().oxb_norm_quant_rows(dx.ptr, _p(dg), eps, n, D, q.ptr, s.ptr, sm.ptr, None),
          "norm_quant_rows")
    sync()
    return q.download(), s.download(), sm.download()


def quantize_rows_tiled(x: DeviceArray, gamma, eps: float, n: int, D: int, Xt: DeviceArray,
                        scales: DeviceArray, sums: DeviceArray, stream=None):
    check(lib().oxb_quantize_rows_tiled(x.ptr, _p(gamma), eps, n, D, Xt.ptr, scales.ptr, sums.ptr,
                                        stream), "quantize_rows_tiled")


def gemm(Wt, x: np.ndarray, gamma, eps: float, wscale: np.ndarray, N: int, K: int,
         epilogue: int = 0, Y0: np.ndarray | None = None):
    """Prefill BitLinear on MFMA: (optional RMSNorm) + quantize rows + GEMM.
    Returns (acc int32 [n, N], Y, xscales)."""
    x = np.ascontiguousarray(np.atleast_2d(x), np.float32)
    n = x.shape[0]
    npad = (n + 63) // 64 * 64
    dx = DeviceArray.from_host(x)
    dg = DeviceArray.from_host(np.ascontiguousarray(gamma, np.float32)) if gamma is not None else None
    Xt = DeviceArray((npad * K,), np.int8, zero=True)
    sc = DeviceArray((npad,), np.float32)
    sm = DeviceArray((npad,), np.int32)
    check(lib().oxb_quantize_rows_tiled(dx.ptr, _p(dg), eps, n, K, Xt.ptr, sc.ptr, sm.ptr, None),
          "quantize_rows_tiled")
    dw = DeviceArray.from_host(np.ascontiguousarray(wscale, np.float32))
    ncol = N // 2 if epilogue == 2 else N
    Y = DeviceArray.from_host(np.ascontiguousarray(Y0, np.float32)) if Y0 is not None \
        else DeviceArray((n, ncol), np.float32)
    acc = DeviceArray((n, N), np.int32)
    check(lib().oxb_gemm_i8(Wt.ptr, Xt.ptr, sc.ptr, sm.ptr, dw.ptr, N, K, n, Y.ptr, acc.ptr,
                            epilogue, None), "gemm_i8")
    sync()
    return acc.download(), Y.download(shape=(n, ncol)), sc.download(shape=(n,))


KV_PAD_ROWS = 64   # include/oxbitnet_ops.h OXB_KV_PAD_ROWS


def _padded_cache(c: np.ndarray, hd: int) -> DeviceArray:
    """A cache on the device with OXB_KV_PAD_ROWS rows of zeros past its end."""
    flat = np.ascontiguousarray(c, np.float16).view(np.uint16).reshape(-1)
    return DeviceArray.from_host(np.concatenate([flat, np.zeros(KV_PAD_ROWS * hd, np.uint16)]))


def v_octets(vc: np.ndarray) -> np.ndarray:
    """V cache rows [..., Hkv, S, hd] (f16) in the decode P.V's octet layout:
    per head round8(S) x hd elements, (position s, dim d) at ((s // 8) * hd +
    d) * 8 + s % 8 (positions past S zero)."""
    vc = np.asarray(vc, np.float16)
    *lead, hkv, S, hd = vc.shape
    S8 = (S + 7) // 8 * 8
    pad = np.zeros((*lead, hkv, S8, hd), np.float16)
    pad[..., :S, :] = vc
    o = pad.reshape(*lead, hkv, S8 // 8, 8, hd).swapaxes(-1, -2)   # [.., oct, hd, 8]
    return np.ascontiguousarray(o).view(np.uint16).reshape(*lead, hkv * S8 * hd)


def attn_decode(q: np.ndarray, kcache: np.ndarray, vcache: np.ndarray, pos: int, H: int, Hkv: int,
                hd: int, max_seq: int, fused: bool = False, head: bool = False, s_max: int = 0,
                octets: bool = False):
    """q [H*hd] f32; caches [Hkv][max_seq][hd] f16; attends over pos+1 positions.
    fused: the one-kernel variant (oxb_attn_decode_fused); head: one workgroup
    per query head (oxb_attn_decode_head, caches padded as it requires);
    octets: with the octet copy of V as well (oxb_attn_decode_head_v8 /
    oxb_attn_decode_batch_v8)."""
    dq = DeviceArray.from_host(np.ascontiguousarray(q, np.float32))
    dk = _padded_cache(kcache, hd)
    dv = _padded_cache(vcache, hd)
    dpos = DeviceArray.from_host(np.array([pos], np.int32))
    out = DeviceArray((H * hd,), np.float32)
    dv8 = DeviceArray.from_host(v_octets(vcache)) if octets else None
    if head and octets:
        check(lib().oxb_attn_decode_head_v8(dq.ptr, dk.ptr, dv.ptr, dv8.ptr, dpos.ptr, 0, 0, 0, 1,
                                            H, Hkv, hd, max_seq, s_max or pos + 1, out.ptr, None),
              "attn_decode_head_v8")
    elif head:
        check(lib().oxb_attn_decode_head(dq.ptr, dk.ptr, dv.ptr, dpos.ptr, 0, 0, 1, H, Hkv, hd,
                                         max_seq, s_max or pos + 1, out.ptr, None),
              "attn_decode_head")
    elif octets:
        sc = DeviceArray((H * max_seq,), np.float32)
        check(lib().oxb_attn_decode_batch_v8(dq.ptr, dk.ptr, dv.ptr, dv8.ptr, dpos.ptr, 0, 0, 0, 1,
                                             H, Hkv, hd, max_seq, sc.ptr, out.ptr, None),
              "attn_decode_batch_v8")
    elif fused:
        check(lib().oxb_attn_decode_fused(dq.ptr, dk.ptr, dv.ptr, dpos.ptr, H, Hkv, hd, max_seq,
                                          out.ptr, None), "attn_decode_fused")
    else:
        sc = DeviceArray((H * max_seq,), np.float32)
        check(lib().oxb_attn_decode(dq.ptr, dk.ptr, dv.ptr, dpos.ptr, H, Hkv, hd, max_seq, sc.ptr,
                                    out.ptr, None), "attn_decode")
    sync()
    return out.download()


def attn_prefill(q: np.ndarray, kcache: np.ndarray, vcache: np.ndarray, n_tok: int, pos0: int,
                 H: int, Hkv: int, hd: int, max_seq: int):
    dq = DeviceArray.from_host(np.ascontiguousarray(q, np.float32))
    dk = DeviceArray.from_host(np.ascontiguousarray(kcache, np.float16).view(np.uint16))
    dv = DeviceArray.from_host(np.ascontiguousarray(vcache, np.float16).view(np.uint16))
    out = DeviceArray((n_tok, H * hd), np.float32)
    check(lib().oxb_attn_prefill(dq.ptr, dk.ptr, dv.ptr, n_tok, pos0, H, Hkv, hd, max_seq, out.ptr,
                                 None), "attn_prefill")
    sync()
    return out.download()


KV8_INT8, KV8_E4M3, KV8_BLOCK = 0, 1, 32   # include/oxbitnet_ops.h OXB_KV8_*


def _require(ok, what: str) -> None:
    if not ok:
        raise ValueError(what)


class Kv8Cache:
    """A batch's 8-bit KV cache (oxb_kv8_*, oxb_attn_*_kv8): numpy rows in, numpy out."""

    def __init__(self, batch: int, Hkv: int, max_seq: int, fmt: int = KV8_INT8, hd: int = 128):
        self.batch, self.Hkv, self.max_seq, self.fmt, self.hd = batch, Hkv, max_seq, fmt, hd
        self.stride = lib().oxb_kv8_bytes(Hkv, hd, max_seq)
        if not self.stride:
            raise NativeError(f"no 8-bit cache of {Hkv} heads of {hd}, {max_seq} positions")
        self.data = DeviceArray((batch, self.stride), np.uint8)

    def _per_seq(self, x, what: str) -> np.ndarray:
        x = np.ascontiguousarray(x, np.int32)
        _require(x.shape == (self.batch,), f"{what}: {x.shape} for {self.batch} sequences")
        return x

    def _heads(self, q: np.ndarray) -> int:
        _require(q.shape[1] % (self.hd * self.Hkv) == 0 and q.shape[1] > 0,
                 f"q rows of {q.shape[1]} for {self.Hkv} KV heads of {self.hd}")
        return q.shape[1] // self.hd

    def append(self, k: np.ndarray, v: np.ndarray, pos, counts=None, stream=None) -> None:
        """f16 rows [batch][Hkv][n][128] at each sequence's position."""
        k, v = (np.ascontiguousarray(x, np.float16) for x in (k, v))
        _require(k.ndim == 4 and k.shape == v.shape == (self.batch, self.Hkv, k.shape[2], self.hd),
                 f"k {k.shape} and v {v.shape} for [{self.batch}][{self.Hkv}][n][{self.hd}]")
        n = k.shape[2]
        pos = self._per_seq(pos, "pos")
        counts = self._per_seq(counts, "counts") if counts is not None else None
        dk, dv = (DeviceArray.from_host(x.view(np.uint16)) for x in (k, v))
        dp = DeviceArray.from_host(pos)
        dc = DeviceArray.from_host(counts) if counts is not None else None
        check(lib().oxb_kv8_append(self.data.ptr, self.stride, self.fmt, self.batch, self.Hkv, self.hd,
                                   self.max_seq, dk.ptr, dv.ptr, self.Hkv * n * self.hd, n * self.hd, 0,
                                   dp.ptr, 1, 0, n, _p(dc), stream), "kv8_append")
        sync()

    def read(self, pos, n: int, length=None):
        """The values of n positions from each sequence's pos on: k, v f32 [batch][Hkv][n][128]."""
        pos = self._per_seq(pos, "pos")
        length = self._per_seq(length, "length") if length is not None else None
        dp = DeviceArray.from_host(pos)
        dl = DeviceArray.from_host(length) if length is not None else None
        k, v = (DeviceArray((self.batch, self.Hkv, n, self.hd), np.float32) for _ in "kv")
        check(lib().oxb_kv8_read(self.data.ptr, self.stride, self.fmt, self.batch, self.Hkv, self.hd,
                                 self.max_seq, dp.ptr, 1, 0, n, _p(dl), 1, k.ptr, v.ptr, None), "kv8_read")
        sync()
        return k.download(), v.download()

    def weights(self) -> np.ndarray:
        """Each block's accumulated attention weight [batch][Hkv][blocks]."""
        nb, al = (self.max_seq + KV8_BLOCK - 1) // KV8_BLOCK, lambda b: (b + 255) // 256 * 256
        at = al(self.Hkv * nb * 8192) + al(self.Hkv * nb * 8)
        raw = self.data.download()[:, at:at + self.Hkv * nb * 4]
        return np.ascontiguousarray(raw).view(np.float32).reshape(self.batch, self.Hkv, nb)

    def attn_decode(self, q: np.ndarray, pos, add_weights: bool = False) -> np.ndarray:
        """q f32 [batch][H*128]; sequence z attends over pos[z] + 1 positions."""
        q = np.ascontiguousarray(q, np.float32).reshape(self.batch, -1)
        H, pos = self._heads(q), self._per_seq(pos, "pos")
        dq, dp = DeviceArray.from_host(q), DeviceArray.from_host(pos)
        out = DeviceArray(q.shape, np.float32)
        n = lib().oxb_attn_decode_kv8_ws_bytes(self.batch, H, self.Hkv, self.hd, self.max_seq)
        ws = DeviceArray((max(n, 16),), np.uint8, zero=True)
        check(lib().oxb_attn_decode_kv8(dq.ptr, self.data.ptr, self.stride, self.fmt, dp.ptr, 1, self.batch,
                                        H, self.Hkv, self.hd, self.max_seq, int(add_weights), out.ptr,
                                        ws.ptr, n, None), "attn_decode_kv8")
        sync()
        return out.download()

    def attn_prefill(self, q: np.ndarray, pos0: int, slot: int = 0, add_weights: bool = False) -> np.ndarray:
        """q f32 [n][H*128] of sequence `slot` at positions pos0.., causal."""
        q = np.ascontiguousarray(np.atleast_2d(q), np.float32)
        _require(0 <= slot < self.batch, f"sequence {slot} of {self.batch}")
        n, H = q.shape[0], self._heads(q)
        dq, out = DeviceArray.from_host(q), DeviceArray(q.shape, np.float32)
        b = lib().oxb_attn_prefill_kv8_ws_bytes(n, pos0, H, self.Hkv, self.hd, int(add_weights))
        ws = DeviceArray((max(b, 16),), np.uint8, zero=True)
        check(lib().oxb_attn_prefill_kv8(dq.ptr, self.data.offset(slot * self.stride), self.fmt, n, pos0, H,
                                         self.Hkv, self.hd, self.max_seq, int(add_weights), out.ptr, ws.ptr,
                                         b, None), "attn_prefill_kv8")
        sync()
        return out.download()

    def evict(self, length, budget: int, sink: int = 1, recent: int = 1, dst: "Kv8Cache | None" = None):
        """Cut to `budget` blocks, in place or into dst; returns the new lengths."""
        dst = dst or self
        _require((dst.batch, dst.Hkv, dst.hd, dst.fmt) == (self.batch, self.Hkv, self.hd, self.fmt),
                 "dst is a cache of another shape or format")
        dl = DeviceArray.from_host(self._per_seq(length, "length"))
        n = lib().oxb_kv8_evict_ws_bytes(self.batch, self.Hkv, self.max_seq, budget)
        ws = DeviceArray((max(n, 16),), np.uint8)
        check(lib().oxb_kv8_evict(self.data.ptr, self.stride, self.max_seq, dst.data.ptr, dst.stride,
                                  dst.max_seq, dl.ptr, 1, dl.ptr, 1, self.batch, self.Hkv, self.hd, budget,
                                  sink, recent, ws.ptr, n, None), "kv8_evict")
        sync()
        return dl.download()


F32, F16 = 0, 1   # include/oxbitnet_ops.h OXB_F32, OXB_F16
# OXB_PAGED_UNIT, OXB_PAGED_MAX_SEQ, OXB_PAGED_MAX_BATCH, OXB_PAGED_MAX_PREFILL
PAGED_UNIT, PAGED_MAX_SEQ, PAGED_MAX_BATCH, PAGED_MAX_PREFILL = 32, 1 << 24, 4096, 128


class PagedCache:
    """A batch's f16 KV cache in pages of one pool (oxb_paged_*, oxb_attn_*_paged):
    numpy rows in, numpy out."""

    def __init__(self, batch: int, Hkv: int, n_pages: int, page_size: int, table_pages: int, hd: int = 128):
        self.batch, self.Hkv, self.n_pages, self.page_size, self.hd = batch, Hkv, n_pages, page_size, hd
        n = lib().oxb_paged_bytes(n_pages, page_size, Hkv, hd)
        if not n:
            raise NativeError(f"no pool of {n_pages} pages of {page_size} positions, {Hkv} heads of {hd}")
        _require(1 <= batch <= PAGED_MAX_BATCH, f"batch {batch}")
        _require(1 <= table_pages <= PAGED_MAX_SEQ // page_size, f"block table of {table_pages} pages a sequence")
        self.pool = DeviceArray((n // 2,), np.uint16)
        self.table = DeviceArray.from_host(np.full((batch, table_pages), -1, np.int32))
        self.free = DeviceArray.from_host(np.arange(n_pages, dtype=np.int32)[::-1])
        self.n_free = DeviceArray.from_host(np.array([n_pages], np.int32))
        self.len = DeviceArray((batch,), np.int32, zero=True)
        self._ws = None

    def _workspace(self, n: int) -> tuple:
        """One for all calls, of the largest so far."""
        _require(n > 0, "no workspace for this shape")
        if self._ws is None or self._ws.nbytes < n:
            if self._ws is not None:
                sync()
                self._ws.free()
            self._ws = None   # (should the allocation fail)
            self._ws = DeviceArray((n,), np.uint8, zero=True)
        return self._ws.ptr, self._ws.nbytes

    def step(self, delta, n_max: int | None = None) -> dict:
        """Grow, keep or shrink each sequence: granted tokens, and the packed tokens'
        starts (cu), slots and positions."""
        delta = np.ascontiguousarray(delta, np.int32)
        _require(delta.shape == (self.batch,), f"delta {delta.shape} for {self.batch} sequences")
        n = int(np.maximum(delta, 0).sum()) if n_max is None else n_max
        dd = DeviceArray.from_host(delta)
        cu, granted = DeviceArray((self.batch + 1,), np.int32), DeviceArray((self.batch,), np.int32)
        slots, pos = (DeviceArray((n,), np.int32) for _ in "sp")
        check(lib().oxb_paged_update(self.page_size, self.batch, self.len.ptr, dd.ptr, self.table.ptr,
                                     self.table.shape[1], self.free.ptr, self.n_pages, self.n_free.ptr, self.len.ptr,
                                     self.n_free.ptr, cu.ptr, granted.ptr, slots.ptr, pos.ptr, n, None),
              "paged_update")
        sync()
        return {"cu": cu.download(), "granted": granted.download(), "slots": slots.download(),
                "pos": pos.download()}

    def append(self, k: np.ndarray, v: np.ndarray, slots) -> None:
        """f16 rows [n][Hkv][128] of packed tokens into their slots."""
        k, v = (np.ascontiguousarray(x, np.float16) for x in (k, v))
        slots = np.ascontiguousarray(slots, np.int32)
        _require(k.shape == v.shape == (slots.size, self.Hkv, self.hd) and slots.ndim == 1,
                 f"k {k.shape} and v {v.shape} for [{slots.size}][{self.Hkv}][{self.hd}]")
        if not slots.size:
            return
        dk, dv = (DeviceArray.from_host(x.view(np.uint16)) for x in (k, v))
        ds = DeviceArray.from_host(slots)
        check(lib().oxb_paged_append(self.pool.ptr, self.n_pages, self.page_size, self.Hkv, self.hd, dk.ptr, dv.ptr,
                                     self.Hkv * self.hd, self.hd, None, ds.ptr, slots.size, None), "paged_append")
        sync()

    def _q(self, q: np.ndarray) -> tuple:
        q = np.ascontiguousarray(q)
        _require(q.dtype in (np.float32, np.float16) and q.ndim == 2, f"q is {q.dtype} {q.shape}")
        _require(q.shape[1] % (self.hd * self.Hkv) == 0 and q.shape[1] > 0,
                 f"q rows of {q.shape[1]} for {self.Hkv} KV heads of {self.hd}")
        return q, F32 if q.dtype == np.float32 else F16, q.shape[1] // self.hd

    def attn_decode(self, q: np.ndarray) -> np.ndarray:
        """q f32 or f16 [batch][H*128]; each sequence attends over all it holds."""
        q, dtype, H = self._q(q)
        _require(q.shape[0] == self.batch, f"{q.shape[0]} queries for {self.batch} sequences")
        dq, out = DeviceArray.from_host(q), DeviceArray(q.shape, q.dtype)
        ws = self._workspace(lib().oxb_attn_decode_paged_ws_bytes(self.batch, H, self.Hkv, self.hd))
        check(lib().oxb_attn_decode_paged(dq.ptr, dtype, self.pool.ptr, self.n_pages, self.page_size, self.table.ptr,
                                          self.table.shape[1], self.len.ptr, self.batch, H, self.Hkv, self.hd,
                                          out.ptr, *ws, None), "attn_decode_paged")
        sync()
        return out.download()

    def attn_prefill(self, q: np.ndarray, cu, out: np.ndarray | None = None) -> np.ndarray:
        """q f32 or f16 [n][H*128] packed, sequence z's newest tokens at cu[z]..cu[z+1]-1,
        causal; out: what the rows of no sequence hold before (and after)."""
        q, dtype, H = self._q(q)
        cu = np.ascontiguousarray(cu, np.int32)
        _require(cu.shape == (self.batch + 1,), f"cu {cu.shape} for {self.batch} sequences")
        dq, dc = DeviceArray.from_host(q), DeviceArray.from_host(cu)
        do = DeviceArray.from_host(np.zeros_like(q) if out is None else np.ascontiguousarray(out, q.dtype))
        _require(do.shape == q.shape, f"out {do.shape} for {q.shape}")
        # as many sequences a call as one takes
        parts = [(z, min(PAGED_MAX_PREFILL, self.batch - z)) for z in range(0, self.batch, PAGED_MAX_PREFILL)]
        ws = self._workspace(max(lib().oxb_attn_prefill_paged_ws_bytes(q.shape[0], b, H, self.Hkv, self.hd)
                                 for _, b in parts))
        for z, b in parts:
            check(lib().oxb_attn_prefill_paged(dq.ptr, dtype, self.pool.ptr, self.n_pages, self.page_size,
                                               self.table.offset(4 * z * self.table.shape[1]), self.table.shape[1],
                                               dc.offset(4 * z), self.len.offset(4 * z), q.shape[0], b, H, self.Hkv,
                                               self.hd, do.ptr, *ws, None), "attn_prefill_paged")
        sync()
        return do.download()


def logits_rules(logits: np.ndarray, penalties=None, history=None, bias=None, mask=None) -> np.ndarray:
    """Rules on logits [n][V] (oxb_logits_rules).  penalties: [n][3] repeat, frequency,
    presence; history: a list of ids per row; bias: a list of (id, value) per row;
    mask: uint32 words [n][w], or [w] for every row."""
    x = np.ascontiguousarray(np.atleast_2d(logits), np.float32)
    n, V = x.shape

    def csr(lists, dtype):
        _require(len(lists) == n, f"{len(lists)} lists for {n} rows")
        off = np.concatenate([[0], np.cumsum([len(r) for r in lists])]).astype(np.int32)
        flat = np.concatenate([np.asarray(r, dtype).reshape(-1) for r in lists]).astype(dtype)
        return flat, off

    pen = np.asarray(penalties, np.float32).reshape(n, 3) if penalties is not None else None
    h, ho = csr(history, np.int32) if history is not None else (np.empty(0, np.int32), None)
    bi, bo = csr([[i for i, _ in r] for r in bias], np.int32) if bias is not None else (np.empty(0, np.int32), None)
    bv = csr([[b for _, b in r] for r in bias], np.float32)[0] if bias is not None else None
    words = 0
    if mask is not None:
        mask = np.ascontiguousarray(mask, np.uint32)
        _require(mask.shape[-1] >= (V + 31) // 32 and mask.shape[:-1] in ((), (n,)),
                 f"mask {mask.shape} for {n} rows of {V}")
        words = mask.shape[1] if mask.ndim == 2 else 0
    up = lambda a: DeviceArray.from_host(a) if a is not None and a.size else None  # noqa: E731
    dx, dpen, dh, dho, dbi, dbo, dbv, dm = (up(a) for a in (x, pen, h, ho, bi, bo, bv, mask))
    out = DeviceArray((n, V), np.float32)
    check(lib().oxb_logits_rules(dx.ptr, V, n, V, _p(dpen), _p(dh), _p(dho), h.size, _p(dbi), _p(dbv),
                                 _p(dbo), bi.size, _p(dm), words, out.ptr, V, None), "logits_rules")
    sync()
    return out.download()


def lm_head_argmax(x: np.ndarray, gamma: np.ndarray, eps: float, E_f16: np.ndarray):
    """Returns (logits [V], token, state)."""
    V, D = E_f16.shape
    dx = DeviceArray.from_host(np.ascontiguousarray(x, np.float32))
    dg = DeviceArray.from_host(np.ascontiguousarray(gamma, np.float32))
    dE0 = DeviceArray.from_host(np.ascontiguousarray(E_f16).view(np.uint16))
    dE = DeviceArray((lib().oxb_lm_bytes(V, D),), np.uint8)
    check(lib().oxb_repack_lm(dE0.ptr, dE.ptr, V, D, None), "repack_lm")
    dE0.free()
    logits = DeviceArray((V,), np.float32)
    st = np.zeros(STATE_INTS, np.int32)
    st[STATE_HIST_CAP] = 4
    dst = DeviceArray.from_host(st)
    hist = DeviceArray((4,), np.int32, zero=True)
    check(lib().oxb_lm_head_argmax(dx.ptr, dg.ptr, eps, dE.ptr, V, D, logits.ptr, dst.ptr,
                                   hist.ptr, 1, None), "lm_head_argmax")
    sync()
    s = dst.download()
    return logits.download(), int(s[STATE_TOKEN]), s, hist.download()


def embedding(E_f16: np.ndarray, ids: np.ndarray):
    V, D = E_f16.shape
    ids = np.ascontiguousarray(ids, np.int32)
    dE = DeviceArray.from_host(np.ascontiguousarray(E_f16).view(np.uint16))
    di = DeviceArray.from_host(ids)
    x = DeviceArray((ids.size, D), np.float32)
    check(lib().oxb_embedding(dE.ptr, V, D, di.ptr, ids.size, None, x.ptr, None), "embedding")
    sync()
    return x.download()

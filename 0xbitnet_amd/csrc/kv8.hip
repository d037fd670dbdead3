// The 8-bit KV cache for gfx950: appending rows, reading values back, and
// eviction of whole blocks by accumulated attention weight.  No counterpart in
// the reference (its cache is f32 rows that are never dropped,
// nn/attention.rs:23-48).
//
// A block is 32 positions of one KV head; its K codes and its V codes have a
// scale each.  With a = max|x| over the block's rows so far,
//   int8: scale = a / 127, code = round(127 x / a)
//   e4m3: scale = a / 448, code = e4m3(448 x / a)
// both rounded to nearest, ties to even.  x is f16, so 127 x and 448 x are
// exact in f32 and x's quotient by a (11 bits) differs from a rounding
// boundary (at most 9 bits) by at least 2^-20 of itself unless it is one: the
// f32 division, correctly rounded, never moves it onto or across one, and
// the code is that of the real quotient.
//
// An unfinished block grows row by row and its scale with it.  Its rows stay
// in f16 beside the codes (the tail, 16 KB per KV head), and each append
// quantizes the whole block again from them, so the cache depends on the rows
// alone, not on how they were split over calls, and no value is rounded twice.
// The tail keeps a completed block's rows too, until the next block's first ones
// take their place: rows may be taken back within it.
#include "kv8.h"
#include "radix_select.h"

#include <algorithm>

namespace oxb {

constexpr int kKvThreads = 256;

struct Kv8AppendArgs {
    uint8_t *cache;
    size_t stride;
    int Hkv, max_seq, nb;
    const uint16_t *k, *v;          // the new rows
    size_t src_stride, src_head;    // elements between sequences, between heads
    int src_at_pos;                 // row i of the call is source row pos + i (else i)
    const int *pos;
    int pos_stride, pos0, n;
    const int *counts;
};

// Where sequence z's new rows start and how many the cache takes.
__device__ inline void kv8_span(const Kv8AppendArgs &a, int z, int &p0, int &cnt) {
    const int64_t p = (int64_t)(a.pos ? a.pos[(size_t)z * a.pos_stride] : 0) + a.pos0;
    int c = a.counts ? min(max(a.counts[z], 0), a.n) : a.n;
    if (p < 0 || p >= a.max_seq) {
        p0 = 0;
        cnt = 0;
        return;
    }
    p0 = (int)p;
    cnt = min(c, a.max_seq - p0);
}

// One workgroup per (block, K or V, head, sequence).  A thread holds 4 dims of 4
// consecutive positions, so that it has the 4 bytes that a V row keeps together
// (and 4 of a K row).  Latency bound for one row (a block's rows come from L2),
// by the rows' and codes' bytes for a prompt: the quotient is two products and
// its own remainder's correction,
//   y = t (1/a),  y' = y + (t - y a) (1/a),  t = top x (exact),
// off by 2^-24 of itself at most and exact where the quotient is an f32 number,
// ties among them: the same codes as the f32 division's, in a third of its
// instructions.  One row: 3.4 us.  Four prompts of up to 2048 rows, 5 heads (16 MB
// in, 8 out): 8.5-9.1 us, 2.7-2.9 TB/s; 13.9 with divisions and V's bytes stored one
// by one.  Short of the copy's rate as nothing of another block is in flight while a
// workgroup waits for its rows, their maximum and its two barriers.
template <int FMT>
__global__ __launch_bounds__(kKvThreads) void kv8_append_kernel(Kv8AppendArgs a) {
    __shared__ uint32_t vt[kKv8Hd * 9];   // V codes, [dim][9 dwords]: 8, and one against bank conflicts
    __shared__ int red[4];
    const int z = blockIdx.z, h = blockIdx.y, isv = blockIdx.x & 1;
    int p0, cnt;
    kv8_span(a, z, p0, cnt);
    const int first = p0 / kKv8Block, b = first + (int)(blockIdx.x >> 1);
    const int end = p0 + cnt;                        // one past the last new position
    if (cnt == 0 || b * kKv8Block >= end) return;    // uniform over the workgroup
    const Kv8Layout l = kv8_layout(a.Hkv, a.nb);
    uint8_t *seq = a.cache + (size_t)z * a.stride;
    uint16_t *tail = (uint16_t *)(seq + l.tails) + ((size_t)h * 2 + isv) * kKv8Half;
    const uint16_t *src = (isv ? a.v : a.k) + (size_t)z * a.src_stride + (size_t)h * a.src_head;
    const int row0 = a.src_at_pos ? 0 : p0;          // source row = position - row0
    const int tid = threadIdx.x, d = (tid & 31) * 4, t0 = (tid >> 5) * 4;

    u32x2_t x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int t = t0 + i, p = b * kKv8Block + t;
        x[i] = u32x2_t{0, 0};
        if (p < p0)
            x[i] = *(const u32x2_t *)(tail + t * kKv8Hd + d);
        else if (p < end)
            x[i] = *(const u32x2_t *)(src + (size_t)(p - row0) * kKv8Hd + d);
    }
    // |x| as the f16's low 15 bits: ordered like the values, 0x7c00 and up not finite
    int m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        m = max(m, max((int)(x[i].x & 0x7fff), (int)(x[i].x >> 16 & 0x7fff)));
        m = max(m, max((int)(x[i].y & 0x7fff), (int)(x[i].y >> 16 & 0x7fff)));
    }
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) m = max(m, __shfl_xor(m, s, 64));
    if ((tid & 63) == 0) red[tid >> 6] = m;
    __syncthreads();
    m = max(max(red[0], red[1]), max(red[2], red[3]));
    constexpr float kTop = FMT == OXB_KV8_INT8 ? 127.0f : 448.0f;
    const bool finite = m < 0x7c00;
    const float amax = finite ? __half2float(__ushort_as_half((unsigned short)m)) : 1.0f;
    const float div = amax > 0.0f ? amax : 1.0f, rdiv = 1.0f / div;
    uint32_t c[4];   // 4 dims of a position
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float r[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t bits = (j < 2 ? x[i].x : x[i].y) >> (16 * (j & 1)) & 0xffff;
            const float t = finite ? __half2float(__ushort_as_half((unsigned short)bits)) * kTop : 0.0f;
            const float y = t * rdiv;
            r[j] = __builtin_fmaf(__builtin_fmaf(-y, div, t), rdiv, y);
            if constexpr (FMT == OXB_KV8_E4M3) r[j] = __builtin_copysignf(r[j], t);   // -0 stays
        }
        if constexpr (FMT == OXB_KV8_INT8) {
            // 2^23 + 2^22 + 128: the sum's rounding is the quotient's to a whole
            // number, and its low byte the code's
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = __float_as_uint(r[j] + 12583040.0f);
            const uint32_t lo = __builtin_amdgcn_perm(w[1], w[0], 0x0c0c0400u);
            const uint32_t hi = __builtin_amdgcn_perm(w[3], w[2], 0x0c0c0400u);
            c[i] = lo | hi << 16;
        } else {
            const int q = __builtin_amdgcn_cvt_pk_fp8_f32(r[0], r[1], 0, false);
            c[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(r[2], r[3], q, true);
        }
    }
    const size_t blk = (size_t)h * a.nb + b;
    uint8_t *codes = seq + blk * kKv8Codes;
    if (isv) {
        // bytes to positions: dword j holds dim d + j of positions t0 .. t0 + 3
        const uint32_t l0 = __builtin_amdgcn_perm(c[1], c[0], 0x05010400u);   // c0.0 c1.0 c0.1 c1.1
        const uint32_t l1 = __builtin_amdgcn_perm(c[3], c[2], 0x05010400u);
        const uint32_t h0 = __builtin_amdgcn_perm(c[1], c[0], 0x07030602u);   // c0.2 c1.2 c0.3 c1.3
        const uint32_t h1 = __builtin_amdgcn_perm(c[3], c[2], 0x07030602u);
        uint32_t *at = vt + d * 9 + kv8_v_byte(t0) / 4;
        at[0] = __builtin_amdgcn_perm(l1, l0, 0x05040100u);
        at[9] = __builtin_amdgcn_perm(l1, l0, 0x07060302u);
        at[18] = __builtin_amdgcn_perm(h1, h0, 0x05040100u);
        at[27] = __builtin_amdgcn_perm(h1, h0, 0x07060302u);
        __syncthreads();
        const uint32_t *w = vt + (tid >> 1) * 9 + (tid & 1) * 4;
        ((uint4 *)(codes + kKv8Half))[tid] = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) *(uint32_t *)(codes + (t0 + i) * kKv8Hd + d) = c[i];
    }
    if (tid == 0) {
        ((float *)(seq + l.scales))[2 * blk + isv] = finite ? amax / kTop : __builtin_nanf("");
        if (!isv && b * kKv8Block >= p0) ((float *)(seq + l.weights))[blk] = 0.0f;
    }
    // the last block's new rows join the tail, written by the workgroup that
    // has read the tail (of the first block), so that no other one reads it
    // while it changes
    const int last = (end - 1) / kKv8Block;
    if (b == first) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int t = t0 + i, p = last * kKv8Block + t;
            if (p >= p0 && p < end) {
                u32x2_t y = x[i];
                if (last != first) y = *(const u32x2_t *)(src + (size_t)(p - row0) * kKv8Hd + d);
                *(u32x2_t *)(tail + t * kKv8Hd + d) = y;
            }
        }
    }
}

struct Kv8ReadArgs {
    const uint8_t *cache;
    size_t stride;
    int Hkv, max_seq, nb;
    const int *pos;
    int pos_stride, pos0, n;
    const int *len;
    int len_stride;
    float *k, *v;
};

// One workgroup per (block, K or V, head, sequence): its positions among the
// asked ones as f32 rows, 4 dims of 4 positions a thread as in the append.
// Bound by the rows' bytes: 32 sequences of 1024 positions, 5 heads (43 MB in,
// 168 out) 31 us, 6.7 TB/s.
template <int FMT>
__global__ __launch_bounds__(kKvThreads) void kv8_read_kernel(Kv8ReadArgs a) {
    __shared__ uint32_t vt[kKv8Hd * 9];
    const int z = blockIdx.z, h = blockIdx.y, isv = blockIdx.x & 1, tid = threadIdx.x;
    const int64_t p0 = (int64_t)(a.pos ? a.pos[(size_t)z * a.pos_stride] : 0) + a.pos0;
    int64_t limit = a.max_seq;
    if (a.len) limit = min(limit, (int64_t)a.len[(size_t)z * a.len_stride]);
    const int64_t b = (p0 >> 5) + (blockIdx.x >> 1);   // (a negative position's block too)
    if (b * kKv8Block >= p0 + a.n) return;
    const bool there = b >= 0 && b * kKv8Block < limit;
    const Kv8Layout l = kv8_layout(a.Hkv, a.nb);
    const uint8_t *seq = a.cache + (size_t)z * a.stride;
    const size_t blk = (size_t)h * a.nb + (there ? (int)b : 0);
    const uint8_t *codes = seq + blk * kKv8Codes + (isv ? kKv8Half : 0);
    const float scale = there ? ((const float *)(seq + l.scales))[2 * blk + isv] : 0.0f;
    const int d = (tid & 31) * 4, t0 = (tid >> 5) * 4;
    uint32_t c[4] = {0, 0, 0, 0};
    if (there && isv) {
        const uint4 v = ((const uint4 *)codes)[tid];
        uint32_t *w = vt + (tid >> 1) * 9 + (tid & 1) * 4;
        w[0] = v.x;
        w[1] = v.y;
        w[2] = v.z;
        w[3] = v.w;
        __syncthreads();   // (uniform)
        const uint32_t *at = vt + d * 9 + kv8_v_byte(t0) / 4;
        const uint32_t l0 = __builtin_amdgcn_perm(at[9], at[0], 0x05010400u);
        const uint32_t l1 = __builtin_amdgcn_perm(at[27], at[18], 0x05010400u);
        const uint32_t h0 = __builtin_amdgcn_perm(at[9], at[0], 0x07030602u);
        const uint32_t h1 = __builtin_amdgcn_perm(at[27], at[18], 0x07030602u);
        c[0] = __builtin_amdgcn_perm(l1, l0, 0x05040100u);
        c[1] = __builtin_amdgcn_perm(l1, l0, 0x07060302u);
        c[2] = __builtin_amdgcn_perm(h1, h0, 0x05040100u);
        c[3] = __builtin_amdgcn_perm(h1, h0, 0x07060302u);
    } else if (there) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] = *(const uint32_t *)(codes + (t0 + i) * kKv8Hd + d);
    }
    float *out = (isv ? a.v : a.k) + ((size_t)z * a.Hkv + h) * (size_t)a.n * kKv8Hd;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t p = b * kKv8Block + t0 + i;
        if (p < p0 || p >= p0 + a.n) continue;
        float4 v = make_float4(0, 0, 0, 0);
        if (p >= 0 && p < limit) {
            half2_t x, y;
            kv8_unpack4<FMT>(c[i], x, y);
            v = make_float4((float)x.x * scale, (float)x.y * scale, (float)y.x * scale, (float)y.y * scale);
        }
        *(float4 *)(out + (size_t)(p - p0) * kKv8Hd + d) = v;
    }
}

// ---------------------------------------------------------------------------
// eviction
// ---------------------------------------------------------------------------
// Two launches: the selection (one workgroup per head and sequence), which
// lists the kept blocks in order and moves their scales and weights, then
// the move of codes.  A cache may be compacted in place: kept block j comes
// from a block at j or later, so a workgroup that takes blocks in rising
// groups, reading a whole group before it writes it, overwrites nothing that
// is still to be read.  The selection is a chain of short steps (the weights'
// load, four digits of a radix select, two counts over waves): 5.6 us for 128
// blocks; ranks by comparison of all weights in LDS took 6.6.
struct Kv8EvictArgs {
    const uint8_t *cache;
    uint8_t *dst;
    size_t stride, dst_stride;
    int Hkv, max_seq, nb, dst_nb;
    const int *len;
    int len_stride;
    int *len_out;
    int len_out_stride;
    int budget, sink, recent;
    int *list;     // [batch][Hkv][budget] the kept blocks' old places
    int *head;     // [batch][Hkv][2] kept blocks, the new length
};

constexpr int kEvThreads = 256;

__global__ __launch_bounds__(kEvThreads) void kv8_select_kernel(Kv8EvictArgs a) {
    __shared__ uint32_t hist[256];
    __shared__ uint32_t s_prefix;
    __shared__ int s_rem, s_cnt[2][kEvThreads / 64];
    const int h = blockIdx.x, z = blockIdx.y, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int len = min(max(a.len[(size_t)z * a.len_stride], 0), a.max_seq);
    const int n = kv8_blocks(len), drop = max(n - a.budget, 0);
    const Kv8Layout ls = kv8_layout(a.Hkv, a.nb), ld = kv8_layout(a.Hkv, a.dst_nb);
    const uint8_t *seq = a.cache + (size_t)z * a.stride;
    uint8_t *dseq = a.dst + (size_t)z * a.dst_stride;
    const float2 *sc = (const float2 *)(seq + ls.scales) + (size_t)h * a.nb;
    const float *w = (const float *)(seq + ls.weights) + (size_t)h * a.nb;
    float2 *dsc = (float2 *)(dseq + ld.scales) + (size_t)h * a.dst_nb;
    float *dw = (float *)(dseq + ld.weights) + (size_t)h * a.dst_nb;
    const size_t zh = (size_t)z * a.Hkv + h;
    int *list = a.list + zh * a.budget;
    if (tid == 0) {
        a.head[2 * zh] = n - drop;
        a.head[2 * zh + 1] = len - drop * kKv8Block;
    }
    // the rest of the budget goes to the largest weights between the sink and
    // the recent blocks; a weight that is not a number goes first
    const int lo = a.sink, hi = n - a.recent, k = a.budget - a.sink - a.recent;
    auto key = [&](int i) {
        const float v = w[lo + i];
        return v == v ? smp_ord(v) : 0u;
    };
    uint32_t thr = 0;
    int ties = 0;   // how many blocks of weight thr are kept: the first ones
    if (drop > 0 && k > 0) {
        thr = smp_select<kEvThreads>(hi - lo, k, key, hist, &s_prefix, &s_rem);
        ties = s_rem;
    }
    int kept = 0, equal = 0;   // of the blocks before this group
    for (int i0 = 0; i0 < n; i0 += kEvThreads) {
        const int i = i0 + tid;
        bool keep = i < n, tie = false;
        float2 s = make_float2(0, 0);
        float wt = 0;
        if (i < n) {
            s = sc[i];
            wt = w[i];
            if (drop > 0 && i >= lo && i < hi) {
                const uint32_t o = wt == wt ? smp_ord(wt) : 0u;
                keep = k > 0 && o > thr;
                tie = k > 0 && o == thr;
            }
        }
        const uint64_t below = (1ull << lane) - 1;
        const uint64_t tb = __ballot(tie);
        if (lane == 0) s_cnt[0][wave] = __popcll(tb);
        __syncthreads();
        int before = equal + __popcll(tb & below);
#pragma unroll
        for (int v = 0; v < kEvThreads / 64; ++v) {
            if (v < wave) before += s_cnt[0][v];
            equal += s_cnt[0][v];
        }
        keep |= tie && before < ties;
        const uint64_t kb = __ballot(keep);
        if (lane == 0) s_cnt[1][wave] = __popcll(kb);
        __syncthreads();   // every thread's scales and weights are read
        int at = kept + __popcll(kb & below);
#pragma unroll
        for (int v = 0; v < kEvThreads / 64; ++v) {
            if (v < wave) at += s_cnt[1][v];
            kept += s_cnt[1][v];
        }
        if (keep) {
            list[at] = i;
            dsc[at] = s;
            dw[at] = wt;
        }
    }
}

// A workgroup moves a 256-byte column of a head's kept blocks, 16 blocks a pass
// and 4 passes in flight.  Bound by the codes' bytes, and by the list's and the
// codes' loads one behind the other: 32 sequences of 5 heads and 32 kept blocks
// (89 MB in all) 22.7 us, 3.9 TB/s; with 1 KB columns in a quarter of the
// workgroups 24.0.  The same cut in place, behind a copy that has left the codes in
// the caches: 13.5 us, and the blocks that stay where they are not written.
constexpr int kMvCols = 32;
constexpr int kMvLanes = kKv8Codes / kMvCols / 16;   // 16-byte lanes of a column
constexpr int kMvRows = kKvThreads / kMvLanes;       // blocks per pass
constexpr int kMvUnroll = 4;

__global__ __launch_bounds__(kKvThreads) void kv8_move_kernel(Kv8EvictArgs a) {
    const int col = blockIdx.x, h = blockIdx.y, z = blockIdx.z, tid = threadIdx.x;
    const size_t zh = (size_t)z * a.Hkv + h;
    const int kept = a.head[2 * zh];
    const int *list = a.list + zh * a.budget;
    const bool inplace = a.cache == a.dst;
    const uint8_t *seq = a.cache + (size_t)z * a.stride;
    uint8_t *dseq = a.dst + (size_t)z * a.dst_stride;
    const size_t off = (size_t)col * (kKv8Codes / kMvCols) + (tid % kMvLanes) * 16;
    const uint8_t *src = seq + (size_t)h * a.nb * kKv8Codes + off;
    uint8_t *dst = dseq + (size_t)h * a.dst_nb * kKv8Codes + off;
    for (int j0 = 0; j0 < kept; j0 += kMvRows * kMvUnroll) {
        u32x4_t v[kMvUnroll];
        int from[kMvUnroll];
#pragma unroll
        for (int u = 0; u < kMvUnroll; ++u)   // (clamped; not written past the kept ones)
            if (j0 + u * kMvRows < kept) from[u] = list[min(j0 + u * kMvRows + tid / kMvLanes, kept - 1)];
#pragma unroll
        for (int u = 0; u < kMvUnroll; ++u)
            if (j0 + u * kMvRows < kept) v[u] = *(const u32x4_t *)(src + (size_t)from[u] * kKv8Codes);
        if (inplace) __syncthreads();   // the group is read before any of it is overwritten
#pragma unroll
        for (int u = 0; u < kMvUnroll; ++u) {
            const int j = j0 + u * kMvRows + tid / kMvLanes;
            if (j < kept && !(inplace && from[u] == j)) *(u32x4_t *)(dst + (size_t)j * kKv8Codes) = v[u];
        }
    }
    if (!inplace) {   // the newest block's f16 rows, 16 KB over the columns
        const Kv8Layout ls = kv8_layout(a.Hkv, a.nb), ld = kv8_layout(a.Hkv, a.dst_nb);
        const size_t t = (size_t)h * 2 * kKv8Half * 2 + (size_t)col * (16384 / kMvCols) + tid * 16;
        if (tid < 1024 / kMvCols) *(uint4 *)(dseq + ld.tails + t) = *(const uint4 *)(seq + ls.tails + t);
    }
    if (col == 0 && h == 0 && tid == 0) a.len_out[(size_t)z * a.len_out_stride] = a.head[2 * zh + 1];
}

}  // namespace oxb

using namespace oxb;

extern "C" size_t oxb_kv8_bytes(int Hkv, int hd, int max_seq) {
    if (Hkv < 1 || Hkv > 4096 || hd != kKv8Hd || max_seq < 1 || max_seq > OXB_KV8_MAX_SEQ) return 0;
    return kv8_layout(Hkv, kv8_blocks(max_seq)).bytes;
}

extern "C" int oxb_kv8_append(void *cache, size_t cache_stride, int fmt, int batch, int Hkv, int hd,
                              int max_seq, const uint16_t *k, const uint16_t *v, size_t src_stride,
                              size_t src_head_stride, int src_at_pos, const int *pos, int pos_stride,
                              int pos0, int n, const int *counts, void *stream) {
    clear_error();
    if (kv8_check(cache, cache_stride, fmt, batch, Hkv, hd, max_seq)) return -1;
    OXB_REQUIRE(k && v, "kv8 append: k or v is NULL");
    OXB_REQUIRE((((uintptr_t)k | (uintptr_t)v) & 15) == 0 && ((src_stride | src_head_stride) & 7) == 0,
                "kv8 append: k and v rows must be 16-byte aligned");
    OXB_REQUIRE(n >= 1 && n <= max_seq, "kv8 append: %d rows", n);
    OXB_REQUIRE(pos_stride >= 0, "kv8 append: pos stride %d", pos_stride);
    OXB_REQUIRE(pos || (pos0 >= 0 && pos0 <= max_seq - n), "kv8 append: rows %d..%d of %d positions",
                pos0, pos0 + n - 1, max_seq);
    Kv8AppendArgs a{(uint8_t *)cache, cache_stride, Hkv, max_seq, kv8_blocks(max_seq), k, v,
                    src_stride, src_head_stride, src_at_pos != 0, pos, pos_stride, pos0, n, counts};
    // the most blocks that n rows touch: 31 rows may stand before them
    const int span = pos ? kv8_blocks(n + kKv8Block - 1)
                         : (pos0 + n - 1) / kKv8Block - pos0 / kKv8Block + 1;
    const dim3 grid(2 * span, Hkv, batch);
    if (fmt == OXB_KV8_INT8)
        hipLaunchKernelGGL(kv8_append_kernel<OXB_KV8_INT8>, grid, dim3(kKvThreads), 0,
                           (hipStream_t)stream, a);
    else
        hipLaunchKernelGGL(kv8_append_kernel<OXB_KV8_E4M3>, grid, dim3(kKvThreads), 0,
                           (hipStream_t)stream, a);
    OXB_CHECK_HIP(hipGetLastError());
    return 0;
}

extern "C" int oxb_kv8_read(const void *cache, size_t cache_stride, int fmt, int batch, int Hkv,
                            int hd, int max_seq, const int *pos, int pos_stride, int pos0, int n,
                            const int *len, int len_stride, float *k, float *v, void *stream) {
    clear_error();
    if (kv8_check(cache, cache_stride, fmt, batch, Hkv, hd, max_seq)) return -1;
    OXB_REQUIRE(k && v && (((uintptr_t)k | (uintptr_t)v) & 15) == 0,
                "kv8 read: k or v is NULL or not 16-byte aligned");
    OXB_REQUIRE(n >= 1 && n <= OXB_KV8_MAX_SEQ, "kv8 read: %d rows", n);
    OXB_REQUIRE(pos_stride >= 0 && len_stride >= 0, "kv8 read: stride %d, %d", pos_stride, len_stride);
    Kv8ReadArgs a{(const uint8_t *)cache, cache_stride, Hkv, max_seq, kv8_blocks(max_seq), pos,
                  pos_stride, pos0, n, len, len_stride, k, v};
    const dim3 grid(2 * kv8_blocks(n + kKv8Block - 1), Hkv, batch);
    if (fmt == OXB_KV8_INT8)
        hipLaunchKernelGGL(kv8_read_kernel<OXB_KV8_INT8>, grid, dim3(kKvThreads), 0,
                           (hipStream_t)stream, a);
    else
        hipLaunchKernelGGL(kv8_read_kernel<OXB_KV8_E4M3>, grid, dim3(kKvThreads), 0,
                           (hipStream_t)stream, a);
    OXB_CHECK_HIP(hipGetLastError());
    return 0;
}

extern "C" size_t oxb_kv8_evict_ws_bytes(int batch, int Hkv, int max_seq, int budget) {
    if (batch < 1 || Hkv < 1 || max_seq < 1 || max_seq > OXB_KV8_MAX_SEQ || budget < 1) return 0;
    budget = std::min(budget, kv8_blocks(max_seq));   // no more are kept
    return kv8_align((size_t)batch * Hkv * budget * 4) + kv8_align((size_t)batch * Hkv * 8);
}

extern "C" int oxb_kv8_evict(const void *cache, size_t cache_stride, int max_seq, void *dst,
                             size_t dst_stride, int dst_max_seq, const int *len, int len_stride,
                             int *len_out, int len_out_stride, int batch, int Hkv, int hd, int budget,
                             int sink, int recent, void *ws, size_t ws_bytes, void *stream) {
    clear_error();
    if (kv8_check(cache, cache_stride, OXB_KV8_INT8, batch, Hkv, hd, max_seq) ||
        kv8_check(dst, dst_stride, OXB_KV8_INT8, batch, Hkv, hd, dst_max_seq))
        return -1;
    OXB_REQUIRE(len && len_out, "kv8 evict: len or len_out is NULL");
    OXB_REQUIRE(len_stride >= 0 && len_out_stride >= (batch > 1 ? 1 : 0),
                "kv8 evict: length stride %d, %d", len_stride, len_out_stride);
    OXB_REQUIRE(budget >= 1 && sink >= 0 && recent >= 1 && sink <= budget && recent <= budget - sink,
                "kv8 evict: a budget of %d blocks does not hold %d first and %d last ones (at least 1)",
                budget, sink, recent);
    const int nb = kv8_blocks(max_seq), dnb = kv8_blocks(dst_max_seq);
    OXB_REQUIRE(dst_max_seq >= max_seq || dst_max_seq / kKv8Block >= budget,
                "kv8 evict: %d positions do not hold a budget of %d blocks", dst_max_seq, budget);
    if (cache == dst) {
        OXB_REQUIRE(max_seq == dst_max_seq && (batch == 1 || cache_stride == dst_stride),
                    "kv8 evict: a cache cut in place keeps its max_seq and stride");
    } else {
        const uintptr_t s = (uintptr_t)cache, d = (uintptr_t)dst;
        const size_t sb = (batch - 1) * cache_stride + kv8_layout(Hkv, nb).bytes;
        const size_t db = (batch - 1) * dst_stride + kv8_layout(Hkv, dnb).bytes;
        OXB_REQUIRE(s + sb <= d || d + db <= s, "kv8 evict: dst overlaps the cache");
    }
    OXB_REQUIRE(ws && ((uintptr_t)ws & 15) == 0 &&
                    ws_bytes >= oxb_kv8_evict_ws_bytes(batch, Hkv, max_seq, budget),
                "kv8 evict: workspace is NULL, unaligned or %zu bytes < %zu", ws_bytes,
                oxb_kv8_evict_ws_bytes(batch, Hkv, max_seq, budget));
    budget = std::min(budget, nb);   // (then nothing is dropped)
    Kv8EvictArgs a{(const uint8_t *)cache, (uint8_t *)dst, cache_stride, dst_stride, Hkv, max_seq, nb,
                   dnb, len, len_stride, len_out, len_out_stride, budget, sink, recent, (int *)ws,
                   (int *)((char *)ws + kv8_align((size_t)batch * Hkv * budget * 4))};
    hipStream_t s = (hipStream_t)stream;
    hipLaunchKernelGGL(kv8_select_kernel, dim3(Hkv, batch), dim3(kEvThreads), 0, s, a);
    OXB_CHECK_HIP(hipGetLastError());
    hipLaunchKernelGGL(kv8_move_kernel, dim3(kMvCols, Hkv, batch), dim3(kKvThreads), 0, s, a);
    OXB_CHECK_HIP(hipGetLastError());
    return 0;
}

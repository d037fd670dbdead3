// Attention over the 8-bit KV cache for gfx950 (layout: kv8.h): one decode
// token of a batch, and causal prefill of n tokens of a sequence, each with
// the blocks' attention weights accumulated on request.  No counterpart in the
// reference, whose attention reads f32 rows (nn/attention.rs:109-118).
//
//   out = sum_t p_t V_t,  p = softmax over the visible t of q.K_t / sqrt(128)
//
// One pass over the cache with a running reference m of the row's maximum:
// p' = 2^(x - m), l += p', O += p' V, and O and l are rescaled when a score
// passes m by 8 (in log2 units) -- a fixed m is as good as the exact maximum as
// long as nothing overflows, and the test costs less than a maximum over lanes
// for every tile.
//
// Arithmetic: codes are exact in f16 (8 bits), so both products run on f16
// MFMA with f32 sums.  The f32 operands, q and p', go in as two f16 parts
// hi + lo (22 bits of each value; one part alone, 11 bits, would cost the f32
// result three digits): q's row is first scaled by a power of two to a maximum
// in [2^13, 2^14), p' is at most 2^14, so that lo's own rounding stays 2^-25
// absolute, 2^-39 of the largest.  K's block scale multiplies the scores.  V's
// goes into p' for the product only, which has a reference of its own, m2 over
// x + e (2^e the scale's power of two): p' keeps its 22 bits where p V is large,
// not where p is, however far apart the blocks' values lie.  O = sum of
// 2^(x - m2) vs V is then o / (l r), r = 2^(m - m2).
#include "kv8.h"

namespace oxb {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr float kScoreUnit = 1.44269504088896340736f * 0.08838834764831844f;   // log2(e) / sqrt(128)
constexpr float kStep = 8.0f;      // a score may pass the reference by this much
constexpr int kQExp = 14;          // q rows are scaled below 2^kQExp

__device__ __forceinline__ float kv8_ror8(float v) {   // lane i of 16 takes lane i ^ 8
    const int i = __float_as_int(v);
    return __int_as_float(__builtin_amdgcn_update_dpp(i, i, 0x128, 0xf, 0xf, false));
}

// A block's V scale as a power of two not below it; scales of 0 and NaN as one
// below every other (f16's smallest value over 448 is 2^-33).
__device__ __forceinline__ float kv8_scale_exp(float s) {
    return s > 0.0f ? (float)__builtin_amdgcn_frexp_expf(s) : -40.0f;
}

// The references of a row and what they make of a tile: mx, mx2 are the lane's
// largest x and x + e.  Where any row of the wave passes a reference by kStep,
// all take their row's maxima (over LANES lane groups) and al, al2 are what l
// and o shrink by.
struct Kv8Ref {
    float m = -__builtin_inff(), m2 = -__builtin_inff(), r = 1.0f;
    __device__ __forceinline__ bool passed(float mx, float mx2) const {
        return __any(mx > m + kStep || mx2 > m2 + kStep || (m == -__builtin_inff() && mx > m));
    }
    template <int LANES>
    __device__ __forceinline__ void raise(float mx, float mx2, float &al, float &al2) {
#pragma unroll
        for (int s = 64 / LANES; s < 64; s <<= 1) {
            mx = fmaxf(mx, __shfl_xor(mx, s, 64));
            mx2 = fmaxf(mx2, __shfl_xor(mx2, s, 64));
        }
        const float n = fmaxf(m, mx), n2 = fmaxf(m2, mx2);
        al = n == m ? 1.0f : __builtin_amdgcn_exp2f(m - n);
        al2 = n2 == m2 ? 1.0f : __builtin_amdgcn_exp2f(m2 - n2);
        m = n;
        m2 = n2;
        // (a row that has seen nothing, or nothing but NaN: any r will do)
        r = n == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(n - n2);
    }
    __device__ __forceinline__ float off() const { return m == -__builtin_inff() ? 0.0f : m; }
};

// The exponent that scales a row of maximum a below 2^kQExp (0 and values that
// are not finite: none).
__device__ __forceinline__ int kv8_row_exp(float a) {
    return a > 0.0f && a < __builtin_inff() ? __builtin_amdgcn_frexp_expf(a) - kQExp : 0;
}

// ---------------------------------------------------------------------------
// decode
// ---------------------------------------------------------------------------
// Workgroup: four waves over a run of blocks, wave w taking every fourth; one
// KV head, up to 8 of its query heads (K and V are read once for all of them).
// 16x16x32 MFMA: the 16 columns are the 8 heads' hi and lo parts, for q and
// for p' alike, so the two-part products cost nothing over one.
//   scores: A = 16 K rows x 32 dims, B = q; column c + (c ^ 8) is the score.
//   K rows are taken in an order that leaves lane group g (of 4) the scores of
//   the positions that bytes 8g .. 8g + 7 of a V row hold;
//   P.V: A = 16 dims x the block's 32 positions (8 bytes a lane), B = the lane's
//   own eight p' -- no exchange between lanes.
constexpr int kDecWaves = 4;
constexpr int kDecThreads = 64 * kDecWaves;
constexpr int kDecRows = 8;            // query heads of a workgroup
constexpr int kDecQs = kKv8Hd + 8;     // q row stride in LDS (f16)
constexpr float kDecBase = 6.0f;       // p' <= 2^(6 + kStep)

struct Kv8DecodeArgs {
    const float *q;
    uint8_t *cache;
    size_t stride;
    const int *pos;
    int pos_stride, H, Hkv, G, HC, max_seq, nb, splits, weights;
    float *out;
    float2 *ml;      // [batch][Hkv * HC][splits][8] reference and sum
    float *o;        // [batch][Hkv * HC][splits][8][128]
    float2 *bw;      // [batch][H][nb] a block's sum of p' and its reference
};

__device__ __forceinline__ int kv8_len(const Kv8DecodeArgs &a, int z) {
    const int64_t p = (int64_t)a.pos[(size_t)z * a.pos_stride] + 1;
    return (int)(p < 0 ? 0 : p > a.max_seq ? a.max_seq : p);
}
// Blocks of a workgroup: the sequence's blocks over all workgroups, at least
// one per wave.
__device__ __forceinline__ int kv8_per(int nblk, int splits) {
    return max(kDecWaves, (nblk + splits - 1) / splits);
}

template <int FMT, bool WEIGHTS>
__global__ __launch_bounds__(kDecThreads) void kv8_decode_kernel(Kv8DecodeArgs a) {
    __shared__ _Float16 sq[2 * kDecRows * kDecQs];
    __shared__ float sqs[kDecRows];
    __shared__ float2 sml[kDecWaves][kDecRows];
    __shared__ float4 so[kDecWaves][kDecRows][kKv8Hd / 4];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int z = blockIdx.z, hv = blockIdx.y, kvh = hv / a.HC, split = blockIdx.x;
    const int g0 = kvh * a.G + (hv % a.HC) * kDecRows;      // first query head
    const int ng = min(kDecRows, (kvh + 1) * a.G - g0);
    const int len = kv8_len(a, z), nblk = kv8_blocks(len), per = kv8_per(nblk, a.splits);
    const int b0 = split * per, b1 = min(nblk, b0 + per);
    const bool direct = a.splits == 1 && !WEIGHTS;
    const int orow = tid >> 5, od = (tid & 31) * 4;         // the row and dims a thread writes
    float *out = a.out + ((size_t)z * a.H + g0 + orow) * kKv8Hd + od;
    if (b0 >= b1) {
        if (direct && orow < ng) *(float4 *)out = make_float4(0, 0, 0, 0);
        return;
    }
    {   // q rows: scaled, split, and their score units
        float4 v = make_float4(0, 0, 0, 0);
        if (orow < ng) v = *(const float4 *)(a.q + ((size_t)z * a.H + g0 + orow) * kKv8Hd + od);
        float m = fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w)));
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) m = fmaxf(m, __shfl_xor(m, s, 64));
        const int e = kv8_row_exp(m);
        const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float x = ldexpf(f[j], -e);
            const _Float16 hi = (_Float16)x;
            sq[orow * kDecQs + od + j] = hi;
            sq[(orow + kDecRows) * kDecQs + od + j] = (_Float16)(x - (float)hi);
        }
        if ((tid & 31) == 0) sqs[orow] = ldexpf(kScoreUnit, e);
    }
    __syncthreads();
    const int rr = lane & 15, g = lane >> 4;
    half8_t qf[4];
#pragma unroll
    for (int s = 0; s < 4; ++s)
        qf[s] = *(const half8_t *)(sq + rr * kDecQs + 64 * (s >> 1) + 16 * g + 8 * (s & 1));
    const float qs = sqs[rr & 7];

    const Kv8Layout l = kv8_layout(a.Hkv, a.nb);
    const uint8_t *seq = a.cache + (size_t)z * a.stride;
    const uint8_t *codes = seq + (size_t)kvh * a.nb * kKv8Codes;
    const float2 *sc = (const float2 *)(seq + l.scales) + (size_t)kvh * a.nb;
    // K row of this lane in 16-row tile 0 (tile 1: 8 positions on), V bytes of dim rr
    const int krow = ((rr >> 2) & 1) * 16 + (rr >> 3) * 4 + (rr & 3);
    const int koff = krow * kKv8Hd + 16 * g, voff = kKv8Half + rr * kKv8Block + 8 * g;

    struct Blk {
        uint4 k[4];
        uint2 v[8];
        float2 s;
    };
    auto load = [&](int b) {
        Blk x;
        const uint8_t *p = codes + (size_t)b * kKv8Codes;
#pragma unroll
        for (int i = 0; i < 4; ++i)   // tile i / 2, dims 64 (i % 2) ..
            x.k[i] = *(const uint4 *)(p + koff + (i >> 1) * 8 * kKv8Hd + (i & 1) * 64);
#pragma unroll
        for (int i = 0; i < 8; ++i) x.v[i] = *(const uint2 *)(p + voff + i * 16 * kKv8Block);
        x.s = sc[b];
        return x;
    };

    f32x4 o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = f32x4{0, 0, 0, 0};
    Kv8Ref ref;
    float lsum = 0.0f;

    Blk cur;
    if (b0 + wave < b1) cur = load(b0 + wave);
    for (int b = b0 + wave; b < b1; b += kDecWaves) {
        const Blk nxt = load(min(b + kDecWaves, b1 - 1));
        f32x4 s0{0, 0, 0, 0}, s1{0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const uint4 k0 = cur.k[s >> 1], k1 = cur.k[2 + (s >> 1)];
            const half8_t f0 = (s & 1) ? kv8_unpack8<FMT>(k0.z, k0.w) : kv8_unpack8<FMT>(k0.x, k0.y);
            const half8_t f1 = (s & 1) ? kv8_unpack8<FMT>(k1.z, k1.w) : kv8_unpack8<FMT>(k1.x, k1.y);
            s0 = __builtin_amdgcn_mfma_f32_16x16x32_f16(f0, qf[s], s0, 0, 0, 0);
            s1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(f1, qf[s], s1, 0, 0, 0);
        }
        float x[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = s0[i] + kv8_ror8(s0[i]);
            x[4 + i] = s1[i] + kv8_ror8(s1[i]);
        }
        // lane's positions in the block: slot 4 t + i is (g & 1) 16 + 8 t + (g >> 1) 4 + i
        const int left = len - b * kKv8Block - ((g & 1) * 16 + (g >> 1) * 4);
        const bool partial = len - b * kKv8Block < kKv8Block;
        const float ck = cur.s.x * qs;
        float mx = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float v = x[i] * ck;
            if (!partial || (i >> 2) * 8 + (i & 3) < left) mx = fmaxf(mx, v);
        }
        const float mx2 = mx + kv8_scale_exp(cur.s.y);
        if (ref.passed(mx, mx2)) {
            float al, al2;
            ref.raise<4>(mx, mx2, al, al2);
            lsum *= al;
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] *= al2;
        }
        const float moff = ref.off() - kDecBase, vs = cur.s.y * ref.r;
        float ps = 0.0f;
        half8_t pf;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float p = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], ck, -moff));
            if (partial && (i >> 2) * 8 + (i & 3) >= left) p = 0.0f;
            ps += p;
            p *= vs;
            const _Float16 hi = (_Float16)p;
            pf[i] = rr < kDecRows ? hi : (_Float16)(p - (float)hi);
        }
        lsum += ps;
        if constexpr (WEIGHTS) {
            ps += __shfl_xor(ps, 16, 64);
            ps += __shfl_xor(ps, 32, 64);
            if (lane < ng) a.bw[((size_t)z * a.H + g0 + lane) * a.nb + b] = make_float2(ps, moff);
        }
        if (partial) {   // bytes behind the last position may hold anything
            uint32_t mk[2] = {0, 0};
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if ((i >> 2) * 8 + (i & 3) < left) mk[i >> 2] |= 0xffu << (8 * (i & 3));
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                cur.v[i].x &= mk[0];
                cur.v[i].y &= mk[1];
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
            o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kv8_unpack8<FMT>(cur.v[i].x, cur.v[i].y), pf,
                                                          o[i], 0, 0, 0);
        cur = nxt;
    }
    // the four waves' parts
    lsum += __shfl_xor(lsum, 16, 64);
    lsum += __shfl_xor(lsum, 32, 64);
    const bool some = b0 + wave < b1;
    if (lane < kDecRows)
        sml[wave][lane] = make_float2(some ? ref.off() - kDecBase : -__builtin_inff(), lsum);
    const float ri = 1.0f / ref.r;   // o in l's units
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float4 t;
        t.x = (o[i][0] + kv8_ror8(o[i][0])) * ri;
        t.y = (o[i][1] + kv8_ror8(o[i][1])) * ri;
        t.z = (o[i][2] + kv8_ror8(o[i][2])) * ri;
        t.w = (o[i][3] + kv8_ror8(o[i][3])) * ri;
        if (rr < kDecRows) so[wave][rr][4 * i + g] = t;
    }
    __syncthreads();
    float M = -__builtin_inff();
#pragma unroll
    for (int w = 0; w < kDecWaves; ++w) M = fmaxf(M, sml[w][orow].x);
    float lt = 0.0f;
    float4 t = make_float4(0, 0, 0, 0);
#pragma unroll
    for (int w = 0; w < kDecWaves; ++w) {
        const float2 p = sml[w][orow];
        const float f = __builtin_amdgcn_exp2f(p.x - M);
        const float4 v = so[w][orow][od >> 2];
        lt = __builtin_fmaf(p.y, f, lt);
        t.x = __builtin_fmaf(v.x, f, t.x);
        t.y = __builtin_fmaf(v.y, f, t.y);
        t.z = __builtin_fmaf(v.z, f, t.z);
        t.w = __builtin_fmaf(v.w, f, t.w);
    }
    if (direct) {
        if (orow < ng) *(float4 *)out = make_float4(t.x / lt, t.y / lt, t.z / lt, t.w / lt);
        return;
    }
    const size_t part = (((size_t)z * a.Hkv * a.HC + hv) * a.splits + split) * kDecRows + orow;
    *(float4 *)(a.o + part * kKv8Hd + od) = t;
    if (od == 0) a.ml[part] = make_float2(M, lt);
}

// Joins the splits: workgroup y < H writes a query head's output; the others
// add to 128 blocks' weights each (their KV head's query heads in order).
constexpr int kJoinThreads = 128;
__global__ __launch_bounds__(kJoinThreads) void kv8_decode_join_kernel(Kv8DecodeArgs a) {
    const int z = blockIdx.y, tid = threadIdx.x;
    const int len = kv8_len(a, z), nblk = kv8_blocks(len), per = kv8_per(nblk, a.splits);
    const int ns = (nblk + per - 1) / per;
    auto row = [&](int h) {   // the first split's part of a query head
        const int kvh = h / a.G, i = h % a.G, hv = kvh * a.HC + i / kDecRows;
        return (((size_t)z * a.Hkv * a.HC + hv) * a.splits) * kDecRows + i % kDecRows;
    };
    auto total = [&](size_t r, float &M, float &lt) {
        M = -__builtin_inff();
        for (int s = 0; s < ns; ++s) M = fmaxf(M, a.ml[r + (size_t)s * kDecRows].x);
        lt = 0.0f;
        for (int s = 0; s < ns; ++s) {
            const float2 p = a.ml[r + (size_t)s * kDecRows];
            lt = __builtin_fmaf(p.y, __builtin_amdgcn_exp2f(p.x - M), lt);
        }
    };
    if ((int)blockIdx.x < a.H) {
        const int h = blockIdx.x;
        float *out = a.out + ((size_t)z * a.H + h) * kKv8Hd + tid;
        if (len == 0) {
            *out = 0.0f;
            return;
        }
        const size_t r = row(h);
        float M, lt, t = 0.0f;
        total(r, M, lt);
        for (int s = 0; s < ns; ++s) {
            const size_t p = r + (size_t)s * kDecRows;
            t = __builtin_fmaf(a.o[p * kKv8Hd + tid], __builtin_amdgcn_exp2f(a.ml[p].x - M), t);
        }
        *out = t / lt;
        return;
    }
    const int chunks = (a.nb + kJoinThreads - 1) / kJoinThreads;
    const int c = blockIdx.x - a.H, kvh = c / chunks, b = (c % chunks) * kJoinThreads + tid;
    if (b >= nblk) return;
    float add = 0.0f;
    for (int i = 0; i < a.G; ++i) {
        const int h = kvh * a.G + i;
        float M, lt;
        total(row(h), M, lt);
        const float2 p = a.bw[((size_t)z * a.H + h) * a.nb + b];
        add += p.x * __builtin_amdgcn_exp2f(p.y - M) / lt;
    }
    uint8_t *seq = a.cache + (size_t)z * a.stride;
    float *w = (float *)(seq + kv8_layout(a.Hkv, a.nb).weights) + (size_t)kvh * a.nb + b;
    *w += add;
}

// Workgroups per KV head and sequence: about four per CU over the launch, none
// with fewer than one block per wave.
static int decode_splits(int batch, int Hkv, int HC, int nb) {
    const int64_t target = 4 * (int64_t)device_cus(), rows = (int64_t)batch * Hkv * HC;
    int64_t s = (target + rows - 1) / rows;
    const int64_t most = (nb + kDecWaves - 1) / kDecWaves;
    if (s > most) s = most;
    return (int)(s < 1 ? 1 : s);
}

struct DecodeWs {
    size_t ml, o, bw, bytes;
};
static DecodeWs decode_ws(int batch, int H, int Hkv, int nb) {
    const int HC = (H / Hkv + kDecRows - 1) / kDecRows;
    const size_t parts = (size_t)batch * Hkv * HC * decode_splits(batch, Hkv, HC, nb) * kDecRows;
    DecodeWs w;
    w.ml = 0;
    w.o = kv8_align(parts * 8);
    w.bw = w.o + kv8_align(parts * kKv8Hd * 4);
    w.bytes = w.bw + kv8_align((size_t)batch * H * nb * 8);
    return w;
}

// ---------------------------------------------------------------------------
// prefill
// ---------------------------------------------------------------------------
// Rows of a KV head are (token, query head of the group) pairs, token-major, so
// that a K/V tile serves all of the group's heads.  A workgroup takes 128 rows,
// 32 per wave, and a run of 64-position tiles.  Each tile's codes are unpacked
// to f16 once, by all four waves, into LDS in the order the MFMA operands are
// read (every read is 1 KB contiguous); the next tile's codes are in flight
// meanwhile.
//   scores: 32x32x16 MFMA, A = 32 K rows, B = q (in registers, hi and lo);
//   P.V: A = 32 dims x 16 positions, B = the lane's own p' (kv8_v_byte's order).
// Rows that see different lengths finish at different tiles; long rows are
// split over workgroups where the rows alone leave CUs idle, and joined after.
constexpr int kPreWaves = 4;
constexpr int kPreThreads = 64 * kPreWaves;
constexpr int kPreRows = 32 * kPreWaves;
constexpr int kPreTile = 2 * kKv8Block;
constexpr int kPreTileBytes = 2 * 2 * kKv8Codes;   // a tile's K and V as f16
constexpr float kPreBase = 6.0f;                   // p' <= 2^(6 + kStep)

struct Kv8PrefillArgs {
    const float *q;
    uint8_t *cache;
    int n, pos0, H, Hkv, G, nb, rows, splits, per, weights;
    float *out;
    float2 *ml;     // [splits][Hkv][rows]
    float *o;       // [splits][Hkv][rows][128]
    float2 *lse;    // [Hkv][rows32] log2 of the row's softmax sum, its score unit
    uint4 *qf;      // [Hkv][rows32 / 32][8][2][64] q as MFMA operands
    float *part;    // [row splits][Hkv][blocks of the call] weights
    int rsplits;
};

__host__ __device__ inline int pre_rows32(int rows) { return (rows + 31) & ~31; }

template <int FMT>
__global__ __launch_bounds__(kPreThreads, 2) void kv8_prefill_kernel(Kv8PrefillArgs a) {
    extern __shared__ uint4 sbuf[];   // two tiles: K operands [2][8][64], V operands [2][4][2][64]
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kvh = blockIdx.y;
    const int rtile = gridDim.x - 1 - blockIdx.x;   // the longest rows first
    const int split = blockIdx.z;
    const int r0 = rtile * kPreRows, row = r0 + wave * 32 + (lane & 31), h = lane >> 5;
    const int total = a.pos0 + a.n;
    const int lastrow = min(r0 + kPreRows, a.rows) - 1;
    const int seen = a.pos0 + lastrow / a.G + 1;    // positions the tile's last row sees
    const int tiles = (seen + kPreTile - 1) / kPreTile;
    const int t0 = split * a.per, t1 = min(tiles, t0 + a.per);
    if (t0 >= t1) return;
    const bool live = row < a.rows;
    const int tok = min(row, a.rows - 1) / a.G, head = kvh * a.G + min(row, a.rows - 1) % a.G;
    const int qpos = a.pos0 + tok;

    // q: dims 32 c + 16 h + 8 e + j are operand s = 2 c + e
    half8_t qh[8], ql[8];
    float qs;
    {
        const float *q = a.q + ((size_t)tok * a.H + head) * kKv8Hd + 16 * h;
        float m = 0.0f;
        float v[64];
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float4 f = *(const float4 *)(q + 32 * c + 4 * j);
                v[16 * c + 4 * j] = f.x;
                v[16 * c + 4 * j + 1] = f.y;
                v[16 * c + 4 * j + 2] = f.z;
                v[16 * c + 4 * j + 3] = f.w;
            }
#pragma unroll
        for (int i = 0; i < 64; ++i) m = fmaxf(m, fabsf(v[i]));
        m = fmaxf(m, __shfl_xor(m, 32, 64));
        const int e = kv8_row_exp(m);
        qs = ldexpf(kScoreUnit, e);
#pragma unroll
        for (int s = 0; s < 8; ++s)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float x = ldexpf(v[8 * s + j], -e);
                const _Float16 hi = (_Float16)x;
                qh[s][j] = hi;
                ql[s][j] = (_Float16)(x - (float)hi);
            }
    }
    if (a.weights && split == 0) {
        const int r32 = pre_rows32(a.rows);
        if (r0 + wave * 32 < r32) {
            uint4 *f = a.qf + (((size_t)kvh * r32 + r0 + wave * 32) / 32) * (8 * 2 * 64) + lane;
#pragma unroll
            for (int s = 0; s < 8; ++s) {
                f[(2 * s) * 64] = __builtin_bit_cast(uint4, qh[s]);
                f[(2 * s + 1) * 64] = __builtin_bit_cast(uint4, ql[s]);
            }
            if (h == 0) a.lse[(size_t)kvh * r32 + row].y = qs;
        }
    }

    const Kv8Layout l = kv8_layout(a.Hkv, a.nb);
    const uint8_t *codes = a.cache + (size_t)kvh * a.nb * kKv8Codes;
    const float2 *sc = (const float2 *)(a.cache + l.scales) + (size_t)kvh * a.nb;
    const int lastblk = kv8_blocks(total) - 1;
    // wave 0, 1: K of the tile's blocks; 2, 3: V
    const int lb = wave & 1, isv = wave >> 1;
    const int goff = isv ? kKv8Half + (lane & 31) * kKv8Block + 16 * h : (lane & 31) * kKv8Hd + 16 * h;
    const int gstep = isv ? 32 * kKv8Block : 32;
    uint4 c[4];
    auto fetch = [&](int t) {
        const int b = min(2 * t + lb, lastblk);
        const uint8_t *p = codes + (size_t)b * kKv8Codes + goff;
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] = *(const uint4 *)(p + i * gstep);
    };
    auto stage = [&](int t, int buf) {
        const int b = min(2 * t + lb, lastblk), left = total - b * kKv8Block;
        if (isv && left < kKv8Block) {   // bytes behind the last position may hold anything
            uint32_t mk[4] = {0, 0, 0, 0};
#pragma unroll
            for (int p = 0; p < 16; ++p)   // byte 16 h + p: position 16 (p / 8) + 8 (p / 4 % 2) + 4 h + p % 4
                if (16 * (p >> 3) + 8 * (p >> 2 & 1) + 4 * h + (p & 3) < left)
                    mk[p >> 2] |= 0xffu << (8 * (p & 3));
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                c[i].x &= mk[0];
                c[i].y &= mk[1];
                c[i].z &= mk[2];
                c[i].w &= mk[3];
            }
        }
        // operands 2 i and 2 i + 1 of the block
        uint4 *s = sbuf + buf * (kPreTileBytes / 16) + (isv * 2 + lb) * 512 + lane;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            s[(2 * i) * 64] = __builtin_bit_cast(uint4, kv8_unpack8<FMT>(c[i].x, c[i].y));
            s[(2 * i + 1) * 64] = __builtin_bit_cast(uint4, kv8_unpack8<FMT>(c[i].z, c[i].w));
        }
    };

    f32x16 o[4];
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;
    Kv8Ref ref;
    float lsum = 0.0f;
    const int wseen = a.pos0 + min(r0 + wave * 32 + 31, a.rows - 1) / a.G + 1;   // the wave's last row
    const int wfull = a.pos0 + min(r0 + wave * 32, a.rows - 1) / a.G + 1;        // its first row

    fetch(t0);
    stage(t0, 0);
    __syncthreads();
    for (int t = t0; t < t1; ++t) {
        const int buf = (t - t0) & 1;
        if (t + 1 < t1) fetch(t + 1);
        if (t * kPreTile < wseen) {   // uniform over the wave
            const uint4 *kb = sbuf + buf * (kPreTileBytes / 16) + lane;
            const uint4 *vb = kb + 1024;
            f32x16 s[2];
#pragma unroll
            for (int b = 0; b < 2; ++b) {
#pragma unroll
                for (int i = 0; i < 16; ++i) s[b][i] = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const half8_t k = __builtin_bit_cast(half8_t, kb[(b * 8 + i) * 64]);
                    s[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, qh[i], s[b], 0, 0, 0);
                    s[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, ql[i], s[b], 0, 0, 0);
                }
            }
            const float2 sc0 = sc[min(2 * t, lastblk)], sc1 = sc[min(2 * t + 1, lastblk)];
            const float ck[2] = {sc0.x * qs, sc1.x * qs};
            // positions of the lane's scores: 32 b + (i & 3) + 8 (i >> 2) + 4 h
            const bool masked = (t + 1) * kPreTile > wfull;
            const int left = qpos + 1 - t * kPreTile - 4 * h;
            float mb[2];
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                mb[b] = -__builtin_inff();
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float v = s[b][i] * ck[b];
                    if (!masked || 32 * b + (i & 3) + 8 * (i >> 2) < left) mb[b] = fmaxf(mb[b], v);
                }
            }
            const float mx = fmaxf(mb[0], mb[1]);
            const float mx2 = fmaxf(mb[0] + kv8_scale_exp(sc0.y), mb[1] + kv8_scale_exp(sc1.y));
            if (ref.passed(mx, mx2)) {
                float al, al2;
                ref.raise<2>(mx, mx2, al, al2);
                lsum *= al;
#pragma unroll
                for (int d = 0; d < 4; ++d)
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[d][i] *= al2;
            }
            const float moff = ref.off() - kPreBase;
            const float vs[2] = {sc0.y * ref.r, sc1.y * ref.r};
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int gr = 0; gr < 2; ++gr) {
                    half8_t ph, pl;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int i = 8 * gr + j;
                        float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][i], ck[b], -moff));
                        const bool hide = masked && 32 * b + (i & 3) + 8 * (i >> 2) >= left;
                        lsum += hide ? 0.0f : p;
                        p = hide ? 0.0f : p * vs[b];   // (vs may be NaN)
                        const _Float16 hi = (_Float16)p;
                        ph[j] = hi;
                        pl[j] = (_Float16)(p - (float)hi);
                    }
#pragma unroll
                    for (int d = 0; d < 4; ++d) {
                        const half8_t v = __builtin_bit_cast(half8_t, vb[((b * 4 + d) * 2 + gr) * 64]);
                        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, ph, o[d], 0, 0, 0);
                        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, pl, o[d], 0, 0, 0);
                    }
                }
        }
        if (t + 1 < t1) stage(t + 1, buf ^ 1);
        __syncthreads();
    }
    lsum += __shfl_xor(lsum, 32, 64);
    if (!live) return;
    // lane's dims: 32 d + 8 k + 4 h + 0..3
    const float moff = ref.off() - kPreBase, f = 1.0f / ref.r;
    const bool direct = a.splits == 1;
    float *dst;
    if (direct) {
        dst = a.out + ((size_t)tok * a.H + head) * kKv8Hd;
        if (a.weights && h == 0)
            a.lse[(size_t)kvh * pre_rows32(a.rows) + row].x = moff + __builtin_amdgcn_logf(lsum);
    } else {
        const size_t p = ((size_t)split * a.Hkv + kvh) * a.rows + row;
        dst = a.o + p * kKv8Hd;
        // (a wave may see nothing of a split that others see)
        if (h == 0) a.ml[p] = make_float2(t0 * kPreTile < wseen ? moff : -__builtin_inff(), lsum);
    }
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float4 v = make_float4(o[d][4 * k] * f, o[d][4 * k + 1] * f, o[d][4 * k + 2] * f,
                                   o[d][4 * k + 3] * f);
            if (direct) v = make_float4(v.x / lsum, v.y / lsum, v.z / lsum, v.w / lsum);
            *(float4 *)(dst + 32 * d + 8 * k + 4 * h) = v;
        }
}

// Joins a row's splits: 32 threads a row, 4 dims each.
__global__ __launch_bounds__(256) void kv8_prefill_join_kernel(Kv8PrefillArgs a) {
    const int row = blockIdx.x * 8 + (threadIdx.x >> 5), kvh = blockIdx.y, d = (threadIdx.x & 31) * 4;
    if (row >= a.rows) return;
    const int tok = row / a.G, head = kvh * a.G + row % a.G;
    // splits that the row's workgroup had tiles in
    const int lastrow = min((row / kPreRows + 1) * kPreRows, a.rows) - 1;
    const int tiles = (a.pos0 + lastrow / a.G + kPreTile) / kPreTile;
    const int ns = (tiles + a.per - 1) / a.per;
    const size_t step = (size_t)a.Hkv * a.rows, r = (size_t)kvh * a.rows + row;
    float M = -__builtin_inff();
    for (int s = 0; s < ns; ++s) M = fmaxf(M, a.ml[r + s * step].x);
    float lt = 0.0f;
    float4 t = make_float4(0, 0, 0, 0);
    for (int s = 0; s < ns; ++s) {
        const float2 p = a.ml[r + s * step];
        const float4 v = *(const float4 *)(a.o + (r + s * step) * kKv8Hd + d);
        const float f = __builtin_amdgcn_exp2f(p.x - M);
        lt = __builtin_fmaf(p.y, f, lt);
        t.x = __builtin_fmaf(v.x, f, t.x);
        t.y = __builtin_fmaf(v.y, f, t.y);
        t.z = __builtin_fmaf(v.z, f, t.z);
        t.w = __builtin_fmaf(v.w, f, t.w);
    }
    *(float4 *)(a.out + ((size_t)tok * a.H + head) * kKv8Hd + d) =
        make_float4(t.x / lt, t.y / lt, t.z / lt, t.w / lt);
    if (a.weights && d == 0)
        a.lse[(size_t)kvh * pre_rows32(a.rows) + row].x = M + __builtin_amdgcn_logf(lt);
}

// A block's weight from the rows' softmax sums: the scores again, K in
// registers (two blocks a wave), q's operands streamed.  Sums are in a fixed
// order: rows of a lane, then lanes, then row splits.
template <int FMT>
__global__ __launch_bounds__(256) void kv8_weights_kernel(Kv8PrefillArgs a) {
    const int lane = threadIdx.x & 63, kvh = blockIdx.y, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int nblk = kv8_blocks(a.pos0 + a.n), b0 = (blockIdx.x * 4 + wave) * 2;
    if (b0 >= nblk) return;
    const Kv8Layout l = kv8_layout(a.Hkv, a.nb);
    const float2 *sc = (const float2 *)(a.cache + l.scales) + (size_t)kvh * a.nb;
    half8_t kf[2][8];
    float ks[2], acc[2] = {0.0f, 0.0f};
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        const int blk = min(b0 + b, nblk - 1);
        const uint8_t *p = a.cache + ((size_t)kvh * a.nb + blk) * kKv8Codes + (lane & 31) * kKv8Hd + 16 * h;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint4 c = *(const uint4 *)(p + 32 * i);
            kf[b][2 * i] = kv8_unpack8<FMT>(c.x, c.y);
            kf[b][2 * i + 1] = kv8_unpack8<FMT>(c.z, c.w);
        }
        ks[b] = sc[blk].x;
    }
    const int r32 = pre_rows32(a.rows), groups = r32 / 32;
    const int per = (groups + a.rsplits - 1) / a.rsplits;
    // rows before the block see nothing of it
    const int first = max(0, b0 * kKv8Block - a.pos0) * a.G / 32;
    const int g1 = min(groups, (int)(blockIdx.z + 1) * per);
    for (int g = max(first, (int)blockIdx.z * per); g < g1; ++g) {
        const uint4 *f = a.qf + ((size_t)kvh * groups + g) * (8 * 2 * 64) + lane;
        const int row = 32 * g + (lane & 31);
        const float2 ls = a.lse[(size_t)kvh * r32 + row];
        f32x16 s[2];
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[b][i] = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const half8_t q = __builtin_bit_cast(half8_t, f[i * 64]);
            s[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[0][i >> 1], q, s[0], 0, 0, 0);
            s[1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[1][i >> 1], q, s[1], 0, 0, 0);
        }
        // positions that the row sees, from the lane's first one on
        const int left = row < a.rows ? a.pos0 + row / a.G + 1 - b0 * kKv8Block - 4 * h : -1000;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const float ck = ks[b] * ls.y;
            float ps = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][i], ck, -ls.x));
                ps += 32 * b + (i & 3) + 8 * (i >> 2) < left ? p : 0.0f;
            }
            acc[b] += ps;
        }
    }
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        acc[b] = wave_sum(acc[b]);
        if (lane == 0 && b0 + b < nblk)
            a.part[((size_t)blockIdx.z * a.Hkv + kvh) * nblk + b0 + b] = acc[b];
    }
}

__global__ __launch_bounds__(256) void kv8_weights_add_kernel(Kv8PrefillArgs a) {
    const int b = blockIdx.x * 256 + threadIdx.x, kvh = blockIdx.y;
    const int nblk = kv8_blocks(a.pos0 + a.n);
    if (b >= nblk) return;
    float s = 0.0f;
    for (int i = 0; i < a.rsplits; ++i) s += a.part[((size_t)i * a.Hkv + kvh) * nblk + b];
    ((float *)(a.cache + kv8_layout(a.Hkv, a.nb).weights))[(size_t)kvh * a.nb + b] += s;
}

// The launch shapes of a prefill call and its workspace.
struct PrefillPlan {
    int rows, rtiles, splits, per, rsplits;
    size_t ml, o, lse, qf, part, bytes;
};
static PrefillPlan prefill_plan(int n, int pos0, int H, int Hkv, bool weights) {
    PrefillPlan p{};
    const int G = H / Hkv, total = pos0 + n, nblk = kv8_blocks(total);
    p.rows = n * G;
    p.rtiles = (p.rows + kPreRows - 1) / kPreRows;
    const int tiles = (total + kPreTile - 1) / kPreTile;
    // two workgroups per CU are resident; splits of at least four tiles
    const int64_t wgs = (int64_t)p.rtiles * Hkv, target = 2 * (int64_t)device_cus();
    int64_t s = (target + wgs - 1) / wgs;
    if (s > (tiles + 3) / 4) s = (tiles + 3) / 4;
    if (s < 1) s = 1;
    p.per = (int)((tiles + s - 1) / s);
    p.splits = (tiles + p.per - 1) / p.per;
    size_t at = 0;
    auto take = [&](size_t b) {
        const size_t o = at;
        at += kv8_align(b);
        return o;
    };
    if (p.splits > 1) {
        p.ml = take((size_t)p.splits * Hkv * p.rows * 8);
        p.o = take((size_t)p.splits * Hkv * p.rows * kKv8Hd * 4);
    }
    if (weights) {
        const size_t r32 = pre_rows32(p.rows);
        p.lse = take(Hkv * r32 * 8);
        p.qf = take(Hkv * r32 * kKv8Hd * 4);
        const int64_t w = (int64_t)((nblk + 7) / 8) * Hkv, groups = r32 / 32;
        int64_t rs = (4 * (int64_t)device_cus() + w - 1) / w;
        if (rs > (groups + 3) / 4) rs = (groups + 3) / 4;
        p.rsplits = (int)(rs < 1 ? 1 : rs);
        p.part = take((size_t)p.rsplits * Hkv * nblk * 4);
    }
    p.bytes = at;
    return p;
}

static int heads_check(int H, int Hkv) {
    OXB_REQUIRE(Hkv > 0 && H > 0 && H % Hkv == 0, "attention: heads %d not a multiple of kv heads %d", H, Hkv);
    OXB_REQUIRE(H <= 65535, "attention: %d heads", H);
    return 0;
}

}  // namespace oxb

using namespace oxb;

extern "C" size_t oxb_attn_decode_kv8_ws_bytes(int batch, int H, int Hkv, int hd, int max_seq) {
    if (batch < 1 || batch > 65535 || Hkv < 1 || H < 1 || H % Hkv || H > 65535 || hd != kKv8Hd ||
        max_seq < 1 || max_seq > OXB_KV8_MAX_SEQ)
        return 0;
    return decode_ws(batch, H, Hkv, kv8_blocks(max_seq)).bytes;
}

extern "C" int oxb_attn_decode_kv8(const float *q, void *cache, size_t cache_stride, int fmt,
                                   const int *pos, int pos_stride, int batch, int H, int Hkv, int hd,
                                   int max_seq, int add_weights, float *out, void *ws,
                                   size_t ws_bytes, void *stream) {
    clear_error();
    if (kv8_check(cache, cache_stride, fmt, batch, Hkv, hd, max_seq) || heads_check(H, Hkv)) return -1;
    OXB_REQUIRE(q && out && (((uintptr_t)q | (uintptr_t)out) & 15) == 0,
                "attention: q or out is NULL or not 16-byte aligned");
    OXB_REQUIRE(pos && pos_stride >= 0, "attention: pos is NULL or its stride %d", pos_stride);
    const int nb = kv8_blocks(max_seq), G = H / Hkv, HC = (G + kDecRows - 1) / kDecRows;
    const DecodeWs w = decode_ws(batch, H, Hkv, nb);
    OXB_REQUIRE(ws && ((uintptr_t)ws & 255) == 0 && ws_bytes >= w.bytes,
                "attention: workspace is NULL, not 256-byte aligned or %zu bytes < %zu", ws_bytes, w.bytes);
    Kv8DecodeArgs a{q, (uint8_t *)cache, cache_stride, pos, pos_stride, H, Hkv, G, HC, max_seq, nb,
                    decode_splits(batch, Hkv, HC, nb), add_weights != 0, out,
                    (float2 *)((char *)ws + w.ml), (float *)((char *)ws + w.o),
                    (float2 *)((char *)ws + w.bw)};
    hipStream_t s = (hipStream_t)stream;
    const dim3 grid(a.splits, Hkv * HC, batch), th(kDecThreads);
    if (fmt == OXB_KV8_INT8) {
        if (add_weights)
            hipLaunchKernelGGL((kv8_decode_kernel<OXB_KV8_INT8, true>), grid, th, 0, s, a);
        else
            hipLaunchKernelGGL((kv8_decode_kernel<OXB_KV8_INT8, false>), grid, th, 0, s, a);
    } else {
        if (add_weights)
            hipLaunchKernelGGL((kv8_decode_kernel<OXB_KV8_E4M3, true>), grid, th, 0, s, a);
        else
            hipLaunchKernelGGL((kv8_decode_kernel<OXB_KV8_E4M3, false>), grid, th, 0, s, a);
    }
    OXB_CHECK_HIP(hipGetLastError());
    if (a.splits > 1 || add_weights) {
        const int chunks = add_weights ? Hkv * ((nb + kJoinThreads - 1) / kJoinThreads) : 0;
        hipLaunchKernelGGL(kv8_decode_join_kernel, dim3(H + chunks, batch), dim3(kJoinThreads), 0, s, a);
        OXB_CHECK_HIP(hipGetLastError());
    }
    return 0;
}

extern "C" size_t oxb_attn_prefill_kv8_ws_bytes(int n_tok, int pos0, int H, int Hkv, int hd,
                                                int add_weights) {
    if (n_tok < 1 || pos0 < 0 || pos0 > OXB_KV8_MAX_SEQ - n_tok || Hkv < 1 || H < 1 || H % Hkv ||
        H > 65535 || hd != kKv8Hd || (int64_t)n_tok * (H / Hkv) > (1 << 30))
        return 0;
    return prefill_plan(n_tok, pos0, H, Hkv, add_weights != 0).bytes;
}

extern "C" int oxb_attn_prefill_kv8(const float *q, void *cache, int fmt, int n_tok, int pos0, int H,
                                    int Hkv, int hd, int max_seq, int add_weights, float *out,
                                    void *ws, size_t ws_bytes, void *stream) {
    clear_error();
    if (kv8_check(cache, 0, fmt, 1, Hkv, hd, max_seq) || heads_check(H, Hkv)) return -1;
    OXB_REQUIRE(q && out && (((uintptr_t)q | (uintptr_t)out) & 15) == 0,
                "attention: q or out is NULL or not 16-byte aligned");
    OXB_REQUIRE(n_tok >= 1 && pos0 >= 0 && n_tok <= max_seq && pos0 <= max_seq - n_tok,
                "prefill attention: bad range");
    OXB_REQUIRE((int64_t)n_tok * (H / Hkv) <= (1 << 30), "prefill attention: %d tokens", n_tok);
    const PrefillPlan p = prefill_plan(n_tok, pos0, H, Hkv, add_weights != 0);
    OXB_REQUIRE(p.bytes == 0 || (ws && ((uintptr_t)ws & 255) == 0 && ws_bytes >= p.bytes),
                "attention: workspace is NULL, not 256-byte aligned or %zu bytes < %zu", ws_bytes, p.bytes);
    char *w = (char *)ws;
    Kv8PrefillArgs a{q, (uint8_t *)cache, n_tok, pos0, H, Hkv, H / Hkv, kv8_blocks(max_seq), p.rows,
                     p.splits, p.per, add_weights != 0, out, (float2 *)(w + p.ml), (float *)(w + p.o),
                     (float2 *)(w + p.lse), (uint4 *)(w + p.qf), (float *)(w + p.part), p.rsplits};
    hipStream_t s = (hipStream_t)stream;
    const dim3 grid(p.rtiles, Hkv, p.splits), th(kPreThreads);
    const size_t lds = 2 * kPreTileBytes;
    if (fmt == OXB_KV8_INT8) {
        if (allow_dynamic_lds((const void *)kv8_prefill_kernel<OXB_KV8_INT8>)) return -1;
        hipLaunchKernelGGL(kv8_prefill_kernel<OXB_KV8_INT8>, grid, th, lds, s, a);
    } else {
        if (allow_dynamic_lds((const void *)kv8_prefill_kernel<OXB_KV8_E4M3>)) return -1;
        hipLaunchKernelGGL(kv8_prefill_kernel<OXB_KV8_E4M3>, grid, th, lds, s, a);
    }
    OXB_CHECK_HIP(hipGetLastError());
    if (p.splits > 1) {
        hipLaunchKernelGGL(kv8_prefill_join_kernel, dim3((p.rows + 7) / 8, Hkv), dim3(256), 0, s, a);
        OXB_CHECK_HIP(hipGetLastError());
    }
    if (add_weights) {
        const int nblk = kv8_blocks(pos0 + n_tok);
        const dim3 wg((nblk + 7) / 8, Hkv, p.rsplits);
        if (fmt == OXB_KV8_INT8)
            hipLaunchKernelGGL(kv8_weights_kernel<OXB_KV8_INT8>, wg, dim3(256), 0, s, a);
        else
            hipLaunchKernelGGL(kv8_weights_kernel<OXB_KV8_E4M3>, wg, dim3(256), 0, s, a);
        OXB_CHECK_HIP(hipGetLastError());
        hipLaunchKernelGGL(kv8_weights_add_kernel, dim3((nblk + 255) / 256, Hkv), dim3(256), 0, s, a);
        OXB_CHECK_HIP(hipGetLastError());
    }
    return 0;
}

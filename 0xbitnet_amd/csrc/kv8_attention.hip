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

#include <algorithm>

namespace oxb {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr float kScoreUnit = 1.44269504088896340736f * 0.08838834764831844f;   // log2(e) / sqrt(128)
constexpr int kArrivals = 1024; // arrival counters at a workspace's start
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
// Workgroup: four waves over a run of a KV head's blocks, wave w taking every
// fourth, for up to 8 of its query heads at a time (K and V are read once for
// all of them; more than 8 go round again over the run, which L2 then holds).
// 16x16x32 MFMA: the 16 columns are the 8 heads' hi and lo parts, for q and
// for p' alike, so the two-part products cost nothing over one.
//   scores: A = 16 K rows x 32 dims, B = q; column c + (c ^ 8) is the score.
//   K rows are taken in an order that leaves lane group g (of 4) the scores of
//   the positions that bytes 8g .. 8g + 7 of a V row hold;
//   P.V: A = 16 dims x the block's 32 positions (8 bytes a lane), B = the lane's
//   own eight p' -- no exchange between lanes.
// Bound by the cache's bytes; a wave keeps its next block's 8 KB in flight
// under the current one's arithmetic (32 sequences of up to 2304 positions, H 20
// over 5, with weights: 22.2 us; 33.4 with no block in flight, 25.0 with two).  A
// sequence's runs meet in the workspace: each stores its part and counts in,
// and the last one joins them in order, so the sum does not depend on which is
// last.  Those 32 read 73 MB, 3.2 TB/s, of which about 8 us are no bytes' time:
// the position, the first block, the hand-over, the join (one sequence of 2304
// alone: 8.9 us).  Four sequences of up to 100001: 77 us, 415 MB, 5.4 TB/s.
constexpr int kDecWaves = 4;
constexpr int kDecThreads = 64 * kDecWaves;
constexpr int kDecRows = 8;            // query heads of a pass
constexpr int kDecQs = kKv8Hd + 8;     // q row stride in LDS (f16)
constexpr float kDecBase = 6.0f;       // p' <= 2^(6 + kStep)

struct Kv8DecodeArgs {
    const float *q;
    uint8_t *cache;
    size_t stride;
    const int *pos;
    int pos_stride, H, Hkv, G, max_seq, nb, splits, many, least;
    float *out;
    int *cnt;        // [batch * Hkv] zero between calls
    uint64_t *ml;    // [batch][H][splits] reference and sum (two floats)
    uint64_t *o;     // [batch][H][splits][64] pairs of dims
    uint64_t *bw;    // [batch][H][nb] a block's sum of p' and its reference
};

__device__ __forceinline__ uint64_t kv8_pair(float a, float b) {
    return (uint64_t)__float_as_uint(a) | ((uint64_t)__float_as_uint(b) << 32);
}
__device__ __forceinline__ float2 kv8_unpair(uint64_t p) {
    return make_float2(__uint_as_float((uint32_t)p), __uint_as_float((uint32_t)(p >> 32)));
}
// Hand-over between workgroups (and, for a block's weight, between the threads
// of one) goes through agent-scope stores and loads.
__device__ __forceinline__ void kv8_put(uint64_t *p, float a, float b) {
    __hip_atomic_store(p, kv8_pair(a, b), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 kv8_get(const uint64_t *p) {
    return kv8_unpair(__hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}

// The softmax weights of a pass's heads (rows' references and sums in sml) join
// the weights of the sequence's blocks, the heads in order.
__device__ __forceinline__ void kv8_add_weights(const Kv8DecodeArgs &a, int z, int kvh, int g0, int ng,
                                                int nblk, const float2 *sml) {
    uint8_t *seq = a.cache + (size_t)z * a.stride;
    float *w = (float *)(seq + kv8_layout(a.Hkv, a.nb).weights) + (size_t)kvh * a.nb;
    const uint64_t *bw = a.bw + ((size_t)z * a.H + g0) * a.nb;
    for (int b = threadIdx.x; b < nblk; b += kDecThreads) {
        float add = 0.0f;
#pragma unroll
        for (int i = 0; i < kDecRows; ++i) {
            if (i >= ng) break;
            const float2 p = kv8_get(bw + (size_t)i * a.nb + b);
            add += p.x * __builtin_amdgcn_exp2f(p.y - sml[i].x) / sml[i].y;
        }
        w[b] += add;
    }
}

template <int FMT, bool WEIGHTS>
__global__ __launch_bounds__(kDecThreads) void kv8_decode_kernel(Kv8DecodeArgs a) {
    __shared__ _Float16 sq[2 * kDecRows * kDecQs];
    __shared__ float sqs[kDecRows];
    __shared__ float2 sml[kDecWaves][kDecRows];
    __shared__ float4 so[kDecWaves][kDecRows][kKv8Hd / 4];
    __shared__ float2 stot[kDecRows];
    __shared__ int s_last;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kvh = blockIdx.x, z = a.many ? blockIdx.y : blockIdx.z, split = a.many ? blockIdx.z : blockIdx.y;
    const int orow = tid >> 5, od = (tid & 31) * 4;         // the row and dims a thread joins
    auto load_q = [&](int hc) {
        float4 v = make_float4(0, 0, 0, 0);
        if (hc + orow < a.G) v = *(const float4 *)(a.q + ((size_t)z * a.H + kvh * a.G + hc + orow) * kKv8Hd + od);
        return v;
    };
    float4 qv = load_q(0);   // with pos, before the cache's loads: loads return in order
    const int64_t p1 = (int64_t)a.pos[(size_t)z * a.pos_stride] + 1;
    const int len = (int)(p1 < 0 ? 0 : p1 > a.max_seq ? a.max_seq : p1), nblk = kv8_blocks(len);
    // blocks of a run: an even share of `least` or more, or all of a short sequence
    const int share = max(a.least, (nblk + a.splits - 1) / a.splits);
    const int per = nblk <= 2 * a.least ? max(nblk, 1) : share, runs = (nblk + per - 1) / per;
    const int b0 = split * per, b1 = min(nblk, b0 + per);
    if (b0 >= b1) {
        if (split == 0)
            for (int i = tid; i < a.G * kKv8Hd; i += kDecThreads)
                a.out[((size_t)z * a.H + kvh * a.G) * kKv8Hd + i] = 0.0f;
        return;
    }
    const Kv8Layout l = kv8_layout(a.Hkv, a.nb);
    const uint8_t *seq = a.cache + (size_t)z * a.stride;
    const uint8_t *codes = seq + (size_t)kvh * a.nb * kKv8Codes;
    const float2 *sc = (const float2 *)(seq + l.scales) + (size_t)kvh * a.nb;
    const int rr = lane & 15, g = lane >> 4;
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

    for (int hc = 0; hc < a.G; hc += kDecRows) {
        const int g0 = kvh * a.G + hc, ng = min(kDecRows, a.G - hc);
        // the first block is on its way while q is made ready
        Blk cur = load(min(b0 + wave, b1 - 1));
        {   // q rows: scaled, split, and their score units
            const float4 v = qv;
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
        lds_barrier();
        half8_t qf[4];
#pragma unroll
        for (int s = 0; s < 4; ++s)
            qf[s] = *(const half8_t *)(sq + rr * kDecQs + 64 * (s >> 1) + 16 * g + 8 * (s & 1));
        const float qs = sqs[rr & 7];

        f32x4 o[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = f32x4{0, 0, 0, 0};
        Kv8Ref ref;
        float lsum = 0.0f;
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
                // hi and lo of p' vs, each rounded once from the exact product
                const _Float16 hi = (_Float16)__builtin_fmaf(p, vs, 0.0f);
                pf[i] = rr < kDecRows ? hi : (_Float16)__builtin_fmaf(p, vs, -(float)hi);
            }
            lsum += ps;
            if constexpr (WEIGHTS) {
                ps += __shfl_xor(ps, 16, 64);
                ps += __shfl_xor(ps, 32, 64);
                if (lane < ng) kv8_put(a.bw + ((size_t)z * a.H + g0 + lane) * a.nb + b, ps, moff);
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
        lds_barrier();
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
        const size_t row = (size_t)z * a.H + g0 + orow;
        if (runs == 1) {
            if (orow < ng)
                *(float4 *)(a.out + row * kKv8Hd + od) =
                    make_float4(t.x / lt, t.y / lt, t.z / lt, t.w / lt);
            if constexpr (WEIGHTS) {
                if (od == 0) stot[orow] = make_float2(M, lt);
                __syncthreads();
                kv8_add_weights(a, z, kvh, g0, ng, nblk, stot);
            }
        } else if (orow < ng) {
            const size_t part = row * a.splits + split;
            kv8_put(a.o + part * 64 + (od >> 1), t.x, t.y);
            kv8_put(a.o + part * 64 + (od >> 1) + 1, t.z, t.w);
            if (od == 0) kv8_put(a.ml + part, M, lt);
        }
        lds_barrier();   // LDS is free for the next heads
        qv = load_q(hc + kDecRows);
    }
    if (runs == 1) return;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();   // every thread's part has arrived
    if (tid == 0) {
        int *cnt = a.cnt + (size_t)z * a.Hkv + kvh;
        const int old = __hip_atomic_fetch_add(cnt, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        s_last = old == runs - 1;
        if (s_last) __hip_atomic_store(cnt, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!s_last) return;
    for (int hc = 0; hc < a.G; hc += kDecRows) {
        const int g0 = kvh * a.G + hc, ng = min(kDecRows, a.G - hc);
        // 32 lanes a head; the lanes that fewer than 8 heads leave take every
        // second, fourth or eighth run of one
        const int np = ng > 4 ? 8 : ng > 2 ? 4 : ng, step = kDecRows / np, jr = orow % np;
        if (jr < ng) {
            const size_t row = (size_t)z * a.H + g0 + jr;
            const uint64_t *ml = a.ml + row * a.splits, *op = a.o + row * a.splits * 64 + (od >> 1);
            float M = -__builtin_inff(), lt = 0.0f;
            float4 t = make_float4(0, 0, 0, 0);
            constexpr int kB = 16;   // runs in flight
            for (int s0 = orow / np; s0 < runs; s0 += kB * step) {
                float2 p[kB], lo[kB], hi[kB];
#pragma unroll
                for (int j = 0; j < kB; ++j) {
                    p[j] = make_float2(-__builtin_inff(), 0.0f);
                    lo[j] = hi[j] = make_float2(0, 0);
                    const int s = s0 + j * step;
                    if (s < runs) {
                        p[j] = kv8_get(ml + s);
                        lo[j] = kv8_get(op + (size_t)s * 64);
                        hi[j] = kv8_get(op + (size_t)s * 64 + 1);
                    }
                }
                float m = M;
#pragma unroll
                for (int j = 0; j < kB; ++j) m = fmaxf(m, p[j].x);
                const float f0 = m == M ? 1.0f : __builtin_amdgcn_exp2f(M - m);
                M = m;
                lt *= f0;
                t = make_float4(t.x * f0, t.y * f0, t.z * f0, t.w * f0);
#pragma unroll
                for (int j = 0; j < kB; ++j) {
                    if (s0 + j * step >= runs) break;
                    const float f = __builtin_amdgcn_exp2f(p[j].x - M);
                    lt = __builtin_fmaf(p[j].y, f, lt);
                    t.x = __builtin_fmaf(lo[j].x, f, t.x);
                    t.y = __builtin_fmaf(lo[j].y, f, t.y);
                    t.z = __builtin_fmaf(hi[j].x, f, t.z);
                    t.w = __builtin_fmaf(hi[j].y, f, t.w);
                }
            }
            so[0][orow][od >> 2] = t;
            if (od == 0) sml[0][orow] = make_float2(M, lt);
        }
        lds_barrier();
        if (orow < ng) {
            float M = -__builtin_inff(), lt = 0.0f;
            float4 t = make_float4(0, 0, 0, 0);
            for (int i = orow; i < kDecRows; i += np) M = fmaxf(M, sml[0][i].x);
            for (int i = orow; i < kDecRows; i += np) {
                const float2 p = sml[0][i];
                const float f = __builtin_amdgcn_exp2f(p.x - M);
                const float4 v = so[0][i][od >> 2];
                lt = __builtin_fmaf(p.y, f, lt);
                t.x = __builtin_fmaf(v.x, f, t.x);
                t.y = __builtin_fmaf(v.y, f, t.y);
                t.z = __builtin_fmaf(v.z, f, t.z);
                t.w = __builtin_fmaf(v.w, f, t.w);
            }
            *(float4 *)(a.out + ((size_t)z * a.H + g0 + orow) * kKv8Hd + od) =
                make_float4(t.x / lt, t.y / lt, t.z / lt, t.w / lt);
            if (od == 0) stot[orow] = make_float2(M, lt);
        }
        lds_barrier();
        if constexpr (WEIGHTS) {
            kv8_add_weights(a, z, kvh, g0, ng, nblk, stot);
            lds_barrier();
        }
    }
}

// Runs per KV head and sequence: two workgroups per CU over the launch (what
// the registers let reside; the 32 sequences above: 22.2 us, with one per CU
// 28.6, with four 28.4), none with fewer blocks than waves.  The division is
// rounded down and knows no lengths.  51 sequences of up to 2304 have two runs
// each and take 28.0 us; 52 have one, half of the places stay empty, and they take
// 35.3 (64: 40.1, 96: 45.8).  A long sequence among many short ones gets their few
// runs: 100000 positions beside 63 of 500, H 64 over 8, 770 us (alone 50).
static int decode_splits(int batch, int Hkv, int nb) {
    const int64_t rows = (int64_t)batch * Hkv, most = (nb + kDecWaves - 1) / kDecWaves;
    int64_t s = 2 * (int64_t)device_cus() / rows;
    if (s > most) s = most;
    return (int)(s < 1 || rows > kArrivals ? 1 : s);
}

// Many rows (sequence and KV head) fill a good part of the CUs by themselves.  Then
// a run has 8 blocks at least (else 4), and twice as many are not cut: the
// hand-over and the join take 3-5 us, a workgroup's next four blocks 1.  H 20
// over 5, with runs of 4 and of 8: 8 sequences of up to 600 positions 8.2, 8.9
// us; 16 of 640 9.4, 8.8; 32 of 512 11.2, 8.5; just past the uncut lengths it
// loses, 32 of 700 by 3%, 48 of 600 with weights by 4%.  And a sequence's second runs,
// which it may not have, are started after all first ones, so that those are on
// all XCDs alike (16 of 640: 8.8 against 10.9 with a sequence's runs side by
// side); of few rows each has its runs side by side (4 of 100001: 75 us against
// 82 the other way, on one box).
static bool decode_many(int batch, int Hkv) { return (int64_t)batch * Hkv >= 64; }

// Parts are as many as a batch of up to this size leaves at most, whatever its own
// cut: fewer sequences have more runs each (51 of 5 KV heads two, 52 one), and a
// workspace of the largest batch serves every smaller one.
struct DecodeWs {
    size_t ml, o, bw, bytes;
};
static DecodeWs decode_ws(int batch, int H, int Hkv, int nb) {
    const int64_t rows = (int64_t)batch * Hkv, most = (nb + kDecWaves - 1) / kDecWaves;
    const size_t parts = H / Hkv * std::max(rows, std::min<int64_t>(2 * device_cus(), rows * most));
    DecodeWs w;
    w.ml = kArrivals * 4;
    w.o = w.ml + kv8_align(parts * 8);
    w.bw = w.o + kv8_align(parts * kKv8Hd * 4);
    w.bytes = w.bw + kv8_align((size_t)batch * H * nb * 8);
    return w;
}

// ---------------------------------------------------------------------------
// prefill
// ---------------------------------------------------------------------------
// Rows of a KV head are (token, query head of the group) pairs, token-major, so
// that a block of K and V serves all of the group's heads.  A workgroup takes
// 128 rows, 32 per wave, and a run of blocks.  A block's codes are unpacked to
// f16 once, a quarter by each wave, into LDS in the order the MFMA operands are
// read (every read is 1 KB contiguous).
//   scores: 32x32x16 MFMA, A = 32 K rows, B = q (in registers, hi and lo);
//   P.V: A = 32 dims x 16 positions, B = the lane's own p' (kv8_v_byte's order).
// Bound by the MFMAs (32 of 32 cycles per wave and block, twice the one-part
// products) as long as the softmax's VALU work runs under them: the next
// block's score products alternate with this block's exponentials, and P.V with
// the rest of them and the unpacking, instruction by instruction (a wave that
// issues 16 MFMAs and then 128 VALU instructions takes 395 ns, one that
// alternates them 349, the MFMAs alone 261; two waves per SIMD).  K runs a
// block ahead of V; rings of four blocks of each leave one barrier per two
// blocks.  8192 tokens, H 20 over 5: 612 us, 1124 TFLOP/s of MFMA work (a large
// f16 product of the library: 1330); 2048 tokens 54 us and 9 for the join; 333
// behind 20011 137-153 us and 9.  The MFMAs are busy for two thirds of a wave's time
// and the clock falls under them, so what saves VALU instructions saves time.
// Row tiles see different lengths; where they alone leave CUs idle or finish
// far apart, the launch cuts them into runs (prefill_plan), and a second launch
// joins the parts.  More tiles than resident workgroups are not cut at all: behind
// a long context, where all are equally long, a few too many cost a second round
// (3264 tokens behind 20000, 510 workgroups: 1221 us; 3300, 520: 1781; 4096: 1950).
// From position 0 the lengths differ and the last ones are short (3264 tokens 125
// us, 3300 127).
constexpr int kPreWaves = 4;
constexpr int kPreThreads = 64 * kPreWaves;
constexpr int kPreRows = 32 * kPreWaves;
constexpr int kPreRing = 4;
constexpr int kPreOps = kKv8Half * 2 / 16;   // 16-byte operands of a block's K (or V) as f16
constexpr float kPreBase = 6.0f;             // p' <= 2^(6 + kStep)

struct Kv8PrefillArgs {
    const float *q;
    uint8_t *cache;
    int n, pos0, H, Hkv, G, nb, rows, rtiles, planned, per, nblk;
    float *out;
    float2 *ml;     // [splits][Hkv][rows] a row's reference and sum
    float *o;       // [splits][Hkv][rows][128]
    float *rsum;    // [Hkv][rows] 1 / the row's softmax sum, or NULL: no weights
    float2 *bw;     // [Hkv][nblk][rtiles * 128] a block's sum of p' in a row, its reference
};

// A row's final reference and softmax sum, for its blocks' weights: the sum's
// reciprocal, and the reference in the pair of the row's first block, whose own sum
// is brought to it.  (One f32 logarithm of both in their place has steps of 2^-20
// from 16 on, and the instruction's error leans to one side: the weights of 333
// tokens behind 20011 were 5.9e-7 from the 64-bit ones; this way 6e-8, as f32
// torch, in the same time.)
__device__ __forceinline__ void kv8_row_total(const Kv8PrefillArgs &a, int kvh, int row, float M, float l) {
    a.rsum[(size_t)kvh * a.rows + row] = 1.0f / l;
    float2 *p = a.bw + (size_t)kvh * a.nblk * a.rtiles * kPreRows + row;
    *p = make_float2(p->x * __builtin_amdgcn_exp2f(p->y - M), M);
}

// A row tile's blocks in even runs, of `per` blocks at most and cut as few times as
// that takes: the last of k + 1 has (k per + 1) / (k + 1) blocks or more, (per + 1) / 2
// at least, rounded up.  The tile's rows end in at most kPreRows / 32 + 1 blocks, so
// with runs of kPreLeast or more each row sees some position of each run, and its
// reference is a score's.
constexpr int kPreLeast = 8;
static_assert((kPreLeast + 2) / 2 >= kPreRows / kKv8Block + 1, "a row sees nothing of its tile's last run");
__host__ __device__ inline int pre_run_start(int blocks, int runs, int i) {
    return (int)((int64_t)blocks * i / runs);
}
// The order in which runs are started: row tile | run << 16.  By value with the
// launch, so that a captured graph keeps it.
constexpr int kPreOrder = 512;
struct Kv8PrefillOrder {
    uint32_t run[kPreOrder];
};

template <int FMT, bool WEIGHTS>
__global__ __launch_bounds__(kPreThreads, 2) void kv8_prefill_kernel(Kv8PrefillArgs a, const Kv8PrefillOrder order) {
    // rings of K [8][64] and V operands [4 dims][2][64]: block b of the run in slot
    // b % 4; the rows of q before
    __shared__ uint4 lds[2][kPreRing][kPreOps];
    static_assert(sizeof lds == sizeof(float) * kPreRows * kKv8Hd, "q rows fill the rings");
    auto &sk = lds[0], &sv = lds[1];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // workgroups take the plan's runs in its order, the KV heads side by side
    const int kvh = blockIdx.x % a.Hkv;
    int rtile = a.rtiles - 1 - (int)(blockIdx.x / a.Hkv), split = 0;
    if (a.planned) {
        const uint32_t e = order.run[blockIdx.x / a.Hkv];
        rtile = e & 0xffff;
        split = e >> 16;
    }
    const int r0 = rtile * kPreRows, row = r0 + wave * 32 + (lane & 31), h = lane >> 5;
    const int total = a.pos0 + a.n;
    const int lastrow = min(r0 + kPreRows, a.rows) - 1;
    const int blocks = kv8_blocks(a.pos0 + lastrow / a.G + 1);   // that the tile's last row sees
    const int runs = a.planned ? (blocks + a.per - 1) / a.per : 1;
    const int b0 = pre_run_start(blocks, runs, split), b1 = pre_run_start(blocks, runs, split + 1);
    const int tok = min(row, a.rows - 1) / a.G, head = kvh * a.G + min(row, a.rows - 1) % a.G;
    const int qpos = a.pos0 + tok;

    const Kv8Layout l = kv8_layout(a.Hkv, a.nb);
    const uint8_t *codes = a.cache + (size_t)kvh * a.nb * kKv8Codes;
    const float2 *sc = (const float2 *)(a.cache + l.scales) + (size_t)kvh * a.nb;
    // a wave unpacks 32 dims of K and of V of each block: operands 2 wave, 2 wave + 1
    const uint32_t koff = (lane & 31) * kKv8Hd + 32 * wave + 16 * h;
    const uint32_t voff = kKv8Half + (32 * wave + (lane & 31)) * kKv8Block + 16 * h;
    uint4 ck4[2], cv4[2];
    // (buffer loads: a scalar address and one register of offset)
    auto fetch = [&](int b, uint32_t off) {
        const uint8_t *p = codes + (size_t)__builtin_amdgcn_readfirstlane(min(b, b1 - 1)) * kKv8Codes;
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void *)p, 0, kKv8Codes, 0x00027000);
        return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
    };
    const int slot = 128 * wave + lane;
    auto stage = [&](uint4 *ring, const uint4 &c) {
        ring[slot] = __builtin_bit_cast(uint4, kv8_unpack8<FMT>(c.x, c.y));
        ring[slot + 64] = __builtin_bit_cast(uint4, kv8_unpack8<FMT>(c.z, c.w));
    };
    auto clear_v = [&](int b, uint4 &c) {   // bytes behind the last position may hold anything
        const int left = total - b * kKv8Block, hh = 4 * h + opaque_zero();
        if (left >= kKv8Block) return;   // uniform
        uint32_t mk[4] = {0, 0, 0, 0};
#pragma unroll
        for (int p = 0; p < 16; ++p)   // byte 16 h + p: position 16 (p / 8) + 8 (p / 4 % 2) + 4 h + p % 4
            if (16 * (p >> 3) + 8 * (p >> 2 & 1) + (p & 3) + hh < left) mk[p >> 2] |= 0xffu << (8 * (p & 3));
        c.x &= mk[0];
        c.y &= mk[1];
        c.z &= mk[2];
        c.w &= mk[3];
    };
    // q first, through the rings' LDS, 16 KB a wave: two of its rows a load, row r's
    // 16-byte piece c at c ^ r, so that the rows' reads of one piece meet no bank
    // twice (a lane loading its own row, 64 pieces of 32 rows at a time: 101 tokens
    // 11.0 us against 10.5, 300 behind 500 22.9 against 22.6)
    uint4 *sq = &lds[0][0][0] + 1024 * wave;
    const uint32_t qrow = (uint32_t)tok * a.H + head;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const uint32_t ra = __builtin_amdgcn_readlane(qrow, 2 * i), rb = __builtin_amdgcn_readlane(qrow, 2 * i + 1);
        const int c = (lane & 31) ^ (2 * i + h);
        lds_dma16(a.q + (size_t)(h ? rb : ra) * kKv8Hd + 4 * c, sq + 64 * i);
    }
    ck4[0] = fetch(b0, koff);
    ck4[1] = fetch(b0 + 1, koff);
    cv4[0] = fetch(b0, voff);
    cv4[1] = fetch(b0 + 1, voff);
    const uint4 ck2 = fetch(b0 + 2, koff);

    // q: dims 32 c + 16 h + 8 e + j are operand s = 2 c + e
    half8_t qh[8], ql[8];
    float qs;
    {
        float m = 0.0f;
        float v[64];
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int p = (8 * (i >> 2) + 4 * h + (i & 3)) ^ (lane & 31);
            const float4 f = __builtin_bit_cast(float4, sq[32 * (lane & 31) + p]);
            v[4 * i] = f.x;
            v[4 * i + 1] = f.y;
            v[4 * i + 2] = f.z;
            v[4 * i + 3] = f.w;
        }
#pragma unroll
        for (int i = 0; i < 64; i += 2) m = fmaxf(fmaxf(fabsf(v[i]), fabsf(v[i + 1])), m);
        m = fmaxf(m, __shfl_xor(m, 32, 64));
        const int e = max(kv8_row_exp(m), -127);   // (a row below 2^-113 stays below 2^kQExp)
        const float up = ldexpf(1.0f, -e);
        qs = ldexpf(kScoreUnit, e);
#pragma unroll
        for (int s = 0; s < 8; ++s)
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const float x = v[8 * s + j], y = v[8 * s + j + 1];
                half2_t hi, lo;
                hi.x = (_Float16)__builtin_fmaf(x, up, 0.0f);
                hi.y = (_Float16)__builtin_fmaf(y, up, 0.0f);
                asm("" : "+v"(hi));
                lo.x = (_Float16)__builtin_fmaf(x, up, -(float)hi.x);
                lo.y = (_Float16)__builtin_fmaf(y, up, -(float)hi.y);
                qh[s][j] = hi.x;
                qh[s][j + 1] = hi.y;
                ql[s][j] = lo.x;
                ql[s][j + 1] = lo.y;
            }
    }
    // where the row's sums of the blocks go: the first half's lanes and the second's
    // store the same
    const int wrows = a.rtiles * kPreRows, woff = row * 8;

    f32x16 o[4];
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;
    Kv8Ref ref;
    float lsum = 0.0f;
    const int wseen = a.pos0 + min(r0 + wave * 32 + 31, a.rows - 1) / a.G + 1;   // the wave's last row
    const int wfull = a.pos0 + min(r0 + wave * 32, a.rows - 1) / a.G + 1;        // its first row

    lds_barrier();   // every wave has its q
    clear_v(b0, cv4[0]);
    clear_v(b0 + 1, cv4[1]);
    stage(sk[0], ck4[0]);
    stage(sk[1], ck4[1]);
    stage(sv[0], cv4[0]);
    stage(sv[1], cv4[1]);
    stage(sk[2], ck2);
    // codes in flight at the start of a pair b, b + 1: K of b + 3, b + 4, V of b + 2, b + 3
    auto fetch_pair = [&](int b) {
        ck4[0] = fetch(b + 3, koff);
        ck4[1] = fetch(b + 4, koff);
        cv4[0] = fetch(b + 2, voff);
        cv4[1] = fetch(b + 3, voff);
    };
    fetch_pair(b0);
    lds_barrier();
    f32x16 s0, s1;
#pragma unroll
    for (int i = 0; i < 16; ++i) s0[i] = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const half8_t k = __builtin_bit_cast(half8_t, sk[0][i * 64 + lane]);
        s0 = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, qh[i], s0, 0, 0, 0);
        s0 = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, ql[i], s0, 0, 0, 0);
    }
    lds_barrier();   // the first K slot is free
    const int wb = min(b1, kv8_blocks(wseen));   // blocks that some row of the wave sees
    float2 sb = sc[b0];
    // the running maximum with four more scores (in v_max3's form)
    auto top = [&](float m, const f32x16 &s, int i) {
        m = fmaxf(fmaxf(s[i], s[i + 1]), m);
        return fmaxf(fmaxf(s[i + 2], s[i + 3]), m);
    };
    constexpr float kNone = -__builtin_inff();
    float smax = top(top(top(top(kNone, s0, 0), s0, 4), s0, 8), s0, 12);
    // Block b, its scores in s and their maximum in smax; the next one's go to sn.
    // r: b's place in the run; stage0, stage1: what is unpacked under it.
    auto block = [&](int b, int r, f32x16 &s, f32x16 &sn, auto stage0, auto stage1) {
        const int p0 = b * kKv8Block;
        // (units of 0, of zero blocks, are made positive: hidden scores are -inf)
        float ck = sb.x * qs, vs = sb.y;
        sb = sc[min(b + 1, b1 - 1)];
        ck = ck < 1.2e-38f ? 1.2e-38f : ck;
        if (p0 + kKv8Block > wfull) {   // some rows do not see all of it (uniform)
            // positions of the lane's scores: (i & 3) + 8 (i >> 2) + 4 h
            const int left = qpos + 1 - p0 - 4 * h + opaque_zero();   // (a branch, not 32 selects)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = (i & 3) + 8 * (i >> 2) < left ? s[i] : -__builtin_inff();
            if (qpos < p0) {   // a row that sees none: the block's scales, NaN or not, are nothing to it
                ck = 1.2e-38f;
                vs = 0.0f;
            }
            smax = top(top(top(top(kNone, s, 0), s, 4), s, 8), s, 12);
        }
        const float mx = smax * ck;
        const float mx2 = mx + kv8_scale_exp(vs);
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
        vs *= ref.r;
        // From here on the order is the one written: SLOT ends what may run under
        // the MFMA before it.
#define SLOT() __builtin_amdgcn_sched_barrier(0)
        const uint4 *kb = sk[(r + 1) & 3] + lane, *vb = sv[r & 3] + lane;
        half8_t ph[2], pl[2], v[4], k[2];
        float pa, pb, ps = 0.0f;
        auto exps = [&](int j) {   // elements 2 j, 2 j + 1
            pa = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * j], ck, -moff));
            pb = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * j + 1], ck, -moff));
        };
        auto split = [&](int j) {   // hi and lo of p' vs, each rounded once from the exact product
            ps += pa;
            ps += pb;
            asm volatile("" : "+v"(ps));   // (here, not all sums at the end)
            half2_t hi, lo;
            hi.x = (_Float16)__builtin_fmaf(pa, vs, 0.0f);
            hi.y = (_Float16)__builtin_fmaf(pb, vs, 0.0f);
            asm("" : "+v"(hi));   // (one register for both, or the products are formed twice)
            lo.x = (_Float16)__builtin_fmaf(pa, vs, -(float)hi.x);
            lo.y = (_Float16)__builtin_fmaf(pb, vs, -(float)hi.y);
            ph[j >> 2][2 * (j & 3)] = hi.x;
            ph[j >> 2][2 * (j & 3) + 1] = hi.y;
            pl[j >> 2][2 * (j & 3)] = lo.x;
            pl[j >> 2][2 * (j & 3) + 1] = lo.y;
        };
#pragma unroll
        for (int i = 0; i < 16; ++i) sn[i] = 0.0f;
        k[0] = __builtin_bit_cast(half8_t, kb[0]);
        k[1] = __builtin_bit_cast(half8_t, kb[64]);
        SLOT();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            sn = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[i & 1], qh[i], sn, 0, 0, 0);
            if (i < 6) exps(i);
            SLOT();
            sn = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[i & 1], ql[i], sn, 0, 0, 0);
            if (i < 6) split(i);
            if (i < 6) k[i & 1] = __builtin_bit_cast(half8_t, kb[(i + 2) * 64]);
            else
                for (int d = 2 * (i - 6); d < 2 * (i - 5); ++d) v[d] = __builtin_bit_cast(half8_t, vb[d * 128]);
            SLOT();
        }
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[d], ph[0], o[d], 0, 0, 0);
            if (d & 1) split(6 + (d >> 1));
            else exps(6 + (d >> 1));
            SLOT();
        }
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[d], pl[0], o[d], 0, 0, 0);
            v[d] = __builtin_bit_cast(half8_t, vb[d * 128 + 64]);
            if (d == 1) stage0();
            SLOT();
        }
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[d], ph[1], o[d], 0, 0, 0);
            if (d == 1) stage1();
            SLOT();
        }
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[d], pl[1], o[d], 0, 0, 0);
            smax = top(d == 0 ? kNone : smax, sn, 4 * d);
            if constexpr (WEIGHTS)
                if (d == 1) {
                    const uint32_t u = __float_as_uint(ps);
                    const auto w = __builtin_amdgcn_permlane32_swap(u, u, false, false);   // both halves'
                    const float both = __uint_as_float(w[0]) + __uint_as_float(w[1]);
                    const u32x2_t pair = {__float_as_uint(both), __float_as_uint(moff)};
                    const __amdgpu_buffer_rsrc_t wr = __builtin_amdgcn_make_buffer_rsrc(
                        a.bw + ((size_t)kvh * a.nblk + b) * wrows, 0, wrows * 8, 0x00027000);
                    __builtin_amdgcn_raw_buffer_store_b64(pair, wr, woff, 0, 0);
                }
            SLOT();
        }
#undef SLOT
        lsum += ps;
    };
    auto stage_k = [&](int r) { return [&, r] { stage(sk[(r + 3) & 3], ck4[0]); }; };
    auto stage_k1 = [&](int r) { return [&, r] { stage(sk[r & 3], ck4[1]); }; };
    auto stage_v = [&](int r) { return [&, r] { stage(sv[(r + 2) & 3], cv4[0]); }; };
    auto stage_v1 = [&](int r) { return [&, r] { stage(sv[(r + 3) & 3], cv4[1]); }; };
    // The two waves of a SIMD take turns at priority, a pair of blocks each (their
    // slots differ in the lowest bit as a rule): by age alone one runs at its
    // full speed, 1.35 us a block, and the other, at half of it, finishes late.
    uint32_t hwid;
    asm volatile("s_getreg_b32 %0, hwreg(HW_REG_HW_ID)" : "=s"(hwid));
    int b = b0;
    for (; b + 1 < wb; b += 2) {
        const int r = b - b0;
        if (((r >> 1) ^ hwid) & 1) __builtin_amdgcn_s_setprio(1);
        else __builtin_amdgcn_s_setprio(0);
        clear_v(b + 2, cv4[0]);
        clear_v(b + 3, cv4[1]);
        block(b, r, s0, s1, stage_k(r), stage_k1(r));
        block(b + 1, r + 1, s1, s0, stage_v(r), stage_v1(r));
        fetch_pair(b + 2);
        lds_barrier();
    }
    for (; b < b1; b += 2) {   // a last block alone, and what only other waves see
        const int r = b - b0;
        clear_v(b + 2, cv4[0]);
        clear_v(b + 3, cv4[1]);
        auto none = [] {};
        if (b < wb) block(b, r, s0, s1, none, none);
        stage_k(r)();
        stage_k1(r)();
        stage_v(r)();
        stage_v1(r)();
        fetch_pair(b + 2);
        lds_barrier();
    }
    lsum += __shfl_xor(lsum, 32, 64);
    // the lane's row again (not held in registers over the loop)
    const int elane = lane + opaque_zero(), eh = elane >> 5, erow = r0 + wave * 32 + (elane & 31);
    if (erow >= a.rows) return;
    const float M = ref.off() - kPreBase;
    const bool direct = runs == 1;
    float *dst, f = 1.0f / ref.r;          // o in l's units
    if (direct) {
        dst = a.out + ((size_t)(erow / a.G) * a.H + kvh * a.G + erow % a.G) * kKv8Hd;
        f /= lsum;
        if (WEIGHTS && eh == 0) kv8_row_total(a, kvh, erow, M, lsum);
    } else {
        const size_t part = ((size_t)split * a.Hkv + kvh) * a.rows + erow;
        dst = a.o + part * kKv8Hd;
        if (eh == 0) a.ml[part] = make_float2(M, lsum);
    }
    // lane's dims: 32 d + 8 k + 4 h + 0..3
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int k = 0; k < 4; ++k)
            *(float4 *)(dst + 32 * d + 8 * k + 4 * eh) =
                make_float4(o[d][4 * k] * f, o[d][4 * k + 1] * f, o[d][4 * k + 2] * f, o[d][4 * k + 3] * f);
}

// Joins a row's runs: 32 threads a row, 4 dims each; bound by the parts' bytes
// (2048 tokens: 36 MB in 9 us).  Joined by a tile's last workgroup instead, as in
// decode, the runs' ends stood in one row: 30 us for tiles of 9 runs.
__global__ __launch_bounds__(256) void kv8_prefill_join_kernel(Kv8PrefillArgs a) {
    const int row = blockIdx.x * 8 + (threadIdx.x >> 5), kvh = blockIdx.y, d = (threadIdx.x & 31) * 4;
    if (row >= a.rows) return;
    const int tok = row / a.G, head = kvh * a.G + row % a.G;
    const int lastrow = min((row / kPreRows + 1) * kPreRows, a.rows) - 1;   // of the row's tile
    const int ns = (kv8_blocks(a.pos0 + lastrow / a.G + 1) + a.per - 1) / a.per;   // runs
    if (ns == 1) return;   // written by its only run
    const size_t step = (size_t)a.Hkv * a.rows, r = (size_t)kvh * a.rows + row;
    float M = -__builtin_inff(), lt = 0.0f;
    float4 t = make_float4(0, 0, 0, 0);
    constexpr int kB = 8;   // parts in flight
    for (int i0 = 0; i0 < ns; i0 += kB) {
        float2 p[kB];
        float4 v[kB];
#pragma unroll
        for (int i = 0; i < kB; ++i) {
            p[i] = make_float2(-__builtin_inff(), 0.0f);
            if (i0 + i < ns) {   // (uniform: the workgroup's rows are of one tile)
                const size_t at = r + (i0 + i) * step;
                p[i] = a.ml[at];
                v[i] = *(const float4 *)(a.o + at * kKv8Hd + d);
            }
        }
        float m = M;
#pragma unroll
        for (int i = 0; i < kB; ++i) m = fmaxf(m, p[i].x);
        const float f0 = m == M ? 1.0f : __builtin_amdgcn_exp2f(M - m);
        M = m;
        lt *= f0;
        t = make_float4(t.x * f0, t.y * f0, t.z * f0, t.w * f0);
#pragma unroll
        for (int i = 0; i < kB; ++i) {
            if (i0 + i >= ns) break;
            const float f = __builtin_amdgcn_exp2f(p[i].x - M);
            lt = __builtin_fmaf(p[i].y, f, lt);
            t.x = __builtin_fmaf(v[i].x, f, t.x);
            t.y = __builtin_fmaf(v[i].y, f, t.y);
            t.z = __builtin_fmaf(v[i].z, f, t.z);
            t.w = __builtin_fmaf(v[i].w, f, t.w);
        }
    }
    *(float4 *)(a.out + ((size_t)tok * a.H + head) * kKv8Hd + d) =
        make_float4(t.x / lt, t.y / lt, t.z / lt, t.w / lt);
    if (a.rsum && d == 0) kv8_row_total(a, kvh, row, M, lt);
}

// A block's weight: its sums of p' over the rows that see it, which the
// attention has left, in the units of their softmax sums, known only now.  A
// workgroup a block, in a fixed order; bound by the sums' bytes (333 tokens
// behind 20011, H 20: 35 MB in 9.4-10.8 us; the scores a second time, K in
// registers and q through LDS: 72).
__global__ __launch_bounds__(256) void kv8_prefill_weights_kernel(Kv8PrefillArgs a) {
    __shared__ float red[4];
    const int b = blockIdx.x, kvh = blockIdx.y, tid = threadIdx.x;
    const int first = max(0, b * kKv8Block - a.pos0) * a.G;
    const float2 *bw = a.bw + ((size_t)kvh * a.nblk + b) * a.rtiles * kPreRows;
    const float2 *total = a.bw + (size_t)kvh * a.nblk * a.rtiles * kPreRows;   // the first block's: .y
    const float *rsum = a.rsum + (size_t)kvh * a.rows;
    float s = 0.0f;
    constexpr int kB = 4;   // rows in flight
    for (int r0 = first + tid; r0 < a.rows; r0 += kB * 256) {
        float2 p[kB];
        float m[kB], f[kB];
#pragma unroll
        for (int i = 0; i < kB; ++i) {
            const int r = min(r0 + i * 256, a.rows - 1);
            p[i] = bw[r];
            m[i] = total[r].y;
            f[i] = rsum[r];
        }
#pragma unroll
        for (int i = 0; i < kB; ++i)
            if (r0 + i * 256 < a.rows) s += p[i].x * __builtin_amdgcn_exp2f(p[i].y - m[i]) * f[i];
    }
    s = wave_sum(s);
    if ((tid & 63) == 0) red[tid >> 6] = s;
    __syncthreads();
    if (tid == 0)
        ((float *)(a.cache + kv8_layout(a.Hkv, a.nb).weights))[(size_t)kvh * a.nb + b] +=
            (red[0] + red[1]) + (red[2] + red[3]);
}

// Workgroups of a KV head that are resident at once, two per CU, as far as a plan
// orders them; bytes of a launch's sums of weights.
static int prefill_slots(int Hkv) { return std::min(2 * device_cus() / Hkv, kPreOrder); }
constexpr int64_t kPreSums = 256 << 20;

// The launch shapes of a prefill call and its workspace.
struct PrefillPlan {
    int rows, rtiles, runs, splits, per;
    int64_t wgs;
    size_t ml, o, rsum, bw, bytes;
};
static PrefillPlan prefill_plan(int n, int pos0, int H, int Hkv, bool weights) {
    PrefillPlan p{};
    const int G = H / Hkv, total = pos0 + n;
    p.rows = n * G;
    p.rtiles = (p.rows + kPreRows - 1) / kPreRows;
    // A row tile's blocks may be cut into even runs of `per` at most: the least per,
    // of kPreLeast at least, whose runs all are resident at once.  (2048 tokens: 56
    // us; 850 workgroups of the same work in two rounds 69, as beginning and ending a
    // run takes about 9 us.)
    const int slots = prefill_slots(Hkv), most = kv8_blocks(total);
    auto count = [&](int per) {
        int64_t n = 0;
        for (int r = 0; r < p.rtiles; ++r) {
            const int last = (r + 1) * kPreRows < p.rows ? (r + 1) * kPreRows : p.rows;
            n += (kv8_blocks(pos0 + (last - 1) / G + 1) + per - 1) / per;
        }
        return n;
    };
    int lo = kPreLeast, hi = most;   // runs of `most` blocks are no cut at all
    if (p.rtiles > slots) lo = hi;
    while (lo < hi) {
        const int mid = lo + (hi - lo) / 2;
        if (count(mid) <= slots) hi = mid;
        else lo = mid + 1;
    }
    p.per = hi;
    p.runs = hi == most ? p.rtiles : (int)count(hi);
    p.splits = (most + p.per - 1) / p.per;
    p.wgs = (int64_t)p.runs * Hkv;
    size_t at = kArrivals * 4;
    auto take = [&](size_t b) {
        const size_t o = at;
        at += kv8_align(b);
        return o;
    };
    if (p.splits > 1) {
        const size_t parts = (size_t)p.splits * Hkv * p.rows;
        p.ml = take(parts * 8);
        p.o = take(parts * kKv8Hd * 4);
    }
    if (weights) {
        p.rsum = take((size_t)Hkv * p.rows * 4);
        p.bw = take((size_t)Hkv * most * p.rtiles * kPreRows * 8);
    }
    p.bytes = at;
    return p;
}

// Tokens of a launch: all, but with weights, whose sums take 8 bytes per row and
// block, as many as keep those under kPreSums.
static int prefill_step(int n, int pos0, int H, int Hkv, bool weights) {
    if (!weights) return n;
    const int64_t token = (int64_t)8 * H * kv8_blocks(pos0 + n);
    const int64_t most = std::max<int64_t>(1, kPreSums / token), calls = (n + most - 1) / most;
    return (int)((n + calls - 1) / calls);
}

// The plan's runs, the longest first; of those that run at once, the second half
// the other way round: a CU gets the longest and the shortest.
static void prefill_order(const PrefillPlan &p, int pos0, int G, int Hkv, Kv8PrefillOrder &o) {
    struct Run {
        int len;
        uint32_t id;
    } run[kPreOrder];
    int n = 0;
    for (int r = 0; r < p.rtiles; ++r) {
        const int last = (r + 1) * kPreRows < p.rows ? (r + 1) * kPreRows : p.rows;
        const int b = kv8_blocks(pos0 + (last - 1) / G + 1), k = (b + p.per - 1) / p.per;
        for (int i = 0; i < k; ++i)
            run[n++] = {pre_run_start(b, k, i + 1) - pre_run_start(b, k, i), (uint32_t)r | (uint32_t)i << 16};
    }
    std::sort(run, run + n, [](const Run &x, const Run &y) { return x.len != y.len ? x.len > y.len : x.id > y.id; });
    const int half = device_cus() / Hkv, two = 2 * half < n ? 2 * half : n;
    if (half < two) std::reverse(run + half, run + two);
    for (int i = 0; i < n; ++i) o.run[i] = run[i].id;
}

// What prefill_plan asks for at most over all calls of up to n tokens that end at
// pos0 + n or before, so that a workspace of the largest call serves every smaller one.
// Parts are splits times rows.  A cut launch has `slots` runs at most, of up to per
// blocks, per >= kPreLeast.  With T tokens visible to the last of r tiles, the tiles
// see r T / 64 blocks or more between them, as what they see rises evenly; so r T /
// (64 per) <= slots, and with splits < T / (32 per) + 1, splits r < 2 slots + r <= 3
// slots.  Sums of the weights: a launch's stay under kPreSums (or are one token's), but
// for the last tile's rounding to kPreRows rows.
static size_t prefill_bytes(int n, int pos0, int H, int Hkv, bool weights) {
    const int64_t rows = (int64_t)n * (H / Hkv), most = kv8_blocks(pos0 + n), slots = prefill_slots(Hkv);
    size_t at = kArrivals * 4;
    if (most > kPreLeast && slots > 1) {
        const int64_t uncut = std::min<int64_t>(rows, slots * kPreRows);
        const size_t parts = Hkv * std::min((most + kPreLeast - 1) / kPreLeast * uncut, 3 * slots * kPreRows);
        at += kv8_align(parts * 8) + kv8_align(parts * kKv8Hd * 4);
    }
    if (weights) {
        const int64_t pad = (rows + kPreRows - 1) / kPreRows * kPreRows, token = 8 * H * most;
        const int64_t launch = std::max<int64_t>(kPreSums, token) + 8 * (kPreRows - 1) * Hkv * most;
        at += kv8_align((size_t)Hkv * rows * 4) + kv8_align(std::min(8 * Hkv * most * pad, launch));
    }
    return at;
}

// Tokens pos0 .. pos0 + n - 1 of a call.
static int prefill_launch(const float *q, void *cache, int fmt, int n, int pos0, int H, int Hkv,
                          int max_seq, bool weights, float *out, char *w, size_t ws_bytes, hipStream_t s) {
    const PrefillPlan p = prefill_plan(n, pos0, H, Hkv, weights);
    OXB_REQUIRE(p.bytes <= ws_bytes, "prefill attention: a launch of %zu bytes of workspace, %zu there", p.bytes,
                ws_bytes);
    OXB_REQUIRE(p.wgs < (1 << 24), "prefill attention: %d tokens of %d heads", n, H);
    const int nblk = kv8_blocks(pos0 + n);
    const Kv8PrefillArgs a{q, (uint8_t *)cache, n, pos0, H, Hkv, H / Hkv, kv8_blocks(max_seq), p.rows, p.rtiles,
                           p.rtiles <= kPreOrder, p.per, nblk, out, (float2 *)(w + p.ml), (float *)(w + p.o),
                           weights ? (float *)(w + p.rsum) : nullptr, (float2 *)(w + p.bw)};
    const dim3 grid((unsigned)p.wgs), th(kPreThreads);
    Kv8PrefillOrder order;
    if (a.planned) prefill_order(p, pos0, a.G, Hkv, order);
    if (fmt == OXB_KV8_INT8) {
        if (weights)
            hipLaunchKernelGGL((kv8_prefill_kernel<OXB_KV8_INT8, true>), grid, th, 0, s, a, order);
        else
            hipLaunchKernelGGL((kv8_prefill_kernel<OXB_KV8_INT8, false>), grid, th, 0, s, a, order);
    } else {
        if (weights)
            hipLaunchKernelGGL((kv8_prefill_kernel<OXB_KV8_E4M3, true>), grid, th, 0, s, a, order);
        else
            hipLaunchKernelGGL((kv8_prefill_kernel<OXB_KV8_E4M3, false>), grid, th, 0, s, a, order);
    }
    OXB_CHECK_HIP(hipGetLastError());
    if (p.splits > 1) {
        hipLaunchKernelGGL(kv8_prefill_join_kernel, dim3((p.rows + 7) / 8, Hkv), dim3(256), 0, s, a);
        OXB_CHECK_HIP(hipGetLastError());
    }
    if (weights) {
        hipLaunchKernelGGL(kv8_prefill_weights_kernel, dim3(nblk, Hkv), dim3(256), 0, s, a);
        OXB_CHECK_HIP(hipGetLastError());
    }
    return 0;
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
    const int nb = kv8_blocks(max_seq);
    const DecodeWs w = decode_ws(batch, H, Hkv, nb);
    OXB_REQUIRE(ws && ((uintptr_t)ws & 255) == 0 && ws_bytes >= w.bytes,
                "attention: workspace is NULL, not 256-byte aligned or %zu bytes < %zu", ws_bytes, w.bytes);
    char *wp = (char *)ws;
    const bool many = decode_many(batch, Hkv);
    const Kv8DecodeArgs a{q, (uint8_t *)cache, cache_stride, pos, pos_stride, H, Hkv, H / Hkv, max_seq, nb,
                          decode_splits(batch, Hkv, nb), many, many ? 2 * kDecWaves : kDecWaves, out,
                          (int *)wp, (uint64_t *)(wp + w.ml), (uint64_t *)(wp + w.o), (uint64_t *)(wp + w.bw)};
    hipStream_t s = (hipStream_t)stream;
    const dim3 grid(Hkv, a.many ? batch : a.splits, a.many ? a.splits : batch), th(kDecThreads);
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
    return 0;
}

extern "C" size_t oxb_attn_prefill_kv8_ws_bytes(int n_tok, int pos0, int H, int Hkv, int hd,
                                                int add_weights) {
    if (n_tok < 1 || pos0 < 0 || pos0 > OXB_KV8_MAX_SEQ - n_tok || Hkv < 1 || H < 1 || H % Hkv ||
        H > 65535 || hd != kKv8Hd || (int64_t)n_tok * (H / Hkv) > (1 << 30))
        return 0;
    return prefill_bytes(n_tok, pos0, H, Hkv, add_weights != 0);
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
    const size_t bytes = prefill_bytes(n_tok, pos0, H, Hkv, add_weights != 0);
    OXB_REQUIRE(ws && ((uintptr_t)ws & 255) == 0 && ws_bytes >= bytes,
                "attention: workspace is NULL, not 256-byte aligned or %zu bytes < %zu", ws_bytes, bytes);
    const int step = prefill_step(n_tok, pos0, H, Hkv, add_weights != 0);
    for (int i = 0; i < n_tok; i += step)
        if (prefill_launch(q + (size_t)i * H * hd, cache, fmt, std::min(step, n_tok - i), pos0 + i, H, Hkv,
                           max_seq, add_weights != 0, out + (size_t)i * H * hd, (char *)ws, ws_bytes, (hipStream_t)stream))
            return -1;
    return 0;
}

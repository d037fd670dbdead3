// Attention over the paged KV cache for gfx950 (layout: paged.h): one new token
// per sequence (decode), and causal attention of packed tokens of several
// sequences, each behind the positions it holds already (prefill).  No
// counterpart in the reference, whose attention reads one dense f32 cache
// (nn/attention.rs:109-118).
//
//   out = sum_t p_t V_t,  p = softmax over the visible t of q.K_t / sqrt(128)
//
// One pass over the cache with a running reference m of the row's maximum:
// p' = 2^(x - m), l += p', O += p' V, and O and l are rescaled when a score
// passes m by 8 (in log2 units) -- a fixed m is as good as the exact maximum as
// long as nothing overflows, and the test costs less than a maximum over lanes
// for every tile.
//
// Arithmetic: K and V are f16, so both products run on f16 MFMA with f32 sums.
// f32 operands, q and p', go in as two f16 parts hi + lo (22 bits of each value;
// one part alone, 11 bits, would cost an f32 result three digits): q's row is
// first scaled by a power of two to a maximum in [2^13, 2^14), p' is at most
// 2^14, so that lo's own rounding stays 2^-25 absolute, 2^-39 of the largest.
// With f16 q and output, q is exact in one part; prefill then takes p' in one part
// (2^-12 of each weight, less than the rounding of the output), decode, which is
// bound by bytes, in two.
//
// What a row does not see has no part in it, whatever its bytes are: hidden scores
// become -inf by selection, and V elements that are not finite are taken out of
// units that some row does not see whole (0 times them would be NaN).  A reference
// of -inf says that a row has seen nothing, and its output is zeros; what it does see
// raises the reference to kPgLow at least, so that a row whose scores all are -inf
// has weights and a sum of 0 and ends as 0 / 0, NaN, as a softmax does.
#include "paged.h"
#include "paged_plan.h"

#include <algorithm>
#include <type_traits>

namespace oxb {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));

constexpr float kPgScore = 1.44269504088896340736f * 0.08838834764831844f;   // log2(e) / sqrt(128)
constexpr float kPgStep = 8.0f;       // a score may pass the reference by this much
constexpr float kPgBase = 6.0f;       // p' <= 2^(6 + kPgStep)
constexpr int kPgQExp = 14;           // q rows are scaled below 2^kPgQExp
constexpr float kPgNone = -__builtin_inff();
constexpr float kPgLow = -0x1.fffffep127f;   // the lowest f32

// A row's reference.  mx is the lane's largest score; where any row of the wave
// passes its reference by kPgStep, all take their row's maxima (over LANES lane
// groups), and al is what l and o shrink by.
struct PgRef {
    float m = kPgNone;
    __device__ __forceinline__ bool passed(float mx) const {
        return __any(mx > m + kPgStep || (m == kPgNone && mx > m));
    }
    template <int LANES>
    __device__ __forceinline__ float raise(float mx) {
#pragma unroll
        for (int s = 64 / LANES; s < 64; s <<= 1) mx = fmaxf(mx, __shfl_xor(mx, s, 64));
        const float n = fmaxf(m, mx), al = n == m ? 1.0f : __builtin_amdgcn_exp2f(m - n);
        m = n;
        return al;
    }
    // p' = 2^(x - off)
    __device__ __forceinline__ float off() const { return (m == kPgNone ? 0.0f : m) - kPgBase; }
    // the part's reference for a join: none where the row has seen nothing
    __device__ __forceinline__ float part() const { return m == kPgNone ? kPgNone : m - kPgBase; }
};

// The exponent that scales a row of maximum a below 2^kPgQExp (0 and values that
// are not finite: none).
__device__ __forceinline__ int pg_row_exp(float a) {
    return a > 0.0f && a < __builtin_inff() ? __builtin_amdgcn_frexp_expf(a) - kPgQExp : 0;
}

__device__ __forceinline__ float pg_ror8(float v) {   // lane i of 16 takes lane i ^ 8
    const int i = __float_as_int(v);
    return __int_as_float(__builtin_amdgcn_update_dpp(i, i, 0x128, 0xf, 0xf, false));
}

// Hand-over between workgroups goes through agent-scope stores and loads.
__device__ __forceinline__ void pg_put(uint64_t *p, float a, float b) {
    __hip_atomic_store(p, (uint64_t)__float_as_uint(a) | ((uint64_t)__float_as_uint(b) << 32), __ATOMIC_RELAXED,
                       __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 pg_get(const uint64_t *p) {
    const uint64_t v = __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
}

// Of two f16 in a word: all ones where less than `left` of them come before; 1 in each
// half that is an infinity or NaN.
__device__ __forceinline__ uint32_t pg_first2(int left) { return left >= 2 ? ~0u : left == 1 ? 0xffffu : 0u; }
__device__ __forceinline__ uint32_t pg_wild2(uint32_t w) { return ((w & 0x7c007c00u) + 0x04000400u) >> 15 & 0x10001u; }

__device__ __forceinline__ float4 pg_load4(const float *p) { return *(const float4 *)p; }
__device__ __forceinline__ float4 pg_load4(const _Float16 *p) {
    const half4_t h = *(const half4_t *)p;
    return make_float4((float)h.x, (float)h.y, (float)h.z, (float)h.w);
}
__device__ __forceinline__ void pg_store4(float *p, float x, float y, float z, float w) {
    *(float4 *)p = make_float4(x, y, z, w);
}
__device__ __forceinline__ void pg_store4(_Float16 *p, float x, float y, float z, float w) {
    *(half4_t *)p = half4_t{(_Float16)x, (_Float16)y, (_Float16)z, (_Float16)w};
}

// A row's value from its parts' sum t, softmax sum l and reference m (nothing seen: 0).
__device__ __forceinline__ float pg_quot(float t, float l, float m) { return m == kPgNone ? 0.0f : t / l; }

// What all lanes read and no kernel in flight writes: by scalar loads.
template <typename R>
__device__ __forceinline__ R pg_uniform(const R *p) {
    static_assert(sizeof(R) % 4 == 0, "whole words");
    struct Words {
        int w[sizeof(R) / 4];
    } r;
    const auto *c = (const __attribute__((address_space(4))) int *)p;
#pragma unroll
    for (unsigned i = 0; i < sizeof(R) / 4; ++i) r.w[i] = c[i];
    return __builtin_bit_cast(R, r);
}

// ---------------------------------------------------------------------------
// decode
// ---------------------------------------------------------------------------
// Workgroup: four waves over a run of a sequence's units of a KV head, wave w taking
// every fourth, for ROWS of its query heads at a time (more go round again over the
// run).  16x16x32 MFMA, operands straight from memory to registers:
//   ROWS 8, for groups of up to 8: the 16 columns are the 8 heads' hi and lo parts, for
//   q and for p' alike, so the two-part products cost nothing over one, and column
//   c + (c ^ 8) is the score; ROWS 16: a product for each part;
//   scores: A = 16 K rows x 32 dims, B = q.  K rows are taken in an order that
//   leaves lane group g (of 4) the scores of positions 8 g .. 8 g + 7;
//   P.V: A = 16 dims x 32 positions, B = the lane's own eight p'.
// Bound by the cache's bytes.  The launch is as wide as the card holds, and each
// workgroup finds its run from the lengths themselves: a run has `per` units at
// most, the least that keeps all runs resident at once, so that the work of a
// ragged batch is spread evenly whatever its longest sequence is.  A sequence's
// runs meet in the workspace: each stores its part and counts in, and the last one
// joins them in order, so the sum does not depend on which is last.
// H 20 over 5, pages of 32: 64 sequences of up to 4096, 284 MB, 60 us (4.7 TB/s);
// four of up to 100001, 527 MB, 98.5 us (5.35 TB/s, a copy 4.9); one of 100000 55.5 (4.6);
// one of 2304, 6 MB, 8.2 us, a chain of loads (length, page, K and V, parts) of 0.5 to 1
// us each.  Sequences of up to 16 units are not cut, which saves them the join: 32 of
// 512 positions 8.5 us (cut from 4 units on 10.2), 8 of 300 7.1 (7.7), one of 500 7.6 (7.5);
// uncut up to 32 units, 16 of 1000 take 11.3 for 9.2.  H 32 over 2, 13 of up to 49812: 67
// us, in two passes of 8 heads 107.  Joining 32 runs at once instead of 16 gave nothing
// (one of 100000, its bytes in the 256 MB cache, 47.1 for 47.8 us; 2304 9.3 for 8.6).
constexpr int kDecWaves = 4;
constexpr int kDecThreads = 64 * kDecWaves;
constexpr int kDecRows = 8;            // query heads that the workgroup's threads hold a row of
constexpr int kDecQs = kPgHd + 8;      // q row stride in LDS (f16)
constexpr int kDecLeast = 4;           // units of a run
constexpr int kDecFine = 24;           // units of a run, more of which are cut finer than one round of the card
constexpr int kDecUncut = 16;          // units of a sequence that is not cut
constexpr int kDecSlots = 512;         // runs that are resident at once, at most
constexpr int kDecParts = 4 * kDecSlots;

struct PgDecodeArgs {
    const void *q;
    const _Float16 *pages;
    const int *table, *len;
    int n_pages, page_log, table_stride, batch, H, Hkv, G;
    int runs, most, slots;   // runs beside one a sequence and head: wanted, at most; resident ones, to be filled
    void *out;
    int *cnt;        // [kDecParts] zero between calls
    uint64_t *ml;    // [kDecParts][G] reference and sum (two floats)
    uint64_t *o;     // [kDecParts][G][64] pairs of dims
};

template <typename T, int ROWS>
__global__ __launch_bounds__(kDecThreads, 2) void paged_decode_kernel(PgDecodeArgs a) {
    constexpr int RT = ROWS / kDecRows;    // rows of a thread: orow, orow + 8
    __shared__ _Float16 sq[2 * ROWS * kDecQs];
    __shared__ float sqs[ROWS];
    __shared__ float2 sml[kDecWaves][ROWS];
    __shared__ float4 so[kDecWaves][ROWS][kPgHd / 4];
    __shared__ int s_last;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int orow = tid >> 5, od = (tid & 31) * 4;         // the row and dims a thread joins
    const int64_t cap = (int64_t)a.table_stride << a.page_log;

    // Each wave: the sum of all units, the runs' length from it, and the run of this
    // workgroup.  sum ceil(n / per) <= sum n / per + batch, so per >= sum / (runs beside
    // one a sequence) keeps within the launch.
    auto length = [&](int z) { return z < a.batch ? (int)min(max((int64_t)a.len[z], (int64_t)0), cap) : 0; };
    const int len0 = length(lane);
    uint32_t total = pg_units(len0);   // (2^31 at most)
    for (int c = 64; c < a.batch; c += 64) total += pg_units(length(c + lane));
    total = (uint32_t)wave_isum_dpp((int)total);
    // all / runs or up to 1 more (the product is within 2^-21 of it; whole divisions of 64
    // bits would be a tenth of a short call's time)
    const float all = (float)total * (float)a.Hkv * 1.000001f;
    auto share = [&](int runs) { return (int)fminf(all * __builtin_amdgcn_rcpf((float)runs), 1 << 20) + 1; };
    int per = max(kDecLeast, max(share(a.most), min(share(a.runs), kDecFine)));
    auto runs_of = [&](int units, int per) {
        return units <= kDecUncut ? 1 : pg_div(units + per - 1, __builtin_amdgcn_rcpf((float)per));
    };
    // few sequences, which are in the lanes: the least length that fits (48 of up to 2304
    // 32.0 -> 30.6 us, 32 23.4 -> 22.0)
    if (a.slots) {
        for (int lo = max(kDecLeast, share(a.slots)); lo < per;) {
            const int c = (lo + per) >> 1;
            const int n = wave_isum_dpp(lane < a.batch ? runs_of(pg_units(len0), c) : 0) * a.Hkv;
            if (n <= a.slots) per = c;
            else lo = c + 1;
        }
    }
    int z = -1, len = 0, runs = 0, r = 0, part = 0;
    {
        int base = 0, cut = 0;   // workgroups and parts before the 64 sequences
        for (int c = 0; c < a.batch; c += 64) {
            const int n = c ? length(c + lane) : len0, u = pg_units(n);
            const int k = c + lane < a.batch ? runs_of(u, per) : 0;
            const int upto = wave_iscan(k * a.Hkv), cutto = wave_iscan(k > 1 ? k * a.Hkv : 0);
            const int i = __popcll(__ballot(base + upto <= (int)blockIdx.x));
            if (i < 64) {
                z = c + i;
                len = __builtin_amdgcn_readlane(n, i);
                runs = __builtin_amdgcn_readlane(k, i);
                r = (int)blockIdx.x - (base + __builtin_amdgcn_readlane(upto, i) - runs * a.Hkv);
                part = cut + __builtin_amdgcn_readlane(cutto, i) - runs * a.Hkv;
                break;
            }
            base += __builtin_amdgcn_readlane(upto, 63);
            cut += __builtin_amdgcn_readlane(cutto, 63);
        }
    }
    if (z < 0 || z >= a.batch) return;
    const int run = r / a.Hkv, kvh = r - run * a.Hkv;
    part += kvh * runs;   // the parts of this sequence and head
    const int units = pg_units(len);
    const int b0 = pg_run_start(units, runs, run), b1 = pg_run_start(units, runs, run + 1);
    T *out = (T *)a.out + ((size_t)z * a.H + (size_t)kvh * a.G) * kPgHd;
    if (b0 >= b1) {   // (an idle sequence)
        for (int i = tid; i < a.G * kPgHd; i += kDecThreads) out[i] = (T)0.0f;
        return;
    }
    const T *q = (const T *)a.q + ((size_t)z * a.H + (size_t)kvh * a.G) * kPgHd;
    float4 qv[RT];
    auto load_q = [&](int hc) {
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            const int r = hc + orow + 8 * i;
            qv[i] = r < a.G ? pg_load4(q + (size_t)r * kPgHd + od) : make_float4(0, 0, 0, 0);
        }
    };
    load_q(0);
    const int *table = a.table + (size_t)z * a.table_stride;
    const int in_page = (1 << (a.page_log - 5)) - 1;
    const int rr = lane & 15, g = lane >> 4;
    // K row of this lane in 16-row tile 0 (tile 1: 4 positions on), V octet of dim rr
    const uint32_t koff = paged_k_elem(8 * (rr >> 2) + (rr & 3), 8 * g), voff = paged_v_elem(8 * g, rr);
    struct Blk {
        uint4 k[8], v[8];
        bool there;
    };
    // the pages of the wave's next 64 units, one a lane
    auto load_ids = [&](int b) {
        const int u = b + kDecWaves * lane;
        return u < b1 ? table[u >> (a.page_log - 5)] : 0;
    };

    for (int hc = 0; hc < a.G; hc += ROWS) {
        const int g0 = hc, ng = min(ROWS, a.G - hc);
        int ids = load_ids(b0 + wave), next = 0;   // unit b0 + wave + 4 next is lane next % 64's
        auto load = [&](int b) {
            Blk x;
            const int id = __builtin_amdgcn_readlane(ids, next & 63);
            x.there = (unsigned)id < (unsigned)a.n_pages;
            const _Float16 *p = a.pages + paged_unit(x.there ? id : 0, kvh, b & in_page, a.Hkv, a.page_log);
#pragma unroll
            for (int i = 0; i < 8; ++i)   // tile i & 1, dims 32 (i / 2) ..
                x.k[i] = *(const uint4 *)(p + koff + (i >> 1) * 4 * kPgUnit * 8 + (i & 1) * 32);
#pragma unroll
            for (int i = 0; i < 8; ++i) x.v[i] = *(const uint4 *)(p + voff + i * 16 * 8);
            return x;
        };
        // the first unit is on its way while q is made ready
        Blk cur = load(min(b0 + wave, b1 - 1));
#pragma unroll
        for (int i = 0; i < RT; ++i) {   // q rows: scaled, split, and their score units
            const float4 v = qv[i];
            const int row = orow + 8 * i;
            float m = fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w)));
#pragma unroll
            for (int s = 16; s > 0; s >>= 1) m = fmaxf(m, __shfl_xor(m, s, 64));
            const int e = pg_row_exp(m);
            const float f[4] = {v.x, v.y, v.z, v.w};
            half4_t hi, lo;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float x = ldexpf(f[j], -e);
                hi[j] = (_Float16)x;
                lo[j] = (_Float16)(x - (float)hi[j]);
            }
            *(half4_t *)(sq + row * kDecQs + od) = hi;
            *(half4_t *)(sq + (row + ROWS) * kDecQs + od) = lo;
            if ((tid & 31) == 0) sqs[row] = ldexpf(kPgScore, e);
        }
        lds_barrier();
        half8_t qf[RT][4];
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int s = 0; s < 4; ++s)
                qf[i][s] = *(const half8_t *)(sq + (rr + 16 * i) * kDecQs + 32 * s + 8 * g);
        const float qs = sqs[rr & (ROWS - 1)];

        f32x4 o[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = f32x4{0, 0, 0, 0};
        PgRef ref;
        float lsum = 0.0f;
        for (int b = b0 + wave; b < b1; b += kDecWaves) {
            if ((++next & 63) == 0) ids = load_ids(b + kDecWaves);
            Blk nxt = cur;
            if (b + kDecWaves < b1) nxt = load(b + kDecWaves);
            f32x4 s0{0, 0, 0, 0}, s1{0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int i = 0; i < RT; ++i) {
                    s0 = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, cur.k[2 * s]), qf[i][s], s0, 0, 0, 0);
                    s1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, cur.k[2 * s + 1]), qf[i][s], s1, 0, 0, 0);
                }
            auto whole = [](float v) { return RT == 1 ? v + pg_ror8(v) : v; };   // of both parts
            float x[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = whole(s0[i]);
                x[4 + i] = whole(s1[i]);
            }
            // of the lane's positions 8 g .. 8 g + 7, the first `left` are there
            const bool partial = len - b * kPgUnit < kPgUnit || !cur.there;
            const int left = cur.there ? len - b * kPgUnit - 8 * g : 0;
            float mx = kPgNone;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (!partial || i < left) mx = fmaxf(mx, x[i] * qs);
            if (!partial || left > 0) mx = fmaxf(mx, kPgLow);
            if (ref.passed(mx)) {
                const float al = ref.raise<4>(mx);
                lsum *= al;
#pragma unroll
                for (int i = 0; i < 8; ++i) o[i] *= al;
            }
            const float moff = ref.off();
            half8_t pf[RT];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float p = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], qs, -moff));
                if (partial && i >= left) p = 0.0f;
                lsum += p;
                const _Float16 hi = (_Float16)p;
                const _Float16 lo = (_Float16)(p - (float)hi);
                pf[0][i] = RT == 2 || rr < 8 ? hi : lo;
                pf[RT - 1][i] = RT == 2 || rr >= 8 ? lo : hi;
            }
            if (partial) {   // what is not there may hold anything
                uint32_t mk[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) mk[i] = pg_first2(left - 2 * i);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    cur.v[i].x &= mk[0];
                    cur.v[i].y &= mk[1];
                    cur.v[i].z &= mk[2];
                    cur.v[i].w &= mk[3];
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int j = 0; j < RT; ++j)
                    o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, cur.v[i]), pf[j], o[i], 0, 0, 0);
            cur = nxt;
        }
        // the four waves' parts
        lsum += __shfl_xor(lsum, 16, 64);
        lsum += __shfl_xor(lsum, 32, 64);
        if (lane < ROWS) sml[wave][lane] = make_float2(ref.part(), lsum);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            auto whole = [](float v) { return RT == 1 ? v + pg_ror8(v) : v; };
            const float4 t = make_float4(whole(o[i][0]), whole(o[i][1]), whole(o[i][2]), whole(o[i][3]));
            if (rr < ROWS) so[wave][rr][(4 * i + g) ^ (4 * (rr & 7))] = t;   // (no two rows in a bank)
        }
        lds_barrier();
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            const int row = orow + 8 * i;
            float M = kPgNone;
#pragma unroll
            for (int w = 0; w < kDecWaves; ++w) M = fmaxf(M, sml[w][row].x);
            float lt = 0.0f;
            float4 t = make_float4(0, 0, 0, 0);
#pragma unroll
            for (int w = 0; w < kDecWaves; ++w) {
                const float2 p = sml[w][row];
                const float f = p.x == kPgNone ? 0.0f : __builtin_amdgcn_exp2f(p.x - M);
                const float4 v = so[w][row][(od >> 2) ^ (4 * orow)];
                lt = __builtin_fmaf(p.y, f, lt);
                t.x = __builtin_fmaf(v.x, f, t.x);
                t.y = __builtin_fmaf(v.y, f, t.y);
                t.z = __builtin_fmaf(v.z, f, t.z);
                t.w = __builtin_fmaf(v.w, f, t.w);
            }
            if (row >= ng) continue;
            if (runs == 1) {
                pg_store4(out + (size_t)(g0 + row) * kPgHd + od, pg_quot(t.x, lt, M), pg_quot(t.y, lt, M),
                          pg_quot(t.z, lt, M), pg_quot(t.w, lt, M));
            } else {
                const size_t at = (size_t)(part + run) * a.G + g0 + row;
                pg_put(a.o + at * 64 + (od >> 1), t.x, t.y);
                pg_put(a.o + at * 64 + (od >> 1) + 1, t.z, t.w);
                if (od == 0) pg_put(a.ml + at, M, lt);
            }
        }
        lds_barrier();   // LDS is free for the next heads
        load_q(hc + ROWS);
    }
    if (runs == 1) return;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();   // every thread's part has arrived
    if (tid == 0) {
        int *cnt = a.cnt + part;
        const int old = __hip_atomic_fetch_add(cnt, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        s_last = old == runs - 1;
        if (s_last) __hip_atomic_store(cnt, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!s_last) return;
    for (int hc = 0; hc < a.G; hc += kDecRows) {
        const int ng = min(kDecRows, a.G - hc);
        // 32 lanes a head; the lanes that fewer than 8 heads leave take every
        // second, fourth or eighth run of one
        const int np = ng > 4 ? 8 : ng > 2 ? 4 : ng, step = kDecRows / np, jr = orow % np;
        if (jr < ng) {
            const size_t row = (size_t)part * a.G + hc + jr;
            float M = kPgNone, lt = 0.0f;
            float4 t = make_float4(0, 0, 0, 0);
            constexpr int kB = 16;   // runs in flight
            for (int s0 = orow / np; s0 < runs; s0 += kB * step) {
                float2 p[kB], lo[kB], hi[kB];
#pragma unroll
                for (int j = 0; j < kB; ++j) {
                    p[j] = make_float2(kPgNone, 0.0f);
                    lo[j] = hi[j] = make_float2(0, 0);
                    const int s = s0 + j * step;
                    if (s < runs) {
                        const size_t at = row + (size_t)s * a.G;
                        p[j] = pg_get(a.ml + at);
                        lo[j] = pg_get(a.o + at * 64 + (od >> 1));
                        hi[j] = pg_get(a.o + at * 64 + (od >> 1) + 1);
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
                    const float f = p[j].x == kPgNone ? 0.0f : __builtin_amdgcn_exp2f(p[j].x - M);
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
            float M = kPgNone, lt = 0.0f;
            float4 t = make_float4(0, 0, 0, 0);
            for (int i = orow; i < kDecRows; i += np) M = fmaxf(M, sml[0][i].x);
            for (int i = orow; i < kDecRows; i += np) {
                const float2 p = sml[0][i];
                const float f = p.x == kPgNone ? 0.0f : __builtin_amdgcn_exp2f(p.x - M);
                const float4 v = so[0][i][od >> 2];
                lt = __builtin_fmaf(p.y, f, lt);
                t.x = __builtin_fmaf(v.x, f, t.x);
                t.y = __builtin_fmaf(v.y, f, t.y);
                t.z = __builtin_fmaf(v.z, f, t.z);
                t.w = __builtin_fmaf(v.w, f, t.w);
            }
            pg_store4(out + (size_t)(hc + orow) * kPgHd + od, pg_quot(t.x, lt, M), pg_quot(t.y, lt, M),
                      pg_quot(t.z, lt, M), pg_quot(t.w, lt, M));
        }
        lds_barrier();
    }
}

// Workgroups of a launch, and the runs that are wanted beside one a sequence and head:
// as many as are resident with them.  Where the sequences alone are half of the
// resident workgroups or more, half as many beside them; there runs of more than
// kDecFine units are cut further, as the rounds' ends cost more than a join then (H 20
// over 5, 52 sequences of up to 2304: 31.8 us, cut to 12 units 34.2, to 48 33.9; 96 of
// them 55.0, 56.3, 57.6; 64 of up to 4096 60.4, 62.0, 58.6).
struct DecodePlan {
    int runs, most, slots;
    int64_t wgs;
};
static DecodePlan decode_plan(int batch, int Hkv, int64_t units) {
    const int slots = std::min(2 * device_cus(), kDecSlots);
    const int64_t rows = (int64_t)batch * Hkv;
    DecodePlan p;
    p.runs = rows < slots / 2 ? (int)(slots - rows) : slots / 2;
    p.most = rows < slots / 2 ? p.runs : 2 * slots;
    p.slots = rows < slots / 2 && batch <= 64 ? slots : 0;
    p.wgs = std::min(rows + p.most, rows * (units <= kDecUncut ? 1 : (units + kDecLeast - 1) / kDecLeast));
    return p;
}

// Parts: only a cut sequence's.  k runs where k > 1 are at most 2 (k - 1), and the
// runs past one of each sequence and head are 2 kDecSlots at most.
struct DecodeWs {
    size_t ml, o, bytes;
};
static size_t pg_align(size_t b) { return (b + 255) & ~(size_t)255; }
static DecodeWs decode_ws(int G) {
    DecodeWs w;
    w.ml = kDecParts * 4;
    w.o = w.ml + pg_align((size_t)kDecParts * G * 8);
    w.bytes = w.o + (size_t)kDecParts * G * kPgHd * 4;
    return w;
}

// ---------------------------------------------------------------------------
// prefill
// ---------------------------------------------------------------------------
// Rows of a sequence and KV head are (token, query head of the group) pairs,
// token-major, so that a unit of K and V serves all of the group's heads.  A
// workgroup takes a tile of 128 rows, 32 per wave, and a run of units; K and V go
// from memory to LDS directly, in the order the MFMA operands are read (every read
// is 1 KB contiguous).
//   scores: 32x32x16 MFMA, A = 32 K rows, B = q (in registers), K rows in an order
//   that leaves lane half h the scores of positions 8 h + 16 m + 0..7;
//   P.V: A = 32 dims x 16 positions, B = the lane's own p'.
// Bound by the MFMAs as long as the softmax's VALU work runs under them: the next
// unit's score products alternate with this unit's exponentials, and P.V with the
// rest of them.  K runs a unit ahead of V; rings of four units of each leave one
// barrier per two units.
// H 20 over 5: 8192 tokens 588 us f32 (1170 TFLOP/s of MFMA work, both parts; a large
// f16 product of the library 1153); 12 prompts of up to 4096 507-535 us f32, 320-340
// f16 (1050, 850 TFLOP/s), of which an f16 tile's beginning and end are 14k cycles, 12%
// (20k with q and the output straight from and to memory); the MFMAs are busy for 62-65%
// (f32) and 46% (f16) of all cycles.  101 tokens 12 us; 23 drafts of up to 5 tokens
// behind up to 4000 32 us; 333 tokens behind 30011 and two shorter turns, f16, 148-160.
// With p' in two parts too, f16 takes 416 us for the prompts and 205 for the 333, and is
// as near to 64 bits as its output's rounding (2.0e-4 in the norm; 2.6e-4 to 2.9e-4 as
// it is, half a step of f16 being 4.9e-4).
// Not kept (f32, f16 of the 12 prompts; then 519, 320): 64 rows a wave, one wave a SIMD
// (859, 409: the compiler moves accumulators to and fro); tiles of 256 rows, eight
// waves (532, 317; the 333 tokens 160 against 152); the loads of K and V spread over the
// products (522, 326) or V through registers (531, 343).
//
// What the sequences' lengths are is known on the device only.  A first launch, of
// one workgroup, makes the list of runs: the tiles, each a run where they fill the
// card (but for the last few of equal ones), else cut into runs of `per` units at
// most, the least that keeps all runs resident at once; the longest first.  A last
// launch joins the cut tiles' parts.  (The tiles past whole rounds of equal ones, cut and
// uncut: 3300 tokens behind 20000 1195 and 1622 us, where 3264 take 1174; 4096 1518 and 1704.)
constexpr int kPreRing = 4;
constexpr int kPreOps = kPgHalf * 2 / 16;    // 16-byte operands of a unit's K (or V)
constexpr size_t kPreHead = kDecParts * 4;   // decode's counters, in a workspace of both, then the counts

struct PgPrefillArgs : PgList {
    const void *q;
    const _Float16 *pages;
    const int *table;
    int n_pages, H, rows;
    void *out;
    float2 *ml;     // [slots][Hkv][rows] a row's reference and sum
    float *o;       // [slots][Hkv][rows][128]
};

__global__ __launch_bounds__(kPlanThreads) void paged_plan_kernel(PgList a) { pg_list(a); }

// 16 bytes of each lane from base + off to LDS at m0 + 16 * lane (as lds_dma16, with a
// scalar base).  The load reads m0 a wait state after its write at the earliest, and
// the base five after one by v_readfirstlane; the compiler adds neither inside asm.
__device__ __forceinline__ void pg_dma16(const void *base, uint32_t off, uint32_t lds) {
    // (uniform as they are: for the compiler)
    const uint64_t at = (uint64_t)base;
    const uint64_t sbase = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)at) |
                           (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(at >> 32)) << 32;
    const uint32_t slds = __builtin_amdgcn_readfirstlane((int)lds);
    uint32_t saved;
    asm volatile(
        "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 2\n\tglobal_load_lds_dwordx4 %2, %3\n\ts_mov_b32 m0, %0"
        : "=&s"(saved)
        : "s"(slds), "v"(off), "s"(sbase)
        : "memory");
}

// A row's 16-byte pieces lie in LDS exchanged by the row's number, so that neither a
// piece of all rows nor a row's pieces meet in a bank.
template <int PIECES>
__device__ __forceinline__ int pg_piece(int row, int c) { return row * PIECES + (c ^ (row & (PIECES - 1))); }

template <typename T>
__global__ __launch_bounds__(kPreThreads, 2) void paged_prefill_kernel(PgPrefillArgs a) {
    constexpr int PARTS = std::is_same<T, float>::value ? 2 : 1;
    // rings of K [8][64] and V operands [4 dims][2][64]: unit u of the run in slot u % 4.
    // The rows of q lie in V's ring and in K's behind its first slot before, those of
    // the output in all of them after.
    __shared__ uint4 lds[2 * kPreRing + PARTS - 1][kPreOps];
    uint4(*sk)[kPreOps] = lds, (*sv)[kPreOps] = lds + kPreRing + PARTS - 1;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    PgRun run;
    int kvh;
    // (loaded with the list's arguments, not behind it: 101 tokens 12.1 -> 11.9 us)
    asm volatile("" ::"s"(a.q), "s"(a.pages), "s"(a.table), "s"(a.n_pages), "s"(a.H), "s"(a.out));
    if (a.few) {
        const PgFew p = pg_few(a);
        if (blockIdx.x == 0 && tid == 0) a.counts[1] = p.nt;   // (for the join, of no tiles too)
        if (!pg_few_run(a, p, blockIdx.x, run)) return;
        kvh = run.head;
    } else {
        // Where tiles are cut, a record a workgroup, else one for all KV heads.  (Both are
        // loaded with the counts; past them, whatever is there.)
        struct Counts {
            int runs, cuts, cut;
        };
        const Counts n = pg_uniform((const Counts *)a.counts);
        const int each = blockIdx.x / a.Hkv;
        run = pg_uniform(a.runs + each);
        kvh = blockIdx.x - each * a.Hkv;
        if (n.cut) {
            if ((int)blockIdx.x >= (n.runs * a.Hkv + 7) / 8 * 8) return;
            run = pg_uniform(a.runs + min((int)blockIdx.x, kPreOrder - 1));
            kvh = run.head;
            if (kvh < 0) return;
        } else if (each >= n.runs) {
            return;
        }
    }
    // (uniform all of it: for the compiler)
    auto first = [](int &v) { v = __builtin_amdgcn_readfirstlane(v); };
    first(kvh);
    first(run.tile);
    first(run.u0);
    first(run.u1);
    first(run.part);
    first(run.cu);
    first(run.nq);
    first(run.past);
    first(run.z);
    first(run.tok);
    const int r0 = run.tile * kPreRows, rows = min(kPreRows, run.nq * a.G - r0);   // of the tile
    const int b0 = run.u0, b1 = run.u1, h = lane >> 5;
    const int rest = r0 - run.tok * a.G;
    auto tok_of = [&](int r) { return pg_div(rest + r, a.inv_G); };   // from run.tok on
    T *out = (T *)a.out + ((size_t)(run.cu + run.tok) * a.H + kvh * a.G) * kPgHd;
    const T *q = (const T *)a.q + ((size_t)(run.cu + run.tok) * a.H + kvh * a.G) * kPgHd;
    const int wrow = wave * 32, row = wrow + (lane & 31);   // of the tile
    const int tok = tok_of(min(row, rows - 1));
    const int qrow = tok * a.H + rest + min(row, rows - 1) - tok * a.G;   // its row from q on
    if (b0 >= b1) {   // the tile sees nothing
        for (int r = 0; r < 32; ++r) {
            const int at = __builtin_amdgcn_readlane(qrow, r);
            if (wrow + r < rows)
                for (int i = lane; i < kPgHd; i += 64) out[(size_t)at * kPgHd + i] = (T)0.0f;
        }
        return;
    }
    const int past = run.past + run.tok, qpos = past + tok;
    // positions that the wave's last and first rows see (none: no row at all)
    const bool some = wrow < rows;
    const int wseen = some ? past + tok_of(min(wrow + 31, rows - 1)) + 1 : 0;
    const int wfull = past + tok_of(min(wrow, rows - 1)) + 1;
    const int wb = max(b0, min(b1, pg_units(max(wseen, 0))));

    // Pages: of the run's first units by scalar loads, which wait for no others, and by
    // lanes those of 64 from unit b0 + 3 on, the first that the loop brings.
    const int *table = a.table + (size_t)run.z * a.table_stride;
    const int unit_log = a.page_log - 5, in_page = (1 << unit_log) - 1;
    auto first_id = [&](int u) { return pg_uniform(table + (min(u, b1 - 1) >> unit_log)); };
    auto load_ids = [&](int u) { return table[min(u + lane, b1 - 1) >> unit_log]; };
    const int id0 = first_id(b0), id1 = first_id(b0 + 1), id2 = first_id(b0 + 2);
    int ids = load_ids(b0 + 3);
    uint32_t gone = 0;   // bit u % 32: unit u's page is none
    auto unit = [&](int id, int u) {
        const uint32_t bit = 1u << (u & 31);
        gone &= ~bit;
        if ((unsigned)id >= (unsigned)a.n_pages) {
            gone |= bit;
            id = 0;
        }
        return a.pages + paged_unit(id, kvh, min(u, b1 - 1) & in_page, a.Hkv, a.page_log);
    };
    // a wave brings 32 dims of K and of V of each unit: operands 2 wave, 2 wave + 1.
    // MFMA row i holds position i with bits 2 and 3 exchanged.
    const int kpos = (lane & 19) | ((lane & 4) << 1) | ((lane & 8) >> 1);
    const uint32_t koff = 2 * paged_k_elem(kpos, 8 * (4 * wave + h));
    const uint32_t voff = 2 * paged_v_elem(8 * h, 32 * wave + (lane & 31));
    const uint32_t lds0 = (uint32_t)(size_t)(__attribute__((address_space(3))) void *)&lds[0][0] + 2048 * wave;
    auto bring_k = [&](const _Float16 *p, int r) {
        const uint32_t to = lds0 + (r & 3) * kPreOps * 16;
        pg_dma16(p, koff, to);
        pg_dma16(p, koff + 2 * kPgUnit * 16, to + 1024);
    };
    auto bring_v = [&](const _Float16 *p, int r) {
        const uint32_t to = lds0 + (kPreRing + PARTS - 1 + (r & 3)) * kPreOps * 16;
        pg_dma16(p, voff, to);
        pg_dma16(p, voff + 2 * kPgHd * 16, to + 1024);
    };

    // q through LDS, 256 bytes of each row at a time (a lane loading its own row's
    // pieces meets 32 rows with each load), to operand s: dims 16 s + 8 h + j of row
    // lane % 32
    half8_t qh[8], ql[8];
    float qs = kPgScore;
    uint4 *sq[2] = {&sv[0][0] + 512 * wave, &sk[1][0] + 512 * wave};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = 4 * i + (lane >> 4), c = (lane & 15) ^ (r & 15);
        const uint32_t off = __shfl(qrow, r, 64) * (uint32_t)(kPgHd * sizeof(T)) + 16 * c;
#pragma unroll
        for (int p = 0; p < PARTS; ++p)
            pg_dma16(q, off + 256 * p, lds0 - 2048 * wave + (uint32_t)((char *)(sq[p] + 64 * i) - (char *)&lds[0][0]));
    }
    const _Float16 *u0 = unit(id0, b0), *u1 = unit(id1, b0 + 1), *u2 = unit(id2, b0 + 2);
    bring_k(u0, 0);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if constexpr (PARTS == 1) {
#pragma unroll
        for (int s = 0; s < 8; ++s)
            qh[s] = __builtin_bit_cast(half8_t, sq[0][pg_piece<16>(lane & 31, 2 * s + h)]);
    } else {
        float v[64];
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float4 f = __builtin_bit_cast(float4, sq[i >> 3][pg_piece<16>(lane & 31, 4 * (i >> 1 & 3) + 2 * h + (i & 1))]);
            v[4 * i] = f.x;
            v[4 * i + 1] = f.y;
            v[4 * i + 2] = f.z;
            v[4 * i + 3] = f.w;
        }
#pragma unroll
        for (int i = 0; i < 64; i += 2) m = fmaxf(fmaxf(fabsf(v[i]), fabsf(v[i + 1])), m);
        m = fmaxf(m, __shfl_xor(m, 32, 64));
        const int e = max(pg_row_exp(m), -127);   // (a row below 2^-113 stays below 2^kPgQExp)
        const float up = ldexpf(1.0f, -e);
        qs = ldexpf(kPgScore, e);
        // each part rounded once from the exact product
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
    f32x16 o[4];
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;
    PgRef ref;
    float lsum = 0.0f;

    lds_barrier();   // the first K is there, and every wave has its q
    bring_k(u1, 1);
    bring_k(u2, 2);
    bring_v(u0, 0);
    bring_v(u1, 1);
    f32x16 s0, s1;
#pragma unroll
    for (int i = 0; i < 16; ++i) s0[i] = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const half8_t k = __builtin_bit_cast(half8_t, sk[0][i * 64 + lane]);
        s0 = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, qh[i], s0, 0, 0, 0);
        if constexpr (PARTS == 2) s0 = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, ql[i], s0, 0, 0, 0);
    }
    // the running maximum with four more scores (in v_max3's form)
    auto top = [&](float m, const f32x16 &s, int i) {
        m = fmaxf(fmaxf(s[i], s[i + 1]), m);
        return fmaxf(fmaxf(s[i + 2], s[i + 3]), m);
    };
    float smax = top(top(top(top(kPgNone, s0, 0), s0, 4), s0, 8), s0, 12);
    wait_vmcnt<0>();
    lds_barrier();   // the others are there, and the first K slot is free
    // Unit b, its scores in s and their maximum in smax; the next one's go to sn.
    // r: b's place in the run; SOME: some rows may not see all of it.
    auto block = [&](auto SOME, int b, int r, f32x16 &s, f32x16 &sn) {
        constexpr bool some_hidden = decltype(SOME)::value;
        const int p0 = b * kPgUnit;
        const bool there = !((gone >> (b & 31)) & 1);
        float low = kPgLow;
        if constexpr (some_hidden) {
            // positions of the lane's scores: 16 (i / 8) + 8 h + i % 8
            const int left = there ? qpos + 1 - p0 - 8 * h : 0;
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = (i & 7) + 16 * (i >> 3) < left ? s[i] : kPgNone;
            smax = top(top(top(top(kPgNone, s, 0), s, 4), s, 8), s, 12);
            if (left <= 0) low = kPgNone;
        }
        const float mx = fmaxf(smax * qs, low);
        if (ref.passed(mx)) {
            const float al = ref.raise<2>(mx);
            lsum *= al;
#pragma unroll
            for (int d = 0; d < 4; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] *= al;
        }
        const float moff = ref.off();
        // From here on the order is the one written: SLOT ends what may run under
        // the MFMA before it.
#define SLOT() __builtin_amdgcn_sched_barrier(0)
        const uint4 *kb = sk[(r + 1) & 3] + lane, *vb = sv[r & 3] + lane;
        half8_t ph[2], pl[2], v[4], k[2];
        float pa, pb, ps = 0.0f;
        uint32_t found = 0;   // bits 15 and 31: V that is not finite
        bool wild = false;
        auto exps = [&](int j) {   // elements 2 j, 2 j + 1
            pa = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * j], qs, -moff));
            pb = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * j + 1], qs, -moff));
        };
        auto split = [&](int j) {
            ps += pa;
            ps += pb;
            asm volatile("" : "+v"(ps));   // (here, not all sums at the end)
            half2_t hi;
            hi.x = (_Float16)pa;
            hi.y = (_Float16)pb;
            asm("" : "+v"(hi));
            ph[j >> 2][2 * (j & 3)] = hi.x;
            ph[j >> 2][2 * (j & 3) + 1] = hi.y;
            if constexpr (PARTS == 2) {
                half2_t lo;
                lo.x = (_Float16)(pa - (float)hi.x);
                lo.y = (_Float16)(pb - (float)hi.y);
                pl[j >> 2][2 * (j & 3)] = lo.x;
                pl[j >> 2][2 * (j & 3) + 1] = lo.y;
            }
        };
        auto look = [&](int i) {   // at operand i of V
            const uint4 x = vb[64 * i];
            auto word = [&](uint32_t w) { found |= (w & 0x7c007c00u) + 0x04000400u; };
            word(x.x);
            word(x.y);
            word(x.z);
            word(x.w);
        };
        // (of a unit with V that is not finite, only what the wave's last row sees and
        // is finite)
        auto get_v = [&](int d, int m) {
            uint4 x = vb[d * 128 + 64 * m];
            if constexpr (some_hidden) {
                if (wild) {   // uniform
                    const int left = (there ? wseen - p0 - 8 * h : 0) - 16 * m + opaque_zero();
                    auto word = [&](uint32_t &w, int j) {
                        w &= pg_first2(left - 2 * j);
                        w &= ~(pg_wild2(w) * 0xffffu);
                    };
                    word(x.x, 0);
                    word(x.y, 1);
                    word(x.z, 2);
                    word(x.w, 3);
                }
            }
            return __builtin_bit_cast(half8_t, x);
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
            if (some_hidden && i < 4) look(2 * i);
            if constexpr (PARTS == 2) {
                SLOT();
                sn = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[i & 1], ql[i], sn, 0, 0, 0);
            }
            if (some_hidden && i < 4) look(2 * i + 1);
            if (i < 6) split(i);
            if (some_hidden && i == 5) wild = __any(found & 0x80008000u);
            if (i < 6) k[i & 1] = __builtin_bit_cast(half8_t, kb[(i + 2) * 64]);
            else
                for (int d = 2 * (i - 6); d < 2 * (i - 5); ++d) v[d] = get_v(d, 0);
            SLOT();
        }
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[d], ph[0], o[d], 0, 0, 0);
            if (d & 1) split(6 + (d >> 1));
            else exps(6 + (d >> 1));
            if constexpr (PARTS == 1) v[d] = get_v(d, 1);
            SLOT();
        }
        if constexpr (PARTS == 2) {
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[d], pl[0], o[d], 0, 0, 0);
                v[d] = get_v(d, 1);
                SLOT();
            }
        }
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[d], ph[1], o[d], 0, 0, 0);
            if constexpr (PARTS == 2) {
                SLOT();
                o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[d], pl[1], o[d], 0, 0, 0);
            }
            smax = top(d == 0 ? kPgNone : smax, sn, 4 * d);
            SLOT();
        }
#undef SLOT
        lsum += ps;
        if constexpr (some_hidden) {
            if (wild) {   // a dim of a row that sees such a V is NaN
                const int seen = there ? wseen - p0 - 8 * h : 0, sees = there ? qpos + 1 - p0 - 8 * h : 0;
                for (int d = 0; d < 4; ++d) {
                    f32x16 n;
#pragma unroll
                    for (int i = 0; i < 16; ++i) n[i] = 0.0f;
#pragma unroll
                    for (int m = 0; m < 2; ++m) {
                        const uint4 x = vb[d * 128 + 64 * m];
                        const uint32_t in[4] = {x.x, x.y, x.z, x.w};
                        uint32_t w[4], y[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            w[j] = pg_wild2(in[j] & pg_first2(seen - 16 * m - 2 * j)) * 0x3c00u;   // 1
                            y[j] = pg_first2(sees - 16 * m - 2 * j) & 0x3c003c00u;
                        }
                        n = __builtin_amdgcn_mfma_f32_32x32x16_f16(
                            __builtin_bit_cast(half8_t, make_uint4(w[0], w[1], w[2], w[3])),
                            __builtin_bit_cast(half8_t, make_uint4(y[0], y[1], y[2], y[3])), n, 0, 0, 0);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (e == d)
#pragma unroll
                            for (int i = 0; i < 16; ++i) o[e][i] = n[i] > 0.0f ? __builtin_nanf("") : o[e][i];
                }
            }
        }
    };
    // The two waves of a SIMD take turns at priority, a pair of units each (their
    // slots differ in the lowest bit as a rule): by age alone one runs at its
    // full speed and the other, at half of it, finishes late.
    uint32_t hwid;
    asm volatile("s_getreg_b32 %0, hwreg(HW_REG_HW_ID)" : "=s"(hwid));
    // K of b + 3, b + 4 and V of b + 2, b + 3 come under the pair b, b + 1
    auto bring = [&](int b) {
        const int r = b - b0;
        if (((r >> 1) ^ hwid) & 1) __builtin_amdgcn_s_setprio(1);
        else __builtin_amdgcn_s_setprio(0);
        if (b + 2 >= b1) return;   // uniform
        const _Float16 *u3 = unit(__builtin_amdgcn_readlane(ids, r & 63), b + 3);
        const _Float16 *u4 = unit(__builtin_amdgcn_readlane(ids, (r & 63) + 1), b + 4);
        bring_k(u3, r + 3);
        bring_k(u4, r + 4);
        bring_v(u2, r + 2);
        bring_v(u3, r + 3);
        u2 = u4;
        if ((r & 63) == 62) ids = load_ids(b + 5);   // (waited for with the pair)
    };
    // pairs that every row of the wave sees whole, then the rest of the run (with
    // one loop of both, the registers do not suffice)
    int b = b0;
    const int whole = some ? min(b1, wfull >> 5) : 0;
    for (; b + 1 < whole && !(((gone >> (b & 31)) | (gone >> ((b + 1) & 31))) & 1); b += 2) {
        const int r = b - b0;
        bring(b);
        block(std::false_type{}, b, r, s0, s1);
        block(std::false_type{}, b + 1, r + 1, s1, s0);
        wait_vmcnt<0>();
        lds_barrier();
    }
    for (; b < b1; b += 2) {
        const int r = b - b0;
        bring(b);
        if (b < wb) block(std::true_type{}, b, r, s0, s1);
        if (b + 1 < wb) block(std::true_type{}, b + 1, r + 1, s1, s0);
        wait_vmcnt<0>();
        lds_barrier();
    }
    lsum += __shfl_xor(lsum, 32, 64);
    if (!some) return;
    // The rows of the output whole, through LDS: a lane's dims are 32 d + 8 k + 4 h + 0..3
    // of its row.  (Stored from there, 16 or 32 bytes a row with each store: twice the
    // time.)
    const bool direct = run.part < 0;
    const float f = !direct ? 1.0f : ref.m == kPgNone ? 0.0f : 1.0f / lsum;
    uint4 *so = &lds[0][0] + 1024 * wave;
    const int er = lane & 31;
    if (direct && PARTS == 1) {
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int k = 0; k < 4; ++k)
                pg_store4((_Float16 *)&so[pg_piece<16>(er, 4 * d + k)] + 4 * h, o[d][4 * k] * f, o[d][4 * k + 1] * f,
                          o[d][4 * k + 2] * f, o[d][4 * k + 3] * f);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int r = 4 * i + (lane >> 4), at = __shfl(qrow, r, 64);
            const uint4 x = so[pg_piece<16>(r, lane & 15)];
            if (wrow + r < rows) *(uint4 *)(out + (size_t)at * kPgHd + 8 * (lane & 15)) = x;
        }
        return;
    }
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int k = 0; k < 4; ++k)
            pg_store4((float *)&so[pg_piece<32>(er, 8 * d + 2 * k + h)], o[d][4 * k] * f, o[d][4 * k + 1] * f,
                      o[d][4 * k + 2] * f, o[d][4 * k + 3] * f);
    const size_t prow = ((size_t)run.part * a.Hkv + kvh) * a.rows + wrow;   // (of a part)
    if (!direct && h == 0 && row < rows) a.ml[prow + er] = make_float2(ref.part(), lsum);
    float *dst = direct ? (float *)out : a.o + prow * kPgHd;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int r = 2 * i + h, at = direct ? __shfl(qrow, r, 64) : r;
        const uint4 x = so[pg_piece<32>(r, lane & 31)];
        if (wrow + r < rows) *(uint4 *)(dst + (size_t)at * kPgHd + 4 * (lane & 31)) = x;
    }
}

// Joins a cut tile's parts: 32 threads a row, 4 dims each.  Bound by the parts' bytes
// where there are many (the 333 tokens: 31 MB in 8.2 us), else by the launch (the
// drafts 6.3; 32 rows a workgroup the same).
template <typename T>
__global__ __launch_bounds__(256) void paged_join_kernel(PgPrefillArgs a) {
    const int c = blockIdx.x / (kPreRows / 8), kvh = blockIdx.y, d = (threadIdx.x & 31) * 4;
    const PgCut t = pg_uniform(a.cuts + c);   // (with the count; past it, whatever is there)
    if (c >= pg_uniform(a.counts + 1) || t.runs == 1) return;   // (written by its only run)
    const int lrow = blockIdx.x % (kPreRows / 8) * 8 + (threadIdx.x >> 5), row = t.tile * kPreRows + lrow;
    if (row >= t.nq * a.G) return;
    const size_t step = (size_t)a.Hkv * a.rows, r = ((size_t)t.part * a.Hkv + kvh) * a.rows + lrow;
    float M = kPgNone, lt = 0.0f;
    float4 s = make_float4(0, 0, 0, 0);
    constexpr int kB = 8;   // parts in flight
    for (int i0 = 0; i0 < t.runs; i0 += kB) {
        float2 p[kB];
        float4 v[kB];
#pragma unroll
        for (int i = 0; i < kB; ++i) {
            p[i] = make_float2(kPgNone, 0.0f);
            v[i] = make_float4(0, 0, 0, 0);
            if (i0 + i < t.runs) {   // (uniform)
                const size_t at = r + (i0 + i) * step;
                p[i] = a.ml[at];
                v[i] = *(const float4 *)(a.o + at * kPgHd + d);
            }
        }
        float m = M;
#pragma unroll
        for (int i = 0; i < kB; ++i) m = fmaxf(m, p[i].x);
        const float f0 = m == M ? 1.0f : __builtin_amdgcn_exp2f(M - m);
        M = m;
        lt *= f0;
        s = make_float4(s.x * f0, s.y * f0, s.z * f0, s.w * f0);
#pragma unroll
        for (int i = 0; i < kB; ++i) {
            const float f = p[i].x == kPgNone ? 0.0f : __builtin_amdgcn_exp2f(p[i].x - M);
            lt = __builtin_fmaf(p[i].y, f, lt);
            s.x = __builtin_fmaf(v[i].x, f, s.x);
            s.y = __builtin_fmaf(v[i].y, f, s.y);
            s.z = __builtin_fmaf(v[i].z, f, s.z);
            s.w = __builtin_fmaf(v[i].w, f, s.w);
        }
    }
    pg_store4((T *)a.out + ((size_t)(t.cu + row / a.G) * a.H + kvh * a.G + row % a.G) * kPgHd + d, pg_quot(s.x, lt, M),
              pg_quot(s.y, lt, M), pg_quot(s.z, lt, M), pg_quot(s.w, lt, M));
}

// Workspace of a call of n tokens (of its largest launch, whose sizes an n of the whole
// call gives too): the lists and the parts' rows.
struct PrefillPlan : PgSizes {
    int rows;
    size_t runs_at, cuts_at, ml, o, bytes;
};
static PrefillPlan prefill_plan(int n, int batch, int G, int Hkv) {
    PrefillPlan p{pg_sizes(n, batch, G, Hkv, device_cus())};
    p.rows = (int)std::min<int64_t>(kPreRows, (int64_t)n * G);
    size_t at = kPreHead + 256;
    auto take = [&](size_t b) {
        const size_t o = at;
        at += pg_align(b);
        return o;
    };
    p.runs_at = take(p.runs * sizeof(PgRun));
    p.cuts_at = take(p.cuts * sizeof(PgCut));
    p.ml = take((size_t)p.slots * Hkv * p.rows * 8);
    p.o = take((size_t)p.slots * Hkv * p.rows * kPgHd * 4);
    p.bytes = at;
    return p;
}

static int heads_check(int H, int Hkv) {
    OXB_REQUIRE(Hkv > 0 && H > 0 && H % Hkv == 0, "attention: heads %d not a multiple of kv heads %d", H, Hkv);
    OXB_REQUIRE(H <= 65535, "attention: %d heads", H);
    return 0;
}
static int dtype_check(int dtype, const void *q, const void *out) {
    OXB_REQUIRE(dtype == OXB_F32 || dtype == OXB_F16, "attention: type %d", dtype);
    OXB_REQUIRE(q && out && (((uintptr_t)q | (uintptr_t)out) & 15) == 0,
                "attention: q or out is NULL or not 16-byte aligned");
    return 0;
}

}  // namespace oxb

using namespace oxb;

extern "C" size_t oxb_attn_decode_paged_ws_bytes(int batch, int H, int Hkv, int hd) {
    if (batch < 1 || batch > kPgBatch || Hkv < 1 || Hkv > 4096 || H < 1 || H % Hkv || H > 65535 || hd != kPgHd) return 0;
    return decode_ws(H / Hkv).bytes;
}

extern "C" int oxb_attn_decode_paged(const void *q, int dtype, const void *pages, int n_pages, int page_size,
                                     const int *table, int table_stride, const int *len, int batch, int H, int Hkv,
                                     int hd, void *out, void *ws, size_t ws_bytes, void *stream) {
    clear_error();
    if (paged_check(pages, n_pages, page_size, Hkv, hd) || paged_table_check(table, table_stride, page_size, batch) ||
        heads_check(H, Hkv) || dtype_check(dtype, q, out))
        return -1;
    OXB_REQUIRE(len, "attention: len is NULL");
    const int G = H / Hkv;
    const DecodeWs w = decode_ws(G);
    OXB_REQUIRE(ws && ((uintptr_t)ws & 255) == 0 && ws_bytes >= w.bytes,
                "attention: workspace is NULL, not 256-byte aligned or %zu bytes < %zu", ws_bytes, w.bytes);
    char *wp = (char *)ws;
    const DecodePlan p = decode_plan(batch, Hkv, ((int64_t)table_stride * page_size + kPgUnit - 1) / kPgUnit);
    const PgDecodeArgs a{q, (const _Float16 *)pages, table, len, n_pages, paged_log(page_size), table_stride, batch,
                         H, Hkv, G, p.runs, p.most, p.slots, out, (int *)wp, (uint64_t *)(wp + w.ml), (uint64_t *)(wp + w.o)};
    OXB_REQUIRE(p.wgs < (int64_t)1 << 24, "attention: batch %d of %d kv heads", batch, Hkv);   // (2^32 threads)
    const dim3 grid((unsigned)p.wgs), th(kDecThreads);
    hipStream_t s = (hipStream_t)stream;
    if (dtype == OXB_F32) {
        if (G <= 8) hipLaunchKernelGGL((paged_decode_kernel<float, 8>), grid, th, 0, s, a);
        else hipLaunchKernelGGL((paged_decode_kernel<float, 16>), grid, th, 0, s, a);
    } else {
        if (G <= 8) hipLaunchKernelGGL((paged_decode_kernel<_Float16, 8>), grid, th, 0, s, a);
        else hipLaunchKernelGGL((paged_decode_kernel<_Float16, 16>), grid, th, 0, s, a);
    }
    OXB_CHECK_HIP(hipGetLastError());
    return 0;
}

extern "C" size_t oxb_attn_prefill_paged_ws_bytes(int n_tok, int batch, int H, int Hkv, int hd) {
    if (n_tok < 1 || batch < 1 || batch > kPgPrefill || Hkv < 1 || Hkv > 4096 || H < 1 || H % Hkv || H > 65535 ||
        hd != kPgHd || (int64_t)n_tok * (H / Hkv) > kPreMost)
        return 0;
    return prefill_plan(n_tok, batch, H / Hkv, Hkv).bytes;
}

extern "C" int oxb_attn_prefill_paged(const void *q, int dtype, const void *pages, int n_pages, int page_size,
                                      const int *table, int table_stride, const int *cu, const int *len, int n_tok,
                                      int batch, int H, int Hkv, int hd, void *out, void *ws, size_t ws_bytes,
                                      void *stream) {
    clear_error();
    if (paged_check(pages, n_pages, page_size, Hkv, hd) || paged_table_check(table, table_stride, page_size, batch) ||
        heads_check(H, Hkv) || dtype_check(dtype, q, out))
        return -1;
    OXB_REQUIRE(batch <= kPgPrefill, "prefill attention: batch %d", batch);
    OXB_REQUIRE(cu && len, "prefill attention: cu or len is NULL");
    const int G = H / Hkv;
    OXB_REQUIRE(n_tok >= 1 && (int64_t)n_tok * G <= kPreMost, "prefill attention: %d tokens", n_tok);
    // (q's bytes would pass any device's memory)
    OXB_REQUIRE((int64_t)n_tok * H <= INT32_MAX, "prefill attention: %d tokens of %d heads", n_tok, H);
    const PrefillPlan p = prefill_plan(n_tok, batch, G, Hkv);
    OXB_REQUIRE(ws && ((uintptr_t)ws & 255) == 0 && ws_bytes >= p.bytes,
                "attention: workspace is NULL, not 256-byte aligned or %zu bytes < %zu", ws_bytes, p.bytes);
    char *w = (char *)ws;
    hipStream_t s = (hipStream_t)stream;
    const int window = pg_window(n_tok, batch, G);
    for (int t = 0; t < n_tok; t += std::min(window, n_tok - t)) {
        const int n = std::min(window, n_tok - t);
        const PgSizes z = pg_sizes(n, batch, G, Hkv, device_cus());
        const int few = pg_few_step(z, batch);
        const PgPrefillArgs a{{cu, len, paged_log(page_size), table_stride, batch, n_tok, t, t + n, G, Hkv, z.most, z.slots,
                               (device_cus() + 7) / 8, few, 1.0f / G, (int *)(w + kPreHead), (PgRun *)(w + p.runs_at),
                               (PgCut *)(w + p.cuts_at)},
                              q, (const _Float16 *)pages, table, n_pages, H, p.rows, out, (float2 *)(w + p.ml),
                              (float *)(w + p.o)};
        if (!few) {
            hipLaunchKernelGGL(paged_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, (const PgList &)a);
            OXB_CHECK_HIP(hipGetLastError());
        }
        const dim3 grid((unsigned)z.wgs), th(kPreThreads);
        if (dtype == OXB_F32) hipLaunchKernelGGL((paged_prefill_kernel<float>), grid, th, 0, s, a);
        else hipLaunchKernelGGL((paged_prefill_kernel<_Float16>), grid, th, 0, s, a);
        OXB_CHECK_HIP(hipGetLastError());
        // a tile is cut only where it has more than kPreLeast units
        if ((int64_t)table_stride * page_size > kPreLeast * kPgUnit && z.slots > 1) {
            const dim3 jgrid((unsigned)(few ? z.most : std::min(z.most, z.slots / 2)) * (kPreRows / 8), Hkv);
            if (dtype == OXB_F32) hipLaunchKernelGGL((paged_join_kernel<float>), jgrid, dim3(256), 0, s, a);
            else hipLaunchKernelGGL((paged_join_kernel<_Float16>), jgrid, dim3(256), 0, s, a);
            OXB_CHECK_HIP(hipGetLastError());
        }
    }
    return 0;
}

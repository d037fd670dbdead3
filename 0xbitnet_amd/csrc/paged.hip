// The paged KV cache for gfx950 (layout: paged.h): a step's bookkeeping (block
// tables, slot map, free list) and the append of new rows.  No counterpart in
// the reference, whose cache is one buffer per layer (nn/attention.rs:23-48).
#include "paged.h"

#include <algorithm>

namespace oxb {

// ---------------------------------------------------------------------------
// bookkeeping
// ---------------------------------------------------------------------------
// With pages(n) = ceil(n / page_size), over the sequences in order:
//   end_z  = sum of the growths wanted up to z           (the packed tokens)
//   back_z = sum of the pages given back up to z
//   upto_z = sum of the pages needed up to z by growths that fit table and buffer
//   granted iff no page is needed or upto_z <= n_free + back_last
// Three prefix sums over at most 4096 sequences, which every workgroup forms by
// itself in LDS (a few us; one workgroup of all would write the slots of 100000
// tokens alone, and a launch between would cost as much as the sums).  Then a
// token finds its sequence, and a page taken or given back its owner, by
// bisection; a page's number comes from where it lay before the call, so nothing
// that is written is read.  Only len and n_free may be their own outputs: they
// are written after everything is read, behind a barrier in a call of one
// workgroup, by a second launch in one of several.
// Bound by latency: lengths and growths are loaded once and kept in LDS, a sum over
// the workgroup takes one barrier, and a thread has the pages of four tokens on
// their way at once.  A step of 64 sequences, nine of which end, 549 pages, 6.5 us
// (8.2 with the lengths read from memory by each token and page and two barriers a
// sum, 7.5 with 256 threads); 48 sequences growing by 65000 tokens, two launches, 10.2
// (13.7).
// Sums saturate at kPgMany, past every limit that they are compared with.
constexpr int kUpdThreads = 1024;
constexpr int kUpdWaves = kUpdThreads / 64;
constexpr uint32_t kPgMany = 1u << 30;
constexpr int kUpdTokens = 16384;   // of a call of one workgroup

struct PagedUpdateArgs {
    int page_log, batch, table_stride, free_cap, n_max;
    const int *len, *delta;
    int *table, *free_pages;
    const int *n_free;
    int *len_out, *n_free_out, *cu, *granted, *slots, *pos;
    int lists, lengths;   // what the launch writes
};

__device__ __forceinline__ uint32_t sat_add(uint32_t a, uint32_t b) { return min(a + b, kPgMany); }

// Sums over the lanes up to this one.
__device__ __forceinline__ uint32_t wave_sat_scan(uint32_t v) {
    v = sat_add(v, (uint32_t)dpp0<0x111, 0xf>((int)v));
    v = sat_add(v, (uint32_t)dpp0<0x112, 0xf>((int)v));
    v = sat_add(v, (uint32_t)dpp0<0x114, 0xf>((int)v));
    v = sat_add(v, (uint32_t)dpp0<0x118, 0xf>((int)v));
    v = sat_add(v, (uint32_t)dpp0<0x142, 0xa>((int)v));
    v = sat_add(v, (uint32_t)dpp0<0x143, 0xc>((int)v));
    return v;
}

// A value's sum over the threads before this one, in two steps: up to the lane, with
// the wave's sum to LDS, and behind a barrier the whole.
__device__ __forceinline__ uint32_t block_scan_begin(uint32_t v, uint32_t *to) {
    const uint32_t s = wave_sat_scan(v);
    if ((threadIdx.x & 63) == 63) to[threadIdx.x >> 6] = s;
    const uint32_t before = (uint32_t)__shfl_up((int)s, 1, 64);
    return (threadIdx.x & 63) == 0 ? 0 : before;
}
__device__ __forceinline__ uint32_t block_scan_end(uint32_t v, const uint32_t *to) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t w = wave_sat_scan(lane < kUpdWaves ? to[lane] : 0);
    return wave ? sat_add(v, (uint32_t)__builtin_amdgcn_readlane((int)w, wave - 1)) : v;
}

// The first of n ascending sums above i (n if none).
__device__ __forceinline__ int above(const uint32_t *sum, int n, uint32_t i) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (sum[mid] > i) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

__global__ __launch_bounds__(kUpdThreads) void paged_update_kernel(PagedUpdateArgs a) {
    __shared__ uint32_t end[kPgBatch], back[kPgBatch], upto[kPgBatch];
    __shared__ int s_held[kPgBatch], s_delta[kPgBatch];
    __shared__ uint32_t part[3][kUpdWaves];
    const int tid = threadIdx.x, B = a.batch;
    const int64_t cap = (int64_t)a.table_stride << a.page_log;
    const int round = (1 << a.page_log) - 1;
    const int n_free = min(max(*a.n_free, 0), a.free_cap);
    struct Seq {
        int held, after, delta, need, gone;   // after: the length unless growth is granted
        bool fits;
    };
    auto pages = [&](int64_t n) { return (int)((n + round) >> a.page_log); };
    auto seq = [&](int z) {   // (once end_z is there)
        Seq s;
        s.held = s_held[z];
        s.delta = s_delta[z];
        const int64_t want = (int64_t)s.held + s.delta;
        s.after = s.delta < 0 ? (int)max(want, (int64_t)0) : s.held;
        s.fits = s.delta > 0 && want <= cap && end[z] <= (uint32_t)a.n_max;
        s.need = s.fits ? pages(want) - pages(s.held) : 0;
        s.gone = pages(s.held) - pages(s.after);
        return s;
    };
    // a thread's consecutive sequences
    const int per = (B + kUpdThreads - 1) / kUpdThreads, z0 = tid * per, z1 = min(B, z0 + per);
    uint32_t sum = 0;
    for (int z = z0; z < z1; ++z) {
        const int d = a.delta[z];
        s_held[z] = (int)min(max((int64_t)a.len[z], (int64_t)0), cap);
        s_delta[z] = d;
        sum = sat_add(sum, min((uint32_t)max(d, 0), (uint32_t)a.n_max + 1));
        end[z] = sum;
    }
    sum = block_scan_begin(sum, part[0]);
    __syncthreads();
    sum = block_scan_end(sum, part[0]);
    uint32_t b1 = 0, b2 = 0;
    for (int z = z0; z < z1; ++z) {
        end[z] = sat_add(end[z], sum);
        const Seq s = seq(z);
        back[z] = b1 = sat_add(b1, s.gone);
        upto[z] = b2 = sat_add(b2, s.need);
    }
    b1 = block_scan_begin(b1, part[1]);
    b2 = block_scan_begin(b2, part[2]);
    __syncthreads();
    b1 = block_scan_end(b1, part[1]);
    b2 = block_scan_end(b2, part[2]);
    for (int z = z0; z < z1; ++z) {
        back[z] = sat_add(back[z], b1);
        upto[z] = sat_add(upto[z], b2);
    }
    __syncthreads();
    const uint32_t given = back[B - 1], avail = sat_add(given, n_free);
    const int k = upto[B - 1] <= avail ? B : above(upto, B, avail);
    const uint32_t taken = k ? upto[k - 1] : 0;
    auto granted = [&](int z, const Seq &s) { return s.fits && (s.need == 0 || upto[z] <= avail); };

    if (a.lists) {
        auto given_page = [&](uint32_t i) {   // i-th of those given back
            const int z = above(back, B, i);
            const Seq s = seq(z);
            return a.table + (size_t)z * a.table_stride + pages(s.after) + (i - (back[z] - s.gone));
        };
        auto taken_page = [&](uint32_t r) {   // those given back first, the last first, then the list's end
            return r < given ? given_page(given - 1 - r) : a.free_pages + (n_free - 1 - (int)(r - given));
        };
        const uint32_t at = blockIdx.x * kUpdThreads + tid, step = gridDim.x * kUpdThreads;
        constexpr int kT = 4;   // tokens of a thread at once
        int z = -1;
        for (uint32_t t0 = at; t0 < (uint32_t)a.n_max; t0 += kT * step) {
            const int *from[kT];
            int p[kT], page[kT];
#pragma unroll
            for (int i = 0; i < kT; ++i) {
                const uint32_t t = t0 + i * step;
                p[i] = -1;
                from[i] = nullptr;
                if (t >= (uint32_t)a.n_max) continue;
                if (z < 0 || z >= B || end[z] <= t) z = above(end, B, t);   // (often the same)
                if (z >= B) continue;
                const Seq s = seq(z);
                if (!granted(z, s)) continue;
                p[i] = s.held + (int)(t - (end[z] - s.delta));
                const int b = p[i] >> a.page_log, first = pages(s.held);
                from[i] = b < first ? a.table + (size_t)z * a.table_stride + b
                                    : taken_page(upto[z] - s.need + (b - first));
            }
#pragma unroll
            for (int i = 0; i < kT; ++i) page[i] = from[i] ? *from[i] : -1;
#pragma unroll
            for (int i = 0; i < kT; ++i) {
                const uint32_t t = t0 + i * step;
                if (t >= (uint32_t)a.n_max) break;
                const int64_t x = ((int64_t)page[i] << a.page_log) + (p[i] & round);
                if (a.slots) a.slots[t] = page[i] >= 0 && x <= INT32_MAX ? (int)x : -1;
                if (a.pos) a.pos[t] = p[i];
            }
        }
        for (uint32_t r = at; r < taken; r += step) {
            const int z = above(upto, B, r);
            const Seq s = seq(z);
            a.table[(size_t)z * a.table_stride + pages(s.held) + (r - (upto[z] - s.need))] = *taken_page(r);
        }
        const uint32_t left = given > taken ? given - taken : 0;
        for (uint32_t i = at; i < left && n_free + i < (uint32_t)a.free_cap; i += step)
            a.free_pages[n_free + i] = *given_page(i);
        if (blockIdx.x == 0)
            for (int z = tid; z < B; z += kUpdThreads) {
                if (z == 0) a.cu[0] = 0;
                a.cu[z + 1] = (int)min(end[z], (uint32_t)a.n_max);
                if (a.granted) {
                    const Seq s = seq(z);
                    a.granted[z] = granted(z, s) ? s.delta : 0;
                }
            }
    }
    if (a.lengths) {   // (behind the barriers: every thread has what it reads)
        for (int z = tid; z < B; z += kUpdThreads) {
            const Seq s = seq(z);
            a.len_out[z] = granted(z, s) ? s.held + s.delta : s.after;
        }
        if (tid == 0) *a.n_free_out = (int)min((uint32_t)a.free_cap, avail - taken);
    }
}

// ---------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------
// A workgroup takes 32 packed tokens of a KV head (8 where there are few).  K: 16 bytes of a row go to 16
// bytes of its unit.  V goes through LDS: tokens that follow one another inside an
// octet of positions are written together, a whole octet of a dim as one 16-byte
// store, others (a decode step's single rows) as 2-byte stores.  Bound by the bytes:
// 15700 tokens of 5 KV heads, 80 MB, 15.0 us (5.4 TB/s); 64 single rows 3.5 us (7.0 by
// 32 tokens a workgroup).
constexpr int kAppTokens = 32, kAppFew = 8;
constexpr int kAppThreads = 256;
constexpr int kAppStride = kPgHd + 2;   // of a V row in LDS

struct PagedAppendArgs {
    _Float16 *pages;
    const _Float16 *k, *v;
    size_t tok_stride, head_stride;
    const int *src_pos, *slots;
    int n_tok, n_slots, Hkv, page_log;
};

template <int TOKENS>
__global__ __launch_bounds__(kAppThreads) void paged_append_kernel(PagedAppendArgs a) {
    constexpr int kPieces = TOKENS * 16, kEach = (kPieces + kAppThreads - 1) / kAppThreads;   // of 16 bytes
    __shared__ _Float16 sv[TOKENS * kAppStride];
    __shared__ int sslot[TOKENS], slead[TOKENS], scount[TOKENS], snum;
    const int tid = threadIdx.x, t0 = blockIdx.x * TOKENS, head = blockIdx.y;
    const int round = (1 << a.page_log) - 1;
    auto unit = [&](int s) {
        return a.pages + paged_unit(s >> a.page_log, head, (s & round) >> 5, a.Hkv, a.page_log);
    };
    // rows by 16-byte pieces
    uint4 kr[kEach], vr[kEach];
    int slot[kEach], row[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int l = (tid >> 4) + 16 * i, t = t0 + l;
        const bool some = l < TOKENS && t < a.n_tok;
        slot[i] = some ? a.slots[t] : -1;
        row[i] = some && a.src_pos ? a.src_pos[t] : 0;
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int l = (tid >> 4) + 16 * i;
        if ((unsigned)slot[i] >= (unsigned)a.n_slots || row[i] < 0) slot[i] = -1;
        if (l < TOKENS && (tid & 15) == 0) sslot[l] = slot[i];
        kr[i] = vr[i] = make_uint4(0, 0, 0, 0);
        if (slot[i] >= 0) {
            const size_t at = (size_t)(t0 + l) * a.tok_stride + (size_t)head * a.head_stride + (size_t)row[i] * kPgHd +
                              8 * (tid & 15);
            kr[i] = *(const uint4 *)(a.k + at);
            vr[i] = *(const uint4 *)(a.v + at);
        }
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        if (slot[i] < 0) continue;
        *(uint4 *)(unit(slot[i]) + paged_k_elem(slot[i] & 31, 8 * (tid & 15))) = kr[i];
        uint32_t *row = (uint32_t *)(sv + ((tid >> 4) + 16 * i) * kAppStride + 8 * (tid & 15));
        row[0] = vr[i].x;
        row[1] = vr[i].y;
        row[2] = vr[i].z;
        row[3] = vr[i].w;
    }
    __syncthreads();
    if (tid < 64) {   // the tokens that begin a run inside an octet, and its length
        const int s = tid < TOKENS ? sslot[tid] : -1;
        const bool lead = s >= 0 && (tid == 0 || (s & 7) == 0 || sslot[tid - 1] != s - 1);
        const uint64_t m = __ballot(lead), gap = __ballot(lead || s < 0);
        if (lead) {
            const uint64_t later = gap & ~((2ull << tid) - 1);
            const int i = __popcll(m & ((1ull << tid) - 1));
            slead[i] = tid;
            scount[i] = __builtin_ctzll(later) - tid;   // (the lanes from TOKENS on are gaps)
        }
        if (tid == 0) snum = __popcll(m);
    }
    __syncthreads();
    for (int i = tid; i < snum * kPgHd; i += kAppThreads) {
        const int t = slead[i >> 7], n = scount[i >> 7], d = i & 127, s = sslot[t];
        _Float16 *dst = unit(s) + paged_v_elem(s & 31, d);
        const _Float16 *src = sv + t * kAppStride + d;
        if (n == 8) {
            typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
            half8_t x;
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = src[j * kAppStride];
            *(half8_t *)dst = x;
        } else {
            for (int j = 0; j < n; ++j) dst[j] = src[j * kAppStride];
        }
    }
}

}  // namespace oxb

using namespace oxb;

extern "C" size_t oxb_paged_bytes(int n_pages, int page_size, int Hkv, int hd) {
    if (!paged_size_ok(page_size) || n_pages < 1 || (int64_t)n_pages * page_size > INT32_MAX || hd != kPgHd ||
        Hkv < 1 || Hkv > 4096)
        return 0;
    return (size_t)n_pages * page_size * Hkv * kPgHd * 4;
}

extern "C" int oxb_paged_update(int page_size, int batch, const int *len, const int *delta, int *table,
                                int table_stride, int *free_pages, int free_cap, const int *n_free, int *len_out,
                                int *n_free_out, int *cu, int *granted, int *slots, int *pos, int n_max,
                                void *stream) {
    clear_error();
    OXB_REQUIRE(paged_size_ok(page_size), "paged update: page size %d is not a power of two of %d to %d", page_size,
                kPgUnit, OXB_PAGED_MAX_PAGE);
    if (paged_table_check(table, table_stride, page_size, batch)) return -1;
    OXB_REQUIRE(len && delta && free_pages && n_free && len_out && n_free_out && cu, "paged update: NULL argument");
    OXB_REQUIRE(free_cap >= 1 && free_cap < (1 << 30), "paged update: free list of %d", free_cap);
    OXB_REQUIRE(n_max >= 0 && n_max < (1 << 30), "paged update: %d tokens", n_max);
    PagedUpdateArgs a{paged_log(page_size), batch, table_stride, free_cap, n_max, len,     delta, table, free_pages,
                      n_free,               len_out, n_free_out, cu,      granted, slots, pos,   1,     1};
    hipStream_t s = (hipStream_t)stream;
    const bool one = n_max <= kUpdTokens;
    a.lengths = one;
    const int grid = one ? 1 : std::min(device_cus(), (n_max + 2 * kUpdThreads - 1) / (2 * kUpdThreads));
    hipLaunchKernelGGL(paged_update_kernel, dim3(grid), dim3(kUpdThreads), 0, s, a);
    OXB_CHECK_HIP(hipGetLastError());
    if (!one) {
        a.lists = 0;
        a.lengths = 1;
        hipLaunchKernelGGL(paged_update_kernel, dim3(1), dim3(kUpdThreads), 0, s, a);
        OXB_CHECK_HIP(hipGetLastError());
    }
    return 0;
}

extern "C" int oxb_paged_append(void *pages, int n_pages, int page_size, int Hkv, int hd, const uint16_t *k,
                                const uint16_t *v, size_t tok_stride, size_t head_stride, const int *src_pos,
                                const int *slots, int n_tok, void *stream) {
    clear_error();
    if (paged_check(pages, n_pages, page_size, Hkv, hd)) return -1;
    // (a launch has less than 2^32 threads)
    OXB_REQUIRE(n_tok >= 0 && n_tok <= (1 << 29) - kAppTokens, "paged append: %d tokens", n_tok);
    if (n_tok == 0) return 0;
    OXB_REQUIRE(k && v && slots && (((uintptr_t)k | (uintptr_t)v) & 15) == 0,
                "paged append: k, v or slots is NULL or rows are not 16-byte aligned");
    OXB_REQUIRE(((tok_stride | head_stride) & 7) == 0, "paged append: strides %zu, %zu are not of 16-byte rows",
                tok_stride, head_stride);
    const PagedAppendArgs a{(_Float16 *)pages, (const _Float16 *)k, (const _Float16 *)v, tok_stride, head_stride,
                            src_pos, slots, n_tok, n_pages * page_size, Hkv, paged_log(page_size)};
    // few tokens: more workgroups of fewer
    const bool few = (int64_t)n_tok * Hkv <= (int64_t)device_cus() * kAppFew;
    const int tokens = few ? kAppFew : kAppTokens;
    const dim3 grid((n_tok + tokens - 1) / tokens, Hkv), th(kAppThreads);
    if (few) hipLaunchKernelGGL(paged_append_kernel<kAppFew>, grid, th, 0, (hipStream_t)stream, a);
    else hipLaunchKernelGGL(paged_append_kernel<kAppTokens>, grid, th, 0, (hipStream_t)stream, a);
    OXB_CHECK_HIP(hipGetLastError());
    return 0;
}

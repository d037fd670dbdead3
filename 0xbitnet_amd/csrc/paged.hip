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
// Sums saturate at kPgMany, past every limit that they are compared with.
constexpr int kUpdThreads = 1024;
constexpr uint32_t kPgMany = 1u << 30;
constexpr int kUpdTokens = 8192;   // of a call of one workgroup

struct PagedUpdateArgs {
    int page_log, batch, table_stride, free_cap, n_max;
    const int *len, *delta;
    int *table, *free_pages;
    const int *n_free;
    int *len_out, *n_free_out, *cu, *granted, *slots, *pos;
    int lists, lengths;   // what the launch writes
};

__device__ __forceinline__ uint32_t sat_add(uint32_t a, uint32_t b) { return min(a + b, kPgMany); }

// Sums of two values over the threads before each thread of the workgroup.
__device__ __forceinline__ void block_before2(uint32_t &a, uint32_t &b, uint32_t (*part)[2]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        const uint32_t x = __shfl_up(a, s, 64), y = __shfl_up(b, s, 64);
        if (lane >= s) {
            a = sat_add(a, x);
            b = sat_add(b, y);
        }
    }
    if (lane == 63) {
        part[wave][0] = a;
        part[wave][1] = b;
    }
    a = __shfl_up(a, 1, 64);
    b = __shfl_up(b, 1, 64);
    if (lane == 0) a = b = 0;
    __syncthreads();
    for (int w = 0; w < wave; ++w) {
        a = sat_add(a, part[w][0]);
        b = sat_add(b, part[w][1]);
    }
    __syncthreads();
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
    __shared__ uint32_t part[kUpdThreads / 64][2];
    const int tid = threadIdx.x, B = a.batch;
    const int64_t cap = (int64_t)a.table_stride << a.page_log;
    const int round = (1 << a.page_log) - 1;
    struct Seq {
        int held, after, delta, need, gone;   // after: the length unless growth is granted
        bool fits;
    };
    auto pages = [&](int64_t n) { return (int)((n + round) >> a.page_log); };
    auto seq = [&](int z, uint32_t last) {   // last: end_z
        Seq s;
        s.held = (int)min(max((int64_t)a.len[z], (int64_t)0), cap);
        s.delta = a.delta[z];
        const int64_t want = (int64_t)s.held + s.delta;
        s.after = s.delta < 0 ? (int)max(want, (int64_t)0) : s.held;
        s.fits = s.delta > 0 && want <= cap && last <= (uint32_t)a.n_max;
        s.need = s.fits ? pages(want) - pages(s.held) : 0;
        s.gone = pages(s.held) - pages(s.after);
        return s;
    };
    // a thread's consecutive sequences
    const int per = (B + kUpdThreads - 1) / kUpdThreads, z0 = tid * per, z1 = min(B, z0 + per);
    uint32_t sum = 0, unused = 0;
    for (int z = z0; z < z1; ++z) {
        sum = sat_add(sum, min((uint32_t)max(a.delta[z], 0), (uint32_t)a.n_max + 1));
        end[z] = sum;
    }
    block_before2(sum, unused, part);
    uint32_t b1 = 0, b2 = 0;
    for (int z = z0; z < z1; ++z) {
        end[z] = sat_add(end[z], sum);
        const Seq s = seq(z, end[z]);
        back[z] = b1 = sat_add(b1, s.gone);
        upto[z] = b2 = sat_add(b2, s.need);
    }
    block_before2(b1, b2, part);
    for (int z = z0; z < z1; ++z) {
        back[z] = sat_add(back[z], b1);
        upto[z] = sat_add(upto[z], b2);
    }
    __syncthreads();
    const int n_free = min(max(*a.n_free, 0), a.free_cap);
    const uint32_t given = back[B - 1], avail = sat_add(given, n_free);
    const int k = above(upto, B, avail);
    const uint32_t taken = k ? upto[k - 1] : 0;
    auto granted = [&](int z, const Seq &s) { return s.fits && (s.need == 0 || upto[z] <= avail); };

    if (a.lists) {
        auto given_page = [&](uint32_t i) {   // i-th of those given back
            const int z = above(back, B, i);
            const Seq s = seq(z, end[z]);
            return a.table[(size_t)z * a.table_stride + pages(s.after) + (i - (back[z] - s.gone))];
        };
        auto taken_page = [&](uint32_t r) {   // those given back first, the last first, then the list's end
            return r < given ? given_page(given - 1 - r) : a.free_pages[n_free - 1 - (int)(r - given)];
        };
        const uint32_t at = blockIdx.x * kUpdThreads + tid, step = gridDim.x * kUpdThreads;
        for (uint32_t t = at; t < (uint32_t)a.n_max; t += step) {
            int slot = -1, p = -1;
            const int z = above(end, B, t);
            if (z < B) {
                const Seq s = seq(z, end[z]);
                if (granted(z, s)) {
                    p = s.held + (int)(t - (end[z] - s.delta));
                    const int b = p >> a.page_log, first = pages(s.held);
                    const int page = b < first ? a.table[(size_t)z * a.table_stride + b]
                                               : taken_page(upto[z] - s.need + (b - first));
                    const int64_t x = ((int64_t)page << a.page_log) + (p & round);
                    slot = page >= 0 && x <= INT32_MAX ? (int)x : -1;
                }
            }
            if (a.slots) a.slots[t] = slot;
            if (a.pos) a.pos[t] = p;
        }
        for (uint32_t r = at; r < taken; r += step) {
            const int z = above(upto, B, r);
            const Seq s = seq(z, end[z]);
            a.table[(size_t)z * a.table_stride + pages(s.held) + (r - (upto[z] - s.need))] = taken_page(r);
        }
        const uint32_t left = given > taken ? given - taken : 0;
        for (uint32_t i = at; i < left && n_free + i < (uint32_t)a.free_cap; i += step)
            a.free_pages[n_free + i] = given_page(i);
        if (blockIdx.x == 0)
            for (int z = tid; z < B; z += kUpdThreads) {
                if (z == 0) a.cu[0] = 0;
                a.cu[z + 1] = (int)min(end[z], (uint32_t)a.n_max);
                if (a.granted) {
                    const Seq s = seq(z, end[z]);
                    a.granted[z] = granted(z, s) ? s.delta : 0;
                }
            }
    }
    if (a.lengths) {
        // a thread writes the lengths that only it reads from here on
        __syncthreads();
        for (int z = tid; z < B; z += kUpdThreads) {
            const Seq s = seq(z, end[z]);
            a.len_out[z] = granted(z, s) ? s.held + s.delta : s.after;
        }
        if (tid == 0) *a.n_free_out = (int)min((uint32_t)a.free_cap, avail - taken);
    }
}

// ---------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------
// A workgroup takes 32 packed tokens of a KV head.  K: 16 bytes of a row go to 16
// bytes of its unit.  V goes through LDS: tokens that follow one another inside an
// octet of positions are written together, a whole octet of a dim as one 16-byte
// store, others (a decode step's single rows) as 2-byte stores.
constexpr int kAppTokens = 32;
constexpr int kAppThreads = 256;
constexpr int kAppStride = kPgHd + 2;   // of a V row in LDS

struct PagedAppendArgs {
    _Float16 *pages;
    const _Float16 *k, *v;
    size_t tok_stride, head_stride;
    const int *src_pos, *slots;
    int n_tok, n_slots, Hkv, page_log;
};

__global__ __launch_bounds__(kAppThreads) void paged_append_kernel(PagedAppendArgs a) {
    __shared__ _Float16 sv[kAppTokens * kAppStride];
    __shared__ int sslot[kAppTokens + 1], slead[kAppTokens], scount[kAppTokens], snum;
    const int tid = threadIdx.x, t0 = blockIdx.x * kAppTokens, head = blockIdx.y;
    const int round = (1 << a.page_log) - 1;
    // rows by 16-byte pieces: tokens tid / 16 and 16 on
    uint4 kr[2], vr[2];
    int slot[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int t = t0 + (tid >> 4) + 16 * i;
        slot[i] = t < a.n_tok ? a.slots[t] : -1;
        int row = 0;
        if (a.src_pos && t < a.n_tok) row = a.src_pos[t];
        if ((unsigned)slot[i] >= (unsigned)a.n_slots || row < 0) slot[i] = -1;
        kr[i] = vr[i] = make_uint4(0, 0, 0, 0);
        if (slot[i] >= 0) {
            const size_t at = (size_t)t * a.tok_stride + (size_t)head * a.head_stride + (size_t)row * kPgHd + 8 * (tid & 15);
            kr[i] = *(const uint4 *)(a.k + at);
            vr[i] = *(const uint4 *)(a.v + at);
        }
        if ((tid & 15) == 0) sslot[(tid >> 4) + 16 * i] = slot[i];
    }
    auto unit = [&](int s) {
        return a.pages + paged_unit(s >> a.page_log, head, (s & round) >> 5, a.Hkv, a.page_log);
    };
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if (slot[i] >= 0) *(uint4 *)(unit(slot[i]) + paged_k_elem(slot[i] & 31, 8 * (tid & 15))) = kr[i];
        uint32_t *row = (uint32_t *)(sv + ((tid >> 4) + 16 * i) * kAppStride + 8 * (tid & 15));
        row[0] = vr[i].x;
        row[1] = vr[i].y;
        row[2] = vr[i].z;
        row[3] = vr[i].w;
    }
    __syncthreads();
    if (tid < 64) {   // the tokens that begin a run inside an octet, and its length
        const int s = tid < kAppTokens ? sslot[tid] : -1;
        const bool lead = s >= 0 && (tid == 0 || (s & 7) == 0 || sslot[tid - 1] != s - 1);
        const uint64_t m = __ballot(lead), gap = __ballot(lead || s < 0);
        if (lead) {
            const uint64_t later = gap & ~((2ull << tid) - 1);
            const int i = __popcll(m & ((1ull << tid) - 1));
            slead[i] = tid;
            scount[i] = __builtin_ctzll(later) - tid;   // (lanes from 32 on are gaps)
        }
        if (tid == 0) snum = __popcll(m);
    }
    __syncthreads();
    for (int i = tid; i < snum * kPgHd; i += kAppThreads) {
        const int t = slead[i >> 7], n = scount[i >> 7], d = i & 127, s = sslot[t];
        _Float16 *dst = unit(s) + paged_v_elem(s & 31, d);
        const _Float16 *src = sv + t * kAppStride + d;
        if (n == 8) {
            _Float16 x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = src[j * kAppStride];
            *(uint4 *)dst = __builtin_bit_cast(uint4, *(__attribute__((ext_vector_type(8))) _Float16 *)x);
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
    OXB_REQUIRE(n_tok >= 0 && n_tok < (1 << 30), "paged append: %d tokens", n_tok);
    if (n_tok == 0) return 0;
    OXB_REQUIRE(k && v && slots && (((uintptr_t)k | (uintptr_t)v) & 15) == 0,
                "paged append: k, v or slots is NULL or rows are not 16-byte aligned");
    OXB_REQUIRE(((tok_stride | head_stride) & 7) == 0, "paged append: strides %zu, %zu are not of 16-byte rows",
                tok_stride, head_stride);
    const PagedAppendArgs a{(_Float16 *)pages, (const _Float16 *)k, (const _Float16 *)v, tok_stride, head_stride,
                            src_pos, slots, n_tok, n_pages * page_size, Hkv, paged_log(page_size)};
    hipLaunchKernelGGL(paged_append_kernel, dim3((n_tok + kAppTokens - 1) / kAppTokens, Hkv), dim3(kAppThreads), 0,
                       (hipStream_t)stream, a);
    OXB_CHECK_HIP(hipGetLastError());
    return 0;
}

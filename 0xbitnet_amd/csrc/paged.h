// The paged KV cache: layout and checks shared by paged.hip (bookkeeping,
// append) and paged_attention.hip.
#pragma once

#include "oxb_common.h"
#include "oxb_kernels.h"

namespace oxb {

constexpr int kPgHd = 128;                     // head dimension
constexpr int kPgUnit = OXB_PAGED_UNIT;        // positions of a layout unit
constexpr int kPgHalf = kPgUnit * kPgHd;       // elements of a unit's K (or V)
constexpr int kPgElems = 2 * kPgHalf;          // elements of a unit: K, then V
constexpr int kPgBatch = OXB_PAGED_MAX_BATCH;
constexpr int kPgPrefill = OXB_PAGED_MAX_PREFILL;   // sequences of a prefill call

// Elements inside a unit (include/oxbitnet_ops.h): 8 dims of a K row, 8
// positions of a V dim are 16 bytes, an MFMA operand's share of a lane.
__host__ __device__ inline int paged_k_elem(int t, int d) { return ((d >> 3) * kPgUnit + t) * 8 + (d & 7); }
__host__ __device__ inline int paged_v_elem(int t, int d) {
    return kPgHalf + ((t >> 3) * kPgHd + d) * 8 + (t & 7);
}
// First element of unit u of a page's head.
__host__ __device__ inline size_t paged_unit(int page, int head, int u, int Hkv, int page_log) {
    return ((((size_t)page * Hkv + head) << (page_log - 5)) + u) * kPgElems;
}

inline int paged_log(int page_size) { return __builtin_ctz((unsigned)page_size); }
inline bool paged_size_ok(int page_size) {
    return page_size >= kPgUnit && page_size <= OXB_PAGED_MAX_PAGE && (page_size & (page_size - 1)) == 0;
}

// Host-side checks that the calls on a pool make.
inline int paged_check(const void *pages, int n_pages, int page_size, int Hkv, int hd) {
    OXB_REQUIRE(pages && ((uintptr_t)pages & 255) == 0, "paged: pool is NULL or not 256-byte aligned");
    OXB_REQUIRE(paged_size_ok(page_size), "paged: page size %d is not a power of two of %d to %d", page_size, kPgUnit,
                OXB_PAGED_MAX_PAGE);
    OXB_REQUIRE(n_pages >= 1 && (int64_t)n_pages * page_size <= INT32_MAX, "paged: %d pages of %d positions", n_pages,
                page_size);
    OXB_REQUIRE(hd == kPgHd, "paged: head_dim %d unsupported (128 only)", hd);
    OXB_REQUIRE(Hkv >= 1 && Hkv <= 4096, "paged: kv heads %d", Hkv);
    return 0;
}
inline int paged_table_check(const int *table, int table_stride, int page_size, int batch) {
    OXB_REQUIRE(table, "paged: block table is NULL");
    OXB_REQUIRE(batch >= 1 && batch <= kPgBatch, "paged: batch %d", batch);
    OXB_REQUIRE(table_stride >= 1 && (int64_t)table_stride * page_size <= OXB_PAGED_MAX_SEQ,
                "paged: block table of %d pages a sequence", table_stride);
    return 0;
}

}  // namespace oxb

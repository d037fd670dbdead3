// The 8-bit KV cache: layout and code conversions shared by kv8.hip (append,
// read, eviction) and kv8_attention.hip.
#pragma once

#include "oxb_common.h"
#include "oxb_kernels.h"

namespace oxb {

constexpr int kKv8Hd = 128;                      // head dimension
constexpr int kKv8Block = OXB_KV8_BLOCK;         // positions that share a scale
constexpr int kKv8Half = kKv8Block * kKv8Hd;     // bytes of a block's K (or V) codes
constexpr int kKv8Codes = 2 * kKv8Half;          // bytes of a block: K codes, then V codes

__host__ __device__ inline int kv8_blocks(int positions) {
    return (int)(((int64_t)positions + kKv8Block - 1) / kKv8Block);
}

// Byte offsets inside one sequence's cache (include/oxbitnet_ops.h).
struct Kv8Layout {
    size_t scales, weights, tails, bytes;
};
__host__ __device__ inline size_t kv8_align(size_t b) { return (b + 255) & ~(size_t)255; }
__host__ __device__ inline Kv8Layout kv8_layout(int Hkv, int nb) {
    Kv8Layout l;
    const size_t n = (size_t)Hkv * nb;
    l.scales = kv8_align(n * kKv8Codes);
    l.weights = l.scales + kv8_align(n * 8);
    l.tails = l.weights + kv8_align(n * 4);
    l.bytes = l.tails + kv8_align((size_t)Hkv * 2 * kKv8Half * 2);
    return l;
}

// The byte of a V row (one dim, 32 positions) that holds position t: the
// 32x32x16 MFMA leaves lane half h the scores of positions 4h + 8 hi + 16 grp
// + 0..3, so bytes 16h .. 16h + 15 are the V operand of that half's own
// probabilities, with no exchange between lanes (kv8_attention.hip).
__host__ __device__ inline int kv8_v_byte(int t) {
    return ((t >> 2) & 1) * 16 + (t >> 4) * 8 + ((t >> 3) & 1) * 4 + (t & 3);
}

// Host-side checks that every entry point makes.
inline int kv8_check(const void *cache, size_t stride, int fmt, int batch, int Hkv, int hd,
                     int max_seq) {
    OXB_REQUIRE(cache && ((uintptr_t)cache & 255) == 0, "kv8: cache is NULL or not 256-byte aligned");
    OXB_REQUIRE(fmt == OXB_KV8_INT8 || fmt == OXB_KV8_E4M3, "kv8: format %d", fmt);
    OXB_REQUIRE(hd == kKv8Hd, "kv8: head_dim %d unsupported (128 only)", hd);
    OXB_REQUIRE(batch >= 1 && batch <= 65535, "kv8: batch %d", batch);
    OXB_REQUIRE(Hkv >= 1 && Hkv <= 4096, "kv8: kv heads %d", Hkv);
    OXB_REQUIRE(max_seq >= 1 && max_seq <= OXB_KV8_MAX_SEQ, "kv8: max_seq %d", max_seq);
    OXB_REQUIRE((stride & 255) == 0 &&
                    (batch == 1 || stride >= kv8_layout(Hkv, kv8_blocks(max_seq)).bytes),
                "kv8: cache stride %zu does not hold a sequence or is not a multiple of 256", stride);
    return 0;
}

}  // namespace oxb

#ifdef __HIPCC__
namespace oxb {

typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));

// Four codes (bytes of w) as f16, exactly.  int8 codes are held as q + 128:
// the byte under 0x64 is the f16 number 1024 + byte, and 1152 less is q.
template <int FMT>
__device__ __forceinline__ void kv8_unpack4(uint32_t w, half2_t &a, half2_t &b) {
    if constexpr (FMT == OXB_KV8_INT8) {
        const uint32_t x = __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u);
        const uint32_t y = __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u);
        const half2_t bias = {(_Float16)1152.0f, (_Float16)1152.0f};
        a = __builtin_bit_cast(half2_t, x) - bias;
        b = __builtin_bit_cast(half2_t, y) - bias;
    } else {
        a = __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.0f, false));
        b = __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.0f, true));
    }
}

template <int FMT>
__device__ __forceinline__ half8_t kv8_unpack8(uint32_t lo, uint32_t hi) {
    half2_t p[4];
    kv8_unpack4<FMT>(lo, p[0], p[1]);
    kv8_unpack4<FMT>(hi, p[2], p[3]);
    return half8_t{p[0].x, p[0].y, p[1].x, p[1].y, p[2].x, p[2].y, p[3].x, p[3].y};
}

}  // namespace oxb
#endif

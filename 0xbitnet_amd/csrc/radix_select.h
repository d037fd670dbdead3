// Radix select of the k-th largest key by one workgroup, shared by the device
// sampler and the cache eviction.
#pragma once

#include "oxb_common.h"

#ifdef __HIPCC__
namespace oxb {

// Order-preserving map of a float to u32 (-0 taken as +0, as the float
// comparisons of the reference see them); 0 is below every value and marks
// an empty list slot.
__device__ inline uint32_t smp_ord(float v) {
    if (v == 0.0f) v = 0.0f;
    const uint32_t b = __float_as_uint(v);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// One digit of a radix select, by wave 0 over hist[256] (the counts of the
// current 8-bit digit among the keys that match the digits chosen so far):
// the digit d, largest first, with (count above d) < rem <= (count above d)
// + hist[d]; writes the extended prefix and what remains of rem.
__device__ inline void smp_pick_digit(const uint32_t *hist, int rem, uint32_t prefix, int shift,
                                      uint32_t *s_prefix, int *s_rem) {
    const int lane = threadIdx.x;
    int h[4], local = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        h[j] = (int)hist[255 - 4 * lane - j];
        local += h[j];
    }
    int incl = local;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int v = __shfl_up(incl, o, 64);
        if (lane >= o) incl += v;
    }
    int acc = incl - local;
    if (acc < rem && rem <= incl) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (acc + h[j] >= rem) {
                *s_prefix = prefix | ((uint32_t)(255 - 4 * lane - j) << shift);
                *s_rem = rem - acc;
                break;
            }
            acc += h[j];
        }
    }
}

// The k-th largest of the block's keys key_at(i), i < n (k <= n), by the
// whole block.  hist: 256 words of LDS.  Its barriers order LDS only: the
// keys come from LDS or from memory no thread of the block writes.
template <int NT, typename KeyAt>
__device__ uint32_t smp_select(int n, int k, KeyAt key_at, uint32_t *hist, uint32_t *s_prefix,
                               int *s_rem) {
    uint32_t prefix = 0, mask = 0;
    int rem = k;
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = threadIdx.x; i < 256; i += NT) hist[i] = 0;
        lds_barrier();
        for (int i = threadIdx.x; i < n; i += NT) {
            const uint32_t o = key_at(i);
            if ((o & mask) == prefix) atomicAdd(&hist[(o >> shift) & 255u], 1u);
        }
        lds_barrier();
        if (threadIdx.x < 64) smp_pick_digit(hist, rem, prefix, shift, s_prefix, s_rem);
        lds_barrier();
        prefix = *s_prefix;
        rem = *s_rem;
        mask |= 255u << shift;
    }
    return prefix;
}

}  // namespace oxb
#endif

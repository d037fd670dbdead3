// Rules on logits for gfx950: penalties for tokens that a sequence's history
// holds, biases on single ids and a mask of allowed ids, for a batch of rows
// before the draw (oxb_sample_device) or an argmax.  The reference knows the
// repetition penalty alone, one row at a time on the host
// (rs/sampling.rs:14-24).
//
// One pass: a workgroup takes kLrChunk logits of a row, counts the row's
// history ids that fall among them and finds each id's last bias entry in LDS,
// and writes the ruled values.  Bound by the logits' bytes once there are
// rows enough: 32 rows of 128256 with histories of up to 4096 ids, 34 MB, 10.0 us,
// 3.4 TB/s (10.9 with the lists asked for behind the logits); one row 4.5 us, the
// launch and two round trips.
#include "oxb_common.h"
#include "oxb_kernels.h"

namespace oxb {

constexpr int kLrThreads = 512;
constexpr int kLrPer = 8;                        // logits per thread
constexpr int kLrChunk = kLrThreads * kLrPer;

struct RulesArgs {
    const float *logits;
    size_t stride;
    int V;
    const float *pen;       // [rows][3] repeat, frequency, presence
    const int *hist, *hist_off;
    int n_hist;
    const int *bias_ids;
    const float *bias;
    const int *bias_off;
    int n_bias;
    const uint32_t *mask;
    size_t mask_stride;
    float *out;
    size_t out_stride;
};

__global__ __launch_bounds__(kLrThreads) void logit_rules_kernel(RulesArgs a) {
    __shared__ int cnt[kLrChunk];    // occurrences in the history
    __shared__ int last[kLrChunk];   // 1 + the last bias entry of the id
    const int r = blockIdx.y, base = blockIdx.x * kLrChunk, tid = threadIdx.x;
    const int n = min(kLrChunk, a.V - base);
    // ranges of this row, kept inside the lists whatever the offsets say; unsigned, as
    // a thread's places run past the end of a list, which may be 2^31 - 1 long
    uint32_t h0 = 0, h1 = 0, b0 = 0, b1 = 0;
    if (a.pen && a.n_hist > 0) {
        h0 = min(max(a.hist_off[r], 0), a.n_hist);
        h1 = min(max(a.hist_off[r + 1], 0), a.n_hist);
    }
    if (a.n_bias > 0) {
        b0 = min(max(a.bias_off[r], 0), a.n_bias);
        b1 = min(max(a.bias_off[r + 1], 0), a.n_bias);
    }
    const bool lists = h0 < h1 || b0 < b1;   // uniform
    // The lists' first ids are asked for before the logits: loads return in
    // order, and their counting runs while the logits come.
    int id[kLrPer], bid = -1;
#pragma unroll
    for (int u = 0; u < kLrPer; ++u) {
        const uint32_t j = h0 + tid + u * kLrThreads;
        id[u] = j < h1 ? a.hist[j] : -1;
    }
    if (b0 + tid < b1) bid = a.bias_ids[b0 + tid];
    const float *lg = a.logits + (size_t)r * a.stride + base;
    const uint32_t *mask = a.mask ? a.mask + (size_t)r * a.mask_stride : nullptr;
    float x[kLrPer];
    uint32_t mw[kLrPer];
#pragma unroll
    for (int u = 0; u < kLrPer; ++u) {
        const int i = min(tid + u * kLrThreads, n - 1);
        x[u] = lg[i];
        mw[u] = mask ? mask[(base + i) >> 5] : 0xffffffffu;
    }
    float rep = 1.0f, freq = 0.0f, pres = 0.0f;
    if (a.pen) {
        rep = a.pen[3 * r];
        freq = a.pen[3 * r + 1];
        pres = a.pen[3 * r + 2];
    }
    if (lists) {
#pragma unroll
        for (int u = 0; u < kLrPer; ++u) {
            cnt[tid + u * kLrThreads] = 0;
            last[tid + u * kLrThreads] = 0;
        }
        lds_barrier();
        auto count = [&](int v) {
            const unsigned i = (unsigned)v - (unsigned)base;
            if (i < (unsigned)n) atomicAdd(&cnt[i], 1);
        };
        auto entry = [&](int v, uint32_t j) {
            const unsigned i = (unsigned)v - (unsigned)base;
            if (i < (unsigned)n) atomicMax(&last[i], (int)j + 1);
        };
#pragma unroll
        for (int u = 0; u < kLrPer; ++u) count(id[u]);
        for (uint32_t j = h0 + kLrPer * kLrThreads + tid; j < h1; j += kLrThreads) count(a.hist[j]);
        entry(bid, b0 + tid);
        for (uint32_t j = b0 + kLrThreads + tid; j < b1; j += kLrThreads) entry(a.bias_ids[j], j);
        lds_barrier();
    }
    float *out = a.out + (size_t)r * a.out_stride + base;
#pragma unroll
    for (int u = 0; u < kLrPer; ++u) {
        const int i = tid + u * kLrThreads;
        if (i >= n) continue;
        float y = x[u];
        const int c = lists ? cnt[i] : 0, b = lists ? last[i] : 0;
        if (c > 0) {
            y = y > 0.0f ? y / rep : y * rep;
            y = y - (freq * (float)c + pres);
        }
        if (b > 0) y = y + a.bias[b - 1];
        if (!(mw[u] >> ((base + i) & 31) & 1)) y = -__builtin_inff();
        out[i] = y;
    }
}

}  // namespace oxb

using namespace oxb;

extern "C" int oxb_logits_rules(const float *logits, size_t stride, int n_rows, int V,
                                const float *penalties, const int32_t *history,
                                const int *history_off, int n_history, const int32_t *bias_ids,
                                const float *bias, const int *bias_off, int n_bias,
                                const uint32_t *mask, size_t mask_stride, float *out,
                                size_t out_stride, void *stream) {
    clear_error();
    OXB_REQUIRE(logits && out, "logit rules: logits or out is NULL");
    OXB_REQUIRE(n_rows >= 1 && n_rows <= 65535, "logit rules: %d rows", n_rows);
    OXB_REQUIRE(V >= 1 && V <= (1 << 30), "logit rules: vocabulary %d", V);
    OXB_REQUIRE(n_rows == 1 || (stride >= (size_t)V && out_stride >= (size_t)V),
                "logit rules: row strides %zu and %zu below the vocabulary", stride, out_stride);
    OXB_REQUIRE(n_history >= 0 && (!penalties || n_history == 0 || (history && history_off)),
                "logit rules: a history of %d tokens without ids or offsets", n_history);
    OXB_REQUIRE(n_bias >= 0 && (n_bias == 0 || (bias_ids && bias && bias_off)),
                "logit rules: %d biases without ids, values or offsets", n_bias);
    OXB_REQUIRE(!mask || mask_stride == 0 || mask_stride >= ((size_t)V + 31) / 32,
                "logit rules: mask rows of %zu words for %d ids", mask_stride, V);
    const uintptr_t s = (uintptr_t)logits, d = (uintptr_t)out;
    const size_t sb = 4 * ((n_rows - 1) * stride + V), db = 4 * ((n_rows - 1) * out_stride + V);
    OXB_REQUIRE((s == d && (n_rows == 1 || stride == out_stride)) || s + sb <= d || d + db <= s,
                "logit rules: out overlaps the logits without being them");
    RulesArgs a{logits, stride, V, penalties, history, history_off, n_history, bias_ids, bias,
                bias_off, n_bias, mask, mask_stride, out, out_stride};
    hipLaunchKernelGGL(logit_rules_kernel, dim3((V + kLrChunk - 1) / kLrChunk, n_rows),
                       dim3(kLrThreads), 0, (hipStream_t)stream, a);
    OXB_CHECK_HIP(hipGetLastError());
    return 0;
}

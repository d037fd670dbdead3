// The packed prefill's list of runs (csrc/paged_plan.h) on the host: a workgroup's
// threads are fibers that change places at barriers and wherever lanes exchange
// values.  Arguments: -1, 0 or 1, the steps that reciprocals are off by, and 1 for
// threads that run in descending order.  Reads calls from standard input, whole numbers:
//   cus n_tok batch G Hkv page_log table_stride  cu[batch + 1]  len[batch]
// and writes for each, as int32: its launches' number and for each of these its tokens
// (begin, end), the sizes (most, slots, wgs, runs, cuts), the counts and the entries of runs and of cuts that were written, [index, record ...] and -1 at
// their end.  Where no list is made, count 2 is 2 and the runs are those that the
// workgroups find themselves.  A write outside the entries ends the program.
#include <ucontext.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <vector>

#include "oxbitnet_ops.h"

#define __device__
#define __forceinline__ inline
#define __shared__ static
using std::max, std::min;

struct Fibers {   // those that wait for one another: a wave, a workgroup
    int size, arrived = 0;
    long turn = 0;
};
static int self;
static bool descending;
static ucontext_t back, ctx[1024];
static bool done[1024];
static Fibers group, wave_of[16];

static void meet(Fibers &f) {
    const long turn = f.turn;
    if (++f.arrived == f.size) {
        f.arrived = 0;
        ++f.turn;
        return;
    }
    while (f.turn == turn) swapcontext(&ctx[self], &back);
}
static struct {
    struct {
        operator int() const { return self; }
    } x;
} threadIdx;
static void __syncthreads() { meet(group); }

// All lanes' values, seen by each at once.
template <typename T, typename F>
static auto among(T v, F f) {
    static T at[1024];
    Fibers &w = wave_of[self >> 6];
    at[self] = v;
    meet(w);
    const auto r = f((const T *)at + (self & ~63));
    meet(w);
    return r;
}
static int lane_() { return self & 63; }
static int wave_iscan(int v) {
    return among(v, [](const int *x) {
        int s = 0;
        for (int i = 0; i <= lane_(); ++i) s += x[i];
        return s;
    });
}
static int readlane_(int v, int l) {
    return among(v, [l](const int *x) { return x[l & 63]; });
}
static int wave_isum_dpp(int v) { return readlane_(wave_iscan(v), 63); }
static int wave_imax(int v) {
    return among(v, [](const int *x) { return *std::max_element(x, x + 64); });
}
static float wave_sum(float v) {
    return among(v, [](const float *x) {
        float s = 0;
        for (int i = 0; i < 64; ++i) s += x[i];
        return s;
    });
}
static int __shfl(int v, int l, int) { return readlane_(v, l); }
static int __shfl_xor(int v, int m, int) { return readlane_(v, lane_() ^ m); }
static uint64_t __ballot(bool b) {
    return among(b, [](const bool *x) {
        uint64_t m = 0;
        for (int i = 0; i < 64; ++i) m |= (uint64_t)x[i] << i;
        return m;
    });
}
static int __popcll(uint64_t m) { return __builtin_popcountll(m); }
static int atomicAdd(int *p, int v) {
    const int old = *p;
    *p += v;
    return old;
}
// (the device's reciprocal is within a step of this one)
static int rcp_step;
static float rcp_(float x) {
    float r = 1.0f / x;
    if (rcp_step > 0) r = std::nextafter(r, INFINITY);
    if (rcp_step < 0) r = std::nextafter(r, 0.0f);
    return r;
}
#define __builtin_amdgcn_readlane readlane_
#define __builtin_amdgcn_readfirstlane(v) readlane_(v, 0)
#define __builtin_amdgcn_rcpf rcp_

namespace oxb {
constexpr int kPgUnit = OXB_PAGED_UNIT, kPgPrefill = OXB_PAGED_MAX_PREFILL;
}
#include "../0xbitnet_amd/csrc/paged_plan.h"
using namespace oxb;

static PgList args;
static std::vector<PgRun> few_runs;
static std::vector<char> few_has;

static void body() {
    if (!args.few) {
        pg_list(args);
    } else {
        const PgFew p = pg_few(args);
        if (self == 0) args.counts[0] = p.total, args.counts[1] = p.nt, args.counts[2] = 2;
        for (size_t b = 0; b < few_runs.size(); ++b) {
            PgRun r{};
            const bool some = pg_few_run(args, p, (int)b, r);
            if (self == 0) few_has[b] = some, few_runs[b] = r;
        }
    }
    done[self] = true;
    for (;;) swapcontext(&ctx[self], &back);
}

static void launch(int threads) {
    static std::vector<char> stacks(1024 * (size_t)65536);
    group = {threads};
    for (int i = 0; i < threads / 64; ++i) wave_of[i] = {64};
    for (int t = 0; t < threads; ++t) {
        done[t] = false;
        getcontext(&ctx[t]);
        ctx[t].uc_stack.ss_sp = stacks.data() + (size_t)t * 65536;
        ctx[t].uc_stack.ss_size = 65536;
        ctx[t].uc_link = &back;
        makecontext(&ctx[t], body, 0);
    }
    for (bool any = true; any;) {
        any = false;
        for (int i = 0; i < threads; ++i) {
            self = descending ? threads - 1 - i : i;
            if (done[self]) continue;
            any = true;
            swapcontext(&back, &ctx[self]);
        }
    }
}

static void put(const void *p, size_t ints) { fwrite(p, 4, ints, stdout); }
static void put(int v) { put(&v, 1); }

// The entries that a launch wrote, of n and as many again behind them.
template <typename R>
static void put_written(const std::vector<R> &v, size_t n, const char *what) {
    R none;
    memset(&none, 0x80, sizeof none);
    for (size_t i = 0; i < v.size(); ++i) {
        if (!memcmp(&v[i], &none, sizeof none)) continue;
        if (i >= n) {
            fprintf(stderr, "%s: entry %zu of %zu\n", what, i, n);
            exit(1);
        }
        put((int)i);
        put(&v[i], sizeof(R) / 4);
    }
    put(-1);
}
template <typename R>
static std::vector<R> blank(size_t n) {
    std::vector<R> v(2 * n + 4096);
    memset((void *)v.data(), 0x80, v.size() * sizeof(R));
    return v;
}

int main(int argc, char **argv) {
    rcp_step = argc > 1 ? atoi(argv[1]) : 0;
    descending = argc > 2 && atoi(argv[2]);
    int cus, n, B, G, Hkv, plog, W;
    while (scanf("%d %d %d %d %d %d %d", &cus, &n, &B, &G, &Hkv, &plog, &W) == 7) {
        std::vector<int> cu(B + 1), len(B);
        for (int &x : cu)
            if (scanf("%d", &x) != 1) return 2;
        for (int &x : len)
            if (scanf("%d", &x) != 1) return 2;
        const PgSizes whole = pg_sizes(n, B, G, Hkv, cus);   // (the workspace's)
        const int window = pg_window(n, B, G);
        put((n + window - 1) / window);
        for (int t = 0; t < n; t += window) {
            const int end = min(n, t + window);
            const PgSizes p = pg_sizes(end - t, B, G, Hkv, cus);
            const int sizes[7] = {t, end, p.most, p.slots, (int)p.wgs, (int)whole.runs, (int)whole.cuts};
            put(sizes, 7);
            int counts[4] = {-7, -7, -7, -7};
            auto runs = blank<PgRun>(whole.runs);
            auto cuts = blank<PgCut>(whole.cuts);
            args = PgList{cu.data(), len.data(), plog, W, B, n, t, end, G, Hkv, p.most, p.slots, (cus + 7) / 8,
                          pg_few_step(p, B), 1.0f / G, counts, runs.data(), cuts.data()};
            few_runs.assign(args.few ? p.wgs : 0, PgRun{});
            few_has.assign(few_runs.size(), 0);
            launch(args.few ? 64 : kPlanThreads);
            if (counts[3] != -7) return 3;
            put(counts, 3);
            for (size_t b = 0; b < few_runs.size(); ++b)   // (as the lists of a launch that has them)
                if (few_has[b]) runs[b] = few_runs[b];
            put_written(runs, args.few ? p.wgs : whole.runs, "run");
            put_written(cuts, whole.cuts, "cut");
        }
    }
    return 0;
}

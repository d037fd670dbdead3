// Who does what in the packed prefill: the list of runs, made on the device from the
// sequences' lengths, and a launch's sizes.  Apart from the attention so that it can
// run on a host too: it takes kPgUnit and kPgPrefill (paged.h), and of the device
// threads, barriers, LDS atomics and what passes values between a wave's lanes.
#pragma once

#include <algorithm>
#include <cstddef>
#include <cstdint>

namespace oxb {

// x / d for x below 2^21, with inv within 2^-23 of 1 / d: x + 1/2 is 1 / 2d or more from
// every multiple of d, the product less than that off.
__device__ __forceinline__ int pg_div(int x, float inv) { return (int)(((float)x + 0.5f) * inv); }

// Units before run i of k even runs: units i / k, its whole part apart (units up to
// 2^19, k and i up to 1025).
__device__ __forceinline__ int pg_run_start(int units, int k, int i) {
    const float inv = __builtin_amdgcn_rcpf((float)k);
    const int part = pg_div(units, inv), more = units - part * k;
    return part * i + pg_div(more * i, inv);
}

__device__ __forceinline__ int pg_units(int64_t positions) { return (int)((positions + kPgUnit - 1) >> 5); }

constexpr int kPreWaves = 4;
constexpr int kPreThreads = 64 * kPreWaves;
constexpr int kPreRows = 32 * kPreWaves;
constexpr int kPreLeast = 8;                 // units of a run (8 x 40 tokens behind 2000 36.5 us; 4 37.3, 16 39.0)
constexpr int kPreSlots = 512;               // resident workgroups, at most
constexpr int kPreOrder = kPreSlots;         // (a multiple of 8)
constexpr int kPlanThreads = 1024;
constexpr int kPreList = kPlanThreads;       // tiles and runs of a list, a thread each
constexpr int kFewTiles = 128;
constexpr int64_t kPreMost = 1 << 27;        // rows of a call

// A run: a tile's units u0 .. u1, and a cut tile: its parts.
struct PgRun {
    int tile, u0, u1, part;   // part -1: the tile's only run
    int cu, nq, past, z;
    int tok, head, unused[2]; // the token of the tile's first row; the KV head, -1 where there is no run
};
struct PgCut {
    int tile, part, runs, cu, nq, unused[3];
};

// What a list is made from, and where it goes.
struct PgList {
    const int *cu, *len;
    int page_log, table_stride, batch, n_tok, begin, end;   // of the call's n_tok tokens the launch's begin .. end - 1
    int G, Hkv, most, slots, half;
    int few;        // no plan: the first step of a search among the batch's sequences (0: there is one)
    float inv_G;
    int *counts;    // runs, `cuts`, whether tiles may be cut (then a record a workgroup)
    PgRun *runs;    // [kPreList], or [kPreOrder] in the order of the workgroups
    PgCut *cuts;    // cut tiles, or where there is no plan all tiles
};

// Sequence z's tokens of the launch: the first one's place, their number, positions
// that come before them.
struct PgTokens {
    int cu, nq, past;
};
__device__ __forceinline__ PgTokens pg_tokens(const PgList &a, int z) {
    const int64_t cap = (int64_t)a.table_stride << a.page_log;
    const int end = min(max(a.cu[z + 1], 0), a.n_tok);   // (of all that the call has)
    const int c0 = min(max(a.cu[z], a.begin), a.end), c1 = min(max(end, a.begin), a.end);
    return PgTokens{c0, max(c1 - c0, 0), (int)(min(max((int64_t)a.len[z], (int64_t)0), cap) - (end - c0))};
}

// Latency is all that counts here: lengths are loaded once and kept in LDS, a sum over
// the workgroup takes one barrier, and the search for `per` starts between the bounds
// that the units' sum gives (sum ceil(n / per) lies between sum n / per and that plus
// the tiles), so that one round of candidates decides as a rule.  The 12 prompts' plan
// of 664 tiles: 7.3 us (12.0 with lengths and tiles looked up in memory by each step).
__device__ __forceinline__ void pg_list(const PgList &a) {
    constexpr int kWaves = kPlanThreads / 64;
    static_assert(kPgPrefill <= kPlanThreads && kPreSlots <= kPreList, "a thread a sequence, and a run");
    __shared__ int s_cu[kPgPrefill], s_nq[kPgPrefill], s_past[kPgPrefill];
    __shared__ uint32_t upto[kPgPrefill];               // tiles of the sequences up to z
    __shared__ int cost[kPreSlots], first[kPreSlots];   // of a tile that may be cut: units, runs up to it
    __shared__ uint16_t tile_z[kPreSlots];
    __shared__ int hist[kPlanThreads];
    __shared__ uint32_t wsum[4][kWaves];
    __shared__ int wmax[kWaves], wmin[kWaves], fit[2][kWaves];
    const int tid = threadIdx.x, lane = tid & 63, B = a.batch;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // Inclusive sum over the threads; `all` is the whole one.
    auto scan = [&](int v, uint32_t *to, int &all) {
        v = wave_iscan(v);
        if (lane == 63) to[wave] = v;
        __syncthreads();
        const int w = wave_iscan(lane < kWaves ? (int)to[lane] : 0);
        all = __builtin_amdgcn_readlane(w, kWaves - 1);
        return v + (wave ? __builtin_amdgcn_readlane(w, wave - 1) : 0);
    };
    hist[tid] = 0;
    int nt = 0;
    if (tid < B) {
        const PgTokens k = pg_tokens(a, tid);
        s_cu[tid] = k.cu;
        s_nq[tid] = k.nq;
        s_past[tid] = k.past;
        nt = (k.nq * a.G + kPreRows - 1) / kPreRows;
    }
    const int tiles = scan(nt, wsum[0], nt);
    if (tid < B) upto[tid] = tiles;
    nt = min(nt, a.most);   // (what a cu that ascends has at most)
    __syncthreads();
    const bool cut = nt <= a.slots;
    struct Tile {
        int z, i, units;
    };
    auto tile = [&](int t) {   // sequence, index in it, units that its last row sees
        int lo = 0, hi = B - 1;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (upto[mid] > (uint32_t)t) hi = mid;
            else lo = mid + 1;
        }
        Tile r;
        r.z = lo;
        r.i = t - (lo ? (int)upto[lo - 1] : 0);
        const int last = min((r.i + 1) * kPreRows, s_nq[lo] * a.G) - 1;
        r.units = pg_units(max(s_past[lo] + last / a.G + 1, 0));
        return r;
    };
    Tile own{0, 0, 0};   // a thread's
    int mx = 0, sum = 0;
    if (tid < nt) {
        own = tile(tid);
        mx = sum = own.units;
        if (cut) {
            cost[tid] = own.units;
            tile_z[tid] = own.z;
        }
    }
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) mx = max(mx, __shfl_xor(mx, s, 64));
    if (lane == 0) wmax[wave] = mx;
    scan(sum, wsum[1], sum);
    mx = lane < kWaves ? wmax[lane] : 0;
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) mx = max(mx, __shfl_xor(mx, s, 64));
    int per = max(mx, 1), total = nt, cuts = 0, pieces = 1;
    const int rest = a.slots > 1 ? nt % a.slots : 0;
    if (!cut && rest && 2 * rest <= a.slots) {   // (uniform)
        // Whole rounds of tiles that are nearly equal, and a few more, no more than half a
        // round: those are cut so that they fill a round of their own together.  (H 20 over
        // 5.  Up to a quarter of a round only: 4096 tokens behind 20000 1660 us for 1522; up
        // to three quarters: the same, for lack of pieces.  Nearly equal, a mean of 3/4 of the
        // longest: 4500 tokens from 0, whose mean is half of it, 203.5 us, cut too 210; at
        // 0.9, 4200 behind 8000, f16, 485 for 458.)
        if ((float)sum > 0.75f * (float)mx * (float)nt) {
            int least = tid >= nt - rest && tid < nt ? own.units : INT32_MAX;
#pragma unroll
            for (int s = 32; s > 0; s >>= 1) least = min(least, __shfl_xor(least, s, 64));
            if (lane == 0) wmin[wave] = least;
            __syncthreads();
            for (int w = 0; w < kWaves; ++w) least = min(least, wmin[w]);
            pieces = min(min(a.slots / rest, least / kPreLeast), 1 + (kPreList - nt) / rest);
            if (pieces > 1) {
                cuts = rest;
                total = nt + rest * (pieces - 1);
                const int i = tid - (nt - rest);
                if (i >= 0 && i < rest)
                    a.cuts[i] = PgCut{own.i, i * pieces, pieces, s_cu[own.z], s_nq[own.z], {0, 0, 0}};
            }
        }
    }
    if (cut) {
        // the least run length whose runs all are resident: a candidate a wave
        int lo = max(kPreLeast, nt ? sum / a.slots : 0), hi = per;
        if (nt < a.slots) hi = min(hi, max(lo, (sum + a.slots - nt - 1) / (a.slots - nt)));
        for (int i = 0; lo < hi; i ^= 1) {
            const int step = (hi - lo + kWaves - 1) / kWaves, c = min(hi, lo + wave * step);
            int n = 0;
            const float inv = __builtin_amdgcn_rcpf((float)c);
            for (int t = lane; t < nt; t += 64) n += max(1, pg_div(cost[t] + c - 1, inv));
            n = wave_isum_dpp(n);
            if (lane == 0) fit[i][wave] = n <= a.slots;
            __syncthreads();
            const uint64_t ok = __ballot(lane < kWaves && fit[i][lane & (kWaves - 1)]);
            const int w = ok ? __builtin_ctzll(ok) : kWaves, l = lo;
            if (w < kWaves) hi = min(hi, l + w * step);
            if (w > 0) lo = min(hi, l + (w - 1) * step + 1);
        }
        per = max(hi, 1);
        // runs of the tiles up to each, and cut tiles above bit 16
        const int k = tid < nt ? max(1, pg_div(own.units + per - 1, __builtin_amdgcn_rcpf((float)per))) : 0;
        const int v = scan(k | (k > 1 ? 1 << 16 : 0), wsum[2], total);
        cuts = total >> 16;
        total &= 0xffff;
        if (tid < nt) first[tid] = v & 0xffff;
        if (k > 1) a.cuts[(v >> 16) - 1] = PgCut{own.i, (v & 0xffff) - k, k, s_cu[own.z], s_nq[own.z], {0, 0, 0}};
        __syncthreads();
    }
    if (tid == 0) {
        a.counts[0] = total;
        a.counts[1] = cuts;
        a.counts[2] = cut;
    }
    auto run = [&](int j) {
        int k = 1, i = 0, t = j, part = j;
        if (!cut && j >= nt - cuts) {
            part = j - (nt - cuts);
            k = pieces;
            t = part / k;
            i = part - t * k;
            t += nt - cuts;
        }
        if (cut) {
            int l = 0, h = nt - 1;
            while (l < h) {
                const int mid = (l + h) >> 1;
                if (first[mid] > j) h = mid;
                else l = mid + 1;
            }
            const int before = l ? first[l - 1] : 0;
            t = l;
            k = first[l] - before;
            i = j - before;
        }
        Tile r;
        if (cut) {
            r.z = tile_z[t];
            r.i = t - (r.z ? (int)upto[r.z - 1] : 0);
            r.units = cost[t];
        } else {
            r = tile(t);
        }
        return PgRun{r.i, pg_run_start(r.units, k, i), pg_run_start(r.units, k, i + 1), k > 1 ? part : -1, s_cu[r.z], s_nq[r.z], s_past[r.z],
                     r.z, r.i * kPreRows / a.G, 0, {0, 0}};
    };
    if (cut) {
        // All run at once.  Workgroup b runs on XCD b % 8: each XCD takes an eighth of the
        // (KV head, run) pairs as they follow one another, so that its runs share their
        // sequence's K and V in its L2; there the longest first, and of a CU's two the
        // second the other way round, so that it gets the longest and the shortest.
        const int n = total * a.Hkv, each = (n + 7) / 8, half = a.half;
        const int x = each ? pg_div(tid, __builtin_amdgcn_rcpf((float)each)) : 0, lo = x * each;
        constexpr int kSteps = kPlanThreads / 8;   // of a run's length, to an XCD
        PgRun r{};
        int bucket = 0, head = 0;
        if (tid < n) {
            head = pg_div(tid, __builtin_amdgcn_rcpf((float)total));
            r = run(tid - head * total);
            bucket = x * kSteps + (int)((float)(per - (r.u1 - r.u0)) * ((float)(kSteps - 1) / (float)per));
            atomicAdd(&hist[bucket], 1);
        }
        __syncthreads();
        const int h = hist[tid];
        int all;
        const int v = scan(h, wsum[3], all);
        hist[tid] = v - h;
        __syncthreads();
        if (tid < each * 8) {
            int at = tid - lo;
            r.head = -1;
            if (tid < n) {
                at = atomicAdd(&hist[bucket], 1) - lo;
                const int two = min(2 * half, min(each, n - lo));
                if (at >= half && at < two) at = half + two - 1 - at;
                r.head = head;
            }
            a.runs[at * 8 + x] = r;
        }
        return;
    }
    // the longest first, to a thousandth of the longest
    const float scale = (float)(kPlanThreads - 1) / (float)per;
    auto bucket = [&](const PgRun &r) { return (int)((float)(per - min(per, r.u1 - r.u0)) * scale); };
    PgRun mine{};
    if (tid < total) {
        mine = run(tid);
        atomicAdd(&hist[bucket(mine)], 1);
    }
    __syncthreads();
    const int h = hist[tid];
    int all;
    const int v = scan(h, wsum[3], all);
    hist[tid] = v - h;
    __syncthreads();
    if (tid < total) a.runs[atomicAdd(&hist[bucket(mine)], 1)] = mine;
}

// The same plan of a call of up to 64 sequences and kFewTiles tiles, which a wave
// makes by itself: a lane a sequence, a lane a tile (two), so that no launch comes
// before the attention's (its 4 to 7 us and the gap behind it).  All runs are
// resident at once, so their order matters little: only each XCD's stretch of
// them, and of a CU's two one from either end.  (101 tokens 16.4 -> 12.2 us, the
// drafts 37 -> 33.  The join reads what the first run of each tile leaves: with a plan of
// its own it took 11.3 us for 6.3.)
struct PgFew {
    int nt, total;                     // tiles, runs
    int cu, nq, past;                  // of sequence `lane`
    int z[2], i[2], units[2], k[2], upto[2];   // of tiles `lane` and 64 + `lane`: runs, and up to it
};
__device__ __forceinline__ PgFew pg_few(const PgList &a) {
    const int lane = threadIdx.x & 63;
    PgFew p;
    const PgTokens own = pg_tokens(a, min(lane, a.batch - 1));   // (without a branch that loads wait for)
    p.cu = own.cu;
    p.nq = lane < a.batch ? own.nq : 0;
    p.past = own.past;
    const int tiles = wave_iscan((p.nq * a.G + kPreRows - 1) / kPreRows);
    p.nt = min(__builtin_amdgcn_readlane(tiles, 63), min(a.most, kFewTiles));
    int sum = 0, mx = 0;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        const int t = 64 * c + lane;
        p.z[c] = p.i[c] = p.units[c] = 0;
        if (64 * c >= p.nt) continue;   // (uniform)
        int z = 0;   // the first sequence with more than t tiles up to it
        for (int step = a.few; step > 0; step >>= 1)
            if (__shfl(tiles, z + step - 1, 64) <= t) z += step;
        const int before = __shfl(tiles, z - 1, 64), nq = __shfl(p.nq, z, 64), past = __shfl(p.past, z, 64);
        p.z[c] = z;
        p.i[c] = t - (z ? before : 0);
        const int last = min((p.i[c] + 1) * kPreRows, nq * a.G) - 1;
        p.units[c] = t < p.nt ? pg_units(max(past + pg_div(last, a.inv_G) + 1, 0)) : 0;
        sum += p.units[c];
        mx = max(mx, p.units[c]);
    }
    sum = wave_isum_dpp(sum);
    // (bounds, the lower from below, the upper from above)
    auto share = [&](int n) { return (float)sum * __builtin_amdgcn_rcpf((float)n); };
    int lo = max(kPreLeast, (int)(share(a.slots) * 0.999999f)), hi = max(wave_imax(mx), 1);
    if (p.nt < a.slots) hi = min(hi, max(lo, (int)(share(a.slots - p.nt) * 1.000001f) + 1));
    auto runs = [&](int u, int t, int per) {
        return t < p.nt ? max(1, pg_div(u + per - 1, __builtin_amdgcn_rcpf((float)per))) : 0;
    };
    while (lo < hi) {
        const int per = (lo + hi) >> 1;
        const int n = wave_isum_dpp(runs(p.units[0], lane, per) + runs(p.units[1], 64 + lane, per));
        if (n <= a.slots) hi = per;
        else lo = per + 1;
    }
    p.k[0] = runs(p.units[0], lane, hi);
    p.k[1] = runs(p.units[1], 64 + lane, hi);
    p.upto[0] = wave_iscan(p.k[0]);
    const int half = __builtin_amdgcn_readlane(p.upto[0], 63);
    p.upto[1] = half + wave_iscan(p.k[1]);
    p.total = __builtin_amdgcn_readlane(p.upto[1], 63);
    return p;
}
// Fields of tile t (uniform): of c = t / 64, lane t % 64.
__device__ __forceinline__ int pg_of_tile(const int (&f)[2], int t) {
    return __builtin_amdgcn_readlane(t < 64 ? f[0] : f[1], t & 63);
}

// The run of workgroup `block`, its KV head in run.head; false where it has none.
__device__ __forceinline__ bool pg_few_run(const PgList &a, const PgFew &p, int block, PgRun &run) {
    const int n = p.total * a.Hkv, each = (n + 7) / 8, x = block & 7, i = block >> 3;
    const int there = min(each, n - x * each);   // of this XCD
    if (i >= there) return false;
    const int f = x * each + (i < a.half ? i : there - 1 - (i - a.half));
    run.head = pg_div(f, __builtin_amdgcn_rcpf((float)p.total));
    const int j = f - run.head * p.total;
    const int t = __popcll(__ballot(p.upto[0] <= j)) + __popcll(__ballot(p.upto[1] <= j));
    const int k = pg_of_tile(p.k, t), part = j - (pg_of_tile(p.upto, t) - k), units = pg_of_tile(p.units, t);
    run.z = pg_of_tile(p.z, t);
    run.tile = pg_of_tile(p.i, t);
    run.u0 = pg_run_start(units, k, part);
    run.u1 = pg_run_start(units, k, part + 1);
    run.part = k > 1 ? j : -1;
    run.cu = __builtin_amdgcn_readlane(p.cu, run.z);
    run.nq = __builtin_amdgcn_readlane(p.nq, run.z);
    run.past = __builtin_amdgcn_readlane(p.past, run.z);
    run.tok = pg_div(run.tile * kPreRows, a.inv_G);
    if (run.head == 0 && part == 0 && threadIdx.x == 0)
        a.cuts[t] = PgCut{run.tile, j, k, run.cu, run.nq, {0, 0, 0}};
    return true;
}

// A call's tokens go in launches of `window` each, so that a list has kPreList tiles at
// most, the longest that has run: a call of 4096 tiles, of as many sequences, ended in a
// memory fault, and why is not known.  Even windows, of whole tiles of a sequence where
// one fits.
inline int pg_window(int n, int batch, int G) {
    int64_t whole = kPreRows;   // tokens of whole tiles
    while (whole > 1 && whole / 2 * G % kPreRows == 0) whole /= 2;
    int64_t most = std::max<int64_t>(1, (int64_t)(kPreList - std::min(batch, n)) * kPreRows / G);
    if (n <= most) return n;
    if (most < whole) return (int)most;
    most -= most % whole;
    const int64_t parts = (n + most - 1) / most, even = (n + parts - 1) / parts;
    return (int)((even + whole - 1) / whole * whole);
}

// Sizes of a launch of n tokens on `cus` CUs: tiles at most (a sequence's last one may
// be short), runs that are resident at once, of a KV head, workgroups, and the records'
// entries.
struct PgSizes {
    int most, slots;
    int64_t wgs;
    size_t runs, cuts;
};
inline PgSizes pg_sizes(int n, int batch, int G, int Hkv, int cus) {
    PgSizes p;
    p.most = (int)std::min<int64_t>((int64_t)n * G / kPreRows + std::min(batch, n), kPreList);
    p.slots = std::min(2 * cus, kPreSlots) / Hkv;
    p.runs = std::max(std::min(p.most + p.slots, kPreList), kPreOrder);
    p.wgs = std::max<int64_t>((int64_t)std::min(p.most + p.slots, kPreList) * Hkv, kPreOrder);
    p.cuts = std::max(p.slots / 2 + 1, kFewTiles);
    return p;
}
// The first step of a search of 0 .. batch - 1 (1 without sequences to search) where a
// call has no plan, else 0.
inline int pg_few_step(const PgSizes &p, int batch) {
    int few = 0;
    if (batch <= 64 && p.most <= std::min(p.slots, kFewTiles))
        for (few = 1; 2 * few < batch;) few *= 2;
    return few;
}

}  // namespace oxb

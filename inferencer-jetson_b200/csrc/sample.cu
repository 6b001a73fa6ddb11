// Sampling a token from each row of logits: temperature, top-k, top-p, min-p
// and a given uniform number.
//
// Per row, with m the largest logit (NaN counts as -infinity) and T > 0:
//   t_i = (x_i - m) / T (0 where x_i = m),  w_i = exp(t_i) in fp32, held as the
//   whole number W_i = round(w_i * 2^44).
// Tokens are ordered by logit, the largest first, equal ones by index.  top-k
// keeps the first k; top-p keeps the shortest prefix of those whose mass
// reaches top_p of theirs; min-p keeps the tokens with w_i >= min_p (at most
// what top-p kept; the largest always).  With M the mass kept, the answer is
// the first token whose running mass exceeds floor(u * M).
//
// Masses are 64-bit whole numbers, so a sum is the same in any order: the
// result does not depend on the launch shape, and a cut at a border is exact
// (a running fp32 sum over 128256 tokens is off by as much as a rare token's
// whole share).  2^44 leaves room for 2^19 weights of 1; a weight below 2^-45
// counts as nothing.
//
// One cluster per row: each CTA keeps its part of the row in shared memory, so
// the logits are read from HBM once.  The order is never built.  The tokens are
// counted in 2048 bins of -t (64 a nat, the last open); a bin's tokens weigh
// between exp(-(b + 1) / 64) and exp(-b / 64) each, so the counts alone say, to
// 1.6 %, in which few bins a mass falls.  Those bins' tokens (and all before
// them where they fit) are gathered in the leader CTA, sorted and summed; the
// mass before them is summed in registers.  (Counting masses in the bins too
// took 15 us a row: a 64-bit shared-memory addition a token.)  A range of more
// than kCap tokens is split first, by finer bins of t, then by the bits of the
// logits, down to equal ones, which the order by index decides.
#include <mutex>
#include <string>

#include "../../include/ijb200.h"
#include "common.cuh"
#include "misc.cuh"

namespace ijb {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 2048;
constexpr int kSplit = 1024;          // bins of a split
constexpr int kCap = 1024;            // tokens the leader sorts: two a thread
constexpr int kMaxChunk = 16384;      // logits per CTA
constexpr int kMaxCluster = 8;
constexpr float kBinsPerNat = 64.f;
constexpr float kFixed = 17592186044416.f;  // 2^44
typedef unsigned long long u64;

struct SampleParams {
    const float *x;
    long stride;
    int vocab, chunk;
    const float *u, *temperature;
    const int *top_k;
    const float *top_p, *min_p;
    int *token;
    float *prob;
};

enum Cmd { kDone, kSums, kHist, kGather, kEqual };

// Which tokens an order is about: bins lo..hi of -t; with sub >= 0 the sub-th of
// kSplit equal parts of those; with sh < 32 the logits whose key starts with pref.
struct Range {
    int lo, hi, sub, sh;
    uint32_t pref;
};

struct Ctl {
    // this CTA's part of a reduction
    float max;
    u64 key, total, above, before;
    int equal, found, place;
    // the leader's orders and results
    int cmd, next_sh, list_n, equal_index;
    Range range;
    u64 equal_j;
    // within the CTA
    u64 warp_mass[kWarps];
    float warp_f[kWarps];
    int warp_cnt[kWarps];
};

struct Smem {
    Ctl ctl;
    uint32_t hcnt[kBins];  // this CTA's counts
    uint32_t mcnt[kBins];  // leader: the row's counts up to each bin
    float mlow[kBins];     // leader: the least mass up to each bin
    u64 list[kCap];        // leader: gathered tokens; a split's masses of this CTA
    u64 mass[kCap];        // leader: running masses of the sorted list; a split's masses of the row
    uint32_t scnt[kSplit]; // leader: a split's counts of the row
};
static_assert(kSplit == kCap, "a split's masses lie over the list's");

__device__ __forceinline__ uint32_t ctarank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The same variable in CTA `rank` of the cluster.
template <class T>
__device__ __forceinline__ T *peer(T *p, uint32_t rank) {
    uint64_t out;
    asm("mapa.u64 %0, %1, %2;" : "=l"(out) : "l"(reinterpret_cast<uint64_t>(p)), "r"(rank));
    return reinterpret_cast<T *>(out);
}

// Sum over the cluster of f(q), the reads of all CTAs in flight together.
template <class T, class F>
__device__ __forceinline__ T over_peers(int C, F f) {
    T v[kMaxCluster], sum = 0;
#pragma unroll
    for (int q = 0; q < kMaxCluster; ++q) v[q] = q < C ? f(q) : T(0);
#pragma unroll
    for (int q = 0; q < kMaxCluster; ++q) sum += v[q];
    return sum;
}

// Order-preserving key, ascending from the largest value; -0 and +0 are equal.
__device__ __forceinline__ uint32_t desc_key(float v) {
    if (v == 0.f) v = 0.f;
    const uint32_t b = __float_as_uint(v);
    return ~((b & 0x80000000u) ? ~b : (b | 0x80000000u));
}
__device__ __forceinline__ float desc_value(uint32_t key) {
    const uint32_t o = ~key;
    return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}

struct Row {
    float max, temp, inv;
    bool plain_div;
    // (x - m) / T, rounded to nearest.  With inv = 1 / T rounded to nearest, one
    // residual correction of d * inv gives the quotient rounded to nearest
    // (Markstein), as long as nothing leaves the normal range; else the division.
    __device__ __forceinline__ float t(float x) const {
        const float d = x == max ? 0.f : x - max;
        if (plain_div) return d / temp;
        const float q = d * inv;
        const float r = fmaf(fmaf(-q, temp, d), inv, q);
        return d >= -1e30f ? r : d;  // -infinity, and what exp makes 0 either way
    }
    __device__ __forceinline__ static int bin(float t) {
        return static_cast<int>(fminf(-t * kBinsPerNat, static_cast<float>(kBins - 1)));
    }
    __device__ __forceinline__ static int sub_bin(float t, int lo, int hi) {
        const float f = (-t * kBinsPerNat - static_cast<float>(lo)) * (static_cast<float>(kSplit) / static_cast<float>(hi + 1 - lo));
        return static_cast<int>(fminf(fmaxf(f, 0.f), static_cast<float>(kSplit - 1)));
    }
    // 0 for a NaN (a logit of -infinity at an infinite temperature)
    __device__ __forceinline__ static u64 fixed(float w) {
        return w > 0.f ? static_cast<u64>(__float2ll_rn(w * kFixed)) : 0ull;
    }
    __device__ __forceinline__ bool in(float x, const Range &r) const {
        const float tt = t(x);
        const int b = bin(tt);
        return b >= r.lo && b <= r.hi && (r.sub < 0 || sub_bin(tt, r.lo, r.hi) == r.sub) &&
               (r.sh == 32 || (desc_key(x) >> r.sh) == r.pref);
    }
};

__device__ __forceinline__ u64 warp_sum64(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Inclusive sums over N (kThreads times 1, 2 or 4) values in place.
template <int N, class T>
__device__ __forceinline__ void block_scan(T *v, T *warp_sums) {
    constexpr int PER = N / kThreads;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, base = threadIdx.x * PER;
    T x[PER], m = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        x[i] = v[base + i];
        m += x[i];
    }
    const T own = m;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const T p = __shfl_up_sync(0xffffffffu, m, o);
        if (lane >= o) m += p;
    }
    if (lane == 31) warp_sums[warp] = m;
    __syncthreads();
    T w = lane < warp ? warp_sums[lane] : T(0);  // kWarps <= 32
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
    m += w - own;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        m += x[i];
        v[base + i] = m;
    }
    __syncthreads();
}

// Sum over the CTA, the same in every thread.
__device__ __forceinline__ u64 block_sum(Smem &s, u64 v) {
    v = warp_sum64(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s.ctl.warp_mass[threadIdx.x >> 5] = v;
    __syncthreads();
    const int lane = threadIdx.x & 31;
    return warp_sum64(lane < kWarps ? s.ctl.warp_mass[lane] : 0ull);
}

// First i of n (a multiple of kThreads) at which the rising predicate f holds,
// n - 1 if none; every thread calls it.
template <class F>
__device__ __forceinline__ int first_of(int n, F f) {
    int at = 0;
    for (int i = threadIdx.x; i < n; i += kThreads) at += __syncthreads_count(!f(i));
    return min(at, n - 1);
}

// Counts the CTA's tokens by bin; with SUMS also its mass, and the mass of what
// min_p keeps.
template <bool SUMS>
__device__ __forceinline__ void count_bins(Smem &s, const float *xs, int len, const Row &row, float min_p) {
    for (int i = threadIdx.x; i < kBins; i += kThreads) s.hcnt[i] = 0;
    __syncthreads();
    u64 total = 0, above = 0;
#pragma unroll 4
    for (int i0 = 0; i0 < len; i0 += kThreads) {
        const int i = i0 + threadIdx.x;
        const bool live = i < len;
        const float x = live ? xs[i] : -INFINITY;
        const float t = row.t(x);
        const int b = Row::bin(t);
        if (SUMS) {
            const float w = expf(t);
            const u64 m = live ? Row::fixed(w) : 0ull;
            total += m;
            if (w >= min_p || x == row.max) above += m;
        }
        if (live) atomicAdd(&s.hcnt[b], 1u);
    }
    if (SUMS) {
        total = block_sum(s, total);
        above = block_sum(s, above);
        if (threadIdx.x == 0) {
            s.ctl.total = total;
            s.ctl.above = above;
        }
    }
}

// What every CTA of the cluster does for one order of the leader.
__device__ __forceinline__ void execute(Smem &s, const float *xs, int len, int begin, const Row &row, float min_p, int C, int rank) {
    const Ctl *lead = peer(&s.ctl, 0);
    const int cmd = lead->cmd;
    const Range range = lead->range;
    if (cmd == kSums) {  // the mass, and the mass of what min_p keeps
        u64 total = 0, above = 0;
        for (int i = threadIdx.x; i < len; i += kThreads) {
            const float x = xs[i], w = expf(row.t(x));
            const u64 m = Row::fixed(w);
            total += m;
            if (w >= min_p || x == row.max) above += m;
        }
        total = block_sum(s, total);
        above = block_sum(s, above);
        if (threadIdx.x == 0) {
            s.ctl.total = total;
            s.ctl.above = above;
        }
        cluster_sync();
    } else if (cmd == kHist) {  // counts and masses of a split: by finer bins (next_sh 32) or by key bits
        const int sh = lead->next_sh;
        for (int i = threadIdx.x; i < kSplit; i += kThreads) {
            s.list[i] = 0;
            s.hcnt[i] = 0;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < len; i += kThreads) {
            const float x = xs[i];
            if (!row.in(x, range)) continue;
            const float t = row.t(x);
            const int d = sh == 32 ? Row::sub_bin(t, range.lo, range.hi)
                                   : static_cast<int>((desc_key(x) >> sh) & ((1u << (range.sh - sh)) - 1u));
            const u64 m = Row::fixed(expf(t));
            atomicAdd(&s.hcnt[d], 1u);
            if (m) atomicAdd(&s.list[d], m);
        }
        cluster_sync();
        const int per = kSplit / C;
        for (int i = rank * per + threadIdx.x; i < (rank + 1) * per; i += kThreads) {
            *peer(&s.mass[i], 0) = over_peers<u64>(C, [&](int q) { return *peer(&s.list[i], q); });
            *peer(&s.scnt[i], 0) = over_peers<uint32_t>(C, [&](int q) { return *peer(&s.hcnt[i], q); });
        }
        cluster_sync();
    } else if (cmd == kGather) {  // the range's tokens to the leader; the mass of the bins before it
        // first into this CTA's own memory (s.mass, idle now), then in one piece to the leader's list
        u64 before = 0;
        const int lane = threadIdx.x & 31;
        if (threadIdx.x == 0) s.ctl.found = 0;
        __syncthreads();
        // below this no token is in the range (with room for t's rounding)
        const float least = range.hi == kBins - 1 || !(row.max < INFINITY)
                                ? -INFINITY
                                : row.max - (static_cast<float>(range.hi + 2) / kBinsPerNat) * row.temp * 1.0001f -
                                      fabsf(row.max) * 1e-5f;
#pragma unroll 4
        for (int i0 = 0; i0 < len; i0 += kThreads) {
            const int i = i0 + threadIdx.x;
            const float x = i < len ? xs[i] : -INFINITY;
            bool take = i < len && x >= least;
            if (!__any_sync(0xffffffffu, take)) continue;
            if (take) {
                const float t = row.t(x);
                if (range.lo > 0 && Row::bin(t) < range.lo) before += Row::fixed(expf(t));
                take = row.in(x, range);
            }
            const uint32_t all = __ballot_sync(0xffffffffu, take);
            if (all == 0) continue;
            int at = 0;
            if (lane == 0) at = atomicAdd(&s.ctl.found, __popc(all));
            at = __shfl_sync(0xffffffffu, at, 0) + __popc(all & ((1u << lane) - 1u));
            if (take && at < kCap) s.mass[at] = (static_cast<u64>(desc_key(x)) << 32) | static_cast<uint32_t>(begin + i);
        }
        __syncthreads();
        const int found = min(s.ctl.found, kCap);
        if (threadIdx.x == 0 && found) s.ctl.place = atomicAdd(peer(&s.ctl.list_n, 0), found);
        __syncthreads();
        u64 *list = peer(s.list, 0);
        for (int i = threadIdx.x; i < found; i += kThreads)
            if (s.ctl.place + i < kCap) list[s.ctl.place + i] = s.mass[i];
        if (range.lo > 0) {
            before = block_sum(s, before);
            if (threadIdx.x == 0) s.ctl.before = before;
        }
        cluster_sync();
    } else if (cmd == kEqual) {
        // the range's tokens (one logit) in index order: a run of the part per thread
        const int per = (len + kThreads - 1) / kThreads, i0 = min(len, static_cast<int>(threadIdx.x) * per),
                  i1 = min(len, i0 + per);
        int c = 0;
        for (int i = i0; i < i1; ++i) c += desc_key(xs[i]) == range.pref ? 1 : 0;
        int *runs = reinterpret_cast<int *>(s.hcnt);
        __syncthreads();
        runs[threadIdx.x] = c;
        __syncthreads();
        block_scan<kThreads>(runs, s.ctl.warp_cnt);
        if (threadIdx.x == kThreads - 1) s.ctl.equal = runs[kThreads - 1];
        cluster_sync();
        long j = static_cast<long>(lead->equal_j);
        for (int q = 0; q < rank; ++q) j -= *peer(&s.ctl.equal, q);
        const long before = runs[threadIdx.x] - c;
        if (j >= before && j < before + c) {
            for (int i = i0; i < i1; ++i)
                if (desc_key(xs[i]) == range.pref && j-- == before) {
                    *peer(&s.ctl.equal_index, 0) = begin + i;
                    break;
                }
        }
        cluster_sync();
    }
}

// ------------------------------------------------------------- the leader --

struct List {  // tokens of bins [lo, hi] in order, with what comes before them
    int lo, hi, n;
    u64 base_mass;
    int base_cnt;
};

// Sorts the n gathered tokens and leaves their running masses in s.mass.  Up to
// kFew tokens: each thread finds its token's place, and the mass before it, by
// looking at all; more: bitonic, elements t and t + kThreads in thread t, strides
// below 32 by shuffle.
constexpr int kFew = 128;
__device__ __forceinline__ void sort_list(Smem &s, int n, const Row &row) {
    const int t = threadIdx.x;
    auto weight = [&](u64 v) { return Row::fixed(expf(row.t(desc_value(static_cast<uint32_t>(v >> 32))))); };
    if (n <= kFew) {
        u64 *w = reinterpret_cast<u64 *>(s.scnt);
        static_assert(kFew * 8 <= sizeof(s.scnt), "weights of a short list");
        u64 mine = 0, m = 0;
        if (t < n) {
            mine = s.list[t];
            w[t] = m = weight(mine);
        }
        __syncthreads();
        int place = 0;
        if (t < n) {
#pragma unroll 4
            for (int i = 0; i < n; ++i) {
                const bool before = s.list[i] < mine;
                place += before ? 1 : 0;
                m += before ? w[i] : 0ull;
            }
        }
        __syncthreads();
        if (t < n) {
            s.list[place] = mine;
            s.mass[place] = m;
        }
        __syncthreads();
        return;
    }
    int p2 = kFew;
    while (p2 < n) p2 <<= 1;
    const bool two = p2 > kThreads;
    u64 v[2];
    v[0] = t < n ? s.list[t] : ~0ull;
    v[1] = t + kThreads < n ? s.list[t + kThreads] : ~0ull;
    __syncthreads();
#pragma unroll 1
    for (int k = 2; k <= p2; k <<= 1) {
#pragma unroll 1
        for (int j = k >> 1; j > 0; j >>= 1) {
            if (j == kThreads) {  // k = 2 * kThreads: ascending
                if (v[0] > v[1]) {
                    const u64 w = v[0];
                    v[0] = v[1];
                    v[1] = w;
                }
                continue;
            }
            if (j >= 32) {
                if (t < p2) s.list[t] = v[0];
                if (two) s.list[t + kThreads] = v[1];
                __syncthreads();
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                if (e == 1 && !two) break;
                const int i = t + e * kThreads;
                u64 o;
                if (j >= 32) o = i < p2 ? s.list[i ^ j] : ~0ull;
                else o = __shfl_xor_sync(0xffffffffu, v[e], j);
                const bool low = ((i & j) == 0) == ((i & k) == 0);  // keeps the smaller
                v[e] = low ? (o < v[e] ? o : v[e]) : (o > v[e] ? o : v[e]);
            }
            if (j >= 32) __syncthreads();
        }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const int i = t + e * kThreads;
        s.list[i] = v[e];
        s.mass[i] = i < n ? weight(v[e]) : 0ull;
    }
    __syncthreads();
    block_scan<kCap>(s.mass, s.ctl.warp_mass);
}

// The leader's cuts, one after another (top-k, top-p, the draw), as steps
// between orders: next() goes on until it has an order for the cluster (in
// s.ctl) or the answer.  All of the leader's threads run it with the same
// values.  One loop of order and execution, and not a call for each order, keeps
// the code small: most of it runs once a row, and fetching it costs more than
// running it.
struct Leader {
    enum Step { kTopK, kTopP, kDraw };
    enum Phase { kBegin, kSummed, kLook, kGathered, kBefore, kSplitNext, kSplitDone, kOnly, kEqualDone, kCut };
    Row row;
    float min_p, top_p, u;
    int k, vocab, C;
    bool few;  // the row's sums are not there yet
    int step = kTopK, phase = kBegin;
    // the list: tokens of bins [lo, hi] in order, with what comes before them
    int list_lo = 0, list_hi = -1, list_n = 0, list_cnt = 0;
    u64 list_mass = 0;
    u64 total = 0, above = 0, kept = 0;  // the row's mass and what min_p keeps (0: unknown); the mass kept so far
    int limit = kBins - 1;               // no cut falls behind this bin
    // the cut at work: where the running count reaches `target`, or the running mass first exceeds it
    bool by_count = false;
    u64 target = 0;
    Range r{0, kBins - 1, -1, 32, 0u};
    bool split = false;
    u64 base_m = 0;
    int base_c = 0;
    // its token
    u64 cut_mass = 0, cut_w = 0;
    int cut_index = -1;

    __device__ __forceinline__ void order(Smem &s, int cmd, int then, Range range, int next_sh = 32, u64 j = 0) {
        __syncthreads();  // what the last order left has been read
        if (threadIdx.x == 0) {
            Ctl &c = s.ctl;
            c.cmd = cmd;
            c.range = range;
            c.next_sh = next_sh;
            c.list_n = 0;
            c.equal_j = j;
        }
        phase = then;
    }
    __device__ __forceinline__ void read_sums(Smem &s) {
        total = over_peers<u64>(C, [&](int q) { return peer(&s.ctl, q)->total; });
        above = over_peers<u64>(C, [&](int q) { return peer(&s.ctl, q)->above; });
        few = false;
    }
    // The bins that a mass falls in.  A bin's true running mass lies between low - count and
    // low * e^(1/64) + count (in units of 2^-44, where a weight is rounded by half), give or take
    // fp32 sums; with the row's mass known, what follows the bin is bounded the same way.
    __device__ __forceinline__ void mass_range(Smem &s) {
        const float want = static_cast<float>(target), all_low = s.mlow[kBins - 1], slack = 4e-6f * all_low;
        const float rest = total ? static_cast<float>(total - target) : INFINITY;
        const float all_cnt = static_cast<float>(s.mcnt[kBins - 1]);
        r.lo = first_of(kBins, [&](int i) {
            const float c = static_cast<float>(s.mcnt[i]), low = s.mlow[i];
            return low * 1.0161f + c + slack > want && (all_low - low) * 0.9997f - (all_cnt - c) - slack < rest;
        });
        r.hi = first_of(kBins, [&](int i) {
            const float c = static_cast<float>(s.mcnt[i]), low = s.mlow[i];
            return i >= r.lo && (low * 0.9997f - c - slack > want || (all_low - low) * 1.0161f + (all_cnt - c) + slack < rest);
        });
        r.lo = min(r.lo, limit);
        r.hi = min(r.hi, limit);
    }
    // True with an order, false with the answer.
    __device__ __forceinline__ bool next(Smem &s) {
        while (true) {
            if (phase == kBegin) {
                if (few && (k <= 0 || k >= vocab)) {  // all are kept: the mass is needed
                    order(s, kSums, kSummed, r);
                    return true;
                }
                if (step == kTopK) {
                    if (!few && total == 0) {
                        read_sums(s);
                        kept = total;
                    }
                    by_count = true;
                    target = k;
                    if (k <= 0 || k >= vocab) {
                        step = kTopP;
                        continue;
                    }
                } else if (step == kTopP) {
                    by_count = false;
                    if (!(top_p < 1.f)) {
                        step = kDraw;
                        continue;
                    }
                    const double want = ceil(static_cast<double>(top_p) * static_cast<double>(kept));
                    target = want < 1.0 ? 0ull : min(kept, static_cast<u64>(want)) - 1;
                } else {
                    by_count = false;
                    if (min_p > 0.f) {
                        if (few && list_hi >= 0 && list_lo == 0) {  // the list holds all that is kept
                            u64 m = 0;
                            for (int i = threadIdx.x; i < list_n; i += kThreads) {
                                const float x = desc_value(static_cast<uint32_t>(s.list[i] >> 32)), w = expf(row.t(x));
                                if (w >= min_p || x == row.max) m += Row::fixed(w);
                            }
                            above = block_sum(s, m);
                        } else if (few) {
                            order(s, kSums, kSummed, r);
                            return true;
                        }
                        kept = min(kept, above);
                    }
                    const double at = floor(static_cast<double>(u) * static_cast<double>(kept));
                    target = at > 0.0 ? min(kept - 1, static_cast<u64>(at)) : 0ull;
                }
                phase = kLook;
            } else if (phase == kSummed) {
                read_sums(s);
                if (step == kTopK) kept = total;
                phase = kBegin;
            } else if (phase == kLook) {
                r = Range{0, 0, -1, 32, 0u};
                if (by_count) r.lo = r.hi = first_of(kBins, [&](int i) { return s.mcnt[i] >= static_cast<uint32_t>(target); });
                else mass_range(s);
                limit = r.hi;
                if (r.lo >= list_lo && r.hi <= list_hi) {
                    phase = kCut;
                    continue;
                }
                const int upto = static_cast<int>(s.mcnt[r.hi]);
                if (upto <= kCap) r.lo = 0;  // everything up to here fits: later cuts need no gather
                base_c = r.lo ? static_cast<int>(s.mcnt[r.lo - 1]) : 0;
                base_m = 0;
                list_hi = -1;
                split = upto - base_c > kCap;
                Range get = r;
                if (split) get.hi = get.lo;  // for the mass before the range alone
                order(s, kGather, split ? kBefore : kGathered, get);
                return true;
            } else if (phase == kGathered) {
                list_lo = r.lo;
                list_hi = r.hi;
                list_n = static_cast<int>(s.mcnt[r.hi]) - base_c;
                list_cnt = base_c;
                list_mass = r.lo ? over_peers<u64>(C, [&](int q) { return peer(&s.ctl, q)->before; }) : 0;
                sort_list(s, list_n, row);
                phase = kCut;
            } else if (phase == kBefore) {
                if (r.lo) base_m = over_peers<u64>(C, [&](int q) { return peer(&s.ctl, q)->before; });
                order(s, kHist, kSplitDone, r, 32);
                return true;
            } else if (phase == kSplitDone) {
                const int sh = s.ctl.next_sh;
                block_scan<kSplit>(s.mass, s.ctl.warp_mass);
                block_scan<kSplit>(s.scnt, reinterpret_cast<uint32_t *>(s.ctl.warp_cnt));
                const int d = by_count ? first_of(kSplit, [&](int i) { return s.scnt[i] >= static_cast<uint32_t>(target - base_c); })
                                       : first_of(kSplit, [&](int i) { return s.mass[i] > target - base_m; });
                const u64 dm = d ? s.mass[d - 1] : 0, in_m = s.mass[d] - dm;
                const int dc = d ? static_cast<int>(s.scnt[d - 1]) : 0, in_c = static_cast<int>(s.scnt[d]) - dc;
                base_m += dm;
                base_c += dc;
                if (sh == 32) {
                    r.sub = d;
                } else {
                    r.pref = r.sh == 32 ? static_cast<uint32_t>(d) : (r.pref << (r.sh - sh)) | static_cast<uint32_t>(d);
                    r.sh = sh;
                }
                if (in_c <= kCap) {
                    list_n = in_c;
                    list_cnt = base_c;
                    list_mass = base_m;
                    order(s, kGather, kOnly, r);
                    return true;
                }
                if (r.sh == 0) {  // equal logits
                    const u64 w = in_m / static_cast<u64>(in_c);
                    const u64 j = by_count ? target - 1 - base_c : (w ? (target - base_m) / w : 0);
                    cut_mass = base_m + (j + 1) * w;
                    cut_w = w;
                    order(s, kEqual, kEqualDone, r, 32, j);
                    return true;
                }
                order(s, kHist, kSplitDone, r, r.sh == 2 ? 0 : r.sh - 10);
                return true;
            } else if (phase == kOnly) {  // a list of use to this cut only
                sort_list(s, list_n, row);
                phase = kCut;
            } else {
                if (phase == kEqualDone) {
                    cut_index = s.ctl.equal_index;
                } else {
                    const int i = by_count ? static_cast<int>(target) - 1 - list_cnt
                                           : min(list_n - 1, first_of(kCap, [&](int i) { return i >= list_n || s.mass[i] > target - list_mass; }));
                    cut_mass = list_mass + s.mass[i];
                    cut_w = s.mass[i] - (i ? s.mass[i - 1] : 0);
                    cut_index = static_cast<int>(s.list[i] & 0xffffffffull);
                }
                if (step == kDraw) return false;
                kept = cut_mass;
                ++step;
                phase = kBegin;
            }
        }
    }
};

__global__ void __launch_bounds__(kThreads, 2) ijb_sample_kernel(const __grid_constant__ SampleParams p) {
    extern __shared__ __align__(16) uint8_t raw[];
    Smem &s = *reinterpret_cast<Smem *>(raw);
    float *xs = reinterpret_cast<float *>(raw + sizeof(Smem));
    const int rank = static_cast<int>(ctarank());
    uint32_t csize;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(csize));
    const int C = static_cast<int>(csize), r = blockIdx.x / C;
    const int begin = min(p.vocab, rank * p.chunk), len = min(p.vocab, begin + p.chunk) - begin;
    const float *x = p.x + r * p.stride + begin;
    const float temp = p.temperature ? p.temperature[r] : 1.f;
    const bool greedy = !(temp > 0.f);

    float m = -INFINITY;
    u64 key = 0;
    auto take = [&](int i, float v) {
        if (v != v) v = -INFINITY;
        xs[i] = v;
        m = fmaxf(m, v);
        if (greedy) {
            const u64 k = argmax_key(v, begin + i);
            key = k > key ? k : key;
        }
    };
    if (reinterpret_cast<uintptr_t>(x) % 16 == 0) {
        const int n4 = len / 4;
#pragma unroll 4
        for (int i = threadIdx.x; i < n4; i += kThreads) {
            const float4 v = reinterpret_cast<const float4 *>(x)[i];
            take(4 * i, v.x);
            take(4 * i + 1, v.y);
            take(4 * i + 2, v.z);
            take(4 * i + 3, v.w);
        }
        for (int i = n4 * 4 + threadIdx.x; i < len; i += kThreads) take(i, x[i]);
    } else {
        for (int i = threadIdx.x; i < len; i += kThreads) take(i, x[i]);
    }
    m = warp_max(m);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const u64 other = __shfl_xor_sync(0xffffffffu, key, o);
        key = other > key ? other : key;
    }
    if (threadIdx.x == 0) {
        s.ctl.max = -INFINITY;
        s.ctl.key = 0;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) {
        s.ctl.warp_mass[threadIdx.x >> 5] = key;
        s.ctl.warp_cnt[threadIdx.x >> 5] = __float_as_int(m);
    }
    __syncthreads();
    if (threadIdx.x == 0)
        for (int w = 0; w < kWarps; ++w) {
            s.ctl.max = fmaxf(s.ctl.max, __int_as_float(s.ctl.warp_cnt[w]));
            s.ctl.key = s.ctl.warp_mass[w] > s.ctl.key ? s.ctl.warp_mass[w] : s.ctl.key;
        }
    cluster_sync();
    Row row;
    row.max = -INFINITY;
    row.temp = temp;
#pragma unroll
    for (int q = 0; q < kMaxCluster; ++q) row.max = fmaxf(row.max, peer(&s.ctl, q < C ? q : 0)->max);
    if (row.max == -INFINITY || greedy) {  // nothing to choose from, or the largest
        if (rank == 0 && threadIdx.x == 0) {
            u64 best = 0;
            for (int q = 0; q < C; ++q) best = max(best, peer(&s.ctl, q)->key);
            p.token[r] = row.max == -INFINITY ? -1 : argmax_key_index(best);
            if (p.prob) p.prob[r] = row.max == -INFINITY ? 0.f : 1.f;
        }
        cluster_sync();  // no CTA leaves while the leader reads it
        return;
    }
    row.inv = 1.f / temp;
    row.plain_div = !(temp >= 1e-6f && temp <= 1e6f);
    const float min_p = p.min_p ? p.min_p[r] : 0.f;
    const int k = p.top_k ? p.top_k[r] : 0;
    const bool few = k > 0 && k <= kCap / 2;  // usually the list holds all that is kept: no sums over the row
    if (few) count_bins<false>(s, xs, len, row, min_p);
    else count_bins<true>(s, xs, len, row, min_p);
    cluster_sync();
    {  // CTA r adds a slice of the counts
        const int per = kBins / C;
        for (int i = rank * per + threadIdx.x; i < (rank + 1) * per; i += kThreads) {
            const uint32_t c = over_peers<uint32_t>(C, [&](int q) { return *peer(&s.hcnt[i], q); });
            *peer(&s.mcnt[i], 0) = c;
            *peer(&s.mlow[i], 0) = i == kBins - 1 ? 0.f : static_cast<float>(c) * exp2f(static_cast<float>(i + 1) * (-1.4426950408889634f / kBinsPerNat) + 44.f);
        }
    }
    cluster_sync();
    Leader lead;
    if (rank == 0) {
        block_scan<kBins>(s.mcnt, reinterpret_cast<uint32_t *>(s.ctl.warp_cnt));
        block_scan<kBins>(s.mlow, s.ctl.warp_f);
        lead.row = row;
        lead.min_p = min_p;
        lead.top_p = p.top_p ? p.top_p[r] : 1.f;
        lead.u = p.u[r];
        lead.k = k;
        lead.vocab = p.vocab;
        lead.C = C;
        lead.few = few;
    }
    while (true) {
        if (rank == 0 && !lead.next(s)) {
            if (threadIdx.x == 0) {
                s.ctl.cmd = kDone;
                p.token[r] = lead.cut_index;
                if (p.prob) p.prob[r] = static_cast<float>(static_cast<double>(lead.cut_w) / static_cast<double>(lead.kept));
            }
        }
        cluster_sync();  // the order is there
        if (peer(&s.ctl, 0)->cmd == kDone) break;
        execute(s, xs, len, begin, row, min_p, C, rank);
    }
    cluster_sync();  // the others have read the leader's last order
}

}  // namespace

cudaError_t sample_launch(const float *x, long stride, int n, int vocab, const float *u, const float *temperature,
                          const int *top_k, const float *top_p, const float *min_p, int *token, float *prob,
                          cudaStream_t stream) {
    SampleParams p{x, stride, vocab, 0, u, temperature, top_k, top_p, min_p, token, prob};
    int c = 1;  // parts of at most 2048 logits where the cluster may be that large
    while (c < kMaxCluster && (vocab + c - 1) / c > 2048) c *= 2;
    p.chunk = ((vocab + c - 1) / c + 3) / 4 * 4;
    const int smem = static_cast<int>(sizeof(Smem)) + p.chunk * 4;
    static bool ready[64];
    static std::mutex mu;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    {
        std::lock_guard<std::mutex> lock(mu);
        if (!ready[dev]) {
            e = cudaFuncSetAttribute(ijb_sample_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     static_cast<int>(sizeof(Smem)) + kMaxChunk * 4);
            if (e == cudaSuccess)
                e = cudaFuncSetAttribute(ijb_sample_kernel, cudaFuncAttributePreferredSharedMemoryCarveout,
                                         cudaSharedmemCarveoutMaxShared);
            if (e != cudaSuccess) return e;
            ready[dev] = true;
        }
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(n) * c);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = c;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, ijb_sample_kernel, p);
}

}  // namespace ijb

extern "C" int ijb_sample(const float *logits_dev, long stride, int n, int vocab, const float *u_dev,
                          const float *temperature_dev, const int *top_k_dev, const float *top_p_dev,
                          const float *min_p_dev, int *token_dev, float *prob_dev, void *stream) {
    using namespace ijb;
    try {
        const char *bad = nullptr;
        if (n < 0 || n > (1 << 24)) bad = "ijb_sample: n must be 0..2^24";
        else if (vocab < 1 || vocab > kMaxCluster * kMaxChunk) bad = "ijb_sample: vocab must be 1..131072";
        else if (stride < vocab) bad = "ijb_sample: the stride is shorter than a row";
        else if (n > 0 && (!logits_dev || !u_dev || !token_dev)) bad = "ijb_sample: null pointer";
        if (bad) {
            set_thread_error(bad);
            return IJB_ERR_INVALID;
        }
        if (n == 0) return IJB_OK;
        const cudaError_t e = sample_launch(logits_dev, stride, n, vocab, u_dev, temperature_dev, top_k_dev, top_p_dev,
                                            min_p_dev, token_dev, prob_dev, static_cast<cudaStream_t>(stream));
        if (e != cudaSuccess) {
            set_thread_error(std::string("ijb_sample: ") + cudaGetErrorString(e));
            return IJB_ERR_CUDA;
        }
        count_launches(1);
        return IJB_OK;
    } catch (...) {
        return IJB_ERR_NOMEM;
    }
}

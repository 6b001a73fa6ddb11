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
// counted and weighed in 1024 bins of -t (64 a nat, the last open), which says in
// which bin a cut falls.  That bin's tokens (and all before them where they fit)
// are gathered in the leader CTA, which narrows them by finer bins to at most
// kFew and finds each one's place by looking at all.  A bin of too many tokens is
// split over the cluster first, by finer bins of t, then by the bits of the
// logits, down to equal ones, which the order by index decides.  A row with a
// small top-k weighs only what its list holds: then the first pass only counts.
//
// What bounds it: the chain of steps, most of them for the whole cluster: one row of
// 128256 takes 18 us, 256 of them (37 at a time on 148 SMs) 221 us, with 32 % of the
// issue slots and 29 % of the shared-memory cycles in use.  Two CTAs of 512 threads
// an SM were the fastest shape (one of 1024: 415 us; three of 256: 254; clusters of
// 16: 431), and rows read again from L2 in place of a copy in shared memory, for
// fewer CTAs a row, took 236 to 566 us.
#include <mutex>
#include <string>

#include "../../include/ijb200.h"
#include "common.cuh"
#include "misc.cuh"

namespace ijb {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 1024;
constexpr int kCap = 1024;            // tokens of the leader's list
constexpr int kFew = 128;             // tokens that are put in order
constexpr int kMaxVocab = 131072;
constexpr int kMaxCluster = 16;
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

enum Cmd { kDone, kMass, kHist, kGather, kEqual };

// Which tokens an order is about: bins lo..hi of -t; with sub >= 0 the sub-th of
// kBins equal parts of those; with sh < 32 the logits whose key starts with pref.
struct Range {
    int lo, hi, sub, sh;
    uint32_t pref;
};

struct Ctl {
    // this CTA's part of a reduction
    float max;
    u64 key, above;
    int equal, found, place;
    // the leader's orders and results
    int cmd, next_sh, list_n, index;
    Range range;
    u64 equal_j, cut_mass, cut_w;
    // within the CTA
    u64 warp_mass[kWarps];
    int warp_cnt[kWarps];
};

struct Smem {
    Ctl ctl;
    uint32_t hcnt[kBins];  // this CTA's counts and masses
    u64 hmass[kBins];
    uint32_t mcnt[kBins];  // leader: the row's, up to each bin
    u64 mmass[kBins];
    uint32_t scnt[kBins];  // leader: a split's, up to each part
    u64 smass[kBins];      // (also where a CTA collects what it gathers)
    u64 few[kFew], few_w[kFew];
    // the leader's list lies over its hmass
};
static_assert(kCap <= kBins, "the list lies over a histogram");

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
// Sum over the cluster of f(q), the reads of eight CTAs in flight together.
template <class T, class F>
__device__ __forceinline__ T over_peers(int C, F f) {
    T sum = 0;
#pragma unroll 1
    for (int q0 = 0; q0 < C; q0 += 8) {
        T v[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = q0 + q < C ? f(q0 + q) : T(0);
#pragma unroll
        for (int q = 0; q < 8; ++q) sum += v[q];
    }
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
    float max, temp, inv;  // max finite, temp within 1e-15 .. 1e15
    // (x - m) / T, rounded to nearest: with inv = 1 / T rounded to nearest, one
    // residual correction of d * inv gives the quotient rounded to nearest
    // (Markstein).  Differences below -1e20, -infinity included, count as that:
    // exp makes 0 of all of them.
    __device__ __forceinline__ float t(float x) const {
        const float d = fmaxf(x - max, -1e20f);
        const float q = d * inv;
        return fmaf(fmaf(-q, temp, d), inv, q);
    }
    // Nearest whole number of -64 t, kBins - 1 at most (adding 2^23 leaves it in the low bits).
    __device__ __forceinline__ static int bin(float t) {
        const float c = fmaxf(t, -static_cast<float>(kBins - 1) / kBinsPerNat);
        return __float_as_int(fmaf(c, -kBinsPerNat, 8388608.f)) & (2 * kBins - 1);
    }
    // Which of kBins equal parts of bins lo..hi, the open bin taken to end at -t = 32 (where
    // weights end), its rest in the last part.
    __device__ __forceinline__ static int part(float t, int lo, int hi) {
        const float end = hi == kBins - 1 ? 32.f * kBinsPerNat : static_cast<float>(hi) + 0.5f;
        const float begin = static_cast<float>(lo) - 0.5f;
        const float f = (-t * kBinsPerNat - begin) * (static_cast<float>(kBins) / (end - begin));
        return static_cast<int>(fminf(fmaxf(f, 0.f), static_cast<float>(kBins - 1)));
    }
    __device__ __forceinline__ static u64 fixed(float w) { return __float2ull_rn(w * kFixed); }
    __device__ __forceinline__ bool in(float x, const Range &r) const {
        const float tt = t(x);
        const int b = bin(tt);
        return b >= r.lo && b <= r.hi && (r.sub < 0 || part(tt, r.lo, r.hi) == r.sub) &&
               (r.sh == 32 || (desc_key(x) >> r.sh) == r.pref);
    }
    // Bounds on the logits of bins lo..hi, with room for t's rounding.
    __device__ __forceinline__ float least(int hi) const {
        return hi == kBins - 1
                   ? -INFINITY
                   : max - (static_cast<float>(hi + 2) / kBinsPerNat) * temp * 1.0001f - fabsf(max) * 1e-5f;
    }
    __device__ __forceinline__ float most(int lo) const {
        return lo == 0
                   ? INFINITY
                   : max - (static_cast<float>(lo - 1) / kBinsPerNat) * temp * 0.9999f + fabsf(max) * 1e-5f;
    }
};

__device__ __forceinline__ u64 warp_sum64(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
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
// Inclusive sums over N (a multiple of kThreads) pairs in place.
template <int N>
__device__ __forceinline__ void block_scan(Smem &s, u64 *mass, uint32_t *cnt) {
    constexpr int PER = N / kThreads;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, base = threadIdx.x * PER;
    u64 x[PER], m = 0;
    uint32_t y[PER], c = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        x[i] = mass ? mass[base + i] : 0ull;
        y[i] = cnt[base + i];
        m += x[i];
        c += y[i];
    }
    const u64 own_m = m;
    const uint32_t own_c = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 pm = __shfl_up_sync(0xffffffffu, m, o);
        const uint32_t pc = __shfl_up_sync(0xffffffffu, c, o);
        if (lane >= o) {
            m += pm;
            c += pc;
        }
    }
    if (lane == 31) {
        s.ctl.warp_mass[warp] = m;
        s.ctl.warp_cnt[warp] = static_cast<int>(c);
    }
    __syncthreads();
    u64 wm = lane < warp ? s.ctl.warp_mass[lane] : 0ull;  // kWarps <= 32
    uint32_t wc = lane < warp ? static_cast<uint32_t>(s.ctl.warp_cnt[lane]) : 0u;
    wm = warp_sum64(wm);
    wc = __reduce_add_sync(0xffffffffu, wc);
    m += wm - own_m;
    c += wc - own_c;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        m += x[i];
        c += y[i];
        if (mass) mass[base + i] = m;
        cnt[base + i] = c;
    }
    __syncthreads();
}
// First i of n (a multiple of kThreads) at which the rising predicate f holds,
// n - 1 if none; every thread calls it.
template <class F>
__device__ __forceinline__ int first_of(int n, F f) {
    int at = 0;
    for (int i = threadIdx.x; i < n; i += kThreads) at += __syncthreads_count(!f(i));
    return min(at, n - 1);
}

__device__ __forceinline__ void clear_hist(uint32_t *cnt, u64 *mass) {
    for (int i = threadIdx.x; i < kBins; i += kThreads) {
        cnt[i] = 0;
        mass[i] = 0;
    }
    __syncthreads();
}

// 64-bit addition in shared memory by its two words (shared memory has no 64-bit
// addition of its own; a loop of compare-and-swap took four times as long).
__device__ __forceinline__ void add64(u64 *p, u64 m) {
    uint32_t *w = reinterpret_cast<uint32_t *>(p);
    const uint32_t lo = static_cast<uint32_t>(m), old = atomicAdd(w, lo);
    const uint32_t hi = static_cast<uint32_t>(m >> 32) + (old + lo < old ? 1u : 0u);
    if (hi) atomicAdd(w + 1, hi);
}

// Counts (and weighs) the CTA's tokens by bin; with MASS also what min_p keeps.
template <bool MASS>
__device__ __forceinline__ void local_hist(Smem &s, const float *xs, int len, const Row &row, float min_p) {
    clear_hist(s.hcnt, s.hmass);
    u64 above = 0, last = 0;
    uint32_t last_n = 0;
#pragma unroll 4
    for (int i = threadIdx.x; i < len; i += kThreads) {
        const float x = xs[i], t = row.t(x);
        const int b = Row::bin(t);
        u64 m = 0;
        if (MASS) {
            const float w = expf(t);
            m = Row::fixed(w);
            if (min_p > 0.f && (w >= min_p || x == row.max)) above += m;
        }
        if (b == kBins - 1) {  // the open bin may hold most of the row
            ++last_n;
            last += m;
        } else {
            atomicAdd(&s.hcnt[b], 1u);
            if (MASS) add64(&s.hmass[b], m);
        }
    }
    last_n = __reduce_add_sync(0xffffffffu, last_n);
    if (MASS) last = warp_sum64(last);
    if ((threadIdx.x & 31) == 0 && last_n) {
        atomicAdd(&s.hcnt[kBins - 1], last_n);
        if (MASS) add64(&s.hmass[kBins - 1], last);
    }
    if (MASS && min_p > 0.f) {
        above = block_sum(s, above);
        if (threadIdx.x == 0) s.ctl.above = above;
    }
}

// Adds the cluster's histograms into the leader's (cnt, mass): CTA r a slice.
__device__ __forceinline__ void merge_hist(Smem &s, uint32_t *cnt, u64 *mass, int C, int rank, bool masses = true) {
    cluster_sync();  // every CTA's is there
    const int per = kBins / C;
    for (int i = rank * per + threadIdx.x; i < (rank + 1) * per; i += kThreads) {
        *peer(&cnt[i], 0) = over_peers<uint32_t>(C, [&](int q) { return *peer(&s.hcnt[i], q); });
        if (masses) *peer(&mass[i], 0) = over_peers<u64>(C, [&](int q) { return *peer(&s.hmass[i], q); });
    }
    cluster_sync();
}

// What every CTA of the cluster does for one order of the leader.
__device__ __forceinline__ void execute(Smem &s, const float *xs, int len, int begin, const Row &row, float min_p, int C,
                                        int rank) {
    const Ctl *lead = peer(&s.ctl, 0);
    const int cmd = lead->cmd;
    const Range range = lead->range;
    if (cmd == kMass) {
        local_hist<true>(s, xs, len, row, min_p);
        merge_hist(s, s.mcnt, s.mmass, C, rank);
    } else if (cmd == kHist) {  // counts and masses of a split: by parts (next_sh 32) or by key bits
        const int sh = lead->next_sh;
        const float least = row.least(range.hi), most = row.most(range.lo);
        clear_hist(s.hcnt, s.hmass);
        for (int i = threadIdx.x; i < len; i += kThreads) {
            const float x = xs[i];
            if (x < least || x > most || !row.in(x, range)) continue;
            const float t = row.t(x);
            const int d = sh == 32 ? Row::part(t, range.lo, range.hi)
                                   : static_cast<int>((desc_key(x) >> sh) & ((1u << (range.sh - sh)) - 1u));
            const u64 m = Row::fixed(expf(t));
            atomicAdd(&s.hcnt[d], 1u);
            if (m) add64(&s.hmass[d], m);
        }
        merge_hist(s, s.scnt, s.smass, C, rank);
    } else if (cmd == kGather) {  // the range's tokens, first together here, then in one piece to the leader's list
        const float least = row.least(range.hi), most = row.most(range.lo);
        if (threadIdx.x == 0) s.ctl.found = 0;
        __syncthreads();
#pragma unroll 4
        for (int i = threadIdx.x; i < len; i += kThreads) {
            const float x = xs[i];
            if (x >= least && x <= most && row.in(x, range)) {
                const int at = atomicAdd(&s.ctl.found, 1);
                if (at < kCap) s.smass[at] = (static_cast<u64>(desc_key(x)) << 32) | static_cast<uint32_t>(begin + i);
            }
        }
        __syncthreads();
        const int found = min(s.ctl.found, kCap);
        if (threadIdx.x == 0 && found) s.ctl.place = atomicAdd(peer(&s.ctl.list_n, 0), found);
        __syncthreads();
        u64 *list = peer(s.hmass, 0);
        for (int i = threadIdx.x; i < found; i += kThreads)
            if (s.ctl.place + i < kCap) list[s.ctl.place + i] = s.smass[i];
        cluster_sync();
    } else if (cmd == kEqual) {
        // the range's tokens (one logit) in index order: a run of the part per thread
        const int per = (len + kThreads - 1) / kThreads, i0 = min(len, static_cast<int>(threadIdx.x) * per),
                  i1 = min(len, i0 + per);
        uint32_t c = 0;
        for (int i = i0; i < i1; ++i) c += desc_key(xs[i]) == range.pref ? 1u : 0u;
        __syncthreads();
        s.hcnt[threadIdx.x] = c;
        __syncthreads();
        block_scan<kThreads>(s, nullptr, s.hcnt);
        if (threadIdx.x == kThreads - 1) s.ctl.equal = static_cast<int>(s.hcnt[kThreads - 1]);
        cluster_sync();
        long j = static_cast<long>(lead->equal_j);
        for (int q = 0; q < rank; ++q) j -= *peer(&s.ctl.equal, q);
        const long before = static_cast<long>(s.hcnt[threadIdx.x]) - c;
        if (j >= before && j < before + static_cast<long>(c)) {
            for (int i = i0; i < i1; ++i)
                if (desc_key(xs[i]) == range.pref && j-- == before) {
                    *peer(&s.ctl.index, 0) = begin + i;
                    break;
                }
        }
        cluster_sync();
    }
}

// The leader's cuts, one after another (top-k, top-p, the draw), as steps
// between orders: next() goes on until it has an order for the cluster (in
// s.ctl) or the answer.  All of the leader's threads run it with the same
// values.  One loop of order and execution, and not a call for each order, keeps
// the code small: most of it runs once a row, and fetching it costs more than
// running it.
struct Leader {
    enum Step { kTopK, kTopP, kDraw };
    enum Phase { kBegin, kWeighed, kLook, kGathered, kInList, kSplitDone, kOrder, kEqualDone, kCut };
    Row row;
    float min_p, top_p, u;
    int k, vocab, C;
    bool weighed;  // the bins' masses are there
    int step = kTopK, phase = kBegin;
    int list_lo = 0, list_hi = -1, list_n = 0;  // the list: tokens of bins [lo, hi]
    bool sorted = false;                        // the whole list is in s.few, in order, with its running masses
    u64 kept = 0, above = 0;
    // the cut at work: where the running count reaches `target`, or the running mass first exceeds it
    bool by_count = false;
    u64 target = 0;
    Range r{0, 0, -1, 32, 0u};
    u64 base_m = 0;  // what comes before the tokens looked at
    int base_c = 0;

    __device__ __forceinline__ void order(Smem &s, int cmd, int then, int next_sh = 32, u64 j = 0) {
        __syncthreads();  // what the last order left has been read
        if (threadIdx.x == 0) {
            Ctl &c = s.ctl;
            c.cmd = cmd;
            c.range = r;
            c.next_sh = next_sh;
            c.list_n = 0;
            c.equal_j = j;
        }
        phase = then;
    }
    __device__ __forceinline__ u64 weight(u64 v) const {
        return Row::fixed(expf(row.t(desc_value(static_cast<uint32_t>(v >> 32)))));
    }
    // Part d (of a scanned split) holds the cut: moves the base there; its tokens.
    __device__ __forceinline__ int enter(Smem &s, int &d) {
        d = by_count ? first_of(kBins, [&](int i) { return s.scnt[i] >= static_cast<uint32_t>(target - base_c); })
                     : first_of(kBins, [&](int i) { return s.smass[i] > target - base_m; });
        const int before = d ? static_cast<int>(s.scnt[d - 1]) : 0, n = static_cast<int>(s.scnt[d]) - before;
        base_m += d ? s.smass[d - 1] : 0ull;
        base_c += before;
        return n;
    }
    // True with an order, false with the answer (s.ctl.index, cut_w; kept).
    __device__ __forceinline__ bool next(Smem &s) {
        u64 *list = s.hmass;
        while (true) {
            if (phase == kBegin) {
                by_count = step == kTopK;
                if (!by_count && !weighed && list_hi < 0) {  // no list that holds all that is kept
                    order(s, kMass, kWeighed);
                    return true;
                }
                if (step == kTopK) {
                    if (weighed) kept = s.mmass[kBins - 1];
                    if (k <= 0 || k >= vocab) {
                        if (!weighed) {
                            order(s, kMass, kWeighed);
                            return true;
                        }
                        step = kTopP;
                        continue;
                    }
                    target = k;
                } else if (step == kTopP) {
                    if (!(top_p < 1.f)) {
                        step = kDraw;
                        continue;
                    }
                    const double want = ceil(static_cast<double>(top_p) * static_cast<double>(kept));
                    target = want < 1.0 ? 0ull : min(kept, static_cast<u64>(want)) - 1;
                } else {
                    if (min_p > 0.f) {
                        if (weighed) {
                            above = over_peers<u64>(C, [&](int q) { return peer(&s.ctl, q)->above; });
                        } else {  // the list holds all that is kept
                            u64 m = 0;
                            for (int i = threadIdx.x; i < list_n; i += kThreads) {
                                const float x = desc_value(static_cast<uint32_t>(list[i] >> 32)), w = expf(row.t(x));
                                if (w >= min_p || x == row.max) m += Row::fixed(w);
                            }
                            above = block_sum(s, m);
                        }
                        kept = min(kept, above);
                    }
                    const double at = floor(static_cast<double>(u) * static_cast<double>(kept));
                    target = at > 0.0 ? min(kept - 1, static_cast<u64>(at)) : 0ull;
                }
                phase = kLook;
            } else if (phase == kWeighed) {
                block_scan<kBins>(s, s.mmass, s.mcnt);
                weighed = true;
                list_hi = -1;  // the histogram lay over it
                sorted = false;
                phase = kBegin;
            } else if (phase == kLook) {
                r = Range{list_lo, list_hi, -1, 32, 0u};
                base_m = 0;
                base_c = 0;
                if (!weighed && !by_count) {  // a list from bin 0 on holds all that is kept
                    phase = kInList;
                    continue;
                }
                const int b = by_count ? first_of(kBins, [&](int i) { return s.mcnt[i] >= static_cast<uint32_t>(target); })
                                       : first_of(kBins, [&](int i) { return s.mmass[i] > target; });
                if (list_hi >= 0 && b >= list_lo && b <= list_hi) {
                    base_m = list_lo ? s.mmass[list_lo - 1] : 0ull;
                    base_c = list_lo ? static_cast<int>(s.mcnt[list_lo - 1]) : 0;
                    phase = kInList;
                    continue;
                }
                const int upto = static_cast<int>(s.mcnt[b]);
                r.hi = b;
                r.lo = upto <= kCap ? 0 : b;  // everything up to here fits: later cuts need no gather
                if (r.lo && !weighed) {
                    order(s, kMass, kWeighed);
                    return true;
                }
                base_c = r.lo ? static_cast<int>(s.mcnt[r.lo - 1]) : 0;
                base_m = r.lo ? s.mmass[r.lo - 1] : 0ull;
                list_lo = r.lo;
                list_hi = -1;
                sorted = false;
                list_n = upto - base_c;
                if (list_n <= kCap) {
                    order(s, kGather, kGathered);
                } else {
                    order(s, kHist, kSplitDone);
                }
                return true;
            } else if (phase == kGathered) {
                list_hi = r.hi;
                phase = kInList;
            } else if (phase == kInList) {
                if (list_n <= kFew) {
                    if (!sorted) {
                        for (int i = threadIdx.x; i < list_n; i += kThreads) s.few[i] = list[i];
                        if (threadIdx.x == 0) s.ctl.list_n = list_n;
                        __syncthreads();
                    }
                    phase = kOrder;
                    continue;
                }
                clear_hist(s.scnt, s.smass);
                for (int i = threadIdx.x; i < list_n; i += kThreads) {
                    const u64 v = list[i];
                    const int d = Row::part(row.t(desc_value(static_cast<uint32_t>(v >> 32))), r.lo, r.hi);
                    atomicAdd(&s.scnt[d], 1u);
                    add64(&s.smass[d], weight(v));
                }
                __syncthreads();
                block_scan<kBins>(s, s.smass, s.scnt);
                int d;
                const int n = enter(s, d);
                r.sub = d;
                if (n > kFew) {
                    order(s, kHist, kSplitDone, 22);
                    list_hi = -1;
                    return true;
                }
                if (threadIdx.x == 0) s.ctl.list_n = 0;
                __syncthreads();
                for (int i = threadIdx.x; i < list_n; i += kThreads) {
                    const u64 v = list[i];
                    if (Row::part(row.t(desc_value(static_cast<uint32_t>(v >> 32))), r.lo, r.hi) == d)
                        s.few[atomicAdd(&s.ctl.list_n, 1)] = v;
                }
                __syncthreads();
                phase = kOrder;
            } else if (phase == kSplitDone) {
                const int sh = s.ctl.next_sh;
                block_scan<kBins>(s, s.smass, s.scnt);
                const u64 m0 = base_m;
                int d;
                const int n = enter(s, d);
                if (sh == 32) {
                    r.sub = d;
                } else {
                    r.pref = r.sh == 32 ? static_cast<uint32_t>(d) : (r.pref << (r.sh - sh)) | static_cast<uint32_t>(d);
                    r.sh = sh;
                }
                if (n <= kFew) {
                    list_n = n;
                    order(s, kGather, kInList);  // a list of use to this cut only
                    return true;
                }
                if (r.sh == 0) {  // equal logits
                    const u64 w = (m0 + s.smass[d] - base_m) / static_cast<u64>(n);
                    const u64 j = by_count ? target - 1 - base_c : (w ? (target - base_m) / w : 0);
                    order(s, kEqual, kEqualDone, 32, j);
                    if (threadIdx.x == 0) {
                        s.ctl.cut_mass = base_m + (j + 1) * w;
                        s.ctl.cut_w = w;
                    }
                    return true;
                }
                order(s, kHist, kSplitDone, r.sh == 32 ? 22 : (r.sh == 2 ? 0 : r.sh - 10));
                return true;
            } else if (phase == kOrder) {
                const int n = s.ctl.list_n, t = threadIdx.x;
                if (!sorted) {  // each of a few tokens finds its place, and the mass before it
                    u64 mine = 0, m = 0;
                    int place = 0;
                    if (t < n) {
                        mine = s.few[t];
                        s.few_w[t] = m = weight(mine);
                    }
                    __syncthreads();
                    if (t < n) {
#pragma unroll 4
                        for (int i = 0; i < n; ++i) {
                            const bool before = s.few[i] < mine;
                            place += before ? 1 : 0;
                            m += before ? s.few_w[i] : 0ull;
                        }
                    }
                    __syncthreads();
                    if (t < n) {
                        s.few[place] = mine;
                        s.few_w[place] = m;
                    }
                    __syncthreads();
                    sorted = list_hi >= 0 && list_n <= kFew;
                }
                if (t < n) {
                    const u64 m = s.few_w[t], before = t ? s.few_w[t - 1] : 0ull;
                    if (by_count ? t == static_cast<int>(target) - 1 - base_c
                                 : before <= target - base_m && target - base_m < m) {
                        s.ctl.cut_mass = base_m + m;
                        s.ctl.cut_w = m - before;
                        s.ctl.index = static_cast<int>(s.few[t] & 0xffffffffull);
                    }
                }
                __syncthreads();
                phase = kCut;
            } else {  // kEqualDone, kCut
                if (step == kDraw) return false;
                kept = s.ctl.cut_mass;
                // The next cut writes it: over a list already in order that is without another
                // barrier on the way (no masses to search, nothing to put in order).
                __syncthreads();
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
    if (greedy) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const u64 other = __shfl_xor_sync(0xffffffffu, key, o);
            key = other > key ? other : key;
        }
    }
    if ((threadIdx.x & 31) == 0) {
        s.ctl.warp_mass[threadIdx.x >> 5] = key;
        s.ctl.warp_cnt[threadIdx.x >> 5] = __float_as_int(m);
    }
    __syncthreads();
    if (threadIdx.x < 32) {
        const int lane = threadIdx.x;
        float v = lane < kWarps ? __int_as_float(s.ctl.warp_cnt[lane]) : -INFINITY;
        u64 k = lane < kWarps ? s.ctl.warp_mass[lane] : 0ull;
        v = warp_max(v);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const u64 other = __shfl_xor_sync(0xffffffffu, k, o);
            k = other > k ? other : k;
        }
        if (lane == 0) {
            s.ctl.max = v;
            s.ctl.key = k;
            s.ctl.above = 0;
        }
    }
    cluster_sync();
    Row row;
    {
        const int lane = threadIdx.x & 31;
        row.max = warp_max(lane < C ? peer(&s.ctl, lane)->max : -INFINITY);
    }
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
    if (row.max == INFINITY) {  // the infinite ones share everything: as logits 0 beside -infinity
        for (int i = threadIdx.x; i < len; i += kThreads) xs[i] = xs[i] == INFINITY ? 0.f : -INFINITY;
        row.max = 0.f;
        __syncthreads();
    }
    row.temp = fminf(fmaxf(temp, 1e-15f), 1e15f);
    row.inv = 1.f / row.temp;
    const float min_p = p.min_p ? p.min_p[r] : 0.f;
    const int k = p.top_k ? p.top_k[r] : 0;
    const bool few = k > 0 && k <= kCap / 2 && k < p.vocab;  // most likely the list holds all that is kept
    if (few) local_hist<false>(s, xs, len, row, 0.f);
    else local_hist<true>(s, xs, len, row, min_p);
    merge_hist(s, s.mcnt, s.mmass, C, rank, !few);
    Leader lead;
    if (rank == 0) {
        block_scan<kBins>(s, few ? nullptr : s.mmass, s.mcnt);
        lead.row = row;
        lead.min_p = min_p;
        lead.top_p = p.top_p ? p.top_p[r] : 1.f;
        lead.u = p.u[r];
        lead.k = k;
        lead.vocab = p.vocab;
        lead.C = C;
        lead.weighed = !few;
    }
    while (true) {
        if (rank == 0 && !lead.next(s)) {
            if (threadIdx.x == 0) {
                s.ctl.cmd = kDone;
                p.token[r] = s.ctl.index;
                if (p.prob) p.prob[r] = static_cast<float>(static_cast<double>(s.ctl.cut_w) / static_cast<double>(lead.kept));
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
    static bool ready[64], wide[64];
    static std::mutex mu;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = kMaxCluster;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.blockDim = dim3(kThreads);
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    bool most;
    {
        std::lock_guard<std::mutex> lock(mu);
        if (!ready[dev]) {
            e = cudaFuncSetAttribute(ijb_sample_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     static_cast<int>(sizeof(Smem)) + kMaxVocab / 8 * 4);
            if (e == cudaSuccess)
                e = cudaFuncSetAttribute(ijb_sample_kernel, cudaFuncAttributePreferredSharedMemoryCarveout,
                                         cudaSharedmemCarveoutMaxShared);
            if (e != cudaSuccess) return e;
            // clusters of 16 only where the device can place one
            cfg.gridDim = dim3(kMaxCluster);
            cfg.dynamicSmemBytes = sizeof(Smem) + kMaxVocab / kMaxCluster * 4;
            int clusters = 0;
            wide[dev] = cudaFuncSetAttribute(ijb_sample_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess &&
                        cudaOccupancyMaxActiveClusters(&clusters, ijb_sample_kernel, &cfg) == cudaSuccess && clusters > 0;
            if (!wide[dev]) cudaGetLastError();
            ready[dev] = true;
        }
        most = n <= 8 && wide[dev];
    }
    // parts of at most 2048 logits, in clusters of up to 8 CTAs; 16 for few rows, where the row's time
    // counts: 128256 logits, in a graph, 24.5 us with 16 and 28.5 with 8 for one row, 26.4 and 28.6 for 4, 28.7
    // each for 8, 47.5 and 30.7 for 16
    int c = 1;
    while (c < (most ? kMaxCluster : 8) && (vocab + c - 1) / c > 2048) c *= 2;
    p.chunk = ((vocab + c - 1) / c + 3) / 4 * 4;
    cfg.gridDim = dim3(static_cast<unsigned>(n) * c);
    cfg.dynamicSmemBytes = sizeof(Smem) + static_cast<size_t>(p.chunk) * 4;
    cfg.stream = stream;
    attr[0].val.clusterDim.x = c;
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
        else if (vocab < 1 || vocab > kMaxVocab) bad = "ijb_sample: vocab must be 1..131072";
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

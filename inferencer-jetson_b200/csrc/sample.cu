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
// the logits are read from HBM once.  The order is never built: a histogram of
// (count, mass) over 1024 bins of -t (32 a nat, the last open) says in which
// bin a cut falls, and only that bin's tokens (and all before them where they
// fit) are gathered in the leader CTA, sorted and summed.  A bin of more than
// kCap tokens is split by the bits of its logits first, down to equal ones,
// which the order by index decides.
#include <string>

#include "../../include/ijb200.h"
#include "common.cuh"
#include "misc.cuh"

namespace ijb {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 1024;
constexpr int kCap = 1024;            // tokens the leader sorts
constexpr int kMaxChunk = 16384;      // logits per CTA
constexpr int kMaxCluster = 8;
constexpr float kBinsPerNat = 32.f;
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

enum Cmd { kDone, kHist, kGather, kEqual };

struct Ctl {
    // this CTA's part of a reduction
    float max;
    u64 key, min_mass;
    int equal;
    // the leader's orders and results
    int cmd, bin_lo, bin_hi, sh, prev_sh;
    uint32_t prev_pref;
    int list_n;
    u64 equal_j;
    int equal_index;
    // broadcast within the CTA
    float row_max;
    u64 warp_mass[kWarps];
    int warp_cnt[kWarps];
};

struct Smem {
    Ctl ctl;
    u64 hmass[kBins];  // local histogram; the leader's list lies over it between histograms
    uint32_t hcnt[kBins];
    u64 mmass[kBins];  // leader: the row's histogram, as inclusive sums
    uint32_t mcnt[kBins];
    u64 smass[kBins];  // leader: a split bin's, then the running masses of the sorted list
    uint32_t scnt[kBins];
};

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
    float max, temp;
    __device__ __forceinline__ float t(float x) const { return x == max ? 0.f : (x - max) / temp; }
    __device__ __forceinline__ static int bin(float t) {
        return static_cast<int>(fminf(-t * kBinsPerNat, static_cast<float>(kBins - 1)));
    }
    // 0 for a NaN (a logit of -infinity at an infinite temperature)
    __device__ __forceinline__ static u64 fixed(float w) {
        return w > 0.f ? static_cast<u64>(__float2ll_rn(w * kFixed)) : 0ull;
    }
};

__device__ __forceinline__ u64 warp_sum64(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Inclusive sums over n (a multiple of kThreads, at most 2 * kThreads) pairs, in place.
__device__ void block_scan(Smem &s, u64 *mass, uint32_t *cnt, int n) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, per = n / kThreads, base = threadIdx.x * per;
    u64 m = 0;
    int c = 0;
    for (int i = 0; i < per; ++i) {
        m += mass[base + i];
        if (cnt) c += cnt[base + i];
    }
    const u64 own_m = m;
    const int own_c = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 pm = __shfl_up_sync(0xffffffffu, m, o);
        const int pc = __shfl_up_sync(0xffffffffu, c, o);
        if (lane >= o) {
            m += pm;
            c += pc;
        }
    }
    if (lane == 31) {
        s.ctl.warp_mass[warp] = m;
        s.ctl.warp_cnt[warp] = c;
    }
    __syncthreads();
    m -= own_m;
    c -= own_c;
    for (int w = 0; w < warp; ++w) {
        m += s.ctl.warp_mass[w];
        c += s.ctl.warp_cnt[w];
    }
    for (int i = 0; i < per; ++i) {
        m += mass[base + i];
        mass[base + i] = m;
        if (cnt) {
            c += cnt[base + i];
            cnt[base + i] = c;
        }
    }
    __syncthreads();
}

// Sum over the CTA, the same in every thread.
__device__ u64 block_sum(Smem &s, u64 v) {
    v = warp_sum64(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s.ctl.warp_mass[threadIdx.x >> 5] = v;
    __syncthreads();
    u64 r = 0;
    for (int w = 0; w < kWarps; ++w) r += s.ctl.warp_mass[w];
    return r;
}

// First i of n inclusive sums with sum > target (n - 1 if none).
template <class T>
__device__ __forceinline__ int first_above(const T *sums, int n, T target) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (sums[mid] > target) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

// Whether x is one of the tokens a command is about.
__device__ __forceinline__ bool in_range(const Row &row, float x, int lo, int hi, int sh, uint32_t pref) {
    const int b = Row::bin(row.t(x));
    return b >= lo && b <= hi && (sh == 32 || (desc_key(x) >> sh) == pref);
}

// Adds (bin, 1, mass) to the CTA's histogram; every lane of the warp calls it.
__device__ __forceinline__ void hist_add(Smem &s, bool live, int bin, u64 mass) {
    const int b0 = __shfl_sync(0xffffffffu, bin, 0);
    if (__all_sync(0xffffffffu, live && bin == b0)) {  // equal logits: one update a warp
        const u64 m = warp_sum64(mass);
        if ((threadIdx.x & 31) == 0) {
            atomicAdd(&s.hcnt[b0], 32u);
            atomicAdd(&s.hmass[b0], m);
        }
    } else if (live) {
        atomicAdd(&s.hcnt[bin], 1u);
        if (mass) atomicAdd(&s.hmass[bin], mass);
    }
}

// The CTA's histogram of level 0 (by bin of -t) or of a split bin (by key bits);
// returns the mass of the tokens that min_p keeps (level 0).
__device__ u64 local_hist(Smem &s, const float *xs, int len, const Row &row, bool level0, float min_p, int bin, int sh,
                          int prev_sh, uint32_t prev_pref) {
    for (int i = threadIdx.x; i < kBins; i += kThreads) {
        s.hmass[i] = 0;
        s.hcnt[i] = 0;
    }
    __syncthreads();
    u64 above = 0;
    const uint32_t mask = level0 ? 0u : (1u << (prev_sh - sh)) - 1u;
    for (int i0 = 0; i0 < len; i0 += kThreads) {
        const int i = i0 + threadIdx.x;
        bool live = i < len;
        const float x = live ? xs[i] : -INFINITY;
        const float t = row.t(x), w = expf(t);
        const u64 m = Row::fixed(w);
        int b = Row::bin(t);
        if (level0) {
            if (live && (w >= min_p || x == row.max)) above += m;
        } else {
            const uint32_t key = desc_key(x);
            live = live && b == bin && (prev_sh == 32 || (key >> prev_sh) == prev_pref);
            b = static_cast<int>((key >> sh) & mask);
        }
        hist_add(s, live, b, m);
    }
    return above;
}

// Sums the cluster's histograms into the leader's (mass, cnt): CTA r sums a slice.
__device__ void merge_hist(Smem &s, u64 *mass, uint32_t *cnt, int C, int rank) {
    cluster_sync();  // every CTA's histogram is there
    const int per = kBins / C;
    for (int i = rank * per + threadIdx.x; i < (rank + 1) * per; i += kThreads) {
        u64 m = 0;
        uint32_t c = 0;
        for (int q = 0; q < C; ++q) {
            m += *peer(&s.hmass[i], q);
            c += *peer(&s.hcnt[i], q);
        }
        *peer(&mass[i], 0) = m;
        *peer(&cnt[i], 0) = c;
    }
    cluster_sync();
}

// What every CTA of the cluster does for one order of the leader.
__device__ void execute(Smem &s, const float *xs, int len, int begin, const Row &row, int C, int rank) {
    const Ctl *lead = peer(&s.ctl, 0);
    const int cmd = lead->cmd, lo = lead->bin_lo, hi = lead->bin_hi, sh = lead->sh, prev_sh = lead->prev_sh;
    const uint32_t pref = lead->prev_pref;
    if (cmd == kHist) {
        local_hist(s, xs, len, row, false, 0.f, lo, sh, prev_sh, pref);
        merge_hist(s, s.smass, s.scnt, C, rank);
    } else if (cmd == kGather) {
        int *n = peer(&s.ctl.list_n, 0);
        u64 *list = peer(s.hmass, 0);
        for (int i = threadIdx.x; i < len; i += kThreads) {
            const float x = xs[i];
            if (!in_range(row, x, lo, hi, prev_sh, pref)) continue;
            const int at = atomicAdd(n, 1);
            if (at < kCap) list[at] = (static_cast<u64>(desc_key(x)) << 32) | static_cast<uint32_t>(begin + i);
        }
        cluster_sync();
    } else if (cmd == kEqual) {
        // tokens with the key prev_pref, in index order: a run of the part per thread
        const int per = (len + kThreads - 1) / kThreads, i0 = min(len, static_cast<int>(threadIdx.x) * per),
                  i1 = min(len, i0 + per);
        int c = 0;
        for (int i = i0; i < i1; ++i) c += desc_key(xs[i]) == pref ? 1 : 0;
        u64 *runs = s.hmass;  // [kThreads] of the local histogram, free now
        __syncthreads();
        runs[threadIdx.x] = c;
        __syncthreads();
        block_scan(s, runs, nullptr, kThreads);
        if (threadIdx.x == kThreads - 1) s.ctl.equal = static_cast<int>(runs[kThreads - 1]);
        cluster_sync();
        u64 j = lead->equal_j;
        for (int q = 0; q < rank; ++q) j -= static_cast<u64>(*peer(&s.ctl.equal, q));  // wraps past zero: not here
        const u64 before = runs[threadIdx.x] - c;
        if (j >= before && j < before + c) {
            for (int i = i0; i < i1; ++i)
                if (desc_key(xs[i]) == pref && j-- == before) {
                    *peer(&s.ctl.equal_index, 0) = begin + i;
                    break;
                }
        }
        cluster_sync();
    }
}

// ------------------------------------------------------------- the leader --

struct List {  // tokens of bins [lo, hi] in order, with what comes before them
    int lo = 0, hi = -1, n = 0;
    u64 base_mass = 0;
    int base_cnt = 0;
};

// Sorts the gathered list and leaves its running masses in smass.
__device__ void sort_list(Smem &s, int n, const Row &row) {
    u64 *list = s.hmass;
    int p2 = 2;
    while (p2 < n) p2 <<= 1;
    for (int i = n + threadIdx.x; i < p2; i += kThreads) list[i] = ~0ull;
    __syncthreads();
    for (int k = 2; k <= p2; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            for (int i = threadIdx.x; i < p2 / 2; i += kThreads) {
                const int a = 2 * i - (i & (j - 1)), b = a + j;
                const u64 x = list[a], y = list[b];
                if ((x > y) == ((a & k) == 0)) {
                    list[a] = y;
                    list[b] = x;
                }
            }
            __syncthreads();
        }
    for (int i = threadIdx.x; i < kCap; i += kThreads)
        s.smass[i] = i < n ? Row::fixed(expf(row.t(desc_value(static_cast<uint32_t>(list[i] >> 32))))) : 0ull;
    __syncthreads();
    block_scan(s, s.smass, nullptr, kCap);
}

__device__ void give(Smem &s, int cmd, int lo, int hi, int sh, int prev_sh, uint32_t pref, u64 j) {
    __syncthreads();
    if (threadIdx.x == 0) {
        Ctl &c = s.ctl;
        c.cmd = cmd;
        c.bin_lo = lo;
        c.bin_hi = hi;
        c.sh = sh;
        c.prev_sh = prev_sh;
        c.prev_pref = pref;
        c.list_n = 0;
        c.equal_j = j;
    }
    cluster_sync();
}

struct Cut {
    u64 mass;  // running mass through the token
    u64 w;
    int index;
};

// The token at which the running count reaches `target` (by_count), or at
// which the running mass first exceeds it.
__device__ Cut select(Smem &s, const float *xs, int len, const Row &row, int C, List &list, bool by_count, u64 target,
                      bool want_index) {
    const int b = by_count ? first_above<uint32_t>(s.mcnt, kBins, static_cast<uint32_t>(target) - 1u)
                           : first_above<u64>(s.mmass, kBins, target);
    if (b < list.lo || b > list.hi) {
        const u64 before_m = b ? s.mmass[b - 1] : 0;
        const int before_c = b ? static_cast<int>(s.mcnt[b - 1]) : 0;
        const int in_bin = static_cast<int>(s.mcnt[b]) - before_c;
        list = List();
        if (in_bin <= kCap) {
            const bool all = static_cast<int>(s.mcnt[b]) <= kCap;  // everything up to here fits: later cuts need no gather
            list.lo = all ? 0 : b;
            list.hi = b;
            list.n = all ? static_cast<int>(s.mcnt[b]) : in_bin;
            list.base_mass = all ? 0 : before_m;
            list.base_cnt = all ? 0 : before_c;
            give(s, kGather, list.lo, b, 32, 32, 0u, 0);
            execute(s, xs, len, 0, row, C, 0);
            sort_list(s, list.n, row);
        } else {
            u64 base_m = before_m;
            int base_c = before_c, prev_sh = 32;
            uint32_t pref = 0;
            while (true) {
                const int sh = prev_sh == 2 ? 0 : prev_sh - 10;
                give(s, kHist, b, b, sh, prev_sh, pref, 0);
                execute(s, xs, len, 0, row, C, 0);
                block_scan(s, s.smass, s.scnt, kBins);
                const int d = by_count ? first_above<uint32_t>(s.scnt, kBins, static_cast<uint32_t>(target - base_c) - 1u)
                                       : first_above<u64>(s.smass, kBins, target - base_m);
                const u64 upto_m = s.smass[d], dm = d ? s.smass[d - 1] : 0;
                const int upto_c = static_cast<int>(s.scnt[d]), dc = d ? static_cast<int>(s.scnt[d - 1]) : 0;
                base_m += dm;
                base_c += dc;
                pref = prev_sh == 32 ? static_cast<uint32_t>(d) : (pref << (prev_sh - sh)) | static_cast<uint32_t>(d);
                prev_sh = sh;
                __syncthreads();  // the sums have been read
                if (upto_c - dc <= kCap) {
                    list.n = upto_c - dc;
                    list.base_mass = base_m;
                    list.base_cnt = base_c;
                    give(s, kGather, b, b, sh, sh, pref, 0);
                    execute(s, xs, len, 0, row, C, 0);
                    sort_list(s, list.n, row);
                    break;  // list.hi stays -1: of use to this cut only
                }
                if (sh == 0) {  // equal logits
                    const u64 w = (upto_m - dm) / static_cast<u64>(upto_c - dc);
                    const u64 j = by_count ? target - 1 - base_c : (w ? (target - base_m) / w : 0);
                    Cut cut;
                    cut.mass = base_m + (j + 1) * w;
                    cut.w = w;
                    cut.index = -1;
                    if (want_index) {
                        give(s, kEqual, b, b, 0, 0, pref, j);
                        execute(s, xs, len, 0, row, C, 0);
                        cut.index = s.ctl.equal_index;
                    }
                    return cut;
                }
            }
        }
    }
    const int i = by_count ? static_cast<int>(target) - 1 - list.base_cnt
                           : first_above<u64>(s.smass, list.n, target - list.base_mass);
    Cut cut;
    cut.mass = list.base_mass + s.smass[i];
    cut.w = s.smass[i] - (i ? s.smass[i - 1] : 0);
    cut.index = static_cast<int>(s.hmass[i] & 0xffffffffull);
    return cut;
}

__global__ void __launch_bounds__(kThreads) ijb_sample_kernel(const __grid_constant__ SampleParams p) {
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
    for (int q = 0; q < C; ++q) row.max = fmaxf(row.max, peer(&s.ctl, q)->max);
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
    const float min_p = p.min_p ? p.min_p[r] : 0.f;
    const u64 above = block_sum(s, local_hist(s, xs, len, row, true, min_p, 0, 0, 32, 0u));
    if (threadIdx.x == 0) s.ctl.min_mass = above;
    merge_hist(s, s.mmass, s.mcnt, C, rank);
    if (rank != 0) {
        while (true) {
            cluster_sync();
            if (peer(&s.ctl, 0)->cmd == kDone) break;
            execute(s, xs, len, begin, row, C, rank);
        }
        cluster_sync();
        return;
    }
    u64 min_mass = 0;
    for (int q = 0; q < C; ++q) min_mass += peer(&s.ctl, q)->min_mass;
    block_scan(s, s.mmass, s.mcnt, kBins);
    u64 kept = s.mmass[kBins - 1];
    List list;
    const int k = p.top_k ? p.top_k[r] : 0;
    if (k > 0 && k < p.vocab) kept = select(s, xs, len, row, C, list, true, k, false).mass;
    const float top_p = p.top_p ? p.top_p[r] : 1.f;
    if (top_p < 1.f) {
        const double want = ceil(static_cast<double>(top_p) * static_cast<double>(kept));
        const u64 least = want < 1.0 ? 1ull : min(kept, static_cast<u64>(want));
        kept = select(s, xs, len, row, C, list, false, least - 1, false).mass;
    }
    kept = min(kept, min_mass);
    const double at = floor(static_cast<double>(p.u[r]) * static_cast<double>(kept));
    const u64 target = at > 0.0 ? min(kept - 1, static_cast<u64>(at)) : 0ull;
    const Cut cut = select(s, xs, len, row, C, list, false, target, true);
    if (threadIdx.x == 0) {
        p.token[r] = cut.index;
        if (p.prob) p.prob[r] = static_cast<float>(static_cast<double>(cut.w) / static_cast<double>(kept));
    }
    give(s, kDone, 0, 0, 0, 0, 0u, 0);
    cluster_sync();  // the others have read the order
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
    cudaError_t e = cudaFuncSetAttribute(ijb_sample_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         static_cast<int>(sizeof(Smem)) + kMaxChunk * 4);
    if (e != cudaSuccess) return e;
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

// Attention of new tokens over the paged K/V cache (fp16, e4m3 or e2m1 rows).
//
// An entry is L new tokens, the last of a sequence's T cached positions.  With
// G query heads to a KV head, its rows for one KV head are the L * G pairs
// (token, head of the group), token first; row r of token i = r / G sees the
// positions t <= T - L + i:
//   s_t = (q . k_t) * scale,   out = sum_t exp(s_t - m) v_t / sum_t exp(s_t - m)
// with the running maximum m and sum of an online softmax in fp32.  A row that
// sees nothing gets zeros.
//
// Two kernels, by rows:
//  * ijb_paged_decode_kernel, up to 16 rows an entry and KV head (single tokens,
//    a few drafted ones): bound by reading the cache.  Every warp streams
//    32-position chunks of its own through shared memory.  For e2m1 rows, whose
//    reading takes less time than their arithmetic, ijb_paged_decode4_kernel (calls of
//    few tiles: in one launch, without what the next paragraph says).
//  * ijb_paged_tile_kernel, more rows (chunks, prompts): bound by the matrix
//    products and the exponentials.  256 rows at a time on tcgen05.
// Both cut all the call's work (tiles of rows x units of positions, over all
// entries and KV heads, in one line) into equal runs, one per worker, so ragged
// lengths and long contexts fill the GPU alike.  A tile counts for `over` units
// more than it has (its queries come in, its output goes out), and a cut that
// would leave less than `least` units of a tile on one side moves to its end.  A tile's run that another
// worker began or goes on with leaves its softmax state in the workspace, and
// ijb_paged_merge_kernel joins the states in order: no atomics, the same result
// every time for the same call.
//
// Arithmetic.  Products are fp16 x fp16 with fp32 sums.  fp32 queries enter as
// two fp16 parts (hi + lo, 22 bits), and so do their probabilities; fp16
// queries enter as they are, their probabilities rounded to fp16 once (the
// output is fp16 too: 2.6e-4 to 2.9e-4 rel-L2 against 64 bits, of which the output's
// rounding alone is 2.1e-4), and their O stays in the tensor core over a worker's run,
// where additions drop bits towards zero: 3e-5 of an output over 131072 positions, 1.4e-4
// over 2^20, 5.5e-4 over 2^22.  Cached rows enter as fp16: fp16 rows exactly, e4m3 values as the
// fp16 number nearest to code * 2^e, as an fp16 cache would hold them: exactly from 2^-14 on (and
// every value of a row whose largest is in [2^-7, 2^15]), else off by 2^-25 at most, infinite from
// 65520 on.  (The decode kernel scales its scores in fp32, so K has no such ends there.)  e2m1 values,
// code * scale, are fp16 numbers.
#include <mutex>
#include <type_traits>

#include "paged.cuh"

namespace ijb {
namespace {

// ------------------------------------------------------------------ plan --

constexpr int kMaxEntries = 4096, kMaxTiles = 8192;

// A place in the line of work: `at` counts units and tiles' `over`; a tile is
// entered past its `over`.
struct Cursor {
    long at, end;
    int e, ti, head, b0;
};

// What a worker leaves to the merge: the tile that its last run begins and does
// not end, as rows row0 .. row0 + rows of the entry whose tokens start at q0, and
// the number of its states (0: there is none); whether any value it computed is
// not finite (1) and any page of its runs names nothing (2); where its runs began.
struct __align__(16) Left {
    int states, q0, row0, rows, head, bad, pad[2];
    Cursor runs;
};

struct AttnArgs {
    KvDev kv;
    const void *q;
    long q_stride;
    void *out;
    long out_stride;
    int heads, group;
    int n_tokens, n_entries;
    const int *q_start, *seq, *kv_len;
    int min_rows, max_rows;  // entries with rows of a KV head in this range are this kernel's
    bool report_long;        // no other kernel takes longer ones: they are beyond the caller's max_q
    int tile_rows, unit;     // rows per tile, positions per unit
    int workers, min_units;
    int over, least;
    float scale_log2;        // scale * log2(e)
    Left *left;              // workspace: per worker, the tile it leaves to be gone on with
    float *part;             // workspace: two states per worker
    float *held;             // workspace: the tile kernel's sums outside TMEM, a worker's 256 rows
    uint32_t *status;
};

struct Entry {
    int q0, len, kv, seq, rows, tiles;
};

__device__ __forceinline__ Entry entry_load(const AttnArgs &a, int e, bool report) {
    Entry x;
    const int q0 = a.q_start[e], q1 = a.q_start[e + 1];
    x.q0 = q0;
    x.len = q1 - q0;
    x.kv = a.kv_len[e];
    x.seq = a.seq ? a.seq[e] : e;
    const bool ok = q0 >= 0 && q1 >= q0 && q1 <= a.n_tokens && x.kv >= 0 &&
                    x.kv <= (a.kv.max_pages << a.kv.page_shift) && x.seq >= 0 && x.seq < a.kv.n_seqs;
    if (!ok && report && a.status) atomicOr(a.status, kDevErrBadIndex);
    const long rows = ok ? static_cast<long>(x.len) * a.group : 0;
    x.rows = rows >= a.min_rows && rows <= a.max_rows ? static_cast<int>(rows) : 0;
    if (rows > a.max_rows && report && a.report_long && a.status) atomicOr(a.status, kDevErrBadIndex);
    x.tiles = (x.rows + a.tile_rows - 1) / a.tile_rows;
    return x;
}

// Positions that tile ti of an entry reads, in units (one at least, so that rows
// that see nothing are written too).
__device__ __forceinline__ int tile_positions(const AttnArgs &a, const Entry &x, int ti) {
    const int last = (min(x.rows, (ti + 1) * a.tile_rows) - 1) / a.group;
    return max(0, x.kv - x.len + last + 1);
}
__device__ __forceinline__ int tile_units(const AttnArgs &a, const Entry &x, int ti) {
    return max(1, (tile_positions(a, x, ti) + a.unit - 1) / a.unit);
}

// One run of a worker: units [b0, b1) of the `units` of tile ti of entry e, KV head h.
struct Segment {
    Entry x;
    int e, ti, head, b0, b1, units;
    long start;  // the tile's place in the line
};

// Inclusive sum over the block's threads of v; *total receives the sum.
template <int NT>
__device__ int block_scan_int(int v, int *warp_sums, int *total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int p = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += p;
    }
    __syncthreads();
    if (lane == 31) warp_sums[warp] = v;
    __syncthreads();
    int sum = 0;
#pragma unroll
    for (int w = 0; w < NT / 32; ++w) {
        const int s = warp_sums[w];
        if (w < warp) v += s;
        sum += s;
    }
    *total = sum;
    return v;
}

// Last index i of n + 1 rising sums with sums[i] <= v (v < sums[n]).
__device__ __forceinline__ int find_le(const int *sums, int n, int v) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (sums[mid] <= v) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

struct PlanOut {
    int warp_sums[32];
    int tiles, units, per;
};

__device__ __forceinline__ void plan_end(const AttnArgs &a, int *sums, PlanOut *po, int tiles, int units) {
    const long all = static_cast<long>(units) * a.kv.kv_heads;
    if (threadIdx.x == 0) {
        sums[tiles] = units;
        po->tiles = tiles;
        po->units = units;
        po->per = static_cast<int>(max(static_cast<long>(a.min_units + a.over), (all + a.workers - 1) / a.workers));
    }
    __syncthreads();
}

// Cuts the call's work: `first` [n_entries + 1] receives each entry's first
// tile, `sums` [tiles + 1] each tile's first unit (of one KV head).  ONE: no entry
// has two tiles, and tiles are entries.  All NT threads call it.
template <int NT, bool ONE>
__device__ void plan_build(const AttnArgs &a, int *first, int *sums, PlanOut *po) {
    const bool lead = blockIdx.x == 0;
    int base = 0;
    if constexpr (ONE) {
        // one tile an entry at most: tiles are entries, some of no units
        for (int e0 = 0; e0 < a.n_entries; e0 += NT) {
            const int e = e0 + static_cast<int>(threadIdx.x);
            int n = 0;
            if (e < a.n_entries) {
                const Entry x = entry_load(a, e, lead);
                n = x.tiles ? tile_units(a, x, 0) + a.over : 0;
            }
            int total;
            const int inc = block_scan_int<NT>(n, po->warp_sums, &total);
            if (e < a.n_entries) sums[e] = base + inc - n;
            base += total;
        }
        plan_end(a, sums, po, a.n_entries, base);
    } else {
        for (int e0 = 0; e0 < a.n_entries; e0 += NT) {
            const int e = e0 + static_cast<int>(threadIdx.x);
            const int n = e < a.n_entries ? entry_load(a, e, lead).tiles : 0;
            int total;
            const int inc = block_scan_int<NT>(n, po->warp_sums, &total);
            if (e < a.n_entries) first[e] = base + inc - n;
            base += total;
        }
        if (threadIdx.x == 0) first[a.n_entries] = base;
        __syncthreads();
        // more tiles than the call's tokens have: starts that fall, whose entries overlap
        if (base > kMaxTiles && lead && threadIdx.x == 0 && a.status) atomicOr(a.status, kDevErrBadIndex);
        const int tiles = base > kMaxTiles ? 0 : base;
        base = 0;
        for (int t0 = 0; t0 < tiles; t0 += NT) {
            const int t = t0 + static_cast<int>(threadIdx.x);
            int n = 0;
            if (t < tiles) {
                const int e = find_le(first, a.n_entries, t);
                n = tile_units(a, entry_load(a, e, false), t - first[e]) + a.over;
            }
            int total;
            const int inc = block_scan_int<NT>(n, po->warp_sums, &total);
            if (t < tiles) sums[t] = base + inc - n;
            base += total;
        }
        plan_end(a, sums, po, tiles, base);
    }
}

// plan_build<NT, true> for up to 32 entries by each warp on its own, without the
// block's barriers: sums in the warp's memory, lane e's entry in x, the rest in *po.
__device__ __forceinline__ void plan_warp(const AttnArgs &a, int *sums, PlanOut *po, bool report, Entry &x) {
    const int lane = threadIdx.x & 31;
    int n = 0;
    x = {};
    if (lane < a.n_entries) {
        x = entry_load(a, lane, report);
        n = x.tiles ? tile_units(a, x, 0) + a.over : 0;
    }
    int inc = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int p = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += p;
    }
    sums[lane] = inc - n;
    const int units = __shfl_sync(0xffffffffu, inc, 31);
    if (lane == 0) sums[a.n_entries] = units;
    const long all = static_cast<long>(units) * a.kv.kv_heads;
    po->tiles = a.n_entries;
    po->units = units;
    po->per = static_cast<int>(max(static_cast<long>(a.min_units + a.over), (all + a.workers - 1) / a.workers));
    __syncwarp();
}

// Where a worker begins: w runs along, or the start or end of the tile there.
template <bool ONE>
__device__ __forceinline__ Cursor cursor_at(const AttnArgs &a, const int *first, const int *sums, const PlanOut &po, int w) {
    Cursor c;
    const long all = static_cast<long>(po.units) * a.kv.kv_heads;
    c.at = c.end = min(all, static_cast<long>(w) * po.per);
    c.e = c.ti = c.head = c.b0 = 0;
    if (c.at >= all) return c;
    c.head = (c.at >> 32) ? static_cast<int>(c.at / po.units)
                          : static_cast<int>(static_cast<uint32_t>(c.at) / static_cast<uint32_t>(po.units));
    const int u = static_cast<int>(c.at - static_cast<long>(c.head) * po.units);
    int t = find_le(sums, po.tiles, u);
    const int in = u - sums[t] - a.over, units = sums[t + 1] - sums[t] - a.over;  // units of the tile before the place
    if (in < a.least) {
        c.at -= u - sums[t];
    } else if (units - in < a.least) {
        c.at += sums[t + 1] - u;
        if (++t == po.tiles) {
            t = 0;
            ++c.head;
        }
    } else {
        c.b0 = in;
    }
    c.e = ONE ? t : find_le(first, a.n_entries, t);
    c.ti = ONE ? 0 : t - first[c.e];
    return c;
}
template <bool ONE>
__device__ __forceinline__ Cursor cursor_start(const AttnArgs &a, const int *first, const int *sums, const PlanOut &po,
                                               int worker) {
    Cursor c = cursor_at<ONE>(a, first, sums, po, worker);
    c.end = cursor_at<ONE>(a, first, sums, po, worker + 1).at;
    return c;
}

// The next run, of entry s.x, and the cursor behind it.
__device__ __forceinline__ void cursor_take(const AttnArgs &a, Cursor &c, Segment &s) {
    s.e = c.e;
    s.ti = c.ti;
    s.head = c.head;
    s.b0 = c.b0;
    s.units = tile_units(a, s.x, c.ti);
    s.start = c.at - (c.b0 > 0 ? a.over + c.b0 : 0);
    const long stop = c.end - s.start - a.over;  // units of the tile before the worker's end
    s.b1 = static_cast<int>(min(static_cast<long>(s.units), stop));
    c.at = s.start + a.over + s.b1;
    c.b0 = 0;
    if (++c.ti >= s.x.tiles) {
        c.ti = 0;
        if (++c.e == a.n_entries) {
            c.e = 0;
            ++c.head;
        }
    }
}
// The next run, and the cursor behind it; false at the end.
__device__ __forceinline__ bool cursor_next(const AttnArgs &a, Cursor &c, Segment &s) {
    if (c.at >= c.end) return false;
    s.x = entry_load(a, c.e, false);
    while (s.x.tiles == 0) {  // entries without rows here
        if (++c.e == a.n_entries) {
            c.e = 0;
            ++c.head;
        }
        s.x = entry_load(a, c.e, false);
    }
    cursor_take(a, c, s);
    return true;
}

// State slot of a run: a worker's first run may go on with a tile that another
// worker began (slot 0), its last may leave one to be gone on with (slot 1).
__device__ __forceinline__ long part_slot(const Segment &s, int worker) { return 2L * worker + (s.b0 > 0 ? 0 : 1); }
template <int ROWS, int HD>
__host__ __device__ constexpr long part_floats() { return static_cast<long>(ROWS) * (HD + 2); }

__device__ __forceinline__ Left left_of(const AttnArgs &a, const Segment &s, int worker, int per) {
    Left x = {};
    if (s.b0 > 0 || s.b1 == s.units) return x;
    // workers w' > worker begin in the tile up to the last w' * per that leaves `least` units of it
    const long last = s.start + a.over + s.units - a.least;
    x.states = 1 + ((last >> 32) ? static_cast<int>(last / per)
                                 : static_cast<int>(static_cast<uint32_t>(last) / static_cast<uint32_t>(per))) - worker;
    x.q0 = s.x.q0;
    x.row0 = s.ti * a.tile_rows;
    x.rows = min(a.tile_rows, s.x.rows - x.row0);
    x.head = s.head;
    return x;
}

__device__ __forceinline__ void store4(float *p, float a, float b, float c, float d) {
    *reinterpret_cast<float4 *>(p) = make_float4(a, b, c, d);
}
__device__ __forceinline__ uint32_t half2_bits(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ void store4(__half *p, float a, float b, float c, float d) {
    *reinterpret_cast<uint2 *>(p) = make_uint2(half2_bits(a, b), half2_bits(c, d));
}
// The same for rows that are aligned to their elements only.
template <typename T>
__device__ __forceinline__ void store4(T *p, bool vec, float a, float b, float c, float d) {
    if (vec) {
        store4(p, a, b, c, d);
    } else {
        p[0] = static_cast<T>(a);
        p[1] = static_cast<T>(b);
        p[2] = static_cast<T>(c);
        p[3] = static_cast<T>(d);
    }
}
__device__ __forceinline__ float4 load4(const float *p, bool vec) {
    return vec ? *reinterpret_cast<const float4 *>(p) : make_float4(p[0], p[1], p[2], p[3]);
}
__device__ __forceinline__ float4 load4(const __half *p, bool vec) {
    if (!vec) return make_float4(__half2float(p[0]), __half2float(p[1]), __half2float(p[2]), __half2float(p[3]));
    const uint2 u = *reinterpret_cast<const uint2 *>(p);
    const float2 x = __half22float2(*reinterpret_cast<const __half2 *>(&u.x)),
                 y = __half22float2(*reinterpret_cast<const __half2 *>(&u.y));
    return make_float4(x.x, x.y, y.x, y.y);
}
// Eight fp16 values as they are.
__device__ __forceinline__ float4 load8_raw(const __half *p, bool vec) {
    if (vec) return *reinterpret_cast<const float4 *>(p);
    __half h[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = p[i];
    return *reinterpret_cast<const float4 *>(h);
}
__device__ __forceinline__ bool aligned16(const void *p, long stride_bytes) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride_bytes % 16 == 0;
}
template <typename T>
__device__ __forceinline__ bool aligned4(const void *p, long stride) {
    return reinterpret_cast<uintptr_t>(p) % (4 * sizeof(T)) == 0 && stride % 4 == 0;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) { return __byte_perm(a, b, sel); }
// Two e4m3 codes (low 16 bits) as fp16, exactly.
__device__ __forceinline__ uint32_t e4m3x2_half2(uint32_t u) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(u), __NV_E4M3);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
    const __half2 r = __hmul2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&r);
}
// A row's scale 2^(s - 127) as factors for its codes.  2^-24 .. 2^15 are fp16 numbers, so that
// one product is code * scale, rounded once.  Beyond that (no row of a model at work) there are
// two: 2^-15 or 2^15, whose product with a code is exact or infinite, and the rest, kept to what
// leaves 0 or infinity as it is: past 2^-39 all is 0, and past 2^30 all but 0 infinite.
__device__ __forceinline__ bool scale_fits(uint32_t s) { return s - 103u <= 39u; }
__device__ __forceinline__ __half scale_half(uint32_t s) {
    return __float2half_rn(kv_scale(s < 103u ? 112u : min(s, 142u)));
}
__device__ __forceinline__ float scale_rest(uint32_t s) {
    return kv_scale(scale_fits(s) ? 127u : s < 103u ? max(s, 88u) + 15u : min(s, 157u) - 15u);
}
// Page id of a position; -1 for one that names no page, which is reported.
__device__ __forceinline__ long page_of(const AttnArgs &a, int seq, int pos) {
    const int page = a.kv.page_table[static_cast<long>(seq) * a.kv.max_pages + (pos >> a.kv.page_shift)];
    if (page >= 0 && page < a.kv.num_pages) return page;
    if (a.status) atomicOr(a.status, kDevErrBadIndex);
    return -1;
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// ---------------------------------------------------------------- decode --
//
// A warp's chunk: 32 positions, rows (up to 16) as the M side of
// mma.m16n8k16:
//   S[row][pos] = Q . K^T: a lane's K fragments are 16-byte pieces of one
//   position's row, so the 16 k slots of a step stand for whichever dims those
//   pieces hold (Q's fragments are loaded in the same order);
//   O[row][dim] += P . V: P comes from the score accumulators as they lie; a
//   lane's V fragments are 16-byte pieces of the four positions its k slots
//   stand for, their bytes paired by position with a permute.
// No operand needs ldmatrix, so 8-bit rows are read as they are stored and
// become fp16 in registers.  Shared rows are XOR-swizzled in 16-byte pieces so
// that both read patterns are free of bank conflicts.
//
// Measured: 16 contexts of 9,001 to 32,768 positions, 8 KV heads of 128 in e4m3, fp16
// queries of 32 heads: 757 MB in 148 us (5.1 TB/s), with the tensor pipe 29 % busy;
// what is left is the loads' latency at the ends of the workers' runs.

constexpr int kChunk = 32;  // positions
constexpr int kDecRows = 16;

// WIDE: more than 8 rows.  Up to 8 leave the upper half of the products' 16 rows
// unused, and with half the registers an SM holds more warps: 64 ragged
// sequences of 4 rows took 25 us with the wide kernel's 8 warps.  Of the e4m3 kernels at
// head_dim 64, fp32 queries' does not fit 16 warps' registers: one token at position 4100, 8 KV heads, took
// 18.0 us with 16 and 14.9 with 12, 16 contexts of 9,001 to 32,768 positions 103 and 98.
template <int HD, int KV, bool WIDE, typename T>
struct Dec {
    static constexpr bool E4M3 = KV == IJB_KV_E4M3;
    static constexpr int kPos = kChunk;
    static constexpr int kRowBytes = kv_row_bytes(KV, HD);
    static constexpr int kTile = kChunk * kRowBytes;
    static constexpr int kStage = 2 * kTile + (E4M3 ? 256 : 0);  // K, V, their scale bytes and what they stand for
    static constexpr int kWarps = kRowBytes == 256 ? 6 : (WIDE || HD == 128 ? 8 : (E4M3 && sizeof(T) == 2 ? 16 : 12));
    static constexpr int kStages = kRowBytes == 256 ? 2 : (kRowBytes == 128 ? (kWarps == 8 ? 3 : 2) : (WIDE ? 4 : 3));
    static constexpr int kSmem = kWarps * kStages * kStage;
    static_assert(kSmem <= 226 * 1024, "stages");
};
constexpr int kDecPlanBytes = (kMaxEntries + 1) * 4;  // entries' first units

// Byte offset of 16-byte piece c of row r in a chunk tile.
template <int RB>
__device__ __forceinline__ uint32_t dec_off(int r, int c) {
    if constexpr (RB == 64)
        return static_cast<uint32_t>((((r >> 3) << 2) | (r & 3)) * 128 + ((((r >> 2) ^ (r >> 1)) & 1) << 6) +
                                     ((c ^ ((r & 1) << 1)) << 4));
    else
        return static_cast<uint32_t>(r * RB + ((c ^ (((r & 3) << 1) ^ (r & 4))) << 4));
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr)
                 : "memory");
    return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void sts64(uint32_t addr, uint32_t a, uint32_t b) {
    asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(addr), "r"(a), "r"(b) : "memory");
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t lds8(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Rows 0..7 alone (the others are zeros): a = {row gid, first and second k pair}.
__device__ __forceinline__ void mma(float (&d)[2], const uint32_t (&a)[2], uint32_t b0, uint32_t b1) {
    [[maybe_unused]] float x, y;
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %8, %5, %8}, {%6, %7}, "
        "{%0, %1, %9, %9};"
        : "+f"(d[0]), "+f"(d[1]), "=f"(x), "=f"(y)
        : "r"(a[0]), "r"(a[1]), "r"(b0), "r"(b1), "r"(0u), "f"(0.f));
}
// fp32 queries' O += (P hi + P lo) V over 16 positions, for two dim tiles.  The products alone
// are summed by the tensor core, whose additions drop bits towards zero, and added to O
// rounded to nearest: left in the product's accumulators, the outputs of 300 entries of 20000
// positions (runs of some thousand a warp) were off by 5e-6 to 2.6e-5 (rel-L2), so they are by
// 8e-7 at most, as a plain fp32 sum's.  16 contexts of 9,001 to 32,768 positions keep their time,
// 64 ragged single tokens take 1 us more.  (volatile: in this order, for the registers.)
__device__ __forceinline__ void add2_in_order(float &x, float &y, float a, float b) {
    float2 o = make_float2(x, y), d = make_float2(a, b);
    asm volatile("add.rn.f32x2 %0, %0, %1;" : "+l"(reinterpret_cast<uint64_t &>(o)) : "l"(reinterpret_cast<uint64_t &>(d)));
    x = o.x;
    y = o.y;
}
__device__ __forceinline__ void value_product(float (&d)[4], const uint32_t (&hi)[4], const uint32_t *lo, uint32_t b0,
                                              uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(hi[0]), "r"(hi[1]), "r"(hi[2]), "r"(hi[3]), "r"(b0), "r"(b1), "f"(0.f));
    if (lo) {
        const uint32_t l[4] = {lo[0], lo[1], lo[2], lo[3]};
        mma(d, l, b0, b1);
    }
}
__device__ __forceinline__ void add_values(float (&o0)[4], float (&o1)[4], const uint32_t (&hi)[4], const uint32_t *lo,
                                           const uint32_t (&b)[4]) {
    float d0[4], d1[4];
    value_product(d0, hi, lo, b[0], b[1]);
    value_product(d1, hi, lo, b[2], b[3]);
    add2_in_order(o0[0], o0[1], d0[0], d0[1]);
    add2_in_order(o0[2], o0[3], d0[2], d0[3]);
    add2_in_order(o1[0], o1[1], d1[0], d1[1]);
    add2_in_order(o1[2], o1[3], d1[2], d1[3]);
}

template <int HD, int KV, bool WIDE, typename T>
__global__ void __launch_bounds__(Dec<HD, KV, WIDE, T>::kWarps * 32, 1)
    ijb_paged_decode_kernel(const __grid_constant__ AttnArgs a) {
    using D = Dec<HD, KV, WIDE, T>;
    constexpr int H = WIDE ? 2 : 1;  // halves of the 16 rows in use
    // up to 8 fp32 rows: their hi parts are rows 0..7 of the products, their lo
    // parts rows 8..15, for the products of one
    constexpr bool PAIR = sizeof(T) == 4 && !WIDE;
    constexpr int C = WIDE || PAIR ? 4 : 2;  // accumulators a lane
    constexpr bool SPLIT = sizeof(T) == 4;  // fp32 queries: hi + lo
    constexpr bool E4M3 = D::E4M3;
    constexpr int NT = D::kWarps * 32, RB = D::kRowBytes, KS = HD / 16, NTILE = HD / 8;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ PlanOut block_po;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gid = lane >> 2, t4 = lane & 3;
    pdl_trigger();
    const int worker = blockIdx.x * D::kWarps + warp;
    Cursor load_c;
    int per;
    if (a.n_entries < 32) {
        int *sums = reinterpret_cast<int *>(smem + warp * D::kStages * D::kStage);
        PlanOut po;
        Entry x;
        plan_warp(a, sums, &po, worker == 0, x);
        load_c = cursor_start<true>(a, nullptr, sums, po, worker);
        per = po.per;
        __syncwarp();  // the plan's shared memory becomes the stages
    } else {
        int *sums = reinterpret_cast<int *>(smem);
        plan_build<NT, true>(a, nullptr, sums, &block_po);
        load_c = cursor_start<true>(a, nullptr, sums, block_po, worker);
        per = block_po.per;
        __syncthreads();
    }
    Cursor use_c = load_c;

    const uint32_t base = smem_u32(smem) + warp * D::kStages * D::kStage;
    const T *qp = static_cast<const T *>(a.q);
    T *op = static_cast<T *>(a.out);
    const bool qvec = aligned4<T>(a.q, a.q_stride), ovec = aligned4<T>(a.out, a.out_stride);
    const long v_off = static_cast<long>(a.kv.kv_heads) << a.kv.page_shift;  // rows from K to V within a page

    // ---- the loading side: one chunk after another, across runs
    Segment ls;
    int lb = 0, stage_in = 0;
    long next_row = 0;  // lane r: cache row (K) of position r of the next chunk, -1 if there is none
    bool gone = false;  // a page was none: the merge computes these runs' rows again, without its positions
    bool more = cursor_next(a, load_c, ls);
    if (more) lb = ls.b0;
    auto find_row = [&]() {
        const int pos = lb * kChunk + lane;
        next_row = -1;
        if (pos < ls.x.kv) {
            const long page = page_of(a, ls.x.seq, pos);
            if (page >= 0) next_row = kv_row(a.kv, page, 0, ls.head, pos & ((1 << a.kv.page_shift) - 1));
            else gone = true;
        }
    };
    if (more) find_row();
    auto issue = [&]() {
        if (more) {
            const uint32_t st = base + stage_in * D::kStage;
            const int left = ls.x.kv - lb * kChunk;  // positions that exist
#pragma unroll
            for (int i = 0; i < kChunk * RB / 512; ++i) {
                const int r = (i * 32 + lane) / (RB / 16), c = lane % (RB / 16);
                // eight rows of a page lie together: their first row's address serves all
                const long row8 = __shfl_sync(0xffffffffu, next_row, r & ~7);
                const bool live = r < left && row8 >= 0;
                const long row = live ? row8 + (r & 7) : 0;
                const uint8_t *src = a.kv.data + row * RB + c * 16;
                const uint32_t off = dec_off<RB>(r, c);
                cp_async16(st + off, src, live);
                cp_async16(st + D::kTile + off, live ? src + v_off * RB : src, live);
            }
            if constexpr (E4M3) {  // 4 scale bytes a copy: lanes 0..7 K, 8..15 V
                const int r = (lane & 7) * 4;
                const long row8 = __shfl_sync(0xffffffffu, next_row, r & ~7);
                if (lane < 16 && r < left && row8 >= 0)
                    cp_async4(st + 2 * D::kTile + lane * 4, a.kv.scale + row8 + (r & 7) + (lane < 8 ? 0 : v_off));
            }
            if (++lb == ls.b1) {
                more = cursor_next(a, load_c, ls);
                lb = ls.b0;
            }
            if (more) find_row();
        }
        cp_async_commit();
        stage_in = stage_in + 1 == D::kStages ? 0 : stage_in + 1;
    };
    for (int i = 0; i < D::kStages - 1; ++i) issue();

    // ---- the computing side
    int stage = 0;
    Left left = {};
    bool bad = false;
    const Cursor runs = use_c;
    Segment s;
    while (cursor_next(a, use_c, s)) {
        const int row0 = s.ti * kDecRows, rows = min(kDecRows, s.x.rows - row0);
        uint32_t qf[KS][C], ql[SPLIT && WIDE ? KS : 1][4];
        int limit[H];  // last position that rows gid and gid + 8 see
#pragma unroll
        for (int hf = 0; hf < H; ++hf) {
            const int r = gid + 8 * hf;
            const int tok = r < rows ? (row0 + r) / a.group : 0, in = r < rows ? (row0 + r) % a.group : 0;
            limit[hf] = r < rows ? s.x.kv - s.x.len + tok : -1;
            const T *src = qp + static_cast<long>(s.x.q0 + tok) * a.q_stride + (s.head * a.group + in) * HD;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const int d = E4M3 ? (t4 + 4 * (ks >> 2)) * 16 + 4 * (ks & 3) : (t4 + 4 * (ks >> 1)) * 8 + 4 * (ks & 1);
                const float4 v = r < rows ? load4(src + d, qvec) : make_float4(0.f, 0.f, 0.f, 0.f);
                const __half2 h0 = __floats2half2_rn(v.x, v.y), h1 = __floats2half2_rn(v.z, v.w);
                qf[ks][hf] = *reinterpret_cast<const uint32_t *>(&h0);
                qf[ks][C / 2 + hf] = *reinterpret_cast<const uint32_t *>(&h1);
                if constexpr (SPLIT) {
                    const float2 f0 = __half22float2(h0), f1 = __half22float2(h1);
                    uint32_t(&lo)[4] = PAIR ? reinterpret_cast<uint32_t(&)[4]>(qf[ks]) : ql[WIDE ? ks : 0];
                    lo[PAIR ? 1 : hf] = half2_bits(v.x - f0.x, v.y - f0.y);
                    lo[PAIR ? 3 : 2 + hf] = half2_bits(v.z - f1.x, v.w - f1.y);
                }
            }
        }
        float m[H], l[H], o[NTILE][C];
#pragma unroll
        for (int hf = 0; hf < H; ++hf) {
            m[hf] = -INFINITY;
            l[hf] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < NTILE; ++i)
#pragma unroll
            for (int k = 0; k < C; ++k) o[i][k] = 0.f;
        const int all_see = s.x.kv - s.x.len + row0 / a.group;  // positions up to here are seen by every row

        for (int b = s.b0; b < s.b1; ++b) {
            issue();  // into the stage used last
            cp_async_wait<D::kStages - 1>();
            __syncwarp();
            const uint32_t kt = base + stage * D::kStage, vt = kt + D::kTile, sc = kt + 2 * D::kTile;
            const int p0 = b * kChunk;
            float kscale[8];         // of positions t4 + 4 i
            uint32_t vscale[4];      // fp16, of positions t4 + 8 i and t4 + 8 i + 4
            bool far = false;        // some need a second factor
            if constexpr (E4M3) {
                // lane r turns position r's scale bytes into numbers, kept so that a lane reads
                // its eight positions' side by side; those behind the last mean nothing
                const bool in = p0 + lane < s.x.kv;
                const int at = (lane & 3) * 8 + (lane >> 2);
                const float ks = in ? kv_scale(lds8(sc + lane)) : 0.f;
                const uint32_t vbyte = lds8(sc + 32 + lane);
                __half vs = in ? __float2half_rn(kv_scale(vbyte)) : __half(0.f);
                far = __any_sync(0xffffffffu, in && !scale_fits(vbyte));
                if (far) vs = scale_half(vbyte);
                const uint32_t nums = kt + 2 * D::kTile + 64;
                asm volatile("st.shared.f32 [%0], %1;" ::"r"(nums + at * 4), "f"(ks * a.scale_log2) : "memory");
                asm volatile("st.shared.u16 [%0], %1;" ::"r"(nums + 128 + at * 2), "h"(__half_as_ushort(vs)) : "memory");
                __syncwarp();
                const uint4 k0 = lds128(nums + t4 * 32), k1 = lds128(nums + t4 * 32 + 16), vv = lds128(nums + 128 + t4 * 16);
                const uint32_t ku[8] = {k0.x, k0.y, k0.z, k0.w, k1.x, k1.y, k1.z, k1.w};
#pragma unroll
                for (int i = 0; i < 8; ++i) kscale[i] = __uint_as_float(ku[i]);
                vscale[0] = vv.x; vscale[1] = vv.y; vscale[2] = vv.z; vscale[3] = vv.w;
            }
            // ---- scores: tile nt, column n is position 16 (nt / 2) + 8 (nt % 2) + n / 2 + 4 (n % 2)
            float p[4][C];
#pragma unroll
            for (int nt = 0; nt < 4; ++nt) {
#pragma unroll
                for (int k = 0; k < C; ++k) p[nt][k] = 0.f;
                const int r = 8 * nt + (gid >> 1) + 4 * (gid & 1);
#pragma unroll
                for (int j = 0; j < RB / 64; ++j) {
                    const uint4 w = lds128(kt + dec_off<RB>(r, t4 + 4 * j));
                    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
                    if constexpr (E4M3) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t b0 = e4m3x2_half2(u[e] & 0xffffu), b1 = e4m3x2_half2(u[e] >> 16);
                            mma(p[nt], qf[4 * j + e], b0, b1);
                            if constexpr (SPLIT && WIDE) mma(p[nt], ql[4 * j + e], b0, b1);
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            mma(p[nt], qf[2 * j + e], u[2 * e], u[2 * e + 1]);
                            if constexpr (SPLIT && WIDE) mma(p[nt], ql[2 * j + e], u[2 * e], u[2 * e + 1]);
                        }
                    }
                }
            }
            // ---- online softmax (base 2) of rows gid and gid + 8
            const bool masked = p0 + kChunk - 1 > all_see;
            float mx[H];
#pragma unroll
            for (int hf = 0; hf < H; ++hf) mx[hf] = -INFINITY;
#pragma unroll
            for (int nt = 0; nt < 4; ++nt) {
#pragma unroll
                for (int i = 0; i < 2 * H; ++i) {
                    float v = PAIR ? p[nt][i] + p[nt][C - 2 + i] : p[nt][i];
                    v *= E4M3 ? kscale[2 * nt + (i & 1)] : a.scale_log2;
                    if (masked && p0 + 8 * nt + t4 + 4 * (i & 1) > limit[i >> 1]) v = -INFINITY;
                    p[nt][i] = v;
                    mx[i >> 1] = fmaxf(mx[i >> 1], v);
                }
            }
            float alpha[H], mu[H];
            bool same = true;
#pragma unroll
            for (int hf = 0; hf < H; ++hf) {
                mx[hf] = fmaxf(mx[hf], __shfl_xor_sync(0xffffffffu, mx[hf], 1));
                mx[hf] = fmaxf(mx[hf], __shfl_xor_sync(0xffffffffu, mx[hf], 2));
                const float mn = fmaxf(m[hf], mx[hf]);
                mu[hf] = mn == -INFINITY ? 0.f : mn;
                alpha[hf] = ex2(m[hf] - mu[hf]);
                m[hf] = mn;
                l[hf] *= alpha[hf];
                same = same && alpha[hf] == 1.f;
            }
#pragma unroll
            for (int nt = 0; nt < 4; ++nt)
#pragma unroll
                for (int i = 0; i < 2 * H; ++i) {
                    p[nt][i] = ex2(p[nt][i] - mu[i >> 1]);
                    l[i >> 1] += p[nt][i];
                }
            if (!__all_sync(0xffffffffu, same)) {
#pragma unroll
                for (int i = 0; i < NTILE; ++i)
#pragma unroll
                    for (int k = 0; k < C; ++k) o[i][k] *= alpha[PAIR ? 0 : k >> 1];
            }
            if (E4M3 && far) {  // second factors go to the weights, which have been summed
#pragma unroll
                for (int nt = 0; nt < 4; ++nt)
#pragma unroll
                    for (int i = 0; i < 2 * H; ++i) p[nt][i] *= scale_rest(lds8(sc + 32 + 8 * nt + t4 + 4 * (i & 1)));
            }
            // ---- values: k slots 2t, 2t+1, 2t+8, 2t+9 are positions 16 st + t, + 4, + 8, + 12
#pragma unroll
            for (int st = 0; st < 2; ++st) {
                uint32_t ph[C], pl[4];
#pragma unroll
                for (int i = 0; i < 2 * H; ++i) {
                    const float x = p[2 * st + i / H][2 * (i % H)], y = p[2 * st + i / H][2 * (i % H) + 1];
                    const __half2 h = __floats2half2_rn(x, y);
                    ph[PAIR ? 2 * i : i] = *reinterpret_cast<const uint32_t *>(&h);
                    if constexpr (SPLIT) {
                        const float2 f = __half22float2(h);
                        const uint32_t lo = half2_bits(x - f.x, y - f.y);
                        if constexpr (PAIR) ph[2 * i + 1] = lo;
                        else pl[i] = lo;
                    }
                }
                auto values = [&](float(&o0)[C], float(&o1)[C], const uint32_t(&b)[4]) {
                    if constexpr (SPLIT) {
                        add_values(o0, o1, ph, WIDE ? pl : nullptr, b);
                    } else {
                        mma(o0, ph, b[0], b[1]);
                        mma(o1, ph, b[2], b[3]);
                    }
                };
                const int r0 = 16 * st + t4;
                if constexpr (E4M3) {
                    const uint32_t sa = vscale[2 * st], sb = vscale[2 * st + 1];
                    uint32_t w[4][HD / 32];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int r = r0 + 4 * i;
                        if constexpr (HD == 128) {
                            const uint4 x = lds128(vt + dec_off<RB>(r, gid));
                            w[i][0] = x.x; w[i][1] = x.y; w[i][2] = x.z; w[i][3] = x.w;
                        } else {
                            const uint2 x = lds64(vt + dec_off<RB>(r, gid >> 1) + 8 * (gid & 1));
                            w[i][0] = x.x; w[i][1] = x.y;
                        }
                    }
#pragma unroll
                    for (int k = 0; k < HD / 32; ++k)
#pragma unroll
                        for (int d = 0; d < 2; ++d) {
                            const uint32_t y0 = prmt(w[0][k], w[1][k], d ? 0x7362 : 0x5140),
                                           y1 = prmt(w[2][k], w[3][k], d ? 0x7362 : 0x5140);
                            const uint32_t vb[4] = {hmul2(e4m3x2_half2(y0 & 0xffffu), sa), hmul2(e4m3x2_half2(y1 & 0xffffu), sb),
                                                   hmul2(e4m3x2_half2(y0 >> 16), sa), hmul2(e4m3x2_half2(y1 >> 16), sb)};
                            values(o[4 * k + 2 * d], o[4 * k + 2 * d + 1], vb);
                        }
                } else {
#pragma unroll
                    for (int h = 0; h < HD / 64; ++h) {
                        uint32_t w[4][4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint4 x = lds128(vt + dec_off<RB>(r0 + 4 * i, gid + 8 * h));
                            w[i][0] = x.x; w[i][1] = x.y; w[i][2] = x.z; w[i][3] = x.w;
                        }
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint32_t vb[4] = {prmt(w[0][k], w[1][k], 0x5410), prmt(w[2][k], w[3][k], 0x5410),
                                                   prmt(w[0][k], w[1][k], 0x7632), prmt(w[2][k], w[3][k], 0x7632)};
                            values(o[8 * h + 2 * k], o[8 * h + 2 * k + 1], vb);
                        }
                    }
                }
            }
            __syncwarp();  // every lane is done with this stage
            stage = stage + 1 == D::kStages ? 0 : stage + 1;
        }

        if constexpr (PAIR) {
#pragma unroll
            for (int i = 0; i < NTILE; ++i) {
                o[i][0] += o[i][C - 2];
                o[i][1] += o[i][C - 1];
            }
        }
        float zero = 0.f;  // NaN once a value is not finite
#pragma unroll
        for (int i = 0; i < NTILE; ++i)
#pragma unroll
            for (int k = 0; k < 2 * H; ++k) zero = fmaf(o[i][k], 0.f, zero);
        bad |= !(zero == 0.f);
        // ---- the run's end: the output, or its state
        left = left_of(a, s, worker, per);
        const bool whole = s.b0 == 0 && s.b1 == s.units;
        float *part = a.part + part_slot(s, worker) * part_floats<kDecRows, HD>();
#pragma unroll
        for (int hf = 0; hf < H; ++hf) {
            l[hf] += __shfl_xor_sync(0xffffffffu, l[hf], 1);
            l[hf] += __shfl_xor_sync(0xffffffffu, l[hf], 2);
            const int r = gid + 8 * hf;
            if (r >= rows) continue;
            const float inv = whole ? (l[hf] > 0.f || l[hf] != l[hf] ? 1.f / l[hf] : 0.f) : 1.f;
            T *dst = op + static_cast<long>(s.x.q0 + (row0 + r) / a.group) * a.out_stride +
                     (s.head * a.group + (row0 + r) % a.group) * HD;
            float *pd = part + r * HD;
            if (!whole && t4 == 0) {
                part[kDecRows * HD + r] = m[hf];
                part[kDecRows * HD + kDecRows + r] = l[hf];
            }
            // lane t4's columns n = 2 t4, 2 t4 + 1 of tile i: dim n * W + i (W dims a piece), pieces of 64 dims apart
            constexpr int W = E4M3 && HD == 128 ? 16 : 8;
#pragma unroll
            for (int h = 0; h < NTILE / W; ++h)
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int i = 0; i < W; i += 4) {
                        const int d = 64 * h + (2 * t4 + c) * W + i;
                        const int j = h * W + i, k = 2 * hf + c;
                        if (whole) store4(dst + d, ovec, o[j][k] * inv, o[j + 1][k] * inv, o[j + 2][k] * inv, o[j + 3][k] * inv);
                        else store4(pd + d, o[j][k], o[j + 1][k], o[j + 2][k], o[j + 3][k]);
                    }
        }
    }
    cp_async_wait<0>();
    left.bad = (__any_sync(0xffffffffu, bad) ? 1 : 0) | (__any_sync(0xffffffffu, gone) ? 2 : 0);
    left.runs = runs;
    if (lane == 0) a.left[worker] = left;
}

// (below)
template <int ROWS, int HD, int NT, int RB, typename T>
__device__ __forceinline__ int merge_block(const AttnArgs &a, const Left &left, int w0, int row0, float *top, float *total,
                                           float4 *sum);
template <int ROWS, int HD, int NT, int RB, int KV, typename T>
__device__ __noinline__ void mend_rows(const AttnArgs &a, int w, int row0, bool all, float4 *shared);

// ------------------------------------------------------- decode, 4 bits --
//
// e2m1 rows have a kernel of their own: with a quarter of an fp16 cache's bytes the
// instructions bound it, not the reading (the general kernel, its operands unpacked in
// place: 170 us for the contexts below).  Positions are the M side of mma.m16n8k16, the
// entry's rows its 8 columns (16 rows: twice 8), so half the products of the other way
// round, where up to 8 rows left half of the M side empty:
//   S^T[pos][row] = K . Q^T: a lane's K fragments are 16 or 8 bytes of one position's
//   row, one scale's block or half of one; the 16 k slots stand for whichever dims those
//   hold (Q's fragments are loaded in the same order);
//   O^T[dim][row] += V^T . P^T: a lane's V fragments are 8 or 4 bytes of each of the four
//   positions of its k slots, whose codes of one dim are put side by side in a byte
//   (two shifts and two bit selections for 16 codes) before they become a pair of fp16
//   numbers.  P^T comes from the score accumulators by movmatrix.
// A byte becomes two fp16 numbers in one instruction, and a second one scales them: 512
// of the 1030 instructions that a warp has for 64 positions of 128 dims.  fp32 rows have
// two parts, hi + lo: up to 4 rows take the 8 columns with both (the parts of a score
// are added by a shuffle), more need a product for each.
// Rows' maxima are raised only when a score passes them by more than 2^8 (see the tile
// kernel), so that a chunk has no shuffles for them.  Page ids are read 256 positions
// at once, a lane for each 8 rows that lie together, and a lane copies 16 bytes at a place
// that is one multiplication away from their number.  What a warp needs between its runs
// only is kept in shared memory, for the registers.  A call of few tiles has a cluster of
// CTAs for each (CLUSTER), which cut it without a plan and join their states behind a
// barrier of the cluster.
//
// Measured in a graph, 8 KV heads: 16 contexts of 11,003 to 40,111 positions, 32 heads of 128: 467 MB in 93 us with
// fp16 queries (5.0 TB/s) and 104 with fp32 ones; heads of 64 63 and 69.  No unit is full (issue slots 63 %, the ALU,
// which converts, 52 %), but the 3 warps a scheduler has wait for one another's instructions, not for memory: of the
// 4.6 clocks from one of a warp's to its next 0.8 go to a pipe that is taken, 0.6 to dispatch, 0.9 to another warp's
// turn, 0.8 to the last result and 0.2 to loads.  64 ragged single tokens behind 23 to 1,499, fp32, heads of 64: 18.3
// us (27.7 with the general kernel).  2 to 5 drafted tokens of 24 heads of 128 in 24 sequences behind 700 to 9,001:
// fp16 55 us, fp32 75, the tensor pipe 46 % busy, for want of more than 2 warps a scheduler beside so many sums.

template <int HD, int ROWS, typename T>
struct Dec4 {
    static constexpr bool WIDE = ROWS == 16;
    // Positions of a chunk: 64 halve what a chunk costs beside its values (16 long contexts, heads of 128, fp16 queries:
    // 93 us, with 32 103); 16 fp32 rows have no registers for them.  Warps: as many as have the registers, the same
    // number on each scheduler; 12 and not 16 at head_dim 64, whose launch costs more than it gains (64 ragged tokens
    // 18.3 and 21.3 us, 16 long contexts 69 and 64), and 8 rather than 12 that spill (8 fp32 rows of 128: 125 and 129 us).
    // Not kept: 10 and 14 warps (uneven), 16 fp32 rows' queries in shared memory for 12 warps (drafts 88 us for 75).
    static constexpr int kRowBytes = HD / 2, kBlocks = HD / kKvBlock;  // of a row: bytes, scales
    static constexpr bool kPair = ROWS == 4, kSplit = sizeof(T) == 4 && !kPair;
    static_assert(!kPair || sizeof(T) == 4, "fp16 rows have one part");
    static constexpr int kPos = WIDE && kSplit ? 32 : 64;
    static constexpr int kTile = kPos * kRowBytes, kScales = kPos * kBlocks;
    static constexpr int kStage = 2 * (kTile + kScales);  // K, V, their scale bytes
    static constexpr int kWarps = HD == 128 && (WIDE || kSplit) ? 8 : 12;
    static constexpr int kFit = 216 * 1024 / (kWarps * kStage), kStages = kFit > 4 ? 4 : kFit;
    static constexpr int kSmem = kWarps * kStages * kStage;
    static_assert(kStages >= 2, "stages");
};

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ void mma_new(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
// (a & m) | (b & ~m)
__device__ __forceinline__ uint32_t select_bits(uint32_t a, uint32_t b, uint32_t m) { return (a & m) | (b & ~m); }

template <int HD, int ROWS, typename T, bool CLUSTER>
__global__ void __launch_bounds__(Dec4<HD, ROWS, T>::kWarps * 32, 1)
    ijb_paged_decode4_kernel(const __grid_constant__ AttnArgs a) {
    using D = Dec4<HD, ROWS, T>;
    constexpr int N = ROWS == 16 ? 2 : 1;  // tiles of 8 rows
    // fp32 queries are hi + lo: products of their own, or (up to 4 rows) columns 4..7 of the same
    constexpr bool SPLIT = D::kSplit, PAIR = D::kPair;
    constexpr int NT = D::kWarps * 32, RB = D::kRowBytes, NB = D::kBlocks, KS = HD / 16, W = HD / 64;  // W: words of V
    constexpr int GROUP = 8 * RB;         // bytes of 8 rows, which lie together
    constexpr int PC = D::kPos, TT = PC / 16, G = PC / 8;  // positions, tiles and groups of a chunk
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ PlanOut block_po;
    // what a warp needs between its runs only: the loading side's place in the line, and the runs from the one
    // being computed to the one being loaded (each chunk that is loaded ahead may end one)
    constexpr int QUEUE = D::kStages + 1;
    __shared__ struct { Cursor load; Segment run[QUEUE]; } state[D::kWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gid = lane >> 2, t4 = lane & 3;
    pdl_trigger();
    const int worker = blockIdx.x * D::kWarps + warp;
    auto &my = state[warp];
    // cursor_start, with the next worker's start found by the odd lanes alongside
    auto cursor_both = [&](const int *sums, const PlanOut &po) {
        Cursor c = cursor_at<true>(a, nullptr, sums, po, worker + (lane & 1));
        c.end = __shfl_sync(0xffffffffu, c.at, 1);
        c.at = __shfl_sync(0xffffffffu, c.at, 0);
        c.e = __shfl_sync(0xffffffffu, c.e, 0);
        c.head = __shfl_sync(0xffffffffu, c.head, 0);
        c.b0 = __shfl_sync(0xffffffffu, c.b0, 0);
        return c;
    };
    Cursor first = {};
    Entry entry;  // of the first run; tiles 0: not read yet
    int per;
    // CLUSTER: the tile, its units, and those of this worker
    [[maybe_unused]] int rank = 0, size = 1, tile = 0, units = 0, b0 = 0, b1 = 0;
    if constexpr (CLUSTER) {
        asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
        asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(size));
        tile = static_cast<int>(blockIdx.x) / size;
        first.e = tile / a.kv.kv_heads;
        first.head = tile % a.kv.kv_heads;
        entry = entry_load(a, first.e, first.head == 0 && rank == 0 && warp == 0);
        if (entry.tiles == 0) return;  // (and so does the rest of the cluster)
        units = tile_units(a, entry, 0);
        per = (units + size * D::kWarps - 1) / (size * D::kWarps);
        b0 = min(units, (rank * D::kWarps + warp) * per);
        b1 = min(units, b0 + per);
        first.end = a.over + units;  // (the whole tile, for mend_rows)
    } else if (a.n_entries < 32) {
        int *sums = reinterpret_cast<int *>(smem + warp * D::kStages * D::kStage);
        PlanOut po;
        plan_warp(a, sums, &po, worker == 0, entry);
        first = cursor_both(sums, po);
        entry.q0 = __shfl_sync(0xffffffffu, entry.q0, first.e);
        entry.len = __shfl_sync(0xffffffffu, entry.len, first.e);
        entry.kv = __shfl_sync(0xffffffffu, entry.kv, first.e);
        entry.seq = __shfl_sync(0xffffffffu, entry.seq, first.e);
        entry.rows = __shfl_sync(0xffffffffu, entry.rows, first.e);
        entry.tiles = __shfl_sync(0xffffffffu, entry.tiles, first.e);
        per = po.per;
        __syncwarp();  // the plan's shared memory becomes the stages
    } else {
        int *sums = reinterpret_cast<int *>(smem);
        plan_build<NT, true>(a, nullptr, sums, &block_po);
        first = cursor_both(sums, block_po);
        entry.tiles = 0;
        per = block_po.per;
        __syncthreads();
    }
    if (lane == 0) {
        my.load = first;
        Left none = {};
        none.runs = first;
        a.left[worker] = none;
    }
    __syncwarp();
    const uint32_t base = smem_u32(smem) + warp * D::kStages * D::kStage;
    const T *qp = static_cast<const T *>(a.q);
    T *op = static_cast<T *>(a.out);
    const bool qvec = aligned4<T>(a.q, a.q_stride), ovec = aligned4<T>(a.out, a.out_stride);

    // ---- the loading side: one chunk after another, across runs
    int l_kv = 0, l_seq = 0, l_head = 0, l_end = 0;  // of the run being loaded
    int lb = 0, stage_in = 0, window = 0;  // window: the first of the 32 / G chunks whose groups the lanes have
    int page_next = -1;     // lane g: page id of group g (8 positions) of the next window
    uint32_t group = 0;     // lane g: number of group g's first row of K / 8 (the cache's memory has fewer than 2^32)
    bool fresh = true;      // the next window becomes the current one
    bool gone = false;      // a page was none: the merge computes these runs' rows again, without its positions
    bool more = false;
    int queued = 0, queue_in = 0;
    auto load_run = [&]() {
        Cursor c = my.load;
        Segment s;
        if constexpr (CLUSTER) {
            more = queued == 0 && b0 < b1;
            s.x = entry;
            s.e = first.e;
            s.ti = 0;
            s.head = first.head;
            s.b0 = b0;
            s.b1 = b1;
            s.units = units;
            s.start = 0;
        } else if (queued == 0 && entry.tiles > 0) {
            more = c.at < c.end;
            s.x = entry;
            if (more) cursor_take(a, c, s);
        } else {
            more = cursor_next(a, c, s);
        }
        if (!more) return;
        l_kv = s.x.kv;
        l_seq = s.x.seq;
        l_head = s.head;
        lb = s.b0;
        l_end = s.b1;
        __syncwarp();
        if (lane == 0) {
            my.load = c;
            my.run[queue_in] = s;
        }
        __syncwarp();
        ++queued;
        queue_in = queue_in + 1 == QUEUE ? 0 : queue_in + 1;
    };
    auto peek = [&]() {
        window = lb;
        const int pos = (lb * G + lane) * 8;
        page_next = 0;
        if (pos < min(l_kv, l_end * PC))
            page_next = a.kv.page_table[static_cast<long>(l_seq) * a.kv.max_pages + (pos >> a.kv.page_shift)];
        fresh = true;
    };
    load_run();
    if (more) peek();
    // 16-byte pieces: of K or V `lane` of 512 bytes side by side, of the scales one for K or V each
    constexpr int C = D::kScales / 16, R = 16 / NB;  // copies of K's scales in a chunk, rows a copy
    const long v_rows = static_cast<long>(a.kv.kv_heads) << a.kv.page_shift;  // from K to V within a page
    const uint8_t *from_k = a.kv.data + (HD == 128 ? lane : lane & 15) * 16, *from_v = from_k + v_rows * RB;
    const uint8_t *from_s = a.kv.scale + ((lane & (C - 1)) * R & 7) * NB + (lane & C ? v_rows * NB : 0);
    const uint32_t to = HD == 128 ? (lane >> 3) * 128 + ((((lane >> 2 & 1) << 2 | (lane & 3)) ^ (lane >> 2 & 6)) << 4)
                                  : (lane >> 3) * 128 + (((lane >> 1 & 3) ^ (lane >> 3 & 1)) << 5) + ((lane & 1) << 4);
    auto issue = [&]() {
        if (more) {
            if (fresh) {
                const int pos = (window * G + lane) * 8;
                const bool ok = page_next >= 0 && page_next < a.kv.num_pages;
                if (!ok) {
                    gone = true;
                    if (a.status) atomicOr(a.status, kDevErrBadIndex);
                }
                const uint32_t off = static_cast<uint32_t>(pos & ((1 << a.kv.page_shift) - 1)) >> 3;
                const uint32_t head = static_cast<uint32_t>(page_next) * 2 * a.kv.kv_heads + l_head;
                group = ok ? (head << (a.kv.page_shift - 3)) + off : 0u;
                fresh = false;
            }
            const uint32_t st = base + stage_in * D::kStage;
            const int g0 = (lb - window) * G;
#pragma unroll
            for (int i = 0; i < PC * RB / 512; ++i) {
                const uint32_t g = __shfl_sync(0xffffffffu, group, g0 + (HD == 128 ? i : 2 * i + (lane >> 4)));
                const uint64_t at = static_cast<uint64_t>(g) * GROUP;
                cp_async16(st + to + i * 512, from_k + at, true);
                cp_async16(st + D::kTile + to + i * 512, from_v + at, true);
            }
            const uint32_t g = __shfl_sync(0xffffffffu, group, g0 + (lane & (C - 1)) * R / 8);
            if (lane < 2 * C) cp_async16(st + 2 * D::kTile + lane * 16, from_s + static_cast<uint64_t>(g) * (8 * NB), true);
            if (++lb == l_end) {
                load_run();
                if (more) peek();
            } else if (lb == window + 32 / G) {
                peek();
            }
        }
        cp_async_commit();
        stage_in = stage_in + 1 == D::kStages ? 0 : stage_in + 1;
    };
    for (int i = 0; i < D::kStages - 1; ++i) issue();

    // ---- the computing side
    // a lane's places in a stage: K rows gid (+ 8), V rows 2 t4 + j (+ 8), their scale bytes
    const uint32_t k_at = HD == 128 ? (gid >> 1) * 128 + ((((gid & 1) << 2 | t4) ^ (gid & 6)) << 4)
                                    : (gid >> 2) * 128 + (((gid & 3) ^ (gid >> 2)) << 5) + t4 * 8;
    uint32_t v_at[2];
#pragma unroll
    for (int j = 0; j < 2; ++j)
        v_at[j] = D::kTile + (HD == 128 ? t4 * 128 + (((j << 2 | gid >> 1) ^ 2 * t4) << 4) + (gid & 1) * 8
                                        : (t4 >> 1) * 128 + (((2 * (t4 & 1) + j) ^ (t4 >> 1)) << 5) + gid * 4);
    constexpr int ROW8 = 8 * RB;  // bytes of 8 rows in a stage too
    const uint32_t ks_at = 2 * D::kTile + gid * NB + t4 * NB / 4, vs_at = 2 * D::kTile + D::kScales + 2 * t4 * NB + gid * NB / 8;
    const float sc = a.scale_log2, raise = fminf(8.f / sc, 3e38f);
    int stage = 0;
    bool bad = false;
    // (the last chunk of a run has been loaded, and the next run been queued, before it is computed)
    for (int run = 0, queue_out = 0; run < queued; ++run, queue_out = queue_out + 1 == QUEUE ? 0 : queue_out + 1) {
        Segment s = my.run[queue_out];  // (read again behind the run, not held)
        const int kv = s.x.kv, b1 = s.b1;
        const int row0 = s.ti * kDecRows, rows = min(kDecRows, s.x.rows - row0);
        uint32_t qh[KS][N][2], ql[SPLIT ? KS : 1][N][2];
        int limit[N][2];  // last position that rows 8 n + 2 t4 + c see
#pragma unroll
        for (int n = 0; n < N; ++n) {
            if constexpr (PAIR) {
                // a row at a time (or two), 4 dims a lane, into the stage that is loaded next, and from there as the
                // products want them: 12 warps that read 16 bytes of each of 32 lines at once took 4800 cycles for
                // this at head_dim 128, 2100 so (but not so for more rows: the loop came out slower)
                constexpr int L = HD / 4, STEP = 32 / L, SQ = 2 * HD + 8;  // SQ: bytes of a part of a row
                const uint32_t qs = base + stage_in * D::kStage;
                float4 v[4 / STEP];
#pragma unroll
                for (int i = 0; i < 4 / STEP; ++i) {
                    const int r = i * STEP + lane / L;
                    const int tok = r < rows ? (row0 + r) / a.group : 0, in = r < rows ? (row0 + r) % a.group : 0;
                    const T *src = qp + static_cast<long>(s.x.q0 + tok) * a.q_stride +
                                   (s.head * a.group + in) * HD + lane % L * 4;
                    v[i] = r < rows ? load4(src, qvec) : make_float4(0.f, 0.f, 0.f, 0.f);
                }
#pragma unroll
                for (int i = 0; i < 4 / STEP; ++i) {
                    const uint32_t at = qs + (i * STEP + lane / L) * SQ + lane % L * 8, h0 = half2_bits(v[i].x, v[i].y),
                                   h1 = half2_bits(v[i].z, v[i].w);
                    const float2 f0 = __half22float2(*reinterpret_cast<const __half2 *>(&h0)),
                                 f1 = __half22float2(*reinterpret_cast<const __half2 *>(&h1));
                    sts64(at, h0, h1);
                    sts64(at + 4 * SQ, half2_bits(v[i].x - f0.x, v[i].y - f0.y), half2_bits(v[i].z - f1.x, v[i].w - f1.y));
                }
                __syncwarp();
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    const uint2 x = lds64(qs + gid * SQ + t4 * (HD / 2) + 8 * ks);  // (rows 4..7: lo parts)
                    qh[ks][n][0] = x.x;
                    qh[ks][n][1] = x.y;
                }
                __syncwarp();
                static_assert(8 * SQ <= D::kStage, "the queries fit a stage");
            } else {
                const int r = gid + 8 * n;
                const int tok = r < rows ? (row0 + r) / a.group : 0, in = r < rows ? (row0 + r) % a.group : 0;
                const T *src = qp + static_cast<long>(s.x.q0 + tok) * a.q_stride + (s.head * a.group + in) * HD + t4 * (HD / 4);
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    const float4 v = r < rows ? load4(src + 4 * ks, qvec) : make_float4(0.f, 0.f, 0.f, 0.f);
                    const __half2 h0 = __floats2half2_rn(v.x, v.y), h1 = __floats2half2_rn(v.z, v.w);
                    qh[ks][n][0] = *reinterpret_cast<const uint32_t *>(&h0);
                    qh[ks][n][1] = *reinterpret_cast<const uint32_t *>(&h1);
                    if constexpr (SPLIT) {
                        const float2 f0 = __half22float2(h0), f1 = __half22float2(h1);
                        ql[ks][n][0] = half2_bits(v.x - f0.x, v.y - f0.y);
                        ql[ks][n][1] = half2_bits(v.z - f1.x, v.w - f1.y);
                    }
                }
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int q = PAIR ? (2 * t4 + c) & 3 : 8 * n + 2 * t4 + c;
                limit[n][c] = q < rows ? s.x.kv - s.x.len + (row0 + q) / a.group : -1;
            }
        }
        // m: the maximum (of raw scores) that weights are relative to, mu the same times sc; l: this lane's positions' sum
        float m[N][2], mu[N][2], l[N][2], o[4 * W][N][4];
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                m[n][c] = -INFINITY;
                mu[n][c] = l[n][c] = 0.f;
            }
#pragma unroll
        for (int i = 0; i < 4 * W; ++i)
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int k = 0; k < 4; ++k) o[i][n][k] = 0.f;
        const int all_see = s.x.kv - s.x.len + row0 / a.group;  // positions up to here are seen by every row

        for (int b = s.b0; b < b1; ++b) {
            issue();  // into the stage used last
            cp_async_wait<D::kStages - 1>();
            __syncwarp();
            const uint32_t st = base + stage * D::kStage;
            const int p0 = b * PC;
            if (p0 + PC > kv) {  // what V's scales behind the last position hold means nothing: zeros
                for (int r = lane; r < PC; r += 32)
                    if (p0 + r >= kv)
#pragma unroll
                        for (int i = 0; i < NB / 2; ++i)
                            asm volatile("st.shared.u16 [%0], %1;" ::"r"(st + 2 * D::kTile + D::kScales + r * NB + 2 * i),
                                         "h"(static_cast<uint16_t>(0))
                                         : "memory");
                __syncwarp();
            }
            // ---- scores: tile t, row gid (+ 8) is position 16 t + gid (+ 8)
            float p[TT][N][4];
#pragma unroll
            for (int t = 0; t < TT; ++t) {
#pragma unroll
                for (int n = 0; n < N; ++n)
#pragma unroll
                    for (int k = 0; k < 4; ++k) p[t][n][k] = 0.f;
                uint32_t u[2][HD / 32], ks2[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t at = st + k_at + (2 * t + h) * ROW8;
                    if constexpr (HD == 128) {
                        const uint4 w = lds128(at);
                        u[h][0] = w.x; u[h][1] = w.y; u[h][2] = w.z; u[h][3] = w.w;
                    } else {
                        const uint2 w = lds64(at);
                        u[h][0] = w.x; u[h][1] = w.y;
                    }
                    ks2[h] = lds8(st + ks_at + (16 * t + 8 * h) * NB) * 0x00800080u;
                }
#pragma unroll
                for (int e = 0; e < HD / 32; ++e) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        uint32_t f[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) f[j] = hmul2(e2m1x2_half2(u[j & 1][e], 2 * i + (j >> 1)), ks2[j & 1]);
                        const int ks = 2 * e + i;
#pragma unroll
                        for (int n = 0; n < N; ++n) {
                            if constexpr (SPLIT) mma(p[t][n], f, ql[ks][n][0], ql[ks][n][1]);
                            mma(p[t][n], f, qh[ks][n][0], qh[ks][n][1]);
                        }
                    }
                }
            }
            if constexpr (PAIR) {
#pragma unroll
                for (int t = 0; t < TT; ++t)
#pragma unroll
                    for (int k = 0; k < 4; ++k) p[t][0][k] += __shfl_xor_sync(0xffffffffu, p[t][0][k], 2);
            }
            // ---- online softmax (base 2)
            if (p0 + PC - 1 > all_see) {
#pragma unroll
                for (int t = 0; t < TT; ++t)
#pragma unroll
                    for (int n = 0; n < N; ++n)
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (p0 + 16 * t + gid + 4 * (k & 2) > limit[n][k & 1]) p[t][n][k] = -INFINITY;
            }
            float mx[N][2];
            bool need = false;
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    mx[n][c] = fmaxf(p[0][n][c], p[0][n][c + 2]);
#pragma unroll
                    for (int t = 1; t < TT; ++t) mx[n][c] = fmaxf(mx[n][c], fmaxf(p[t][n][c], p[t][n][c + 2]));
                    need = need || mx[n][c] > m[n][c] + raise;
                }
            if (__any_sync(0xffffffffu, need)) {
#pragma unroll
                for (int n = 0; n < N; ++n)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        float x = fmaxf(m[n][c], mx[n][c]);
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                        const float f = x == -INFINITY ? 1.f : ex2((m[n][c] - x) * sc);
                        m[n][c] = x;
                        mu[n][c] = x == -INFINITY ? 0.f : x * sc;
                        l[n][c] *= f;
#pragma unroll
                        for (int i = 0; i < 4 * W; ++i) {
                            o[i][n][c] *= f;
                            o[i][n][c + 2] *= f;
                        }
                    }
            }
            // weights as the second product's B: k slots 2 t4, 2 t4 + 1 (+ 8) of tile t, column gid
            uint32_t ph[TT][N][2], pl[SPLIT ? TT : 1][N][2];
#pragma unroll
            for (int t = 0; t < TT; ++t)
#pragma unroll
                for (int n = 0; n < N; ++n)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float e[2];
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            e[c] = ex2(fmaf(p[t][n][2 * h + c], sc, -mu[n][c]));
                            l[n][c] += e[c];
                        }
                        __half2 w = __floats2half2_rn(e[0], e[1]);
                        if constexpr (PAIR) {
                            const float2 f = __half22float2(w);
                            const __half2 lo = __floats2half2_rn(e[0] - f.x, e[1] - f.y);
                            w = t4 & 2 ? lo : w;
                        }
                        ph[t][n][h] = transpose8x8(*reinterpret_cast<const uint32_t *>(&w));
                        if constexpr (SPLIT) {
                            const float2 f = __half22float2(w);
                            pl[t][n][h] = transpose8x8(half2_bits(e[0] - f.x, e[1] - f.y));
                        }
                    }
            // ---- values, 32 positions at a time: tile 4 k + j, rows gid and gid + 8, are the lane's dims 8 k + 2 j and
            // 8 k + 2 j + 1
#pragma unroll
            for (int t0 = 0; t0 < TT; t0 += 2) {
                uint32_t w[2][2][2][W], vs2[2][2];  // [tile][+ 8][j]
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const uint32_t at = st + v_at[j] + (2 * (t0 + t) + h) * ROW8;
                            if constexpr (HD == 128) {
                                const uint2 x = lds64(at);
                                w[t][h][j][0] = x.x; w[t][h][j][1] = x.y;
                            } else {
                                w[t][h][j][0] = lds32(at);
                            }
                        }
                        const uint32_t at = st + vs_at + (16 * (t0 + t) + 8 * h) * NB;
                        vs2[t][h] = lds8(at) * 0x80u + lds8(at + NB) * 0x800000u;
                    }
                constexpr uint32_t LOW = 0x0f0f0f0fu;
#pragma unroll
                for (int k = 0; k < W; ++k) {
                    uint32_t x[2][2][2];  // [tile][+ 8][odd dims]: bytes of codes of positions 2 t4, 2 t4 + 1
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            x[t][h][0] = select_bits(w[t][h][0][k], w[t][h][1][k] << 4, LOW);
                            x[t][h][1] = select_bits(w[t][h][0][k] >> 4, w[t][h][1][k], LOW);
                        }
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        uint32_t f[2][4];
#pragma unroll
                        for (int t = 0; t < 2; ++t)
#pragma unroll
                            for (int i = 0; i < 4; ++i) f[t][i] = hmul2(e2m1x2_half2(x[t][i >> 1][i & 1], j), vs2[t][i >> 1]);
#pragma unroll
                        for (int n = 0; n < N; ++n) {
                            float(&to_o)[4] = o[4 * k + j][n];
                            if constexpr (PAIR) {
                                float d[4];
                                mma_new(d, f[0], ph[t0][n][0], ph[t0][n][1]);
                                mma(d, f[1], ph[t0 + 1][n][0], ph[t0 + 1][n][1]);
                                add2_in_order(to_o[0], to_o[1], d[0], d[1]);
                                add2_in_order(to_o[2], to_o[3], d[2], d[3]);
                            } else if constexpr (SPLIT) {
                                float d[4];
                                mma_new(d, f[0], pl[t0][n][0], pl[t0][n][1]);
                                mma(d, f[1], pl[t0 + 1][n][0], pl[t0 + 1][n][1]);
                                mma(d, f[0], ph[t0][n][0], ph[t0][n][1]);
                                mma(d, f[1], ph[t0 + 1][n][0], ph[t0 + 1][n][1]);
                                add2_in_order(to_o[0], to_o[1], d[0], d[1]);
                                add2_in_order(to_o[2], to_o[3], d[2], d[3]);
                            } else {
                                mma(to_o, f[0], ph[t0][n][0], ph[t0][n][1]);
                                mma(to_o, f[1], ph[t0 + 1][n][0], ph[t0 + 1][n][1]);
                            }
                        }
                    }
                }
            }
            __syncwarp();  // every lane is done with this stage
            stage = stage + 1 == D::kStages ? 0 : stage + 1;
        }

        if constexpr (PAIR) {
#pragma unroll
            for (int i = 0; i < 4 * W; ++i)
#pragma unroll
                for (int k = 0; k < 4; ++k) o[i][0][k] += __shfl_xor_sync(0xffffffffu, o[i][0][k], 2);
        }
        float zero = 0.f;  // NaN once a value is not finite
#pragma unroll
        for (int i = 0; i < 4 * W; ++i)
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int k = 0; k < 4; ++k) zero = fmaf(o[i][n][k], 0.f, zero);
        bad |= !(zero == 0.f);
        // ---- the run's end: the output, or its state
        s = my.run[queue_out];
        const int end_row0 = s.ti * kDecRows, end_rows = min(kDecRows, s.x.rows - end_row0);
        if (!CLUSTER && lane == 0) {
            const Left left = left_of(a, s, worker, per);
            int *to_left = &a.left[worker].states;
            *reinterpret_cast<int4 *>(to_left) = make_int4(left.states, left.q0, left.row0, left.rows);
            to_left[4] = left.head;
        }
        const bool whole = s.b0 == 0 && s.b1 == s.units;
        float *part = a.part + part_slot(s, worker) * part_floats<kDecRows, HD>();
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float sum = l[n][c];
                sum += __shfl_xor_sync(0xffffffffu, sum, 4);
                sum += __shfl_xor_sync(0xffffffffu, sum, 8);
                sum += __shfl_xor_sync(0xffffffffu, sum, 16);
                const int r = 8 * n + 2 * t4 + c;
                if (r >= end_rows || (PAIR && r >= 4)) continue;
                const float inv = whole ? (sum > 0.f || sum != sum ? 1.f / sum : 0.f) : 1.f;
                T *dst = op + static_cast<long>(s.x.q0 + (end_row0 + r) / a.group) * a.out_stride +
                         (s.head * a.group + (end_row0 + r) % a.group) * HD + gid * (HD / 8);
                float *pd = part + r * HD + gid * (HD / 8);
                if (!whole && gid == 0) {
                    part[kDecRows * HD + r] = m[n][c] == -INFINITY ? m[n][c] : mu[n][c];
                    part[kDecRows * HD + kDecRows + r] = sum;
                }
#pragma unroll
                for (int i = 0; i < 4 * W; i += 2) {
                    const float x[4] = {o[i][n][c], o[i][n][c + 2], o[i + 1][n][c], o[i + 1][n][c + 2]};
                    if (whole) store4(dst + 2 * i, ovec, x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
                    else store4(pd + 2 * i, x[0], x[1], x[2], x[3]);
                }
            }
    }
    cp_async_wait<0>();
    const int how = (__any_sync(0xffffffffu, bad) ? 1 : 0) | (__any_sync(0xffffffffu, gone) ? 2 : 0);
    if (lane == 0) a.left[worker].bad = how;
    if constexpr (CLUSTER) {
        // the states are in the workspace: the cluster's CTAs join them, a row each
        __shared__ float top[1], total[1];
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        const int w0 = tile * size * D::kWarps, states = (units + per - 1) / per;
        Left left = {};
        left.states = states;
        left.q0 = entry.q0;
        left.rows = entry.rows;
        left.head = first.head;
        float4 *shared = reinterpret_cast<float4 *>(smem);  // the stages are idle
        static_assert(NT * sizeof(float4) <= D::kSmem, "a value a thread");
        for (int row0 = rank; row0 < entry.rows; row0 += size) {
            const int bad0 = a.left[w0].bad;
            int again = (bad0 ? 1 : 0) | (bad0 & 2);
            if (states > 1) again |= merge_block<kDecRows, HD, NT, 1, T>(a, left, w0, row0, top, total, shared);
            if (again) mend_rows<kDecRows, HD, NT, 1, IJB_KV_E2M1, T>(a, w0, row0, again & 2, shared);
            __syncthreads();
        }
    }
}

// ------------------------------------------------------------------ tile --
//
// 256 rows (two tiles of 128, one softmax warpgroup each) against blocks of
// 128 positions, one CTA per SM:
//   * warps 8..11 bring K and V blocks into a ring of shared-memory buffers, in
//     the tensor cores' 128-byte-swizzled layout, as fp16 (e4m3 rows are
//     converted on the way; rows behind the last position are zeros);
//   * warps 12 and 13, one a tile: S = Q K^T (K-major, from shared memory) and O += P V
//     (P from TMEM, V as it lies: MN-major) with tcgen05.mma, M = 128, sums in
//     TMEM; while one tile's softmax runs, the other's products do;
//   * warps 0..3 and 4..7: one thread a row: maximum, exponentials and sum of
//     its 128 scores, P written over S as fp16 (fp32 queries: hi and lo parts
//     side by side); at the end of a run the output or its state.
// The maximum is raised, and O rescaled, only when a row's scores pass it by
// more than 2^8: until then the weights are relative to an older maximum, at
// most 256, which fp16 and the fp32 sums hold as exactly.  TMEM: S of both
// tiles in columns 0..255, O in 256..511.
//
// The tensor cores' fp32 additions drop the bits that do not fit: each loses half
// a unit of the last place of the sum so far, always towards zero, 4e-8 of O a
// product step.  Over 23000 positions that was 1.5e-5 of an output, too much for
// fp32 queries; so with those O is started anew every few blocks (kFlush) and
// what it held is added, rounded to nearest, to sums kept in TMEM (head_dim 64,
// where half of O's columns are free) or in the workspace (128).
//
// What bounds it: the waits between a tile's products and its softmax.  A block of both
// tiles has 2048 clocks of products at head_dim 128 (1024 at 64; twice that for fp32 queries)
// and 1536 of exponentials (16 a clock and SM, a quarter of them on the FMA pipes; 2048 for fp32
// queries, which leave none to those); the one tile's fill the other's waits but in part, and a
// block takes 3300 to 3600.  Measured in a graph, 32 heads of 128 over 8 KV heads: 512 tokens behind
// 32011 in an e4m3 cache 322 us with fp16 queries (840 TFLOP/s; tensor pipe 40 % and exponential
// unit 32 % busy) and 635 with fp32 ones, a prompt of 8192 641 and 1298.

constexpr int kTileRows = 256, kBlock = 128;
constexpr int kTileThreads = 16 * 32, kMmaWarpId = 12, kLoadWarp0 = 8;
// Registers a thread of each warpgroup; the sum is what the launch gives them:
// 2 * 168 + 112 + 64 = 4 * 128.
constexpr int kSoftmaxRegs = 168, kLoadRegs = 112, kMmaRegs = 64;
static_assert(2 * kSoftmaxRegs + kLoadRegs + kMmaRegs <= 4 * 128, "register shares");

template <int HD, typename T>
struct Tile {
    static constexpr bool kSplit = sizeof(T) == 4;
    static constexpr int kHalf = kBlock * 128;                 // 128 rows x 64 fp16
    static constexpr int kPart = kHalf * (HD / 64);            // a 128-row operand tile
    static constexpr int kQ = 2 * kPart * (kSplit ? 2 : 1);    // both tiles, hi (and lo)
    static constexpr int kFit = (227 * 1024 - 2048 - kQ) / kPart;
    static constexpr int kBufs = kFit > 8 ? 8 : kFit;
    static constexpr int kSmem = kQ + kBufs * kPart + 1024 + 512;
    // blocks that O sums up before they are added to the sums outside
    static constexpr int kFlush = kSplit ? 2 : 0;
    static_assert(kBufs >= 3, "a V block and the next K block are in use while another loads");
    static_assert(kBufs * kPart >= (kMaxEntries + kMaxTiles + 2) * 4, "the plan lies over the buffers");
};

struct TileCtl {
    uint64_t full[8], empty[8], q_full[2], s_full[2], p_half[2], p_full[2], o_full[2];
    uint32_t tmem;
    uint32_t abort;
    uint32_t bad;   // a value of the output is not finite
    uint32_t gone;  // a page was none (see the decode kernel)
};

__device__ __forceinline__ bool try_bar(uint64_t *bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}
// mbar_wait_bounded without its call: a call does not go with warps of
// different register shares.
__device__ __forceinline__ void wait_bar(const AttnArgs &a, TileCtl *ctl, uint64_t *bar, uint32_t parity) {
    if (try_bar(bar, parity)) return;
    volatile uint32_t *abort = &ctl->abort;
    uint64_t start = 0;
#pragma unroll 1
    for (uint32_t n = 1; !try_bar(bar, parity); ++n) {
        if ((n & 255u) != 0) continue;
        if (*abort) return;
        const uint64_t now = global_timer_ns();
        if (start == 0) {
            start = now;
        } else if (now - start > kWaitLimitNs) {
            *abort = 1u;
            if (a.status) atomicOr(a.status, kDevErrWaitTimeout);
            return;
        }
    }
}
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// Shared-memory operand, 128-byte swizzle: 8-row groups 1024 bytes apart;
// `lbo`: bytes between 64-element column blocks of an MN-major operand.
__device__ __forceinline__ uint64_t desc128(uint32_t addr, uint32_t lbo) {
    return static_cast<uint64_t>((addr & 0x3FFFFu) >> 4) | static_cast<uint64_t>((lbo >> 4) & 0x3FFFu) << 16 |
           static_cast<uint64_t>(1024u >> 4) << 32 | 1ull << 46 | 2ull << 61;
}
__device__ __forceinline__ bool elect_one() {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\tselp.u32 %0, 1, 0, e;\n\t}" : "=r"(ok));
    return ok != 0;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}
// 32 columns of this warp's TMEM lanes, one row a thread; tm_wait completes it.
__device__ __forceinline__ void tm_ld32(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
__device__ __forceinline__ void tm_wait(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                   "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                   "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                   "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void tm_st32(uint32_t addr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
        "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
        "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(addr)
        : "memory");
}
__device__ __forceinline__ void tm_st16(uint32_t addr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15};" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(addr)
        : "memory");
}
__device__ __forceinline__ void tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void sts128(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// Byte offset of 16-byte piece c (8 fp16) of row r in a 128-row operand tile.
__device__ __forceinline__ uint32_t tile_off(int r, int c) {
    return static_cast<uint32_t>((c >> 3) * (kBlock * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

// The positions of a 128-position block that one of the 128 loading threads
// copies: LANES 16-byte pieces of a row side by side (an e4m3 row's four then
// fall on different banks than the next row's once they are fp16), HALVES times.
// Page ids are read a block ahead, for their latency.
template <int HD, int KV>
struct Rows {
    static constexpr bool E4M3 = KV == IJB_KV_E4M3, E2M1 = KV == IJB_KV_E2M1;
    static constexpr int LANES = E2M1 ? HD / 32 : (E4M3 ? 4 : 8), HALVES = E2M1 ? 1 : HD / 64;
    static constexpr int RS = 128 / LANES, N = 128 / RS;  // rows a step, rows of a thread
    static constexpr int RB = kv_row_bytes(KV, HD);
    int next[N];   // page ids of the block after this one
    long row[N];   // cache rows (K)
    int live;      // bit k: row k's position exists, and its page
    Segment s;
    int b;
    bool more;
    __device__ __forceinline__ void peek(const AttnArgs &a, int pr) {
        if (!more) return;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int pos = b * kBlock + k * RS + pr;
            next[k] = pos < s.x.kv ? a.kv.page_table[static_cast<long>(s.x.seq) * a.kv.max_pages + (pos >> a.kv.page_shift)] : -1;
        }
    }
    __device__ __forceinline__ void start(const AttnArgs &a, Cursor &c, int pr) {
        more = cursor_next(a, c, s);
        b = s.b0;
        peek(a, pr);
    }
    // Makes the peeked block the current one and peeks the next; false at the end.
    __device__ __forceinline__ bool step(const AttnArgs &a, Cursor &c, int pr, TileCtl *ctl) {
        if (!more) return false;
        live = 0;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int pos = b * kBlock + k * RS + pr;
            const bool in = pos < s.x.kv, ok = next[k] >= 0 && next[k] < a.kv.num_pages;
            if (in && !ok) {
                ctl->gone = 1u;
                if (a.status) atomicOr(a.status, kDevErrBadIndex);
            }
            live |= in && ok ? 1 << k : 0;
            row[k] = in && ok ? kv_row(a.kv, next[k], 0, s.head, pos & ((1 << a.kv.page_shift) - 1)) : 0;
        }
        if (++b == s.b1) {
            more = cursor_next(a, c, s);
            b = s.b0;
        }
        peek(a, pr);
        return true;
    }
};

// Loads the K and V blocks of a worker's runs (128 threads, p of them).
template <int HD, int KV, int BUFS>
__device__ void tile_load(const AttnArgs &a, Cursor c, uint32_t bufs, int part, TileCtl *ctl, int p) {
    using R = Rows<HD, KV>;
    constexpr int STEPS = R::N * R::HALVES, RB = R::RB;
    const int pc = p % R::LANES, pr = p / R::LANES;
    const long v_off = static_cast<long>(a.kv.kv_heads) << a.kv.page_shift;
    R rows;
    rows.start(a, c, pr);
    auto wait_empty = [&](int i) {
        if (i >= BUFS) wait_bar(a, ctl, &ctl->empty[i % BUFS], (i / BUFS - 1) & 1);
    };
    int i = 0;  // buffers filled so far
    if constexpr (R::E4M3 || R::E2M1) {
        uint4 wk[STEPS], wv[STEPS];
        uint32_t sk[R::N], sv[R::N];
        auto load = [&](uint4(&w)[STEPS], uint32_t(&sc)[R::N], long off) {
#pragma unroll
            for (int k = 0; k < STEPS; ++k) {
                const int j = k / R::HALVES, h = k % R::HALVES;
                const bool in = (rows.live >> j) & 1;
                const long r = rows.row[j] + off;
                w[k] = in ? *reinterpret_cast<const uint4 *>(a.kv.data + r * RB + (pc + h * R::LANES) * 16)
                          : make_uint4(0, 0, 0, 0);
                if constexpr (R::E2M1) sc[j] = in ? a.kv.scale[r * R::LANES + pc] : 0u;  // a piece is a block of 32
                else if (h == 0) sc[j] = in ? a.kv.scale[r] : 127u;
            }
        };
        auto store = [&](const uint4(&w)[STEPS], const uint32_t(&sc)[R::N]) {
            wait_empty(i);
            const uint32_t dst = bufs + (i % BUFS) * part;
            if constexpr (R::E2M1) {
#pragma unroll
                for (int k = 0; k < STEPS; ++k) {
                    const uint32_t u[4] = {w[k].x, w[k].y, w[k].z, w[k].w}, sb = sc[k] * 0x00800080u;
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        uint32_t h[4];
                        e2m1x8_half2(u[n], h);
                        sts128(dst + tile_off(k * R::RS + pr, 4 * pc + n), hmul2(h[0], sb), hmul2(h[1], sb), hmul2(h[2], sb),
                               hmul2(h[3], sb));
                    }
                }
                proxy_fence();
                mbar_arrive(&ctl->full[i % BUFS]);
                ++i;
                return;
            }
            [[maybe_unused]] auto scaled = [&](auto twice) {
#pragma unroll
                for (int k = 0; k < STEPS; ++k) {
                    const int j = k / R::HALVES, c2 = 2 * (pc + (k % R::HALVES) * R::LANES);
                    const __half2 s2 = __half2half2(twice.value ? scale_half(sc[j]) : __float2half_rn(kv_scale(sc[j])));
                    const uint32_t sb = *reinterpret_cast<const uint32_t *>(&s2);
                    const uint32_t u[4] = {w[k].x, w[k].y, w[k].z, w[k].w};
                    uint32_t h[8];
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        h[2 * n] = hmul2(e4m3x2_half2(u[n] & 0xffffu), sb);
                        h[2 * n + 1] = hmul2(e4m3x2_half2(u[n] >> 16), sb);
                    }
                    if constexpr (twice.value) {
                        const __half2 rest = __float2half2_rn(scale_rest(sc[j]));
#pragma unroll
                        for (int n = 0; n < 8; ++n) h[n] = hmul2(h[n], *reinterpret_cast<const uint32_t *>(&rest));
                    }
                    const int r = j * R::RS + pr;
                    sts128(dst + tile_off(r, c2), h[0], h[1], h[2], h[3]);
                    sts128(dst + tile_off(r, c2 + 1), h[4], h[5], h[6], h[7]);
                }
            };
            // a loop of its own for the second factor: with a branch a row, or with both factors always,
            // 512 tokens behind 32011 took 404 us in place of 340
            bool far = false;
#pragma unroll
            for (int j = 0; j < R::N; ++j) far |= !scale_fits(sc[j]);
            if (far) scaled(std::true_type{});
            else scaled(std::false_type{});
            proxy_fence();
            mbar_arrive(&ctl->full[i % BUFS]);
            ++i;
        };
        bool more = rows.step(a, c, pr, ctl);
        if (more) load(wk, sk, 0);
        while (more) {
            load(wv, sv, v_off);
            store(wk, sk);
            more = rows.step(a, c, pr, ctl);
            if (more) load(wk, sk, 0);
            store(wv, sv);
        }
    } else {
        // a buffer is handed over once LAG later ones are on their way.  The MMA
        // warp frees a V buffer only when the K buffer behind it is full too, so
        // at most BUFS - 2 may be unannounced.
        constexpr int LAG = BUFS >= 6 ? 3 : (BUFS >= 4 ? 2 : 1);
        while (rows.step(a, c, pr, ctl)) {
#pragma unroll 1
            for (int which = 0; which < 2; ++which, ++i) {
                wait_empty(i);
                const uint32_t dst = bufs + (i % BUFS) * part;
#pragma unroll
                for (int k = 0; k < STEPS; ++k) {
                    const int j = k / R::HALVES, c = pc + (k % R::HALVES) * R::LANES;
                    const bool in = (rows.live >> j) & 1;
                    const long r = in ? rows.row[j] + (which ? v_off : 0) : 0;
                    cp_async16(dst + tile_off(j * R::RS + pr, c), a.kv.data + r * RB + c * 16, in);
                }
                cp_async_commit();
                if (i >= LAG) {
                    cp_async_wait<LAG>();
                    proxy_fence();
                    mbar_arrive(&ctl->full[(i - LAG) % BUFS]);
                }
            }
        }
        cp_async_wait<0>();
        proxy_fence();
        for (int k = max(0, i - LAG); k < i; ++k) mbar_arrive(&ctl->full[k % BUFS]);
    }
}

// Issues tile t's matrix products of a worker's runs (one warp).  A thread gets
// one product in about 130 clocks, whatever its width, and two warps twice as
// many: with one warp for both tiles the products of 128 columns (64 clocks)
// waited for their issue.
template <int HD, bool SPLIT, int BUFS, int FLUSH>
__device__ void tile_mma(const AttnArgs &a, Cursor c, uint32_t q, uint32_t bufs, int part, TileCtl *ctl, uint32_t tmem, int t) {
    constexpr uint32_t kIdS = (1u << 4) | (kBlock / 8) << 17 | (128u / 16) << 24;
    constexpr uint32_t kIdO = (1u << 4) | 1u << 16 | (HD / 8) << 17 | (128u / 16) << 24;  // B is MN-major
    constexpr int kHalf = kBlock * 128;
    q += t * (SPLIT ? 2 : 1) * part;
    const uint32_t ts = tmem + t * 128, to = ts + 256;
    Segment s;
    int i = 0;
    uint32_t runs = 0, blocks = 0;
    auto wait_full = [&](int n) { wait_bar(a, ctl, &ctl->full[n % BUFS], (n / BUFS) & 1); };
    auto score = [&](int n) {  // S = Q K^T, by the elected lane
        const uint64_t qd = desc128(q, 16), kd = desc128(bufs + (n % BUFS) * part, 16);
#pragma unroll
        for (int h = SPLIT ? 1 : 0; h >= 0; --h)  // the small parts first: sums drop bits of their own size
#pragma unroll
            for (int ks = 0; ks < HD / 16; ++ks) {
                const uint32_t off = ((ks >> 2) * kHalf + (ks & 3) * 32) >> 4;
                mma_ss(ts, qd + off + h * (part >> 4), kd + off, kIdS, (SPLIT && h == 0) || ks > 0);
            }
        mma_commit(&ctl->s_full[t]);
    };
    while (cursor_next(a, c, s)) {
        const int n = s.b1 - s.b0;
        if (t == 1 && s.x.rows - s.ti * kTileRows <= 128) {  // no rows here: pass the buffers on
            for (int k = 0; k < 2 * n; ++k, ++i) {
                wait_full(i);
                if (elect_one()) mbar_arrive(&ctl->empty[i % BUFS]);
            }
            continue;
        }
        wait_full(i);
        wait_bar(a, ctl, &ctl->q_full[t], runs++ & 1);
        tc_after();
        if (elect_one()) {
            score(i);
            mma_commit(&ctl->empty[i % BUFS]);
        }
        for (int b = 0; b < n; ++b) {
            const int vi = i + 2 * b + 1, ki = vi + 1;
            wait_full(vi);
            const uint64_t vd = desc128(bufs + (vi % BUFS) * part, kHalf);
            const bool add = FLUSH ? b % (FLUSH ? FLUSH : 1) > 0 : b > 0;  // to what O holds
            auto value = [&](int k0) {  // O += P V over 64 positions
#pragma unroll
                for (int ks = k0; ks < k0 + 4; ++ks) {
                    mma_ts(to, ts + ks * (SPLIT ? 16 : 8), vd + ks * (2048 >> 4), kIdO, add || ks > 0);
                    if constexpr (SPLIT) mma_ts(to, ts + ks * 16 + 8, vd + ks * (2048 >> 4), kIdO, 1);
                }
            };
            wait_bar(a, ctl, &ctl->p_half[t], blocks & 1);
            tc_after();
            if (elect_one()) value(0);
            __syncwarp();
            if (b + 1 < n) wait_full(ki);
            wait_bar(a, ctl, &ctl->p_full[t], blocks++ & 1);
            tc_after();
            if (elect_one()) {
                value(4);
                if (b + 1 < n) score(ki);
                else mma_commit(&ctl->o_full[t]);
                mma_commit(&ctl->empty[vi % BUFS]);
                if (b + 1 < n) mma_commit(&ctl->empty[ki % BUFS]);
            }
        }
        i += 2 * n;
    }
}

__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<uint64_t &>(d))
        : "l"(reinterpret_cast<uint64_t &>(a)), "l"(reinterpret_cast<uint64_t &>(b)), "l"(reinterpret_cast<uint64_t &>(c)));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("add.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<uint64_t &>(d))
        : "l"(reinterpret_cast<uint64_t &>(a)), "l"(reinterpret_cast<uint64_t &>(b)));
    return d;
}

// 2^x of a pair on the FMA pipes, for x <= 8 (see kRaise; below -126: 2^-126 or so): with
// n = round(x) and f = x - n in [-1/2, 1/2], 2^f by a polynomial of degree 4, fitted by least
// squares of the relative error over Chebyshev nodes (off by 1e-5 at most), n added to the
// exponent.  Adding 1.5 * 2^23 rounds x and leaves n in the low bits.
constexpr float kE1 = 0.693121995f, kE2 = 0.240237185f, kE3 = 0.055916894f, kE4 = 0.009600396f;
__device__ __forceinline__ float2 ex2_poly(float2 x) {
    x.x = fmaxf(x.x, -126.f);
    x.y = fmaxf(x.y, -126.f);
    const float2 magic = make_float2(12582912.f, 12582912.f), one = make_float2(1.f, 1.f);
    const float2 k = add2(x, magic);
    const float2 n = add2(k, make_float2(-12582912.f, -12582912.f));
    const float2 f = fma2(n, make_float2(-1.f, -1.f), x);
    float2 p = make_float2(kE4, kE4);
    p = fma2(p, f, make_float2(kE3, kE3));
    p = fma2(p, f, make_float2(kE2, kE2));
    p = fma2(p, f, make_float2(kE1, kE1));
    p = fma2(p, f, one);
    p.x = __int_as_float(__float_as_int(p.x) + (__float_as_int(k.x) << 23));
    p.y = __int_as_float(__float_as_int(p.y) + (__float_as_int(k.y) << 23));
    return p;
}

// The larger, or NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b) {
    float c;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(b));
    return c;
}

// One row's 128 scores (TMEM columns of ts) become its weights there; m and l
// are the row's maximum and sum.  MASK: only columns 0..seen count.
constexpr int kMufuPairs = 6;  // of 8 pairs, on the exponential unit
template <int HD, bool SPLIT, bool MASK>
__device__ __forceinline__ void softmax_block(uint32_t ts, float sc, int seen, uint64_t *half, float &m, float &l) {
    constexpr float kRaise = 8.f;
    uint32_t x[2][32];
    float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    tm_ld32(ts, x[0]);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        tm_wait(x[k & 1]);
        tm_ld32(ts + 32 * ((k + 1) & 3), x[(k + 1) & 1]);  // at the end the first columns again
#pragma unroll
        for (int j = 0; j < 32; ++j) {
            float v = __uint_as_float(x[k & 1][j]);
            if (MASK) v = 32 * k + j <= seen ? v : -INFINITY;
            mx4[j & 3] = max_nan(mx4[j & 3], v);
        }
    }
    float mx = max_nan(max_nan(mx4[0], mx4[1]), max_nan(mx4[2], mx4[3]));
    // a score of NaN or infinity makes the row NaN by its maximum: ex2_poly gives such a pair no weight
    if (!(mx < INFINITY)) m = mx = NAN;
    const bool raise = m != -INFINITY && mx * sc > m * sc + kRaise;
    if (__any_sync(0xffffffffu, raise)) {
        const float alpha = raise ? ex2((m - mx) * sc) : 1.f;
        l *= alpha;
        const uint32_t to = ts + 256;
#pragma unroll 1
        for (int k = 0; k < HD / 32; ++k) {
            uint32_t o[32];
            tm_ld32(to + 32 * k, o);
            tm_wait(o);
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * alpha);
            tm_st32(to + 32 * k, o);
        }
    }
    if (raise || m == -INFINITY) m = mx;
    const float mu = m == -INFINITY ? 0.f : m * sc;
    const float2 sc2 = make_float2(sc, sc), mu2 = make_float2(-mu, -mu);
    float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
    for (int k = 0; k < 4; ++k) {  // two k16 steps of the second product
        tm_wait(x[k & 1]);
        if (k < 3) tm_ld32(ts + 32 * (k + 1), x[(k + 1) & 1]);
        uint32_t w[SPLIT ? 32 : 16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            float2 v = make_float2(__uint_as_float(x[k & 1][2 * j]), __uint_as_float(x[k & 1][2 * j + 1]));
            v = fma2(v, sc2, mu2);
            if (MASK) {
                v.x = 32 * k + 2 * j <= seen ? v.x : -INFINITY;
                v.y = 32 * k + 2 * j + 1 <= seen ? v.y : -INFINITY;
            }
            // some pairs on the FMA pipes, the exponential unit being the busier one
            if (!SPLIT && (j & 7) >= kMufuPairs) {
                v = ex2_poly(v);
            } else {
                v.x = ex2(v.x);
                v.y = ex2(v.y);
            }
            sum[j & 1] = add2(sum[j & 1], v);
            if constexpr (SPLIT) {
                // hi: the weight's first 11 bits, lo: the rest (8 columns each a step)
                const float2 hi = make_float2(__uint_as_float(__float_as_uint(v.x) & 0xffffe000u),
                                              __uint_as_float(__float_as_uint(v.y) & 0xffffe000u));
                const int at = (j >> 3) * 16 + (j & 7);
                w[at] = half2_bits(hi.x, hi.y);
                w[at + 8] = half2_bits(v.x - hi.x, v.y - hi.y);
            } else {
                w[j] = half2_bits(v.x, v.y);
            }
        }
        if constexpr (SPLIT) tm_st32(ts + 32 * k, w);
        else tm_st16(ts + 16 * k, w);
        if (k == 1) {  // the second product may start on the first 64 positions
            tm_wait_st();
            tc_before();
            mbar_arrive(half);
        }
    }
    l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
}

// Writes a warp's 32 rows of O (TMEM columns of `to`, one row a lane), times
// inv, at dst + to_row (each lane its own row's), the first `rows` of them.
// False if one of the lane's own row's values is not finite.
template <int HD, typename O>
__device__ __forceinline__ bool write_rows(uint32_t to, uint32_t st, O *dst, bool vec, long to_row, int rows, float inv,
                                           int lane) {
    float zero = 0.f;
    constexpr int E = 16 / sizeof(O), D = 8 * E;  // elements of a 16-byte piece, of a pass
#pragma unroll 1
    for (int d0 = 0; d0 < HD; d0 += D) {
#pragma unroll
        for (int h = 0; h < D / 32; ++h) {
            uint32_t x[32];
            tm_ld32(to + d0 + 32 * h, x);
            tm_wait(x);
#pragma unroll
            for (int c = 0; c < 32; ++c) zero = fmaf(__uint_as_float(x[c]), 0.f, zero);
#pragma unroll
            for (int c = 0; c < 32 / E; ++c) {
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (sizeof(O) == 4)
                        w[i] = __float_as_uint(__uint_as_float(x[4 * c + i]) * inv);
                    else
                        w[i] = half2_bits(__uint_as_float(x[8 * c + 2 * i]) * inv, __uint_as_float(x[8 * c + 2 * i + 1]) * inv);
                }
                sts128(st + lane * 128 + (((h * (32 / E) + c) ^ (lane & 7)) << 4), w[0], w[1], w[2], w[3]);
            }
        }
        __syncwarp();
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int r = 4 * k + (lane >> 3), c = lane & 7;
            O *p = dst + __shfl_sync(0xffffffffu, to_row, r) + d0 + c * E;
            const uint4 v = lds128(st + r * 128 + ((c ^ (r & 7)) << 4));
            if (r >= rows) continue;
            if (vec) {
                *reinterpret_cast<uint4 *>(p) = v;
            } else {
                const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int i = 0; i < E; ++i) p[i] = reinterpret_cast<const O *>(u)[i];
            }
        }
        __syncwarp();
    }
    return zero == 0.f;
}

// Adds O (relative to the maximum m) to the row's sums outside it (relative to
// held_m; with `more` they hold something), which become relative to m.  LAST: into
// O, for the output.
template <int HD, bool LAST>
__device__ __forceinline__ void hold(uint32_t to, float *held, bool more, float held_m, float m, float sc) {
    const float f = !more || held_m == -INFINITY ? 0.f : ex2((held_m - m) * sc);
#pragma unroll 1
    for (int k = 0; k < HD / 32; ++k) {
        uint32_t x[32];
        tm_ld32(to + 32 * k, x);
        if constexpr (HD == 64) {
            uint32_t y[32];
            tm_ld32(to + 64 + 32 * k, y);
            tm_wait(y);
            tm_wait(x);
            if (more) {
#pragma unroll
                for (int j = 0; j < 32; ++j)
                    x[j] = __float_as_uint(fmaf(__uint_as_float(y[j]), f, __uint_as_float(x[j])));
            }
            tm_st32(to + (LAST ? 0 : 64) + 32 * k, x);
        } else {
            float4 y[8];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                y[j] = more ? *reinterpret_cast<const float4 *>(held + (k * 8 + j) * 512) : make_float4(0.f, 0.f, 0.f, 0.f);
            tm_wait(x);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                y[j].x = fmaf(y[j].x, f, __uint_as_float(x[4 * j]));
                y[j].y = fmaf(y[j].y, f, __uint_as_float(x[4 * j + 1]));
                y[j].z = fmaf(y[j].z, f, __uint_as_float(x[4 * j + 2]));
                y[j].w = fmaf(y[j].w, f, __uint_as_float(x[4 * j + 3]));
                if constexpr (LAST) {
                    x[4 * j] = __float_as_uint(y[j].x);
                    x[4 * j + 1] = __float_as_uint(y[j].y);
                    x[4 * j + 2] = __float_as_uint(y[j].z);
                    x[4 * j + 3] = __float_as_uint(y[j].w);
                } else {
                    *reinterpret_cast<float4 *>(held + (k * 8 + j) * 512) = y[j];
                }
            }
            if constexpr (LAST) tm_st32(to + 32 * k, x);
        }
    }
    if constexpr (LAST || HD == 64) tm_wait_st();
}

// Softmax and output of tile t of a worker's runs (128 threads, row r of them).
template <int HD, typename T>
__device__ void tile_softmax(const AttnArgs &a, Cursor c, int worker, uint32_t q, int part, TileCtl *ctl, uint32_t tmem, int t,
                             int r) {
    constexpr bool SPLIT = sizeof(T) == 4;
    const int warp = r >> 5, lane = r & 31;
    const uint32_t ts = tmem + t * 128 + (static_cast<uint32_t>(warp * 32) << 16), to = ts + 256;
    const T *qp = static_cast<const T *>(a.q);
    T *op = static_cast<T *>(a.out);
    [[maybe_unused]] const bool qvec = aligned4<T>(a.q, a.q_stride);
    [[maybe_unused]] const bool qvec8 = aligned16(a.q, a.q_stride * sizeof(T));
    const bool ovec = aligned16(a.out, a.out_stride * sizeof(T));
    q += t * (SPLIT ? 2 : 1) * part;
    Segment s;
    int runs = 0, blocks = 0;
    while (cursor_next(a, c, s)) {
        const int row0 = s.ti * kTileRows + t * 128;  // of the entry's rows
        if (row0 >= s.x.rows) continue;
        // ---- queries: a warp its own 32 rows, 8 dims a lane; all loads of a batch in flight
        constexpr int P = HD / 8, RQ = 32 / P, B = SPLIT && P > 8 ? 8 : P;  // lanes a row, rows a step, steps a batch
        int tok, in;  // of the lane's row, going on by RQ rows a step
        {
            const int row = row0 + warp * 32 + lane / P;
            tok = row / a.group;
            in = row % a.group;
        }
        const int tok_step = RQ / a.group, in_step = RQ % a.group;
#pragma unroll 1
        for (int k0 = 0; k0 < P; k0 += B) {
            float4 x[B], y[B];
#pragma unroll
            for (int k = 0; k < B; ++k) {
                const int row = row0 + warp * 32 + (k0 + k) * RQ + lane / P;
                x[k] = y[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (row < s.x.rows) {
                    const T *src = qp + static_cast<long>(s.x.q0 + tok) * a.q_stride + (s.head * a.group + in) * HD +
                                   (lane % P) * 8;
                    if constexpr (SPLIT) {
                        x[k] = load4(src, qvec);
                        y[k] = load4(src + 4, qvec);
                    } else {
                        x[k] = load8_raw(src, qvec8);
                    }
                }
                tok += tok_step;
                in += in_step;
                if (in >= a.group) {
                    in -= a.group;
                    ++tok;
                }
            }
#pragma unroll
            for (int k = 0; k < B; ++k) {
                const uint32_t at = q + tile_off(warp * 32 + (k0 + k) * RQ + lane / P, lane % P);
                if constexpr (SPLIT) {
                    const uint32_t h[4] = {half2_bits(x[k].x, x[k].y), half2_bits(x[k].z, x[k].w),
                                           half2_bits(y[k].x, y[k].y), half2_bits(y[k].z, y[k].w)};
                    const float2 f0 = __half22float2(*reinterpret_cast<const __half2 *>(&h[0])),
                                 f1 = __half22float2(*reinterpret_cast<const __half2 *>(&h[1])),
                                 f2 = __half22float2(*reinterpret_cast<const __half2 *>(&h[2])),
                                 f3 = __half22float2(*reinterpret_cast<const __half2 *>(&h[3]));
                    sts128(at, h[0], h[1], h[2], h[3]);
                    sts128(at + part, half2_bits(x[k].x - f0.x, x[k].y - f0.y), half2_bits(x[k].z - f1.x, x[k].w - f1.y),
                           half2_bits(y[k].x - f2.x, y[k].y - f2.y), half2_bits(y[k].z - f3.x, y[k].w - f3.y));
                } else {
                    sts128(at, __float_as_uint(x[k].x), __float_as_uint(x[k].y), __float_as_uint(x[k].z),
                           __float_as_uint(x[k].w));
                }
            }
        }
        proxy_fence();
        mbar_arrive(&ctl->q_full[t]);

        const int row = row0 + r;
        const bool live = row < s.x.rows;
        const int limit = live ? s.x.kv - s.x.len + row / a.group : -1;  // last position this row sees
        const int all_see = s.x.kv - s.x.len + row0 / a.group;
        float m = -INFINITY, l = 0.f;  // maximum in units of the raw scores
        constexpr int FLUSH = Tile<HD, T>::kFlush;
        [[maybe_unused]] float held_m = -INFINITY;  // the maximum that the sums outside O go by
        [[maybe_unused]] float *held = a.held + ((blockIdx.x * 2 + t) * static_cast<long>(HD / 4) * 128 + r) * 4;
        for (int b = s.b0; b < s.b1; ++b) {
            wait_bar(a, ctl, &ctl->s_full[t], blocks++ & 1);
            tc_after();
            if constexpr (FLUSH > 0) {
                const int n = b - s.b0;
                if (n > 0 && n % FLUSH == 0) {
                    hold<HD, false>(to, held, n > FLUSH, held_m, m, a.scale_log2);
                    held_m = m;
                }
            }
            const int p0 = b * kBlock;
            if (p0 + kBlock - 1 > all_see) softmax_block<HD, SPLIT, true>(ts, a.scale_log2, limit - p0, &ctl->p_half[t], m, l);
            else softmax_block<HD, SPLIT, false>(ts, a.scale_log2, 0, &ctl->p_half[t], m, l);
            tm_wait_st();
            tc_before();
            mbar_arrive(&ctl->p_full[t]);
        }
        const float sc = a.scale_log2;
        // ---- the run's end
        wait_bar(a, ctl, &ctl->o_full[t], runs++ & 1);
        tc_after();
        if constexpr (FLUSH > 0)
            if (s.b1 - s.b0 > FLUSH) hold<HD, true>(to, held, true, held_m, m, a.scale_log2);
        // O goes out by way of the queries' shared memory, idle now (128 bytes a row
        // and pass, 4 KB a warp), so that whole rows are written side by side
        const bool whole = s.b0 == 0 && s.b1 == s.units;
        const float inv = whole ? (l > 0.f || l != l ? 1.f / l : 0.f) : 1.f;
        float *state = a.part + part_slot(s, worker) * part_floats<kTileRows, HD>();
        const long to_row = whole ? static_cast<long>(s.x.q0 + (live ? row / a.group : 0)) * a.out_stride +
                                        (s.head * a.group + (live ? row % a.group : 0)) * HD
                                  : static_cast<long>(t * 128 + r) * HD;
        const int rows = min(32, s.x.rows - (row0 + warp * 32));
        const uint32_t st = q + warp * 4096;
        const bool fine = whole ? write_rows<HD, T>(to, st, op, ovec, to_row, rows, inv, lane)
                                : write_rows<HD, float>(to, st, state, true, to_row, rows, 1.f, lane);
        if (live && !fine) ctl->bad = 1u;
        if (!whole && live) {
            state[kTileRows * HD + t * 128 + r] = m == -INFINITY ? m : m * sc;
            state[kTileRows * HD + kTileRows + t * 128 + r] = l;
        }
        tc_before();  // O has been read before the next run's first product
    }
}

template <int HD, int KV, typename T>
__global__ void __launch_bounds__(kTileThreads, 1) ijb_paged_tile_kernel(const __grid_constant__ AttnArgs a) {
    using L = Tile<HD, T>;
    extern __shared__ uint8_t raw[];
    __shared__ PlanOut po;
    __shared__ TileCtl ctl;
    const uint32_t pad = (1024u - (smem_u32(raw) & 1023u)) & 1023u;  // swizzled tiles start on 1024 bytes
    uint8_t *smem = raw + pad;
    const uint32_t q = smem_u32(smem), bufs = q + L::kQ;
    const int warp = threadIdx.x >> 5;
    int *first = reinterpret_cast<int *>(smem + L::kQ), *sums = first + a.n_entries + 1;
    pdl_trigger();
    plan_build<kTileThreads, false>(a, first, sums, &po);
    const Cursor c = cursor_start<false>(a, first, sums, po, blockIdx.x);
    if (threadIdx.x == 0) {  // the last run of this worker
        Left left = {};
        Cursor w = c;
        Segment s;
        while (cursor_next(a, w, s)) left = left_of(a, s, blockIdx.x, po.per);
        left.runs = c;
        a.left[blockIdx.x] = left;
        ctl.bad = ctl.gone = 0u;
    }
    if (c.at >= c.end) return;
    if (threadIdx.x == 0) {
        for (int i = 0; i < 8; ++i) {
            mbar_init(&ctl.full[i], 128);
            mbar_init(&ctl.empty[i], 2);
        }
        for (int t = 0; t < 2; ++t) {
            mbar_init(&ctl.q_full[t], 128);
            mbar_init(&ctl.s_full[t], 1);
            mbar_init(&ctl.p_half[t], 128);
            mbar_init(&ctl.p_full[t], 128);
            mbar_init(&ctl.o_full[t], 1);
        }
        ctl.abort = 0u;
        fence_barrier_init();
    }
    if (warp == kMmaWarpId) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctl.tmem)), "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_before();
    __syncthreads();  // barriers, TMEM; the plan's shared memory becomes the buffers
    tc_after();
    const uint32_t tmem = ctl.tmem;
    if (warp >= kMmaWarpId) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kMmaRegs));
        if (warp < kMmaWarpId + 2)
            tile_mma<HD, L::kSplit, L::kBufs, L::kFlush>(a, c, q, bufs, L::kPart, &ctl, tmem, warp - kMmaWarpId);
    } else if (warp >= kLoadWarp0) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kLoadRegs));
        tile_load<HD, KV, L::kBufs>(a, c, bufs, L::kPart, &ctl, threadIdx.x - kLoadWarp0 * 32);
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        tile_softmax<HD, T>(a, c, blockIdx.x, q, L::kPart, &ctl, tmem, warp >> 2, threadIdx.x & 127);
    }
    tc_before();
    __syncthreads();
    tc_after();
    if (threadIdx.x == 0) a.left[blockIdx.x].bad = ctl.bad + 2 * ctl.gone;
    if (warp == kMmaWarpId)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

// ----------------------------------------------------------------- merge --

// A weight of 0 times a value that is not finite is NaN, so a NaN or an infinity in
// a later token's V reaches the earlier tokens that share its block.  The kernels
// say when a value came out that way, and the merge then computes the rows of those
// tiles again that do not see all of the positions read, one position at a
// time: RB rows a block, for the tiles that worker w begins.  Where a page id named no
// page (nothing was read for it, and its positions counted as zeros), `all` rows of
// the tiles are computed again, without those positions: a mask for them in the kernels' own
// loops would cost every call.
template <int HD, int KV>
__device__ __forceinline__ float cached(const AttnArgs &a, long row, int d) {
    if constexpr (KV == IJB_KV_E2M1) {
        const uint32_t code = a.kv.data[row * (HD / 2) + (d >> 1)] >> (4 * (d & 1));
        const uint32_t h = e2m1x2_half2(code & 15u), s = a.kv.scale[row * (HD / kKvBlock) + d / kKvBlock] << 7;
        return __low2float(__hmul2(*reinterpret_cast<const __half2 *>(&h), *reinterpret_cast<const __half2 *>(&s)));
    } else if constexpr (KV == IJB_KV_E4M3) {
        const uint32_t h = e4m3x2_half2(a.kv.data[row * HD + d]);
        return __half2float(__float2half_rn(__low2float(*reinterpret_cast<const __half2 *>(&h)) * kv_scale(a.kv.scale[row])));
    } else {
        return __half2float(reinterpret_cast<const __half *>(a.kv.data)[row * HD + d]);
    }
}
template <int ROWS, int HD, int NT, int RB, int KV, typename T>
__device__ __noinline__ void mend_rows(const AttnArgs &a, int w, int row0, bool all, float4 *shared) {
    float *weight = reinterpret_cast<float *>(shared), *red = weight + NT;  // 4 * NT floats are there
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    Cursor c = a.left[w].runs;
    Segment s;
    while (cursor_next(a, c, s)) {
        if (s.b0 > 0) continue;
        const int end = static_cast<int>(min(static_cast<long>(s.x.kv), static_cast<long>(s.units) * a.unit));  // read
        for (int r = s.ti * ROWS + row0; r < min(s.x.rows, min((s.ti + 1) * ROWS, s.ti * ROWS + row0 + RB)); ++r) {
            const int tok = r / a.group, h = s.head * a.group + r % a.group;
            const int n = s.x.kv - s.x.len + tok + 1;  // positions it sees
            if (n >= end && !all) continue;
            const T *q = static_cast<const T *>(a.q) + static_cast<long>(s.x.q0 + tok) * a.q_stride + h * HD;
            T *out = static_cast<T *>(a.out) + static_cast<long>(s.x.q0 + tok) * a.out_stride + h * HD;
            const float now = tid < HD ? static_cast<float>(out[tid]) : 0.f;
            if (__syncthreads_and(now * 0.f == 0.f) && !all) continue;
            auto slot = [&](int t) {
                const long page = page_of(a, s.x.seq, t);
                return page < 0 ? -1L : kv_row(a.kv, page, 0, s.head, t & ((1 << a.kv.page_shift) - 1));
            };
            const long v_off = static_cast<long>(a.kv.kv_heads) << a.kv.page_shift;
            float m = -INFINITY, l = 0.f, o = 0.f;  // o: dim tid
            for (int t0 = 0; t0 < n; t0 += NT) {
                float x = -INFINITY;
                const long row = t0 + tid < n ? slot(t0 + tid) : -1;
                if (row >= 0) {
                    x = 0.f;
                    for (int d = 0; d < HD; ++d) x = fmaf(static_cast<float>(q[d]), cached<HD, KV>(a, row, d), x);
                    x *= a.scale_log2;
                }
                const float mx = warp_max(x);  // a NaN is left to its weight
                __syncthreads();  // the weights of the last positions have been used
                if (lane == 0) red[warp] = mx;
                __syncthreads();
                float to = m;
                for (int i = 0; i < NT / 32; ++i) to = fmaxf(to, red[i]);
                const float mu = to == -INFINITY ? 0.f : to, alpha = ex2(m - mu), p = ex2(x - mu);
                m = to;
                weight[tid] = row >= 0 ? p : 0.f;
                const float add = warp_sum(weight[tid]);
                __syncthreads();
                if (lane == 0) red[warp] = add;
                __syncthreads();
                l *= alpha;
                for (int i = 0; i < NT / 32; ++i) l += red[i];
                o *= alpha;
                if (tid < HD)
                    for (int i = 0; i < min(NT, n - t0); ++i) {
                        const long v = slot(t0 + i);
                        if (v >= 0) o = fmaf(weight[i], cached<HD, KV>(a, v + v_off, tid), o);
                    }
            }
            if (tid < HD) out[tid] = static_cast<T>(o * (l > 0.f || l != l ? 1.f / l : 0.f));
            __syncthreads();
        }
    }
}

// Joins the states of the tiles that EACH workers left (few leave one): RB rows of
// them a block of NT threads.  A thread has 4 dims of a row over some of the states,
// whose values it loads (kMergeBatch at a time) before the row's maximum and sum are
// there.  Bound by the latency of its few rounds of loads, so the decode kernel, which
// may leave hundreds of states of a few rows, spreads them: two contexts of 39,000
// positions, 12 rows of 128 each, took 25, 30, 39 and 80 us in all with 1, 2, 4 and 16
// rows a block, and 64 ragged sequences 27, 25, 25 and 27 us.
constexpr int kMergeBatch = 4;

// Joins the states of one tile (`left`, which worker w0 began): its rows row0 .. row0 + RB. Bit 0: rows to look at again;
// bit 1: all of them (a page was none).
template <int ROWS, int HD, int NT, int RB, typename T>
__device__ __forceinline__ int merge_block(const AttnArgs &a, const Left &left, int w0, int row0, float *top, float *total,
                                           float4 *sum) {
    const int n = left.states, rows = min(RB, left.rows - row0);
    constexpr long PF = part_floats<ROWS, HD>();
    auto part = [&](int i) { return a.part + (2L * (w0 + i) + (i == 0 ? 1 : 0)) * PF; };
    // `bad` of the workers that go on with the tile (the first load is not waited for here)
    int theirs = threadIdx.x < n ? a.left[w0 + threadIdx.x].bad : 0;
    for (int i = threadIdx.x + NT; i < n; i += NT) theirs |= a.left[w0 + i].bad;
    constexpr int Q = HD / 4;  // float4 of a row
    const int outs = rows * Q, groups = outs < NT ? NT / outs : 1;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    T *op = static_cast<T *>(a.out);
    const bool vec = aligned4<T>(a.out, a.out_stride);
    bool fine = true;
    for (int o0 = 0; o0 < outs; o0 += NT) {
        const int g = outs < NT ? threadIdx.x / outs : 0, o = outs < NT ? threadIdx.x % outs : o0 + threadIdx.x;
        const int r = min(o / Q, rows - 1), c = o % Q;
        const bool mine = g < groups && o < outs;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int i0 = g; i0 - g < n; i0 += kMergeBatch * groups) {
            float4 v[kMergeBatch];
            float m[kMergeBatch];
#pragma unroll
            for (int k = 0; k < kMergeBatch; ++k) {
                const int i = i0 + k * groups;
                m[k] = -INFINITY;
                v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (mine && i < n) {
                    const float *p = part(i);
                    m[k] = p[ROWS * HD + row0 + r];
                    v[k] = *reinterpret_cast<const float4 *>(p + (row0 + r) * HD + 4 * c);
                }
            }
            if (o0 == 0 && i0 == g) {  // the rows' maxima and sums, a warp a row
                for (int q = warp; q < rows; q += NT / 32) {
                    float mx = -INFINITY, l = 0.f;
                    for (int i = lane; i < n; i += 32) {
                        const float *p = part(i) + ROWS * HD + row0 + q;
                        const float pm = p[0], pl = p[ROWS], to = fmaxf(mx, pm);
                        if (to != -INFINITY) l = l * ex2(mx - to) + pl * ex2(pm - to);
                        mx = to;
                    }
                    const float all = warp_max(mx), mu = all == -INFINITY ? 0.f : all;
                    l = warp_sum(l * ex2(mx - mu));
                    if (lane == 0) {
                        top[q] = mu;
                        total[q] = l;
                    }
                }
                __syncthreads();
            }
#pragma unroll
            for (int k = 0; k < kMergeBatch; ++k) {
                const float f = ex2(m[k] - top[r]);
                if (f != 0.f) {  // a state without positions may hold no values
                    acc.x = fmaf(f, v[k].x, acc.x);
                    acc.y = fmaf(f, v[k].y, acc.y);
                    acc.z = fmaf(f, v[k].z, acc.z);
                    acc.w = fmaf(f, v[k].w, acc.w);
                }
            }
        }
        __syncthreads();
        sum[threadIdx.x] = acc;
        __syncthreads();
        if (g == 0 && o < outs) {
            for (int k = 1; k < groups; ++k) {
                const float4 v = sum[k * outs + o];
                acc.x += v.x;
                acc.y += v.y;
                acc.z += v.z;
                acc.w += v.w;
            }
            const float l = total[r], inv = l > 0.f || l != l ? 1.f / l : 0.f;
            fine = fine && (acc.x * 0.f + acc.y * 0.f + acc.z * 0.f + acc.w * 0.f) * inv == 0.f;
            const int rr = left.row0 + row0 + r;
            store4(op + static_cast<long>(left.q0 + rr / a.group) * a.out_stride +
                       (left.head * a.group + rr % a.group) * HD + 4 * c,
                   vec, acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
        }
    }
    // (also: the shared sums have been read)
    if (!__syncthreads_or(!fine || (theirs & 2))) return 0;
    return __syncthreads_or(theirs & 2) ? 3 : 1;
}

// One tile's rows row0 .. row0 + RB (of `left`'s, which worker w0 began) by a warp, where they have up to kFewStates
// states: a lane has a state's maximum and sum, then HD / 32 dims over all of them.  Bit 0: a value is not finite;
// bit 1: a page was none.
constexpr int kFewStates = 8;
template <int ROWS, int HD, int RB, typename T>
__device__ __forceinline__ int merge_few(const AttnArgs &a, const Left &left, int w0, int row0) {
    constexpr int E = HD / 32;
    constexpr long PF = part_floats<ROWS, HD>();
    const int lane = threadIdx.x & 31, n = left.states, rows = min(RB, left.rows - row0);
    const float *mine = a.part + (2L * (w0 + lane) + (lane == 0 ? 1 : 0)) * PF;  // lane's state, for lane < n
    const int theirs = lane < n ? a.left[w0 + lane].bad : 0;
    T *op = static_cast<T *>(a.out);
    const bool vec = reinterpret_cast<uintptr_t>(op) % (E * sizeof(T)) == 0 && a.out_stride % E == 0;
    bool fine = true;
#pragma unroll
    for (int r = 0; r < RB; ++r) {
        if (r >= rows) break;
        float v[kFewStates][E];
#pragma unroll
        for (int i = 0; i < kFewStates; ++i) {
            const float *p = a.part + (2L * (w0 + i) + (i == 0 ? 1 : 0)) * PF + (row0 + r) * HD + lane * E;
#pragma unroll
            for (int e = 0; e < E; e += 2) {
                const float2 x = i < n ? *reinterpret_cast<const float2 *>(p + e) : make_float2(0.f, 0.f);
                v[i][e] = x.x;
                v[i][e + 1] = x.y;
            }
        }
        const float m = lane < n ? mine[ROWS * HD + row0 + r] : -INFINITY, l = lane < n ? mine[ROWS * HD + ROWS + row0 + r] : 0.f;
        const float top = warp_max(m), f = ex2(m - (top == -INFINITY ? 0.f : top));
        const float sum = warp_sum(f != 0.f ? l * f : 0.f), inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
        float acc[E] = {};
#pragma unroll
        for (int i = 0; i < kFewStates; ++i) {
            const float w = __shfl_sync(0xffffffffu, f, i);
            if (w != 0.f) {  // a state without positions may hold no values
#pragma unroll
                for (int e = 0; e < E; ++e) acc[e] = fmaf(w, v[i][e], acc[e]);
            }
        }
        const int rr = left.row0 + row0 + r;
        T *dst = op + static_cast<long>(left.q0 + rr / a.group) * a.out_stride +
                 (left.head * a.group + rr % a.group) * HD + lane * E;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            fine = fine && acc[e] * 0.f * inv == 0.f;
            acc[e] *= inv;
        }
        if constexpr (E == 4) {
            store4(dst, vec, acc[0], acc[1], acc[2], acc[3]);
        } else {
            if (vec && sizeof(T) == 4) *reinterpret_cast<float2 *>(dst) = make_float2(acc[0], acc[1]);
            else if (vec) *reinterpret_cast<uint32_t *>(dst) = half2_bits(acc[0], acc[1]);
            else
#pragma unroll
                for (int e = 0; e < E; ++e) dst[e] = static_cast<T>(acc[e]);
        }
    }
    return (__all_sync(0xffffffffu, fine) ? 0 : 1) | (__any_sync(0xffffffffu, (theirs & 2) != 0) ? 2 : 0);
}

template <int ROWS, int HD, int NT, int EACH, int RB, int KV, typename T>
__global__ void __launch_bounds__(NT) ijb_paged_merge_kernel(const __grid_constant__ AttnArgs a) {
    __shared__ float top[RB], total[RB];
    __shared__ float4 sum[NT];
    const int row0 = blockIdx.y * RB;
    pdl_wait();
    uint32_t some, again, all;  // bit j: worker j of this block's left a tile; has rows to look at again; all of them
    {
        static_assert(EACH <= 32, "a lane a worker");
        const int j = threadIdx.x & 31, w = blockIdx.x * EACH + j;
        const bool in = j < EACH && w < a.workers;
        const int4 x = in ? *reinterpret_cast<const int4 *>(&a.left[w].states) : make_int4(0, 0, 0, 0);
        some = __ballot_sync(0xffffffffu, x.x > 0 && x.w > row0);
        const int bad = in ? a.left[w].bad : 0;
        again = __ballot_sync(0xffffffffu, bad != 0);
        all = __ballot_sync(0xffffffffu, (bad & 2) != 0);
    }
    static_assert(KV != IJB_KV_E2M1 || ROWS != kDecRows || EACH == NT / 32, "a warp a worker");
    if (KV == IJB_KV_E2M1 && ROWS == kDecRows && (some & (some - 1))) {  // several tiles
        // those of few states are merged at once, a warp each, not one after another: 64 ragged sequences 23.7 -> 19.9 us
        __shared__ uint32_t done, look, whole;
        if (threadIdx.x == 0) done = look = whole = 0u;
        __syncthreads();
        const int j = threadIdx.x >> 5;
        if ((some >> j) & 1u) {
            const Left left = a.left[blockIdx.x * EACH + j];
            if (left.states <= kFewStates) {
                const int how = merge_few<ROWS, HD, RB, T>(a, left, blockIdx.x * EACH + j, row0);
                if ((threadIdx.x & 31) == 0) {
                    atomicOr(&done, 1u << j);
                    if (how) atomicOr(&look, 1u << j);
                    if (how & 2) atomicOr(&whole, 1u << j);
                }
            }
        }
        __syncthreads();
        some &= ~done;
        again |= look;
        all |= whole;
    }
    for (; some; some &= some - 1) {
        const int w0 = blockIdx.x * EACH + __ffs(some) - 1;
        const Left left = a.left[w0];
        if (left.rows <= row0) continue;
        const int how = merge_block<ROWS, HD, NT, RB, T>(a, left, w0, row0, top, total, sum);
        if (how & 1) again |= 1u << (w0 - blockIdx.x * EACH);
        if (how & 2) all |= 1u << (w0 - blockIdx.x * EACH);
    }
    for (; again; again &= again - 1) {
        const int j = __ffs(again) - 1;
        mend_rows<ROWS, HD, NT, RB, KV, T>(a, blockIdx.x * EACH + j, row0, (all >> j) & 1, sum);
    }
}

// ---------------------------------------------------------------- launch --

constexpr int kMaxDevices = 64;
int sm_count() {
    static int sms[kMaxDevices];
    static std::mutex mu;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return 0;
    std::lock_guard<std::mutex> lock(mu);
    if (!sms[dev] && cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) sms[dev] = 0;
    return sms[dev];
}

// Raises a kernel's shared-memory limit, once per device (A, B: tell apart kernels
// of one signature).
template <class K, class A, class B>
cudaError_t allow_smem(K kernel, int bytes) {
    static bool ready[kMaxDevices];
    static std::mutex mu;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    std::lock_guard<std::mutex> lock(mu);
    if (ready[dev]) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    ready[dev] = e == cudaSuccess;
    return e;
}

// The merge behind the kernel just launched, on the GPU early (programmatic
// dependent launch): it waits there for the states.
template <int ROWS, int HD, int KV, typename T>
cudaError_t merge_launch(const AttnArgs &a, cudaStream_t s) {
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    constexpr int NT = 256, EACH = ROWS == kDecRows ? 8 : 1, RB = ROWS == kDecRows ? 2 : 16;
    const int rows = min(a.tile_rows, a.max_rows);
    cfg.gridDim = dim3((a.workers + EACH - 1) / EACH, (rows + RB - 1) / RB);
    cfg.blockDim = dim3(NT);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, ijb_paged_merge_kernel<ROWS, HD, NT, EACH, RB, KV, T>, a);
    count_launches(2);
    return e;
}

// The decode kernel of a cache type for entries of up to ROWS (8 or 16; e2m1, fp32: 4 too) rows, its launch shape and
// its shared memory (the plan's at least).
template <int HD, int KV, int ROWS, typename T>
using DecOf = std::conditional_t<KV == IJB_KV_E2M1, Dec4<HD, ROWS, T>, Dec<HD, KV, ROWS == 16, T>>;
template <int HD, int KV, int ROWS, typename T>
constexpr auto decode_kernel() {
    if constexpr (KV == IJB_KV_E2M1) return ijb_paged_decode4_kernel<HD, ROWS, T, false>;
    else return ijb_paged_decode_kernel<HD, KV, ROWS == 16, T>;
}
template <int HD, int KV, int ROWS, typename T>
constexpr int decode_smem() {
    using D = DecOf<HD, KV, ROWS, T>;
    return D::kSmem > kDecPlanBytes ? D::kSmem : kDecPlanBytes;
}
template <int HD, int KV, int ROWS, typename T>
cudaError_t decode_allow() {
    const auto kernel = decode_kernel<HD, KV, ROWS, T>();
    return allow_smem<decltype(kernel), DecOf<HD, KV, ROWS, T>, T>(kernel, decode_smem<HD, KV, ROWS, T>());
}
template <int HD, int KV, typename T>
cudaError_t tile_allow() {
    auto kernel = ijb_paged_tile_kernel<HD, KV, T>;
    return allow_smem<decltype(kernel), Tile<HD, T>, std::integral_constant<int, KV>>(kernel, Tile<HD, T>::kSmem);
}

// A call of few tiles (entries x KV heads) over an e2m1 cache: a cluster of CTAs for each of them, which joins its
// states itself.  One launch, and no plan.  The lengths are on the device, so the rule goes by the longest there may
// be: a cluster has its own tile only, and long ones of a few tiles want all SMs.  Measured in a graph, 8 KV heads of 64
// (128), 4 fp32 rows each, so and with plan and merge: one sequence of 300 positions 8.0 and 11.3 us (9.5 and 15.0), of
// 2,043 9.4 and 12.3 (11.3 and 16.2), of 30,000 17.2 and 20.3 (23.7 and 25.4), of 40,000 20.7 and 21.8 (29.1 and 28.3);
// two of 8,000 at most 13.1 and 14.5 (17.1 and 18.7), of 16,000 18.5 and 17.6 (25.1 and 23.2); four of 2,043 9.9 and
// 13.6 (11.6 and 17.1), of 16,000 at most 18.7 and 21.3 (27.1 and 30.9).  16 clusters of 8 do not fit the GPU's
// groups of SMs at once (two sequences of 2,043: 15.1).  8 sequences in clusters of 2 gained as much on short ones as
// they lost on ragged ones.
constexpr int kManyCtas = 8, kManyTiles = 8, kFewCtas = 4, kFewTiles = 32;  // CTAs a cluster, up to so many tiles
constexpr long kManyPositions = 32768, kFewPositions = 512;                  // in all; a tile
int cluster_size(const AttnArgs &a, int sms) {
    const long tiles = static_cast<long>(a.n_entries) * a.kv.kv_heads;
    const long positions = static_cast<long>(a.kv.max_pages) << a.kv.page_shift;
    if (tiles <= kManyTiles) return positions <= kManyPositions && tiles * kManyCtas <= sms ? kManyCtas : 0;
    return tiles <= kFewTiles && positions <= kFewPositions * tiles && tiles * kFewCtas <= sms ? kFewCtas : 0;
}
template <int HD, int ROWS, typename T>
cudaError_t cluster_allow() {
    const auto kernel = ijb_paged_decode4_kernel<HD, ROWS, T, true>;
    return allow_smem<decltype(kernel), Dec4<HD, ROWS, T>, std::true_type>(kernel, Dec4<HD, ROWS, T>::kSmem);
}
template <int HD, int ROWS, typename T>
cudaError_t cluster_launch(const AttnArgs &a, int size, cudaStream_t s) {
    using D = Dec4<HD, ROWS, T>;
    cudaError_t e = cluster_allow<HD, ROWS, T>();
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.n_entries * a.kv.kv_heads * size);
    cfg.blockDim = dim3(D::kWarps * 32);
    cfg.dynamicSmemBytes = D::kSmem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = size;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, ijb_paged_decode4_kernel<HD, ROWS, T, true>, a);
    count_launches(1);
    return e;
}

template <int HD, int KV, int ROWS, typename T>
cudaError_t decode_launch(AttnArgs a, int sms, bool all, cudaStream_t s) {
    using D = DecOf<HD, KV, ROWS, T>;
    const cudaError_t e = decode_allow<HD, KV, ROWS, T>();
    if (e != cudaSuccess) return e;
    a.min_rows = 1;
    a.max_rows = ROWS;
    a.report_long = all;
    a.tile_rows = kDecRows;
    a.unit = D::kPos;
    a.workers = sms * D::kWarps;
    // 64 positions a worker at least: one token at position 2043 of an e2m1 cache took 13.1 us so and 15.0 with 128
    // (before such calls had clusters)
    a.min_units = 64 / D::kPos;
    a.over = 1;
    a.least = 1;
    if constexpr (KV == IJB_KV_E2M1) {
        const int size = all ? cluster_size(a, sms) : 0;
        if (size) return cluster_launch<HD, ROWS, T>(a, size, s);
    }
    decode_kernel<HD, KV, ROWS, T>()<<<sms, D::kWarps * 32, decode_smem<HD, KV, ROWS, T>(), s>>>(a);
    return merge_launch<kDecRows, HD, KV, T>(a, s);
}

template <int HD, int KV, typename T>
cudaError_t tile_launch(AttnArgs a, int sms, int min_rows, cudaStream_t s) {
    using L = Tile<HD, T>;
    const cudaError_t e = tile_allow<HD, KV, T>();
    if (e != cudaSuccess) return e;
    a.min_rows = min_rows;
    a.max_rows = 0x7fffffff;
    a.report_long = false;
    a.tile_rows = kTileRows;
    a.unit = kBlock;
    a.workers = sms;
    a.min_units = 2;
    a.over = 4;
    a.least = 2;
    ijb_paged_tile_kernel<HD, KV, T><<<sms, kTileThreads, L::kSmem, s>>>(a);
    return merge_launch<kTileRows, HD, KV, T>(a, s);
}

// Which kernels serve a call.  Entries of up to 16 rows go to the decode kernel, longer ones to the tile kernel; a
// call that may hold longer ones and has few entries leaves them all to the tile kernel, for the launches (up to 4
// fp32 rows of an e2m1 cache have a kernel of their own: see Dec4): entries of 1 to 40 tokens behind 100 to 2000 take
// 49 us so and 55 with both kernels for 2 of them, 51 and 56 for 7, 55 and 59 for 8, 77 and 89 for 16 (so the border
// could lie higher); one of 200 tokens among single ones 54 and 68 for 4, 98 and 83 for 32. Over e2m1 (heads of 64,
// fp32): 38 and 44 for 2, 41 and 47 for 7, 43 and 49 for 8, 64 and 76 for 16, 86 and 102 for 32; one of 200 tokens
// among single ones behind 100 to 2000 35 and 51 for 4, 52 and 60 for 8, 63 and 61 for 16, 93 and 65 for 32, behind
// 8000 to 9000 103 and 93 for 4, 139 and 100 for 7, 149 and 100 for 8, 231 and 124 for 16: long contexts of single
// tokens have the border lower, short entries higher.  The border at 16 rows is the decode kernel's tile, which its
// plan has one of an entry; it is a cliff (24 x 4 and 24 x 5 tokens behind 700 to 9,001, 4 heads to a KV head: 52 and
// 150 us with heads of 64, 80 and 242 with heads of 128), for want of a tile in between.
template <int HD, int KV, typename T>
cudaError_t attention_call(const AttnArgs &a, int max_q, int sms, cudaStream_t s) {
    const long most = static_cast<long>(max_q > 0 ? min(max_q, a.n_tokens) : a.n_tokens) * a.group;
    if constexpr (KV == IJB_KV_E2M1 && sizeof(T) == 4)
        if (most <= 4) return decode_launch<HD, KV, 4, T>(a, sms, true, s);
    if (most <= 8) return decode_launch<HD, KV, 8, T>(a, sms, true, s);
    if (most <= kDecRows) return decode_launch<HD, KV, kDecRows, T>(a, sms, true, s);
    if (a.n_entries < 8) return tile_launch<HD, KV, T>(a, sms, 1, s);
    const cudaError_t e = decode_launch<HD, KV, kDecRows, T>(a, sms, false, s);
    return e != cudaSuccess ? e : tile_launch<HD, KV, T>(a, sms, kDecRows + 1, s);
}
template <int KV, typename T>
cudaError_t attention_call(const AttnArgs &a, int max_q, int sms, cudaStream_t s) {
    return a.kv.head_dim == 64 ? attention_call<64, KV, T>(a, max_q, sms, s) : attention_call<128, KV, T>(a, max_q, sms, s);
}
template <typename T>
cudaError_t attention_call(const AttnArgs &a, int type, int max_q, int sms, cudaStream_t s) {
    if (type == IJB_KV_E2M1) return attention_call<IJB_KV_E2M1, T>(a, max_q, sms, s);
    if (type == IJB_KV_E4M3) return attention_call<IJB_KV_E4M3, T>(a, max_q, sms, s);
    return attention_call<IJB_KV_F16, T>(a, max_q, sms, s);
}

constexpr int kMaxWorkers = 16;  // per SM: the decode kernel's warps

size_t workspace_bytes(int sms, int head_dim) {
    constexpr int rows = kTileRows;
    static_assert(kMaxWorkers * kDecRows <= kTileRows, "the decode kernel's states fit in the tile kernel's");
    // a word per worker, and two states each
    const size_t held = head_dim == 128 ? static_cast<size_t>(sms) * kTileRows * head_dim * sizeof(float) : 0;
    return static_cast<size_t>(sms) * kMaxWorkers * sizeof(Left) + held +
           static_cast<size_t>(sms) * 2 * rows * (head_dim + 2) * sizeof(float);
}

template <int HD, int KV>
cudaError_t prepare() {
    cudaError_t e = decode_allow<HD, KV, 8, float>();
    if (e == cudaSuccess) e = decode_allow<HD, KV, kDecRows, float>();
    if constexpr (KV == IJB_KV_E2M1) {
        if (e == cudaSuccess) e = decode_allow<HD, KV, 4, float>();
        if (e == cudaSuccess) e = cluster_allow<HD, 4, float>();
        if (e == cudaSuccess) e = cluster_allow<HD, 8, float>();
        if (e == cudaSuccess) e = cluster_allow<HD, kDecRows, float>();
    }
    if (e == cudaSuccess) e = tile_allow<HD, KV, float>();
    return e;
}

}  // namespace

cudaError_t paged_attention_prepare(int head_dim, int type) {
    const bool small = head_dim == 64;
    if (type == IJB_KV_E2M1) return small ? prepare<64, IJB_KV_E2M1>() : prepare<128, IJB_KV_E2M1>();
    if (type == IJB_KV_E4M3) return small ? prepare<64, IJB_KV_E4M3>() : prepare<128, IJB_KV_E4M3>();
    return small ? prepare<64, IJB_KV_F16>() : prepare<128, IJB_KV_F16>();
}

}  // namespace ijb

extern "C" {

size_t ijb_paged_attention_workspace(const ijb_kv_view *kv) {
    using namespace ijb;
    KvDev d;
    try {
        return kv_view_check(kv, &d).empty() ? workspace_bytes(sm_count(), kv->head_dim) : 0;
    } catch (...) {
        return 0;
    }
}

int ijb_paged_attention(const ijb_kv_view *kv, int heads, int type, const void *q_dev, long q_stride, void *out_dev,
                        long out_stride, int n_tokens, int n_entries, const int *q_start_dev, const int *seq_dev,
                        const int *kv_len_dev, int max_q, float scale, void *workspace_dev, size_t workspace_size,
                        uint32_t *status_dev, void *stream) {
    using namespace ijb;
    static const char *fn = "ijb_paged_attention";
    try {
        AttnArgs a{};
        const std::string bad = kv_view_check(kv, &a.kv);
        if (!bad.empty()) return kv_fail(IJB_ERR_INVALID, fn, bad);
        if (reinterpret_cast<uintptr_t>(kv->scale_dev) % 4 && kv->type == IJB_KV_E4M3)
            return kv_fail(IJB_ERR_INVALID, fn, "scale bytes must be 4-byte aligned");
        if (reinterpret_cast<uintptr_t>(kv->scale_dev) % 16 && kv->type == IJB_KV_E2M1)
            return kv_fail(IJB_ERR_INVALID, fn, "an e2m1 cache's scale bytes must be 16-byte aligned");
        if (kv->type == IJB_KV_E2M1 && kv->num_pages * 2 * kv->kv_heads > 0xffffffffL / (kv->page_size / 8))
            return kv_fail(IJB_ERR_INVALID, fn, "more than 2^32 groups of 8 rows");
        if (type != IJB_TYPE_F32 && type != IJB_TYPE_F16)
            return kv_fail(IJB_ERR_INVALID, fn, "query type must be IJB_TYPE_F32 or IJB_TYPE_F16");
        if (heads < 1 || heads % kv->kv_heads != 0 || heads / kv->kv_heads > 16)
            return kv_fail(IJB_ERR_INVALID, fn, "heads must be 1 to 16 times kv_heads");
        if (n_entries < 1 || n_entries > kMaxEntries) return kv_fail(IJB_ERR_INVALID, fn, "n_entries must be 1..4096");
        if (n_tokens < 0) return kv_fail(IJB_ERR_INVALID, fn, "negative token count");
        if (n_tokens == 0) return IJB_OK;
        // (times log2(e) it has to be finite, too)
        if (!(scale > 0.f && scale <= 2e38f)) return kv_fail(IJB_ERR_INVALID, fn, "scale must be positive and at most 2e38");
        if (!q_dev || !out_dev || !q_start_dev || !kv_len_dev || !workspace_dev)
            return kv_fail(IJB_ERR_INVALID, fn, "null argument");
        if (q_dev == out_dev) return kv_fail(IJB_ERR_INVALID, fn, "the output must not lie over the queries");
        const int elem = type == IJB_TYPE_F32 ? 4 : 2;
        const long row = static_cast<long>(heads) * kv->head_dim;
        if (q_stride < row || out_stride < row) return kv_fail(IJB_ERR_INVALID, fn, "a stride is shorter than a token's row");
        if (reinterpret_cast<uintptr_t>(q_dev) % elem || reinterpret_cast<uintptr_t>(out_dev) % elem)
            return kv_fail(IJB_ERR_INVALID, fn, "rows must be aligned to their elements");
        if (reinterpret_cast<uintptr_t>(workspace_dev) % 16)
            return kv_fail(IJB_ERR_INVALID, fn, "the workspace must be 16-byte aligned");
        if (static_cast<long>(n_tokens) * (heads / kv->kv_heads) / kTileRows + n_entries > kMaxTiles)
            return kv_fail(IJB_ERR_INVALID, fn, "too many rows for one call");
        // the plan counts units of one KV head, and a worker's units of all, in 32 bits
        const long positions = static_cast<long>(kv->max_pages) * kv->page_size;
        const long units = max(n_entries * (positions / kChunk + 2), kMaxTiles * (positions / kBlock + 5));
        if (units > 0x7fffffffL || units * kv->kv_heads / 64 > 0x7fffffffL)
            return kv_fail(IJB_ERR_INVALID, fn, "max_pages * page_size is too large for this many entries and heads");
        const int sms = sm_count();
        if (sms < 1) return kv_fail(IJB_ERR_CUDA, fn, "no CUDA device");
        if (workspace_size < workspace_bytes(sms, kv->head_dim))
            return kv_fail(IJB_ERR_INVALID, fn, "the workspace is smaller than ijb_paged_attention_workspace says");
        a.q = q_dev;
        a.q_stride = q_stride;
        a.out = out_dev;
        a.out_stride = out_stride;
        a.heads = heads;
        a.group = heads / kv->kv_heads;
        a.n_tokens = n_tokens;
        a.n_entries = n_entries;
        a.q_start = q_start_dev;
        a.seq = seq_dev;
        a.kv_len = kv_len_dev;
        a.scale_log2 = scale * 1.4426950408889634f;
        a.left = static_cast<Left *>(workspace_dev);
        a.part = reinterpret_cast<float *>(a.left + sms * kMaxWorkers);
        a.held = a.part + static_cast<size_t>(sms) * 2 * kTileRows * (kv->head_dim + 2);
        a.status = status_dev;
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        const cudaError_t e = type == IJB_TYPE_F32 ? attention_call<float>(a, kv->type, max_q, sms, s)
                                                   : attention_call<__half>(a, kv->type, max_q, sms, s);
        if (e != cudaSuccess) return kv_fail(IJB_ERR_CUDA, fn, cudaGetErrorString(e));
        return IJB_OK;
    } catch (...) {
        return IJB_ERR_NOMEM;
    }
}

}  // extern "C"

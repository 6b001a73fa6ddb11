// Attention of new tokens over the paged K/V cache (fp16 or e4m3 rows).
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
//    32-position chunks of its own through shared memory.
//  * ijb_paged_tile_kernel, more rows (chunks, prompts): bound by the matrix
//    products and the exponentials.  256 rows at a time on tcgen05.
// Both cut all the call's work (tiles of rows x units of positions, over all
// entries and KV heads, in one line) into equal runs, one per worker, so ragged
// lengths and long contexts fill the GPU alike.  A tile's run that another
// worker began or goes on with leaves its softmax state in the workspace, and
// ijb_paged_merge_kernel joins the states in order: no atomics, the same result
// every time for the same call.
//
// Arithmetic.  Products are fp16 x fp16 with fp32 sums.  fp32 queries enter as
// two fp16 parts (hi + lo, 22 bits), and so do their probabilities; fp16
// queries enter as they are, their probabilities rounded to fp16 once (the
// output is fp16 too).  Cached rows enter as fp16: fp16 rows exactly, e4m3 rows as
// code * 2^e, exact while a row's largest value is in [2^-7, 2^15].
#include <mutex>

#include "paged.cuh"

namespace ijb {
namespace {

// ------------------------------------------------------------------ plan --

constexpr int kMaxEntries = 4096, kMaxTiles = 8192;

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
    int tile_rows, unit;     // rows per tile, positions per unit
    int workers, min_units;
    float scale_log2;        // scale * log2(e)
    int *plan;               // workspace: kPlanHead ints, tile -> entry, tile -> first unit
    float *part;             // workspace: two states per worker
    uint32_t *status;
};
constexpr int kPlanHead = 8;  // tiles, units per KV head, units per worker

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
    if (rows > 0 && x.rows == 0 && report && a.min_rows <= 1 && a.status)
        atomicOr(a.status, kDevErrBadIndex);  // longer than the caller's max_q
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

// Cuts the call's work: `first` [n_entries + 1] receives each entry's first
// tile, `sums` [tiles + 1] each tile's first unit (of one KV head).  Block 0
// keeps them in the workspace for the merge.  All NT threads call it.
template <int NT>
__device__ void plan_build(const AttnArgs &a, int *first, int *sums, PlanOut *po) {
    const bool lead = blockIdx.x == 0;
    int base = 0;
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
    const int tiles = min(base, kMaxTiles);
    base = 0;
    for (int t0 = 0; t0 < tiles; t0 += NT) {
        const int t = t0 + static_cast<int>(threadIdx.x);
        int n = 0, e = 0;
        if (t < tiles) {
            e = find_le(first, a.n_entries, t);
            n = tile_units(a, entry_load(a, e, false), t - first[e]);
        }
        int total;
        const int inc = block_scan_int<NT>(n, po->warp_sums, &total);
        if (t < tiles) {
            sums[t] = base + inc - n;
            if (lead) {
                a.plan[kPlanHead + t] = e;
                a.plan[kPlanHead + kMaxTiles + t] = t - first[e];
                a.plan[kPlanHead + 2 * kMaxTiles + t] = base + inc - n;
            }
        }
        base += total;
    }
    const long all = static_cast<long>(base) * a.kv.kv_heads;
    const int per = static_cast<int>(max(static_cast<long>(a.min_units), (all + a.workers - 1) / a.workers));
    if (threadIdx.x == 0) {
        sums[tiles] = base;
        po->tiles = tiles;
        po->units = base;
        po->per = per;
        if (lead) {
            a.plan[kPlanHead + 2 * kMaxTiles + tiles] = base;
            a.plan[0] = tiles;
            a.plan[1] = base;
            a.plan[2] = per;
        }
    }
    __syncthreads();
}

// A worker's position in the line of work.
struct Cursor {
    long at, end;
    int e, ti, head, b0;
};

__device__ __forceinline__ Cursor cursor_start(const AttnArgs &a, const int *first, const int *sums, const PlanOut &po,
                                               int worker) {
    Cursor c;
    const long all = static_cast<long>(po.units) * a.kv.kv_heads;
    c.at = min(all, static_cast<long>(worker) * po.per);
    c.end = min(all, c.at + po.per);
    c.e = c.ti = c.head = c.b0 = 0;
    if (c.at < c.end) {
        c.head = static_cast<int>(c.at / po.units);
        const int u = static_cast<int>(c.at - static_cast<long>(c.head) * po.units);
        const int t = find_le(sums, po.tiles, u);
        c.e = find_le(first, a.n_entries, t);
        c.ti = t - first[c.e];
        c.b0 = u - sums[t];
    }
    return c;
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
    s.e = c.e;
    s.ti = c.ti;
    s.head = c.head;
    s.b0 = c.b0;
    s.units = tile_units(a, s.x, c.ti);
    s.b1 = static_cast<int>(min(static_cast<long>(s.units), c.b0 + (c.end - c.at)));
    c.at += s.b1 - s.b0;
    c.b0 = 0;
    if (++c.ti >= s.x.tiles) {
        c.ti = 0;
        if (++c.e == a.n_entries) {
            c.e = 0;
            ++c.head;
        }
    }
    return true;
}

// State slot of a run: a worker's first run may go on with a tile that another
// worker began (slot 0), its last may leave one to be gone on with (slot 1).
__device__ __forceinline__ long part_slot(const Segment &s, int worker) { return 2L * worker + (s.b0 > 0 ? 0 : 1); }
template <int ROWS, int HD>
__host__ __device__ constexpr long part_floats() { return static_cast<long>(ROWS) * (HD + 2); }

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
// 2^(s - 127) as fp16, at most 2^15 (a code of 0 must stay 0).
__device__ __forceinline__ __half scale_half(uint32_t s) { return __float2half_rn(fminf(kv_scale(s), 32768.f)); }
// Page id of a position, in bounds whatever the table holds; a bad one is reported.
__device__ __forceinline__ long page_of(const AttnArgs &a, int seq, int pos) {
    const int page = a.kv.page_table[static_cast<long>(seq) * a.kv.max_pages + (pos >> a.kv.page_shift)];
    if (page >= 0 && page < a.kv.num_pages) return page;
    if (a.status) atomicOr(a.status, kDevErrBadIndex);
    return 0;
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

constexpr int kChunk = 32;  // positions
constexpr int kDecRows = 16;

template <int HD, bool E4M3>
struct Dec {
    static constexpr int kRowBytes = HD * (E4M3 ? 1 : 2);
    static constexpr int kTile = kChunk * kRowBytes;
    static constexpr int kStage = 2 * kTile + (E4M3 ? 64 : 0);  // K, V, their scale bytes
    static constexpr int kWarps = kRowBytes == 256 ? 6 : 8;
    static constexpr int kStages = kRowBytes == 256 ? 2 : (kRowBytes == 128 ? 3 : 4);
    static constexpr int kSmem = kWarps * kStages * kStage;
};
constexpr int kDecPlanBytes = (kMaxEntries + kMaxTiles + 2) * 4;  // entries' first tiles and tiles' first units

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

template <int HD, bool E4M3, typename T>
__global__ void __launch_bounds__(Dec<HD, E4M3>::kWarps * 32) ijb_paged_decode_kernel(const __grid_constant__ AttnArgs a) {
    using D = Dec<HD, E4M3>;
    constexpr bool SPLIT = sizeof(T) == 4;  // fp32 queries: hi + lo
    constexpr int NT = D::kWarps * 32, RB = D::kRowBytes, KS = HD / 16, NTILE = HD / 8;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ PlanOut po;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gid = lane >> 2, t4 = lane & 3;
    int *first = reinterpret_cast<int *>(smem), *sums = first + a.n_entries + 1;
    plan_build<NT>(a, first, sums, &po);
    const int worker = blockIdx.x * D::kWarps + warp;
    Cursor load_c = cursor_start(a, first, sums, po, worker), use_c = load_c;
    __syncthreads();  // the plan's shared memory becomes the stages

    const uint32_t base = smem_u32(smem) + warp * D::kStages * D::kStage;
    const T *qp = static_cast<const T *>(a.q);
    T *op = static_cast<T *>(a.out);
    const bool qvec = aligned4<T>(a.q, a.q_stride), ovec = aligned4<T>(a.out, a.out_stride);
    const long v_off = static_cast<long>(a.kv.kv_heads) << a.kv.page_shift;  // rows from K to V within a page

    // ---- the loading side: one chunk after another, across runs
    Segment ls;
    int lb = 0, stage_in = 0;
    long next_row = 0;  // lane r: cache row (K) of position r of the next chunk
    bool more = cursor_next(a, load_c, ls);
    if (more) lb = ls.b0;
    auto find_row = [&]() {
        const int pos = lb * kChunk + lane;
        next_row = pos < ls.x.kv ? kv_row(a.kv, page_of(a, ls.x.seq, pos), 0, ls.head,
                                          pos & ((1 << a.kv.page_shift) - 1))
                                 : -1;
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
                const bool live = r < left;
                const long row = live ? row8 + (r & 7) : 0;
                const uint8_t *src = a.kv.data + row * RB + c * 16;
                const uint32_t off = dec_off<RB>(r, c);
                cp_async16(st + off, src, live);
                cp_async16(st + D::kTile + off, live ? src + v_off * RB : src, live);
            }
            if constexpr (E4M3) {  // 4 scale bytes a copy: lanes 0..7 K, 8..15 V
                const int r = (lane & 7) * 4;
                const long row8 = __shfl_sync(0xffffffffu, next_row, r & ~7);
                if (lane < 16 && r < left)
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
    Segment s;
    while (cursor_next(a, use_c, s)) {
        const int row0 = s.ti * kDecRows, rows = min(kDecRows, s.x.rows - row0);
        uint32_t qf[KS][4], ql[SPLIT ? KS : 1][4];
        int limit[2];  // last position that rows gid and gid + 8 see
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
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
                qf[ks][2 + hf] = *reinterpret_cast<const uint32_t *>(&h1);
                if constexpr (SPLIT) {
                    const float2 f0 = __half22float2(h0), f1 = __half22float2(h1);
                    ql[ks][hf] = half2_bits(v.x - f0.x, v.y - f0.y);
                    ql[ks][2 + hf] = half2_bits(v.z - f1.x, v.w - f1.y);
                }
            }
        }
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[NTILE][4];
#pragma unroll
        for (int i = 0; i < NTILE; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        const int all_see = s.x.kv - s.x.len + row0 / a.group;  // positions up to here are seen by every row

        for (int b = s.b0; b < s.b1; ++b) {
            issue();  // into the stage used last
            cp_async_wait<D::kStages - 1>();
            __syncwarp();
            const uint32_t kt = base + stage * D::kStage, vt = kt + D::kTile, sc = kt + 2 * D::kTile;
            const int p0 = b * kChunk;
            // ---- scores: tile nt, column n is position 16 (nt / 2) + 8 (nt % 2) + n / 2 + 4 (n % 2)
            float p[4][4];
#pragma unroll
            for (int nt = 0; nt < 4; ++nt) {
                p[nt][0] = p[nt][1] = p[nt][2] = p[nt][3] = 0.f;
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
                            if constexpr (SPLIT) mma(p[nt], ql[4 * j + e], b0, b1);
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            mma(p[nt], qf[2 * j + e], u[2 * e], u[2 * e + 1]);
                            if constexpr (SPLIT) mma(p[nt], ql[2 * j + e], u[2 * e], u[2 * e + 1]);
                        }
                    }
                }
            }
            // ---- online softmax (base 2) of rows gid and gid + 8
            const bool masked = p0 + kChunk - 1 > all_see;
            float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int nt = 0; nt < 4; ++nt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = 8 * nt + t4 + 4 * (i & 1);
                    float v = p[nt][i] * a.scale_log2;
                    if constexpr (E4M3) v *= kv_scale(lds8(sc + r));
                    if (masked && p0 + r > limit[i >> 1]) v = -INFINITY;
                    p[nt][i] = v;
                    mx[i >> 1] = fmaxf(mx[i >> 1], v);
                }
            float alpha[2], mu[2];
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                mx[hf] = fmaxf(mx[hf], __shfl_xor_sync(0xffffffffu, mx[hf], 1));
                mx[hf] = fmaxf(mx[hf], __shfl_xor_sync(0xffffffffu, mx[hf], 2));
                const float mn = fmaxf(m[hf], mx[hf]);
                mu[hf] = mn == -INFINITY ? 0.f : mn;
                alpha[hf] = ex2(m[hf] - mu[hf]);
                m[hf] = mn;
                l[hf] *= alpha[hf];
            }
#pragma unroll
            for (int nt = 0; nt < 4; ++nt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    p[nt][i] = ex2(p[nt][i] - mu[i >> 1]);
                    l[i >> 1] += p[nt][i];
                }
            if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
                for (int i = 0; i < NTILE; ++i) {
                    o[i][0] *= alpha[0];
                    o[i][1] *= alpha[0];
                    o[i][2] *= alpha[1];
                    o[i][3] *= alpha[1];
                }
            }
            // ---- values: k slots 2t, 2t+1, 2t+8, 2t+9 are positions 16 st + t, + 4, + 8, + 12
#pragma unroll
            for (int st = 0; st < 2; ++st) {
                uint32_t ph[4], pl[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float x = p[2 * st + (i >> 1)][2 * (i & 1)], y = p[2 * st + (i >> 1)][2 * (i & 1) + 1];
                    const __half2 h = __floats2half2_rn(x, y);
                    ph[i] = *reinterpret_cast<const uint32_t *>(&h);
                    if constexpr (SPLIT) {
                        const float2 f = __half22float2(h);
                        pl[i] = half2_bits(x - f.x, y - f.y);
                    }
                }
                const int r0 = 16 * st + t4;
                if constexpr (E4M3) {
                    __half vs[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i)  // scale bytes behind the last position mean nothing
                        vs[i] = p0 + r0 + 4 * i < s.x.kv ? scale_half(lds8(sc + 32 + r0 + 4 * i)) : __half(0.f);
                    const __half2 s01 = __halves2half2(vs[0], vs[1]), s23 = __halves2half2(vs[2], vs[3]);
                    const uint32_t sa = *reinterpret_cast<const uint32_t *>(&s01),
                                   sb = *reinterpret_cast<const uint32_t *>(&s23);
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
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const uint32_t b0 = hmul2(e4m3x2_half2(e ? y0 >> 16 : y0 & 0xffffu), sa);
                                const uint32_t b1 = hmul2(e4m3x2_half2(e ? y1 >> 16 : y1 & 0xffffu), sb);
                                mma(o[4 * k + 2 * d + e], ph, b0, b1);
                                if constexpr (SPLIT) mma(o[4 * k + 2 * d + e], pl, b0, b1);
                            }
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
                        for (int k = 0; k < 4; ++k)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const uint32_t sel = e ? 0x7632 : 0x5410;
                                const uint32_t b0 = prmt(w[0][k], w[1][k], sel), b1 = prmt(w[2][k], w[3][k], sel);
                                mma(o[8 * h + 2 * k + e], ph, b0, b1);
                                if constexpr (SPLIT) mma(o[8 * h + 2 * k + e], pl, b0, b1);
                            }
                    }
                }
            }
            __syncwarp();  // every lane is done with this stage
            stage = stage + 1 == D::kStages ? 0 : stage + 1;
        }

        // ---- the run's end: the output, or its state
        const bool whole = s.b0 == 0 && s.b1 == s.units;
        float *part = a.part + part_slot(s, worker) * part_floats<kDecRows, HD>();
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
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
}

// ----------------------------------------------------------------- merge --

// Joins the states of one (tile, KV head): 16 of its rows a block.
template <int ROWS, int HD, typename T>
__global__ void __launch_bounds__(256) ijb_paged_merge_kernel(const __grid_constant__ AttnArgs a) {
    __shared__ float top[16], total[16];
    __shared__ float4 sum[256];
    const int tile = blockIdx.x, head = blockIdx.y, row0 = blockIdx.z * 16;
    if (tile >= a.plan[0]) return;
    const int e = a.plan[kPlanHead + tile], ti = a.plan[kPlanHead + kMaxTiles + tile];
    const int *sums = a.plan + kPlanHead + 2 * kMaxTiles;
    const long per = a.plan[2], head_base = static_cast<long>(head) * a.plan[1];
    const long u0 = head_base + sums[tile], u1 = head_base + sums[tile + 1];
    const int w0 = static_cast<int>(u0 / per), n = static_cast<int>((u1 - 1) / per) - w0 + 1;
    if (n == 1) return;  // written by its only worker
    const Entry x = entry_load(a, e, false);
    const int live = min(ROWS, x.rows - ti * ROWS), rows = min(16, live - row0);
    if (rows <= 0) return;
    constexpr long PF = part_floats<ROWS, HD>();
    auto part = [&](int i) { return a.part + (2L * (w0 + i) + (i == 0 ? 1 : 0)) * PF; };
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int r = warp; r < rows; r += 8) {
        float m = -INFINITY, l = 0.f;
        for (int i = lane; i < n; i += 32) m = fmaxf(m, part(i)[ROWS * HD + row0 + r]);
        m = warp_max(m);
        const float mu = m == -INFINITY ? 0.f : m;
        for (int i = lane; i < n; i += 32) {
            const float *p = part(i) + ROWS * HD + row0 + r;
            l += p[ROWS] * ex2(p[0] - mu);
        }
        l = warp_sum(l);
        if (lane == 0) {
            top[r] = mu;
            total[r] = l;
        }
    }
    __syncthreads();
    constexpr int Q = HD / 4;  // float4 of a row
    const int outs = rows * Q, groups = outs < 256 ? 256 / outs : 1;
    T *op = static_cast<T *>(a.out);
    const bool vec = aligned4<T>(a.out, a.out_stride);
    for (int o0 = 0; o0 < outs; o0 += 256) {
        const int g = outs < 256 ? threadIdx.x / outs : 0, o = outs < 256 ? threadIdx.x % outs : o0 + threadIdx.x;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        const int r = o / Q, c = o % Q;
        if (g < groups && o < outs) {
#pragma unroll 4
            for (int i = g; i < n; i += groups) {
                const float *p = part(i);
                const float f = ex2(p[ROWS * HD + row0 + r] - top[r]);
                const float4 v = *reinterpret_cast<const float4 *>(p + (row0 + r) * HD + 4 * c);
                // a state without positions (f = 0) may hold no values
                acc.x = f != 0.f ? fmaf(f, v.x, acc.x) : acc.x;
                acc.y = f != 0.f ? fmaf(f, v.y, acc.y) : acc.y;
                acc.z = f != 0.f ? fmaf(f, v.z, acc.z) : acc.z;
                acc.w = f != 0.f ? fmaf(f, v.w, acc.w) : acc.w;
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
            const int rr = ti * ROWS + row0 + r;
            store4(op + static_cast<long>(x.q0 + rr / a.group) * a.out_stride + (head * a.group + rr % a.group) * HD + 4 * c,
                   vec, acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
        }
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

template <int HD, bool E4M3, typename T>
cudaError_t decode_launch(AttnArgs a, int sms, cudaStream_t s) {
    using D = Dec<HD, E4M3>;
    const int smem = D::kSmem > kDecPlanBytes ? D::kSmem : kDecPlanBytes;
    auto kernel = ijb_paged_decode_kernel<HD, E4M3, T>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    a.min_rows = 1;
    a.max_rows = 0x7fffffff;
    a.tile_rows = kDecRows;
    a.unit = kChunk;
    a.workers = sms * D::kWarps;
    a.min_units = 1;
    kernel<<<sms, D::kWarps * 32, smem, s>>>(a);
    ijb_paged_merge_kernel<kDecRows, HD, T><<<dim3(a.n_tokens * a.group / kDecRows + a.n_entries, a.kv.kv_heads, 1), 256, 0, s>>>(a);
    return cudaGetLastError();
}

template <typename T>
cudaError_t attention_call(const AttnArgs &a, bool e4m3, int sms, cudaStream_t s) {
    if (a.kv.head_dim == 64) return e4m3 ? decode_launch<64, true, T>(a, sms, s) : decode_launch<64, false, T>(a, sms, s);
    return e4m3 ? decode_launch<128, true, T>(a, sms, s) : decode_launch<128, false, T>(a, sms, s);
}

constexpr size_t kPlanBytes = (kPlanHead + 3 * kMaxTiles + 8) * sizeof(int);

size_t workspace_bytes(int sms, int head_dim) {
    return kPlanBytes + static_cast<size_t>(sms) * 8 * 2 * kDecRows * (head_dim + 2) * sizeof(float);
}

}  // namespace
}  // namespace ijb

extern "C" {

size_t ijb_paged_attention_workspace(const ijb_kv_view *kv, int heads, int n_tokens, int n_entries) {
    using namespace ijb;
    KvDev d;
    try {
        if (!kv_view_check(kv, &d).empty() || heads < 1 || n_tokens < 0 || n_entries < 1) return 0;
    } catch (...) {
        return 0;
    }
    return workspace_bytes(sm_count(), kv->head_dim);
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
        if (type != IJB_TYPE_F32 && type != IJB_TYPE_F16)
            return kv_fail(IJB_ERR_INVALID, fn, "query type must be IJB_TYPE_F32 or IJB_TYPE_F16");
        if (heads < 1 || heads % kv->kv_heads != 0 || heads / kv->kv_heads > 16)
            return kv_fail(IJB_ERR_INVALID, fn, "heads must be 1 to 16 times kv_heads");
        if (n_entries < 1 || n_entries > kMaxEntries) return kv_fail(IJB_ERR_INVALID, fn, "n_entries must be 1..4096");
        if (n_tokens < 0) return kv_fail(IJB_ERR_INVALID, fn, "negative token count");
        if (n_tokens == 0) return IJB_OK;
        if (!q_dev || !out_dev || !q_start_dev || !kv_len_dev || !workspace_dev)
            return kv_fail(IJB_ERR_INVALID, fn, "null argument");
        const int elem = type == IJB_TYPE_F32 ? 4 : 2;
        const long row = static_cast<long>(heads) * kv->head_dim;
        if (q_stride < row || out_stride < row) return kv_fail(IJB_ERR_INVALID, fn, "a stride is shorter than a token's row");
        if (reinterpret_cast<uintptr_t>(q_dev) % elem || reinterpret_cast<uintptr_t>(out_dev) % elem)
            return kv_fail(IJB_ERR_INVALID, fn, "rows must be aligned to their elements");
        if (reinterpret_cast<uintptr_t>(workspace_dev) % 16)
            return kv_fail(IJB_ERR_INVALID, fn, "the workspace must be 16-byte aligned");
        if (static_cast<long>(n_tokens) * (heads / kv->kv_heads) / kDecRows + n_entries > kMaxTiles)
            return kv_fail(IJB_ERR_INVALID, fn, "too many rows for one call");
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
        a.plan = static_cast<int *>(workspace_dev);
        a.part = reinterpret_cast<float *>(static_cast<uint8_t *>(workspace_dev) + kPlanBytes);
        a.status = status_dev;
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        const bool e4m3 = kv->type == IJB_KV_E4M3;
        const cudaError_t e = type == IJB_TYPE_F32 ? attention_call<float>(a, e4m3, sms, s)
                                                   : attention_call<__half>(a, e4m3, sms, s);
        if (e != cudaSuccess) return kv_fail(IJB_ERR_CUDA, fn, cudaGetErrorString(e));
        count_launches(2);
        (void)max_q;
        return IJB_OK;
    } catch (...) {
        return IJB_ERR_NOMEM;
    }
}

}  // extern "C"

// Writing rows into the paged K/V cache (quantising to e4m3 on the way) and
// reading them back.
//
// e4m3 rows.  With a = max |x_i| over the row's head_dim values, e is the
// least integer with a <= 448 * 2^e, the row is stored as e4m3(x_i * 2^-e),
// rounded to nearest even, and e + 127 as its scale byte.  448 is e4m3's
// largest value, so nothing saturates; a power of two makes both the scaling
// and its undoing exact, so the only rounding is the one to e4m3 (at most
// 2^-4 of a value in its normal range).  A scale per row (one token, one head)
// and not per page: a page is filled a token at a time, and a later, larger
// token must not change the rows already there.
//
// Both kernels move bytes: 16-byte loads and stores, 8 elements of a row a
// thread, a row per 8 (head_dim 64) or 16 threads.  A thread's loads wait for two
// others (the slot, its page), so with many rows each takes four heads of its
// token at once: 32768 rows of 8 heads x 128 read back as fp16 took 75 us a head
// at a time (2.7 TB/s), and take 47 us (4.2 TB/s); 16383 rows written from fp32 42 us
// (4.0 TB/s).
#include "paged.cuh"

namespace ijb {

constexpr int kRowThreads = 256;

std::string kv_view_check(const ijb_kv_view *v, KvDev *out) {
    if (!v) return "null cache view";
    if (v->type != IJB_KV_F16 && v->type != IJB_KV_E4M3 && v->type != IJB_KV_E2M1)
        return "cache type must be IJB_KV_F16, IJB_KV_E4M3 or IJB_KV_E2M1";
    if (v->head_dim != 64 && v->head_dim != 128) return "head_dim must be 64 or 128";
    if (v->kv_heads < 1 || v->kv_heads > 1024) return "kv_heads must be 1..1024";
    if (v->page_size < 8 || v->page_size > 256 || (v->page_size & (v->page_size - 1)) != 0)
        return "page_size must be 8, 16, 32, 64, 128 or 256";
    if (v->num_pages < 1 || v->num_pages > 0x7fffffffL) return "num_pages must be 1..2^31 - 1";
    if (v->n_seqs < 1 || v->max_pages < 1 || static_cast<long>(v->max_pages) * v->page_size > 0x40000000L)
        return "n_seqs and max_pages must be positive, and max_pages * page_size at most 2^30";
    if (!v->data_dev || !v->page_table_dev) return "null cache data or page table";
    if (reinterpret_cast<uintptr_t>(v->data_dev) % 16 != 0) return "cache data must be 16-byte aligned";
    if (v->type != IJB_KV_F16 && !v->scale_dev) return "an e4m3 or e2m1 cache needs its scale bytes";
    out->data = static_cast<uint8_t *>(v->data_dev);
    out->scale = v->scale_dev;
    out->page_table = v->page_table_dev;
    out->n_seqs = v->n_seqs;
    out->max_pages = v->max_pages;
    out->kv_heads = v->kv_heads;
    out->head_dim = v->head_dim;
    out->page_shift = 0;
    while ((1 << out->page_shift) < v->page_size) ++out->page_shift;
    out->num_pages = v->num_pages;
    return "";
}

namespace {

struct RowsParams {
    KvDev kv;
    void *k, *v;  // [n] tokens of [kv_heads][head_dim], `stride` elements apart
    long stride;
    int n;
    const int *tok_seq, *tok_pos;
    uint32_t *status;
};

// The cache row of token t (which, head 0); -1 when the entry is padding (a
// negative position) or names no slot, which is reported.
__device__ __forceinline__ long slot_row(const RowsParams &p, int t, int which) {
    const int seq = p.tok_seq[t], pos = p.tok_pos[t];
    if (pos < 0) return -1;
    const int pg = pos >> p.kv.page_shift;
    long page = -1;
    if (seq >= 0 && seq < p.kv.n_seqs && pg < p.kv.max_pages)
        page = p.kv.page_table[static_cast<long>(seq) * p.kv.max_pages + pg];
    if (page < 0 || page >= p.kv.num_pages) {
        if (p.status) atomicOr(p.status, kDevErrBadIndex);
        return -1;
    }
    return kv_row(p.kv, page, which, 0, pos & ((1 << p.kv.page_shift) - 1));
}

template <bool VEC>
__device__ __forceinline__ void load_row8(const float *p, float (&f)[8]) {
    if constexpr (VEC) {
        const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
        f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
        f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = p[i];
    }
}
template <bool VEC>
__device__ __forceinline__ void load_row8(const __half *p, float (&f)[8]) {
    __half h[8];
    if constexpr (VEC) {
        *reinterpret_cast<uint4 *>(h) = *reinterpret_cast<const uint4 *>(p);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = p[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = __half2float(h[i]);
}
template <bool VEC>
__device__ __forceinline__ void store_row8(float *p, const float (&f)[8]) {
    if constexpr (VEC) {
        *reinterpret_cast<float4 *>(p) = make_float4(f[0], f[1], f[2], f[3]);
        *reinterpret_cast<float4 *>(p + 4) = make_float4(f[4], f[5], f[6], f[7]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = f[i];
    }
}
template <bool VEC>
__device__ __forceinline__ void store_row8(__half *p, const float (&f)[8]) {
    __half h[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = __float2half_rn(f[i]);
    if constexpr (VEC) {
        *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(h);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = h[i];
    }
}

// Thread -> (token, K or V, U heads, 8 elements of each): rows of one token are
// consecutive, so a block moves whole tokens.  All L threads of a row are of one
// warp and agree on everything but their elements.
template <int HD, int U>
struct Place {
    static constexpr int L = HD / 8;  // threads a row
    int c, t, which, head, n;         // n: heads of this thread, 0 past the end
    __device__ __forceinline__ explicit Place(const RowsParams &p) {
        const long idx = blockIdx.x * static_cast<long>(kRowThreads) + threadIdx.x;
        c = static_cast<int>(idx % L);
        const long row = idx / L;
        const int groups = (p.kv.kv_heads + U - 1) / U, per = 2 * groups;
        t = static_cast<int>(row / per);
        const int r = static_cast<int>(row % per);
        which = r / groups;
        head = (r % groups) * U;
        n = t < p.n ? min(U, p.kv.kv_heads - head) : 0;
    }
};

template <typename T, bool E4M3, bool VEC, int HD, int U>
__global__ void __launch_bounds__(kRowThreads) ijb_kv_append_kernel(const __grid_constant__ RowsParams p) {
    const Place<HD, U> w(p);
    const long src = w.n ? w.t * p.stride + static_cast<long>(w.head) * HD + w.c * 8 : 0;
    const T *from = static_cast<const T *>(w.which ? p.v : p.k) + src;
    float f[U][8];
#pragma unroll
    for (int j = 0; j < U; ++j) {
        if (j < w.n) {
            load_row8<VEC>(from + j * HD, f[j]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) f[j][i] = 0.f;
        }
    }
    const long slot = w.n ? slot_row(p, w.t, w.which) : -1;
    const long to0 = slot + (static_cast<long>(w.head) << p.kv.page_shift);
#pragma unroll
    for (int j = 0; j < U; ++j) {
        const long to = to0 + (static_cast<long>(j) << p.kv.page_shift);
        const bool live = slot >= 0 && j < w.n;
        if constexpr (E4M3) {
            float a = 0.f;  // over the finite values: an infinity saturates, a NaN stays one
#pragma unroll
            for (int i = 0; i < 8; ++i) a = fmaxf(a, fabsf(f[j][i]) <= 3.402823466e38f ? fabsf(f[j][i]) : 0.f);
#pragma unroll
            for (int o = HD / 16; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
            // a = m 2^x with m in [1, 2): 448 = 1.75 * 2^8, so e = x - 8, one more when m > 1.75
            // (a below 2^-126 has x = -127 here and e ends at the floor)
            const uint32_t bits = __float_as_uint(a);
            int e = static_cast<int>(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
            e = max(e, -126);
            const float inv = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
            uint32_t q[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(f[j][4 * h] * inv, f[j][4 * h + 1] * inv),
                                                             __NV_SATFINITE, __NV_E4M3);
                const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(f[j][4 * h + 2] * inv, f[j][4 * h + 3] * inv),
                                                             __NV_SATFINITE, __NV_E4M3);
                q[h] = lo | (hi << 16);
            }
            if (live) {
                *reinterpret_cast<uint2 *>(p.kv.data + to * HD + w.c * 8) = make_uint2(q[0], q[1]);
                if (w.c == 0) p.kv.scale[to] = static_cast<uint8_t>(e + 127);
            }
        } else {
            if (live) store_row8<true>(reinterpret_cast<__half *>(p.kv.data) + to * HD + w.c * 8, f[j]);
        }
    }
}

// Reads back: code * 2^e (exact in fp32), or the fp16 row; rows of padding
// entries and of entries that name no slot are left as they were.
template <typename T, bool E4M3, bool VEC, int HD, int U>
__global__ void __launch_bounds__(kRowThreads) ijb_kv_gather_kernel(const __grid_constant__ RowsParams p) {
    const Place<HD, U> w(p);
    if (w.n == 0) return;
    const long slot = slot_row(p, w.t, w.which);
    if (slot < 0) return;
    const long from0 = slot + (static_cast<long>(w.head) << p.kv.page_shift);
    T *dst = static_cast<T *>(w.which ? p.v : p.k) + w.t * p.stride + static_cast<long>(w.head) * HD + w.c * 8;
    uint4 raw[U];
    uint32_t sc[U];
#pragma unroll
    for (int j = 0; j < U; ++j) {
        if (j >= w.n) continue;
        const long from = from0 + (static_cast<long>(j) << p.kv.page_shift);
        if constexpr (E4M3) {
            const uint2 u = *reinterpret_cast<const uint2 *>(p.kv.data + from * HD + w.c * 8);
            raw[j].x = u.x;
            raw[j].y = u.y;
            sc[j] = p.kv.scale[from];
        } else {
            raw[j] = *reinterpret_cast<const uint4 *>(p.kv.data + (from * HD + w.c * 8) * 2);
        }
    }
#pragma unroll
    for (int j = 0; j < U; ++j) {
        if (j >= w.n) continue;
        float f[8];
        if constexpr (E4M3) {
            const float s = kv_scale(sc[j]);
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                const uint32_t u = h < 2 ? raw[j].x : raw[j].y;
                const __half2_raw x = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(u >> (16 * (h & 1))),
                                                                 __NV_E4M3);
                const float2 v = __half22float2(*reinterpret_cast<const __half2 *>(&x));
                f[2 * h] = v.x * s;
                f[2 * h + 1] = v.y * s;
            }
        } else {
            const __half *h = reinterpret_cast<const __half *>(&raw[j]);
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = __half2float(h[i]);
        }
        store_row8<VEC>(dst + j * HD, f);
    }
}

constexpr int kHeads = 4;              // heads a thread takes of many rows
// A head each fills the GPU about once from here on.  In a graph, e4m3 at head_dim 128 and 8 heads, one
// head and four a thread: 512 rows (2^17 threads of a head) written 8.2 and 9.0 us, read 8.2 and 9.6; 1024 (2^18)
// 10.2 each; 16383 written 50.7 and 47.5, read 50.2 and 43.2.
constexpr long kManyThreads = 1 << 18;

template <bool APPEND, typename T, bool E4M3, bool VEC, int HD, int U>
void rows_launch(const RowsParams &p, cudaStream_t s) {
    const long threads = static_cast<long>(p.n) * 2 * ((p.kv.kv_heads + U - 1) / U) * (HD / 8);
    const unsigned blocks = static_cast<unsigned>((threads + kRowThreads - 1) / kRowThreads);
    if constexpr (APPEND) ijb_kv_append_kernel<T, E4M3, VEC, HD, U><<<blocks, kRowThreads, 0, s>>>(p);
    else ijb_kv_gather_kernel<T, E4M3, VEC, HD, U><<<blocks, kRowThreads, 0, s>>>(p);
}
template <bool APPEND, typename T, bool E4M3, int HD>
void rows_launch(const RowsParams &p, bool vec, cudaStream_t s) {
    const bool many = static_cast<long>(p.n) * 2 * p.kv.kv_heads * (HD / 8) > kManyThreads && p.kv.kv_heads >= kHeads;
    if (!vec) rows_launch<APPEND, T, E4M3, false, HD, 1>(p, s);
    else if (many) rows_launch<APPEND, T, E4M3, true, HD, kHeads>(p, s);
    else rows_launch<APPEND, T, E4M3, true, HD, 1>(p, s);
}
template <bool APPEND, typename T, bool E4M3>
void rows_launch(const RowsParams &p, bool vec, cudaStream_t s) {
    if (p.kv.head_dim == 64) rows_launch<APPEND, T, E4M3, 64>(p, vec, s);
    else rows_launch<APPEND, T, E4M3, 128>(p, vec, s);
}

// ---- e2m1 rows
//
// A block takes whole tokens (part of one when it has many heads), a thread E values of
// each of U heads side by side.
// Threads a block: with few rows (a head a thread) as many as take a token's at once, for the latency.
__host__ __device__ constexpr int append4_threads(int u) { return u == 1 ? 256 : 128; }
__host__ __device__ constexpr int gather4_threads(int u) { return u == 1 ? 256 : 64; }
template <int HD, int U, int E, int NT>
struct Place4 {
    static constexpr int L = HD / E, ROWS = NT / L;  // threads a row, rows a block at a time
    static __host__ __device__ int groups(const KvDev &kv) { return (kv.kv_heads + U - 1) / U; }
    // tokens a block takes
    static __host__ __device__ int tokens(const KvDev &kv) {
        const int n = ROWS / (2 * groups(kv));
        return n > 1 ? n : 1;
    }
    int c, t, which, head, n;  // n: heads of this thread, 0 past the end
    // row: of the block's
    __device__ __forceinline__ Place4(const RowsParams &p, int row) {
        const unsigned g = groups(p.kv), per = 2 * g;
        c = threadIdx.x % L;
        const unsigned in = static_cast<unsigned>(row) / per, r = static_cast<unsigned>(row) % per;
        const long tok = blockIdx.x * static_cast<long>(tokens(p.kv)) + in;
        t = static_cast<int>(tok);
        which = r >= g;
        head = (which ? r - g : r) * U;
        n = tok < p.n && in < tokens(p.kv) ? min(U, p.kv.kv_heads - head) : 0;
    }
};

// The scale byte of 32 dims whose largest finite magnitude is a: the nearest scale to a / 6, ties to even (from
// 2^-14 on the upper bits of the number with 3 of its mantissa, below in steps of 2^-17).  a / 6 is fp32's product of a
// and 1 / 6, a unit of the last place off the quotient at most, which is a millionth of the rounding that follows.
__device__ __forceinline__ uint32_t e2m1_scale_byte(float a) {
    const float r = a * (1.f / 6.f);
    const uint32_t bits = __float_as_uint(r);
    const uint32_t byte = r >= 6.103515625e-5f ? ((bits + 0x7ffffu + ((bits >> 20) & 1u)) >> 20) - ((127u - 15u) << 3)
                                               : __float2uint_rn(r * 131072.f);
    return min(byte, kKvTopScale);
}
// What a value is multiplied by before it becomes a code; 0 where the scale is 0.
__device__ __forceinline__ float e2m1_inverse(uint32_t byte) {
    return byte ? __frcp_rn(half_bits_to_float(static_cast<uint16_t>(byte << 7))) : 0.f;
}
__device__ __forceinline__ float max_abs_nan(float a, float b) {  // the larger magnitude, or NaN if either is
    float c;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(fabsf(b)));
    return c;
}
// 8 codes, rounded to nearest, ties to even, larger values to the largest.
__device__ __forceinline__ uint32_t e2m1_codes(const float (&f)[8], float inv) {
    uint32_t q;
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(q)
        : "f"(f[0] * inv), "f"(f[1] * inv), "f"(f[2] * inv), "f"(f[3] * inv), "f"(f[4] * inv), "f"(f[5] * inv),
          "f"(f[6] * inv), "f"(f[7] * inv));
    return q;
}

// A thread has 8 values of U heads' rows; 4 threads share a block of 32 dims, and each works out the scale of one
// head in 4 for all of them.  Measured: 12289 tokens of 8 heads x 128 from fp32 26 us (4.5 TB/s), from fp16 21 (3.1);
// before, in blocks of 256 threads, 4 on an SM, 28 and 24 us.  No unit is full (DRAM 51 %, issue slots 40 %, the ALU
// 37 %): of the 20 clocks from one of a warp's instructions to its next 12 go to waiting for its loads, and half the
// warps that an SM could hold are there.
template <typename T, bool VEC, int HD, int U>
__global__ void __launch_bounds__(append4_threads(U), U == 1 ? 4 : (sizeof(T) == 4 ? 9 : 10))
    ijb_kv_append4_kernel(const __grid_constant__ RowsParams p) {
    using P = Place4<HD, U, 8, append4_threads(U)>;
    const int rows = P::tokens(p.kv) * 2 * P::groups(p.kv);
    const int lane = threadIdx.x & 31, quad = lane & 28;
    for (int row = threadIdx.x / P::L; row / P::ROWS * P::ROWS < rows; row += P::ROWS) {  // (all threads as often)
        const P w(p, row);
        const T *from = static_cast<const T *>(w.which ? p.v : p.k) +
                        (w.n ? w.t * p.stride + static_cast<long>(w.head) * HD + w.c * 8 : 0);
        float f[U][8], a[U];
#pragma unroll
        for (int j = 0; j < U; ++j) {
            if (j < w.n) {
                load_row8<VEC>(from + j * HD, f[j]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) f[j][i] = 0.f;
            }
        }
        const long slot = w.n ? slot_row(p, w.t, w.which) : -1;
        bool wild = false;  // an infinity or a NaN
#pragma unroll
        for (int j = 0; j < U; ++j) {
            a[j] = fabsf(f[j][0]);
#pragma unroll
            for (int i = 1; i < 8; ++i) a[j] = max_abs_nan(a[j], f[j][i]);
            wild |= !(a[j] <= 3.402823466e38f);
        }
        uint32_t nan = 0;  // bit j: a NaN in this thread's part of head j's block
        if (__any_sync(0xffffffffu, wild)) {
            // infinities count as the largest value of their block, and are left to the conversion; zeros take their
            // place in a block without a scale, and that of a NaN, whose block's scale is NaN
#pragma unroll
            for (int j = 0; j < U; ++j) {
                a[j] = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    a[j] = fmaxf(a[j], fabsf(f[j][i]) <= 3.402823466e38f ? fabsf(f[j][i]) : 0.f);
                    nan |= f[j][i] != f[j][i] ? 1u << j : 0u;
                }
            }
            nan |= __shfl_xor_sync(0xffffffffu, nan, 1);
            nan |= __shfl_xor_sync(0xffffffffu, nan, 2);
        }
        uint32_t byte[(U + 3) / 4];  // of head 4 g + lane % 4 (U 1: of the head)
        float inv[U];
#pragma unroll
        for (int g = 0; g < (U + 3) / 4; ++g) {
            float mine;
            if constexpr (U >= 4) {
                // lane % 4 ends with the maximum of head 4 g + lane % 4
                const bool odd = lane & 1, high = lane & 2;
                float x = odd ? a[4 * g + 1] : a[4 * g], y = odd ? a[4 * g + 3] : a[4 * g + 2];
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, odd ? a[4 * g] : a[4 * g + 1], 1));
                y = fmaxf(y, __shfl_xor_sync(0xffffffffu, odd ? a[4 * g + 2] : a[4 * g + 3], 1));
                mine = fmaxf(high ? y : x, __shfl_xor_sync(0xffffffffu, high ? x : y, 2));
            } else {
                mine = fmaxf(a[0], __shfl_xor_sync(0xffffffffu, a[0], 1));
                mine = fmaxf(mine, __shfl_xor_sync(0xffffffffu, mine, 2));
            }
            byte[g] = e2m1_scale_byte(mine);
            const float x = e2m1_inverse(byte[g]);
            if constexpr (U >= 4) {
#pragma unroll
                for (int j = 0; j < 4; ++j) inv[4 * g + j] = __shfl_sync(0xffffffffu, x, quad + j);
            } else {
                inv[0] = x;
            }
        }
        if (slot < 0) continue;
        const long to0 = slot + (static_cast<long>(w.head) << p.kv.page_shift);
        uint8_t *codes = p.kv.data + to0 * (HD / 2) + w.c * 4;
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const uint32_t q = inv[j] > 0.f ? e2m1_codes(f[j], inv[j]) : 0u;
            if (j < w.n) *reinterpret_cast<uint32_t *>(codes) = q;
            codes += static_cast<long>(HD / 2) << p.kv.page_shift;
        }
#pragma unroll
        for (int g = 0; g < (U + 3) / 4; ++g) {
            const int j = U >= 4 ? 4 * g + (lane & 3) : 0;
            const long to = to0 + (static_cast<long>(j) << p.kv.page_shift);
            if (j < w.n && (U >= 4 || w.c % 4 == 0))
                p.kv.scale[to * (HD / kKvBlock) + w.c / 4] = static_cast<uint8_t>((nan >> j) & 1u ? kKvNanScale : byte[g]);
        }
    }
}

// Code * scale, exact in fp32, and in fp16 for the scales that ijb_kv_append writes (others rounded once).  A thread
// stores 16 bytes of each of U heads' rows, next to its neighbour's.  Bound by the latency of its three loads in a
// row (the slot, its page, the codes; 18 of 25 clocks an instruction go to waiting for them, issue slots 54 %), so
// what counts is how many threads are on an SM, and that a block of few has more than one row each: 32749 tokens of 8
// heads x 128 to fp16 take 34.3 us (5.0 TB/s) and to fp32 53 (5.8), in blocks of 256 threads, 4 on an SM, 49 and 89.
template <typename T, bool VEC, int HD, int U>
__global__ void __launch_bounds__(gather4_threads(U), U == 1 ? 4 : 32)
    ijb_kv_gather4_kernel(const __grid_constant__ RowsParams p) {
    constexpr int E = 16 / sizeof(T);
    using P = Place4<HD, U, E, gather4_threads(U)>;
    const int rows = P::tokens(p.kv) * 2 * P::groups(p.kv);
    for (int row = threadIdx.x / P::L; row < rows; row += P::ROWS) {
        const P w(p, row);
        if (w.n == 0) continue;
        const long slot = slot_row(p, w.t, w.which);
        if (slot < 0) continue;
        const long from0 = slot + (static_cast<long>(w.head) << p.kv.page_shift);
        const uint8_t *from = p.kv.data + from0 * (HD / 2) + w.c * E / 8 * 4;  // (two threads' codes when E is 4)
        const uint8_t *scale = p.kv.scale + from0 * (HD / kKvBlock) + w.c * E / kKvBlock;
        T *dst = static_cast<T *>(w.which ? p.v : p.k) + w.t * p.stride + static_cast<long>(w.head) * HD + w.c * E;
        const long next = static_cast<long>(HD / 2) << p.kv.page_shift,
                   next_scale = static_cast<long>(HD / kKvBlock) << p.kv.page_shift;
        uint32_t raw[U], sc[U];
#pragma unroll
        for (int j = 0; j < U; ++j) {
            if (j < w.n) {
                raw[j] = *reinterpret_cast<const uint32_t *>(from);
                sc[j] = *scale;
            }
            from += next;
            scale += next_scale;
        }
#pragma unroll
        for (int j = 0; j < U; ++j) {
            if (j >= w.n) continue;
            if constexpr (E == 8) {
                const __half2 s = __half2half2(__ushort_as_half(static_cast<uint16_t>(sc[j] << 7)));
                __half2 h[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t x = e2m1x2_half2(raw[j], i);
                    h[i] = __hmul2(*reinterpret_cast<const __half2 *>(&x), s);
                }
                if constexpr (VEC) {
                    *reinterpret_cast<uint4 *>(dst + j * HD) = *reinterpret_cast<const uint4 *>(h);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        dst[j * HD + 2 * i] = __low2half(h[i]);
                        dst[j * HD + 2 * i + 1] = __high2half(h[i]);
                    }
                }
            } else {
                const float s = half_bits_to_float(static_cast<uint16_t>(sc[j] << 7));
                const uint32_t mine = raw[j] >> (w.c % 2 * 16), x = e2m1x2_half2(mine, 0), y = e2m1x2_half2(mine, 1);
                const float2 u = __half22float2(*reinterpret_cast<const __half2 *>(&x)),
                             v = __half22float2(*reinterpret_cast<const __half2 *>(&y));
                if constexpr (VEC) {
                    *reinterpret_cast<float4 *>(dst + j * HD) = make_float4(u.x * s, u.y * s, v.x * s, v.y * s);
                } else {
                    dst[j * HD] = u.x * s;
                    dst[j * HD + 1] = u.y * s;
                    dst[j * HD + 2] = v.x * s;
                    dst[j * HD + 3] = v.y * s;
                }
            }
        }
    }
}

template <bool APPEND, typename T, bool VEC, int HD, int U>
void rows4_launch(const RowsParams &p, cudaStream_t s) {
    constexpr int NT = APPEND ? append4_threads(U) : gather4_threads(U);
    using P = Place4<HD, U, APPEND ? 8 : 16 / static_cast<int>(sizeof(T)), NT>;
    const int each = P::tokens(p.kv);
    const unsigned blocks = static_cast<unsigned>((static_cast<long>(p.n) + each - 1) / each);
    if constexpr (APPEND) ijb_kv_append4_kernel<T, VEC, HD, U><<<blocks, NT, 0, s>>>(p);
    else ijb_kv_gather4_kernel<T, VEC, HD, U><<<blocks, NT, 0, s>>>(p);
}
// Four heads a thread from here on (threads of 8 values of a head).  In a graph, 8 heads, fp32, a head and four a thread:
// head_dim 64, 512 rows (2^16) written 3.1 and 3.3 us, read 3.1 and 3.0; 1024 (2^17) 3.5 and 3.6, 4.1 and 3.6;
// head_dim 128, 512 (2^17) 3.6 and 3.5, 4.0 and 3.8; 1024 (2^18) 4.9 and 4.1, 5.4 and 4.5; 4096 12.7 and 7.8, 13.6
// and 7.9.
constexpr long kMany4Threads = 1 << 17;
template <bool APPEND, typename T, int HD>
void rows4_launch(const RowsParams &p, bool vec, cudaStream_t s) {
    const bool many = static_cast<long>(p.n) * 2 * p.kv.kv_heads * (HD / 8) >= kMany4Threads && p.kv.kv_heads >= kHeads;
    if (!vec) rows4_launch<APPEND, T, false, HD, 1>(p, s);
    else if (many) rows4_launch<APPEND, T, true, HD, kHeads>(p, s);
    else rows4_launch<APPEND, T, true, HD, 1>(p, s);
}

template <bool APPEND, typename T>
void rows_launch(const RowsParams &p, int type, bool vec, cudaStream_t s) {
    if (type == IJB_KV_E2M1 && p.kv.head_dim == 64) rows4_launch<APPEND, T, 64>(p, vec, s);
    else if (type == IJB_KV_E2M1) rows4_launch<APPEND, T, 128>(p, vec, s);
    else if (type == IJB_KV_E4M3) rows_launch<APPEND, T, true>(p, vec, s);
    else rows_launch<APPEND, T, false>(p, vec, s);
}

template <bool APPEND>
int rows_call(const char *fn, const ijb_kv_view *view, int type, void *k, void *v, long stride, int n,
              const int *tok_seq, const int *tok_pos, uint32_t *status, void *stream) {
    try {
        RowsParams p{};
        const std::string bad = kv_view_check(view, &p.kv);
        if (!bad.empty()) return kv_fail(IJB_ERR_INVALID, fn, bad);
        if (type != IJB_TYPE_F32 && type != IJB_TYPE_F16)
            return kv_fail(IJB_ERR_INVALID, fn, "row type must be IJB_TYPE_F32 or IJB_TYPE_F16");
        if (n < 0) return kv_fail(IJB_ERR_INVALID, fn, "negative token count");
        if (n == 0) return IJB_OK;
        if (!k || !v || !tok_seq || !tok_pos) return kv_fail(IJB_ERR_INVALID, fn, "null argument");
        const int elem = type == IJB_TYPE_F32 ? 4 : 2;
        if (reinterpret_cast<uintptr_t>(k) % elem || reinterpret_cast<uintptr_t>(v) % elem)
            return kv_fail(IJB_ERR_INVALID, fn, "rows must be aligned to their elements");
        if (stride < static_cast<long>(view->kv_heads) * view->head_dim)
            return kv_fail(IJB_ERR_INVALID, fn, "the stride is shorter than a token's kv_heads * head_dim elements");
        p.k = k;
        p.v = v;
        p.stride = stride;
        p.n = n;
        p.tok_seq = tok_seq;
        p.tok_pos = tok_pos;
        p.status = status;
        if (static_cast<long>(n) * 2 * view->kv_heads * (view->head_dim / 8) > 0x7fffffffL * kRowThreads)
            return kv_fail(IJB_ERR_INVALID, fn, "too many rows for one call");
        // rows that do not start on 16 bytes are moved an element at a time
        const bool vec = reinterpret_cast<uintptr_t>(k) % 16 == 0 && reinterpret_cast<uintptr_t>(v) % 16 == 0 &&
                         stride * elem % 16 == 0;
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        if (type == IJB_TYPE_F32) rows_launch<APPEND, float>(p, view->type, vec, s);
        else rows_launch<APPEND, __half>(p, view->type, vec, s);
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return kv_fail(IJB_ERR_CUDA, fn, cudaGetErrorString(e));
        count_launches(1);
        return IJB_OK;
    } catch (...) {
        return IJB_ERR_NOMEM;
    }
}

// Copies whole pages, a block a piece of kCopyPiece bytes (or less) of one: four 16-byte loads in flight a thread, and
// bound by the memory: 6007 pages of 8 heads x 16 x 128 in e4m3 (33 KB each) take 63.7 us (6.2 TB/s read and
// written, the rate of a plain copy), 16 fp16 pages of 32 KB 2.4.
struct CopyParams {
    const uint8_t *from, *from_scale;
    uint8_t *to, *to_scale;
    long from_pages, to_pages;
    long data_bytes, scale_bytes;  // of a page
    int n, pieces;                 // pieces a page's data
    const int *src, *dst;
    uint32_t *status;
};
constexpr int kCopyThreads = 128, kCopyEach = 4, kCopyPiece = kCopyThreads * kCopyEach * 16;

__global__ void __launch_bounds__(kCopyThreads) ijb_kv_copy_kernel(const __grid_constant__ CopyParams p) {
    const int i = blockIdx.x / p.pieces, piece = blockIdx.x % p.pieces;
    const int src = p.src[i], dst = p.dst[i];
    if (dst < 0) return;
    if (src < 0 || src >= p.from_pages || dst >= p.to_pages) {
        if (p.status && threadIdx.x == 0) atomicOr(p.status, kDevErrBadIndex);
        return;
    }
    const uint4 *s = reinterpret_cast<const uint4 *>(p.from + src * p.data_bytes);
    uint4 *d = reinterpret_cast<uint4 *>(p.to + dst * p.data_bytes);
    const long at = static_cast<long>(piece) * (kCopyPiece / 16) + threadIdx.x, end = p.data_bytes / 16;
    uint4 x[kCopyEach];
#pragma unroll
    for (int k = 0; k < kCopyEach; ++k)
        if (at + k * kCopyThreads < end) x[k] = s[at + k * kCopyThreads];
#pragma unroll
    for (int k = 0; k < kCopyEach; ++k)
        if (at + k * kCopyThreads < end) d[at + k * kCopyThreads] = x[k];
    if (piece != 0) return;
    const uint8_t *ss = p.from_scale + src * p.scale_bytes;
    uint8_t *sd = p.to_scale + dst * p.scale_bytes;
    const bool vec = ((reinterpret_cast<uintptr_t>(ss) | reinterpret_cast<uintptr_t>(sd) | p.scale_bytes) & 15) == 0;
    if (vec) {
        for (long b = threadIdx.x * 16; b < p.scale_bytes; b += kCopyThreads * 16)
            *reinterpret_cast<uint4 *>(sd + b) = *reinterpret_cast<const uint4 *>(ss + b);
    } else {
        for (long b = threadIdx.x; b < p.scale_bytes; b += kCopyThreads) sd[b] = ss[b];
    }
}

int copy_call(const char *fn, const ijb_kv_view *from, const ijb_kv_view *to, int n, const int *src, const int *dst,
              uint32_t *status, void *stream) {
    try {
        KvDev a, b;
        std::string bad = kv_view_check(from, &a);
        if (bad.empty()) bad = kv_view_check(to, &b);
        if (!bad.empty()) return kv_fail(IJB_ERR_INVALID, fn, bad);
        if (from->type != to->type || from->kv_heads != to->kv_heads || from->head_dim != to->head_dim ||
            from->page_size != to->page_size)
            return kv_fail(IJB_ERR_INVALID, fn, "the two caches' pages differ");
        if (n < 0) return kv_fail(IJB_ERR_INVALID, fn, "negative page count");
        if (n == 0) return IJB_OK;
        if (!src || !dst) return kv_fail(IJB_ERR_INVALID, fn, "null argument");
        CopyParams p;
        const long rows = 2L * from->kv_heads * from->page_size;
        p.from = a.data;
        p.from_scale = a.scale;
        p.to = b.data;
        p.to_scale = b.scale;
        p.from_pages = from->num_pages;
        p.to_pages = to->num_pages;
        p.data_bytes = rows * kv_row_bytes(from->type, from->head_dim);
        p.scale_bytes = from->type == IJB_KV_F16 ? 0 : from->type == IJB_KV_E4M3 ? rows : rows * (from->head_dim / kKvBlock);
        p.pieces = static_cast<int>((p.data_bytes + kCopyPiece - 1) / kCopyPiece);
        p.n = n;
        p.src = src;
        p.dst = dst;
        p.status = status;
        if (static_cast<long>(n) * p.pieces > 0x7fffffffL) return kv_fail(IJB_ERR_INVALID, fn, "too many pages for one call");
        ijb_kv_copy_kernel<<<static_cast<unsigned>(n) * p.pieces, kCopyThreads, 0, static_cast<cudaStream_t>(stream)>>>(p);
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return kv_fail(IJB_ERR_CUDA, fn, cudaGetErrorString(e));
        count_launches(1);
        return IJB_OK;
    } catch (...) {
        return IJB_ERR_NOMEM;
    }
}

}  // namespace
}  // namespace ijb

extern "C" {

int ijb_kv_append(const ijb_kv_view *kv, int src_type, const void *k_dev, const void *v_dev, long stride, int n,
                  const int *tok_seq_dev, const int *tok_pos_dev, uint32_t *status_dev, void *stream) {
    return ijb::rows_call<true>("ijb_kv_append", kv, src_type, const_cast<void *>(k_dev), const_cast<void *>(v_dev),
                                stride, n, tok_seq_dev, tok_pos_dev, status_dev, stream);
}

int ijb_kv_gather(const ijb_kv_view *kv, int dst_type, void *k_dev, void *v_dev, long stride, int n,
                  const int *tok_seq_dev, const int *tok_pos_dev, uint32_t *status_dev, void *stream) {
    return ijb::rows_call<false>("ijb_kv_gather", kv, dst_type, k_dev, v_dev, stride, n, tok_seq_dev, tok_pos_dev,
                                 status_dev, stream);
}

int ijb_kv_copy_pages(const ijb_kv_view *from, const ijb_kv_view *to, int n, const int *src_page_dev,
                      const int *dst_page_dev, uint32_t *status_dev, void *stream) {
    return ijb::copy_call("ijb_kv_copy_pages", from, to ? to : from, n, src_page_dev, dst_page_dev, status_dev, stream);
}

}  // extern "C"

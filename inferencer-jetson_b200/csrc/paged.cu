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
    if (v->type != IJB_KV_F16 && v->type != IJB_KV_E4M3) return "cache type must be IJB_KV_F16 or IJB_KV_E4M3";
    if (v->head_dim != 64 && v->head_dim != 128) return "head_dim must be 64 or 128";
    if (v->kv_heads < 1 || v->kv_heads > 1024) return "kv_heads must be 1..1024";
    if (v->page_size < 8 || v->page_size > 256 || (v->page_size & (v->page_size - 1)) != 0)
        return "page_size must be 8, 16, 32, 64, 128 or 256";
    if (v->num_pages < 1 || v->num_pages > 0x7fffffffL) return "num_pages must be 1..2^31 - 1";
    if (v->n_seqs < 1 || v->max_pages < 1 || static_cast<long>(v->max_pages) * v->page_size > 0x40000000L)
        return "n_seqs and max_pages must be positive, and max_pages * page_size at most 2^30";
    if (!v->data_dev || !v->page_table_dev) return "null cache data or page table";
    if (reinterpret_cast<uintptr_t>(v->data_dev) % 16 != 0) return "cache data must be 16-byte aligned";
    if (v->type == IJB_KV_E4M3 && !v->scale_dev) return "an e4m3 cache needs its scale bytes";
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
        const bool e4m3 = view->type == IJB_KV_E4M3;
        if (type == IJB_TYPE_F32)
            e4m3 ? rows_launch<APPEND, float, true>(p, vec, s) : rows_launch<APPEND, float, false>(p, vec, s);
        else
            e4m3 ? rows_launch<APPEND, __half, true>(p, vec, s) : rows_launch<APPEND, __half, false>(p, vec, s);
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

}  // extern "C"

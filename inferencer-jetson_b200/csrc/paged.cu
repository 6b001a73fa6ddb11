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
// Both kernels move bytes: 8 elements a thread, 16-byte loads and stores, a
// row per 8 (head_dim 64) or 16 threads.
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

// The cache row of token t (which, head); -1 when the entry is padding (a
// negative position) or names no slot, which is reported.
__device__ __forceinline__ long slot_row(const RowsParams &p, int t, int which, int head) {
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
    return kv_row(p.kv, page, which, head, pos & ((1 << p.kv.page_shift) - 1));
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

// Thread -> (token, K or V, head, 8 elements): rows of one token are
// consecutive, so a block reads whole tokens.
template <typename T, bool E4M3, bool VEC, int HD>
__global__ void __launch_bounds__(kRowThreads) ijb_kv_append_kernel(const __grid_constant__ RowsParams p) {
    constexpr int L = HD / 8;  // threads a row
    const long idx = blockIdx.x * static_cast<long>(kRowThreads) + threadIdx.x;
    const int c = static_cast<int>(idx % L);
    const long row = idx / L;
    const int per = 2 * p.kv.kv_heads;
    const bool live = row < static_cast<long>(p.n) * per;  // whole rows: uniform over a row's threads
    const int t = live ? static_cast<int>(row / per) : 0, r = static_cast<int>(row % per);
    const int which = r / p.kv.kv_heads, head = r % p.kv.kv_heads;
    float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    long to = -1;
    if (live) {
        const T *src = static_cast<const T *>(which ? p.v : p.k);
        load_row8<VEC>(src + t * p.stride + static_cast<long>(head) * HD + c * 8, f);
        to = slot_row(p, t, which, head);
    }
    if constexpr (E4M3) {
        float a = 0.f;  // over the finite values: an infinity saturates, a NaN stays one
#pragma unroll
        for (int i = 0; i < 8; ++i) a = fmaxf(a, fabsf(f[i]) <= 3.402823466e38f ? fabsf(f[i]) : 0.f);
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
        if (to < 0) return;
        // a = m 2^x with m in [1, 2): 448 = 1.75 * 2^8, so e = x - 8, one more when m > 1.75
        // (a below 2^-126 has x = -127 here and e ends at the floor)
        const uint32_t bits = __float_as_uint(a);
        int e = static_cast<int>(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
        e = max(e, -126);
        const float inv = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
        uint32_t w[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(f[4 * j] * inv, f[4 * j + 1] * inv),
                                                         __NV_SATFINITE, __NV_E4M3);
            const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(f[4 * j + 2] * inv, f[4 * j + 3] * inv),
                                                         __NV_SATFINITE, __NV_E4M3);
            w[j] = lo | (hi << 16);
        }
        *reinterpret_cast<uint2 *>(p.kv.data + to * HD + c * 8) = make_uint2(w[0], w[1]);
        if (c == 0) p.kv.scale[to] = static_cast<uint8_t>(e + 127);
    } else {
        if (to < 0) return;
        store_row8<true>(reinterpret_cast<__half *>(p.kv.data) + to * HD + c * 8, f);
    }
}

// Reads back: code * 2^e (exact in fp32), or the fp16 row; rows of padding
// entries and of entries that name no slot are left as they were.
template <typename T, bool E4M3, bool VEC, int HD>
__global__ void __launch_bounds__(kRowThreads) ijb_kv_gather_kernel(const __grid_constant__ RowsParams p) {
    constexpr int L = HD / 8;
    const long idx = blockIdx.x * static_cast<long>(kRowThreads) + threadIdx.x;
    const int c = static_cast<int>(idx % L);
    const long row = idx / L;
    const int per = 2 * p.kv.kv_heads;
    if (row >= static_cast<long>(p.n) * per) return;
    const int t = static_cast<int>(row / per), r = static_cast<int>(row % per);
    const int which = r / p.kv.kv_heads, head = r % p.kv.kv_heads;
    const long from = slot_row(p, t, which, head);
    if (from < 0) return;
    float f[8];
    if constexpr (E4M3) {
        const uint2 w = *reinterpret_cast<const uint2 *>(p.kv.data + from * HD + c * 8);
        const float s = kv_scale(p.kv.scale[from]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t u = j < 2 ? w.x : w.y;
            const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(u >> (16 * (j & 1))),
                                                             __NV_E4M3);
            const float2 v = __half22float2(*reinterpret_cast<const __half2 *>(&h));
            f[2 * j] = v.x * s;
            f[2 * j + 1] = v.y * s;
        }
    } else {
        load_row8<true>(reinterpret_cast<const __half *>(p.kv.data) + from * HD + c * 8, f);
    }
    T *dst = static_cast<T *>(which ? p.v : p.k);
    store_row8<VEC>(dst + t * p.stride + static_cast<long>(head) * HD + c * 8, f);
}

template <bool APPEND, typename T, bool E4M3, bool VEC, int HD>
void rows_launch(const RowsParams &p, cudaStream_t s) {
    const long threads = static_cast<long>(p.n) * 2 * p.kv.kv_heads * (HD / 8);
    const unsigned blocks = static_cast<unsigned>((threads + kRowThreads - 1) / kRowThreads);
    if constexpr (APPEND) ijb_kv_append_kernel<T, E4M3, VEC, HD><<<blocks, kRowThreads, 0, s>>>(p);
    else ijb_kv_gather_kernel<T, E4M3, VEC, HD><<<blocks, kRowThreads, 0, s>>>(p);
}
template <bool APPEND, typename T, bool E4M3>
void rows_launch(const RowsParams &p, bool vec, cudaStream_t s) {
    if (p.kv.head_dim == 64)
        vec ? rows_launch<APPEND, T, E4M3, true, 64>(p, s) : rows_launch<APPEND, T, E4M3, false, 64>(p, s);
    else
        vec ? rows_launch<APPEND, T, E4M3, true, 128>(p, s) : rows_launch<APPEND, T, E4M3, false, 128>(p, s);
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

// The paged K/V cache as the stand-alone operators see it: device view, row
// addressing, e4m3 rows and the argument checks they share (paged.cu,
// paged_attention.cu).
#pragma once
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <string>

#include "../../include/ijb200.h"
#include "common.cuh"
#include "misc.cuh"

namespace ijb {

// A row is one token's K or V of one KV head.  Rows of a page are laid out
// [K, V][kv head][position in page][head_dim]; the scale byte of an e4m3 row, or
// the head_dim / 32 of an e2m1 row, have the row's own index in the same order.
struct KvDev {
    uint8_t *data;
    uint8_t *scale;
    const int *page_table;
    int n_seqs, max_pages;
    int kv_heads, head_dim;
    int page_shift;  // log2 of the page size
    long num_pages;
};

// 2^(s - 127) of a scale byte (0..254).
__device__ __forceinline__ float kv_scale(uint32_t s) {
    return __uint_as_float(s ? s << 23 : 0x00400000u);
}

// e2m1 rows: two codes a byte, the even dim's in the low half; kKvBlock dims share a
// scale, the fp16 number of the bits byte << 7 (an unsigned number of 5 exponent and 3
// mantissa bits).  A code has 2 significant bits and a scale 4, so code * scale is an
// fp16 number as long as it is no larger than one: scales up to 10240 (byte kKvTopScale).
constexpr int kKvBlock = 32;
constexpr uint32_t kKvTopScale = 226u, kKvNanScale = 255u;

__host__ __device__ constexpr int kv_row_bytes(int type, int head_dim) {
    return type == IJB_KV_E2M1 ? head_dim / 2 : (type == IJB_KV_E4M3 ? head_dim : 2 * head_dim);
}

// The codes of one byte of u as two fp16 numbers, one instruction (`byte` is a constant); of all four as eight.
__device__ __forceinline__ uint32_t e2m1x2_half2(uint32_t u, int byte = 0) {
    uint32_t h;
    if (byte == 0)
        asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, a;\n\t}" : "=r"(h) : "r"(u));
    else if (byte == 1)
        asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, b;\n\t}" : "=r"(h) : "r"(u));
    else if (byte == 2)
        asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, c;\n\t}" : "=r"(h) : "r"(u));
    else
        asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, d;\n\t}" : "=r"(h) : "r"(u));
    return h;
}
__device__ __forceinline__ void e2m1x8_half2(uint32_t u, uint32_t (&h)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = e2m1x2_half2(u, i);
}

// Row index of (page, which, head, offset); 64 bits: a pool may pass 2^31 rows.
__device__ __forceinline__ long kv_row(const KvDev &kv, long page, int which, int head, int off) {
    return (((page * 2 + which) * kv.kv_heads + head) << kv.page_shift) + off;
}

// Entry-point helper: records `msg` for ijb_last_error(NULL) and returns code.
inline int kv_fail(int code, const char *fn, const std::string &msg) {
    set_thread_error(std::string(fn) + ": " + msg);
    return code;
}
// Checks a caller's view and fills the device view; returns an empty string, or what is wrong.
std::string kv_view_check(const ijb_kv_view *v, KvDev *out);
// Sets the attributes of ijb_paged_attention's fp32 kernels on the current device
// (done by the first call otherwise; an engine does it before it captures one).
cudaError_t paged_attention_prepare(int head_dim, int type);

}  // namespace ijb

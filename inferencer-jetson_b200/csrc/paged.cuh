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
// [K, V][kv head][position in page][head_dim]; the scale byte of an e4m3 row
// has the row's own index in the same order.
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
cudaError_t paged_attention_prepare(int head_dim, bool e4m3);

}  // namespace ijb

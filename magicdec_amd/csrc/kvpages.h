// Where a cache keeps a row, and the block-scaled formats (MD_KV_MXFP8, MD_KV_MXFP4): shared by the kernels that write, read and attend.
#pragma once
#include "md_common.h"

__host__ __device__ constexpr bool kv_is_mx(int kind) { return kind == MD_KV_MXFP8 || kind == MD_KV_MXFP4; }
__host__ __device__ constexpr int kv_element_bytes(int kind, int D) {            // a row's elements
    return kind == MD_KV_BF16 ? 2 * D : kind == MD_KV_MXFP4 ? D / 2 : D;
}
__host__ __device__ constexpr int kv_row_bytes(int kind, int D) { return kv_element_bytes(kind, D) + (kv_is_mx(kind) ? D / 32 : 0); }

// Byte distances inside a cache.  A row of a block-scaled cache keeps its scales behind the page_size rows of elements of its head.
struct KvPages {
    int64_t page, half;      // pages, K to V
    int head, slot;          // kv heads, rows
    int scales;              // from a head's first row to its first scale
};
inline KvPages kv_pages(int kind, int KH, int D, int page_size, bool hnd) {
    KvPages g;
    const int row = kv_row_bytes(kind, D), el = kv_element_bytes(kind, D);
    g.half = (int64_t)page_size * KH * row;
    g.page = 2 * g.half;
    g.head = hnd ? page_size * row : el;
    g.slot = hnd ? el : KH * el;
    g.scales = page_size * el;
    return g;
}

// tokens of a request; what its pages hold of them
__device__ __forceinline__ int kv_len_of(const int32_t* indptr, const int32_t* last, int b, int page_size, int* pg0, int* capacity) {
    const int p0 = indptr[b], np = indptr[b + 1] - p0;
    *pg0 = p0;
    *capacity = np > 0 ? np * page_size : 0;
    return np > 0 ? (np - 1) * page_size + last[b] : 0;
}

// 8 (MD_KV_MXFP4: `x` = 4 bytes), or 4 (8-bit elements) numbers to bf16 pairs, times a power of two: exact (v_cvt_scalef32 keeps subnormal
// results, and a scale of exponent 255 makes NaN)
__device__ __forceinline__ void mx4_to_bf16(unsigned x, float scale, unsigned (&y)[4]) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, scale, 1);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, scale, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, scale, 3);
    y[0] = __builtin_bit_cast(unsigned, a);
    y[1] = __builtin_bit_cast(unsigned, b);
    y[2] = __builtin_bit_cast(unsigned, c);
    y[3] = __builtin_bit_cast(unsigned, d);
}
__device__ __forceinline__ void mx8_to_bf16(unsigned x, float scale, unsigned& lo, unsigned& hi) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, scale, true);
    lo = __builtin_bit_cast(unsigned, a);
    hi = __builtin_bit_cast(unsigned, b);
}
__device__ __forceinline__ float mx_scale(unsigned byte) { return __uint_as_float(byte << 23); }      // 2^(byte - 127); 255: infinity, a NaN to the above

// md_append_paged_kv (cos_sin = null: no queries, no rotation) and md_rope_append over a block-scaled cache (kvpages.hip); `what` names the caller
int md_mx_append(const void* q, const void* k, const void* v, int64_t qs, int64_t ks, int64_t vs, void* q_out, const int32_t* indptr,
                 const int32_t* offsets, int B, int n_max, int H, int KH, int D, const float* cos_sin, int max_pos, void* cache,
                 const int32_t* indices, const int32_t* page_indptr, const int32_t* last, void* cache2, const int32_t* indices2,
                 const int32_t* page_indptr2, const int32_t* last2, int page_size, int kv_dtype, hipStream_t stream, const char* what);

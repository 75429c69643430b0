// Attention over the pages of any cache with a sliding window and first tokens that stay visible (md_window_attn): what its kernels share.
#pragma once
#include "attn_common.h"
#include "kvpages.h"

typedef float f32x16 __attribute__((ext_vector_type(16)));

struct WinParams {
    const bf16_t* q;
    const unsigned char* cache;
    bf16_t* out;
    const int32_t *qo_indptr, *indices, *indptr, *last;
    float *ws_o, *ws_ml;        // of the splits of a row's keys: weighted sums; reference and weight
    int64_t q_row_stride;       // elements
    KvPages g;
    int B, H, KH, group, page_size, nsplit, n_qgroups;
    int window, sinks;          // 0: no window
    float scale_log2;
    const float *k_scale, *v_scale;      // MD_KV_FP8_E4M3
};

// Workgroup -> a (request, kv head) and which of its `of` pieces of work.  Neighbouring workgroups run on different XCDs, those that differ by multiples of
// 8 on one: the pieces of a pair share an XCD's L2, eight pairs at a time.  Of what is left over the pieces lie over all XCDs: on one XCD each, one
// request of 3 764 tokens x 4 heads with a window of 10 28 us, over all 17; 31 965 keys x 1 head for 2 requests 22.9 and 16.6.
__device__ __forceinline__ int win_pair(const WinParams& p, int of, int& sub) {
    const int pairs = p.B * p.KH, whole = pairs & ~7, w = blockIdx.x;
    if (w < whole * of) {
        sub = (w >> 3) % of;
        return ((w >> 3) / of) * 8 + (w & 7);
    }
    const int rest = pairs - whole, t = w - whole * of;
    sub = t / rest;
    return whole + t % rest;
}

constexpr float kLowest = -3.402823466e38f;      // reference of a row without a key: finite, so that differences are no NaN

// MD_KV_FP8_E4M3: the keys' scale is part of the scores' factor, which has to be above 0: a hidden score is -infinity times it, and the largest score is the
// largest before it.  So its size goes there, and its sign to the queries.
__device__ __forceinline__ float size_of_scale(float scale_log2, float k_scale) { return fmaxf(scale_log2 * fabsf(k_scale), 1.17549435e-38f); }
__device__ __forceinline__ bf16x8 with_sign_of(float k_scale, bf16x8 q) {
    const unsigned flip = k_scale < 0.f ? 0x80008000u : 0u;
    return __builtin_bit_cast(bf16x8, __builtin_bit_cast(u32x4, q) ^ u32x4{flip, flip, flip, flip});
}

// Largest of lanes l and l ^ 16, of l and l ^ 32: swaps of 16 and of 32 lanes, no LDS
__device__ __forceinline__ float max_over_16(float x) {
    const unsigned u = __builtin_bit_cast(unsigned, x);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const unsigned a = r[0], b = r[1];
    return fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}
__device__ __forceinline__ float max_over_32(float x) {
    const unsigned u = __builtin_bit_cast(unsigned, x);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const unsigned a = r[0], b = r[1];
    return fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}

// Bits of the halves of a bf16 pair that are infinite or NaN
__device__ __forceinline__ unsigned nonfinite_halves(unsigned u) {
    const unsigned t = ((u & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
    return (t - (t >> 15)) | t;
}
// 1 (bf16) in the halves that are infinite or NaN and not the infinity of the other sign
__device__ __forceinline__ unsigned infinite_halves(unsigned u, bool negative) {
    const unsigned other = negative ? 0x7f80u : 0xff80u;
    unsigned m = nonfinite_halves(u);
    if ((u & 0xffffu) == other) m &= 0xffff0000u;
    if ((u >> 16) == other) m &= 0xffffu;
    return m & 0x3f803f80u;
}

// Weights are exp2(score * factor - reference) in one operation, whose exponent is off by at most 2^-24 of the reference; beyond 2^12 scores are
// rounded in front of it, so that the largest one's weight is 1 however large it is.
template <int N>
__device__ __forceinline__ float exponent_factor(float m, float factor, float (&v)[N]) {
    if (__builtin_amdgcn_ballot_w64(fabsf(m) > 4096.f && m != kLowest) == 0) return factor;
#pragma unroll
    for (int e = 0; e < N; ++e) {
        float x = v[e] * factor;
        asm volatile("" : "+v"(x));          // a branch of the wavefront, not a select
        v[e] = x;
    }
    return 1.0f;
}

// Tiles of KT keys that rows between the positions lo and hi look at: those of the first tokens, then those from the lowest window on
struct Tiles {
    int first, w0, count;       // tiles of the first tokens, the window's first tile, tiles in all
    __device__ __forceinline__ Tiles(int lo, int end, int window, int sinks, int kt) {
        w0 = window > 0 ? max(lo - window + 1, 0) / kt : 0;
        first = min(w0, (min(sinks, end) + kt - 1) / kt);
        count = end > 0 ? first + max((end + kt - 1) / kt - w0, 0) : 0;
    }
    __device__ __forceinline__ int at(int i) const { return i < first ? i : i - first + w0; }
};

// Where a wavefront is in a request's pages: the numbers of 64 of them, one a lane, so that a tile waits for no number of its page.
struct PageCursor {
    const int32_t* list;
    int count, size, base, ids;          // pages of the request, rows of a page; first page that `ids` holds
    int first, page, slot;               // position, number in the request, and row in it
    __device__ __forceinline__ PageCursor(const WinParams& p, int pg0, int room)
        : list(p.indices + pg0), count(room / p.page_size), size(p.page_size), base(-64), ids(0), first(0), page(0), slot(0) {}
    // to position pos, of a page of the request; anywhere, and cheaply where it is less than two pages on
    __device__ __forceinline__ void seek(int pos) {
        slot = pos - first;
        if (slot < 0 || slot >= 2 * size) {
            page = pos / size;
            first = page * size;
            slot = pos - first;
        } else if (slot >= size) {
            ++page;
            first += size;
            slot -= size;
        }
        if (page < base || page >= base + 64) {
            base = page;
            ids = list[min(page + (int)(threadIdx.x & 63), count - 1)];
            asm volatile("" : "+v"(ids));         // waited for here: behind the branch it would be in every tile
        }
    }
    __device__ __forceinline__ int64_t id() const { return __builtin_amdgcn_readlane(ids, page - base); }
};

// winprompt.hip, an object each: calls of more than 32 rows, in workgroups of nw (4 or 8) wavefronts of 32, on tiles of as many keys as divide a page
inline int window_prompt_tile(int D, int nw, int page_size) {
    const int keys = D == 128 && nw == 8 ? 128 : 64;
    return page_size % keys == 0 ? keys : 32;
}
int md_window_prompt_0(const WinParams& p, int D, int nw, int grid, hipStream_t st);      // MD_KV_BF16
int md_window_prompt_1(const WinParams& p, int D, int nw, int grid, hipStream_t st);      // MD_KV_FP8_E4M3
int md_window_prompt_2(const WinParams& p, int D, int nw, int grid, hipStream_t st);      // MD_KV_MXFP8
int md_window_prompt_3(const WinParams& p, int D, int nw, int grid, hipStream_t st);      // MD_KV_MXFP4

// Block-scaled KV pages: rows quantised as they are written (md_append_paged_kv and md_rope_append of MD_KV_MXFP8 / MD_KV_MXFP4), and rows of
// any cache read back (md_read_paged_kv).
//
// A block is 32 consecutive elements of a row.  With 2^e <= amax < 2^(e+1) its largest element and m = amax / 2^e, its scale is
//     2^(e - 8 + (m > 1.8125))  of e4m3 elements (largest 448 = 1.75 * 2^8; what lies up to 464 rounds to it),
//     2^(e - 2 + (m > 1.75))    of e2m1 elements (largest 6 = 1.5 * 2^2; up to 7):
// the smallest at which no element is off by more than half a step of its binade.  The bf16 bits of amax plus 127 - (bits of that m) carry into
// the exponent exactly where m is larger, so the stored byte takes three integer operations.  v_cvt_scalef32 divides by it and rounds to nearest
// even; both are exact but for that rounding, because the scale is a power of two.
//
// Both directions are bound by HBM for prompts and by latency for steps.  A lane holds 8 elements, so a quad of lanes is a block and its
// largest element takes two quad permutations.  A wavefront holds 4 rows of 128 (8 of 64) of one head at a time and goes through heads: the
// rows' cos / sin, their pages and their slots are looked up once for all of them, and the 4 wavefronts of a workgroup hold neighbouring rows,
// whose elements and scales lie side by side in a page, so that no line is written from two XCDs' caches but at a workgroup's ends.
//
// 64 x 128 rows of 32 + 8 + 8 heads of 128, rotated and quantised to 4 bits, take 31 us (177 MB in and out, 5.7 TB/s) and 9 to read back; 8 x 16 032 rows of 4-bit
// pages read back 131 us (665 MB, 5.0 TB/s: what a copy reaches); 256 rows 4.0 and 2.9, a launch's length.
#include "kvpages.h"

#include <algorithm>

unsigned int* md_page_overflow_counter_device();

namespace {

struct RowsParams {
    const bf16_t *q, *k, *v;
    int64_t qs, ks, vs;                 // row strides, elements
    bf16_t *q_out, *k_out, *v_out;
    const int32_t *indptr, *offsets;    // rows of a request; its first position (rotation)
    const float* cos_sin;
    unsigned char* cache;
    const int32_t *indices, *page_indptr, *last;
    bf16_t* cache2;                     // a second, 16-bit cache of pages [2][page][KH][D] that takes the same rows
    const int32_t *indices2, *page_indptr2, *last2;
    const float *k_scale, *v_scale;     // MD_KV_FP8_E4M3
    unsigned int* dropped;
    KvPages g;
    int H, KH, page_size, max_pos;
    int wr, per;                        // wavefronts of a workgroup along the rows; heads a wavefront goes through
};

// 8 elements in pairs to a block-scaled row's elements; the quad's scale byte
template <bool FP4>
__device__ __forceinline__ unsigned mx_quantize(const u32x4 x, unsigned (&y)[2]) {
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    bf16x2 pair[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const unsigned u = x[w];
        pair[w] = __builtin_bit_cast(bf16x2, u);
    }
    u16x2 a = {0, 0};
#pragma unroll
    for (int w = 0; w < 4; ++w) a = __builtin_elementwise_max(a, __builtin_bit_cast(u16x2, x[w] & 0x7fff7fffu));
    int amax = max((int)a[0], (int)a[1]);
    amax = max(amax, __builtin_amdgcn_mov_dpp(amax, 0xB1, 0xf, 0xf, true));       // quad_perm [1, 0, 3, 2]
    amax = max(amax, __builtin_amdgcn_mov_dpp(amax, 0x4E, 0xf, 0xf, true));       // quad_perm [2, 3, 0, 1]
    constexpr int kBinade = FP4 ? 2 : 8, kCarry = 127 - (FP4 ? 96 : 104);
    // from 2^-100, where no conversion is near a subnormal number, up to what the largest finite element takes
    const int byte = min(max(((amax + kCarry) >> 7) - kBinade, 27), 254 - kBinade);
    const bool finite = amax < 0x7f80;
    const float scale = mx_scale(byte);
    if constexpr (FP4) {                                                          // (saturates by itself)
        unsigned r = 0;
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, pair[0], scale, 0);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, pair[1], scale, 1);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, pair[2], scale, 2);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, pair[3], scale, 3);
        y[0] = finite ? r : 0;
    } else {
        typedef short s16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            s16x2 r = {0, 0};
            r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, pair[2 * h], scale, false);
            r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, pair[2 * h + 1], scale, true);
            // beyond 464 (only where the scale is the largest) the conversion gives NaN, 0x7f: the largest number is 0x7e
            const unsigned u = __builtin_bit_cast(unsigned, r);
            y[h] = finite ? u - ((((u & 0x7f7f7f7fu) + 0x01010101u) >> 7) & 0x01010101u) : 0;
        }
    }
    return finite ? byte : 255;
}

// 4 interleaved pairs rotated, every product and sum rounded by itself (as md_rope)
__device__ __forceinline__ u32x4 turn8(const u32x4 x, const f32x4 c0, const f32x4 c1) {
    u32x4 r;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const float xe = __uint_as_float(x[w] << 16), xo = __uint_as_float(x[w] & 0xffff0000u);
        const float co = w < 2 ? c0[(w & 1) * 2] : c1[(w & 1) * 2], si = w < 2 ? c0[(w & 1) * 2 + 1] : c1[(w & 1) * 2 + 1];
        const bf16x2 pk = {f32_to_bf16(__fsub_rn(__fmul_rn(xe, co), __fmul_rn(xo, si))), f32_to_bf16(__fadd_rn(__fmul_rn(xo, co), __fmul_rn(xe, si)))};
        r[w] = __builtin_bit_cast(unsigned, pk);
    }
    return r;
}

// What a lane knows of its row, whatever the head.
template <int D>
struct Lane {
    static constexpr int kChunks = D / 8, kRows = 64 / kChunks;
    int c, j, b, n, a0, unit;
    bool live;
    __device__ __forceinline__ bool init(const RowsParams& p) {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        b = blockIdx.y;
        a0 = p.indptr[b];
        n = p.indptr[b + 1] - a0;
        const int first = (blockIdx.x * p.wr + wave % p.wr) * kRows;
        if (first >= n) return false;
        c = lane % kChunks;
        j = first + lane / kChunks;
        live = j < n;
        unit = blockIdx.z * (4 / p.wr) + wave / p.wr;
        return true;
    }
};

template <int D, bool FP4, bool ROPE>
__global__ __launch_bounds__(256) void mx_append_kernel(const RowsParams p) {
    constexpr int kEl = FP4 ? D / 2 : D;
    Lane<D> at;
    if (!at.init(p)) return;
    const int slots = (ROPE ? p.H : 0) + 2 * p.KH, s0 = at.unit * p.per, s1 = min(slots, s0 + p.per);
    if (s0 >= slots) return;
    const int64_t row = at.a0 + (at.live ? at.j : 0);
    // slots: H query heads, KH key heads, KH value heads
    const int kfirst = ROPE ? p.H : 0, vfirst = kfirst + p.KH;
    auto source = [&](int s) {
        const bf16_t* x = s < kfirst ? p.q + row * p.qs + s * D : s < vfirst ? p.k + row * p.ks + (s - kfirst) * D : p.v + row * p.vs + (s - vfirst) * D;
        return *reinterpret_cast<const u32x4*>(x + at.c * 8);
    };
    u32x4 next = source(s0);
    int pg0, room, pg2 = 0, room2 = 0;
    const int pos = kv_len_of(p.page_indptr, p.last, at.b, p.page_size, &pg0, &room) - at.n + at.j;
    const bool over = at.live && pos >= room, ok = at.live && pos >= 0 && !over;
    const int page = ok ? pos / p.page_size : 0, slot = ok ? pos - page * p.page_size : 0;
    unsigned char* to = p.cache + (ok ? (int64_t)p.indices[pg0 + page] * p.g.page : 0);
    bool ok2 = false, over2 = false;
    bf16_t* to2 = p.cache2;
    if (p.cache2) {
        const int pos2 = kv_len_of(p.page_indptr2, p.last2, at.b, p.page_size, &pg2, &room2) - at.n + at.j;
        over2 = at.live && pos2 >= room2;
        ok2 = at.live && pos2 >= 0 && !over2;
        if (ok2) {
            const int page2 = pos2 / p.page_size;
            to2 += ((int64_t)p.indices2[pg2 + page2] * 2 * p.page_size + (pos2 - page2 * p.page_size)) * (int64_t)(p.KH * D);
        }
    }
    f32x4 c0 = {0.f, 0.f, 0.f, 0.f}, c1 = c0;
    if constexpr (ROPE) {
        const int turn = p.offsets[at.b] + at.j;
        const float* cs = p.cos_sin + (int64_t)min(max(turn, 0), p.max_pos - 1) * D + at.c * 8;
        c0 = *reinterpret_cast<const f32x4*>(cs);
        c1 = *reinterpret_cast<const f32x4*>(cs + 4);
    }
    for (int s = s0; s < s1; ++s) {
        u32x4 x = next;
        if (s + 1 < s1) next = source(s + 1);
        if (ROPE && s < vfirst) x = turn8(x, c0, c1);
        if (s < kfirst) {
            if (at.live) *reinterpret_cast<u32x4*>(p.q_out + (row * p.H + s) * D + at.c * 8) = x;
            continue;
        }
        const bool v = s >= vfirst;
        const int h = s - (v ? vfirst : kfirst);
        unsigned y[2];
        const unsigned scale = mx_quantize<FP4>(x, y);
        if (ok) {
            unsigned char* head = to + (v ? p.g.half : 0) + (int64_t)h * p.g.head;
            if constexpr (FP4)
                *reinterpret_cast<unsigned*>(head + slot * kEl + at.c * 4) = y[0];
            else
                *reinterpret_cast<u32x2*>(head + slot * kEl + at.c * 8) = u32x2{y[0], y[1]};
            if ((at.c & 3) == 0) head[p.g.scales + slot * (D / 32) + (at.c >> 2)] = (unsigned char)scale;
        }
        if (ok2) *reinterpret_cast<u32x4*>(to2 + (v ? (int64_t)p.page_size * p.KH * D : 0) + h * D + at.c * 8) = x;
        if (!v && h == 0 && at.c == 0 && (over || over2)) atomicAdd(p.dropped, (unsigned)over + (unsigned)over2);
    }
}

template <int D, int KIND>
__global__ __launch_bounds__(256) void read_kernel(const RowsParams p) {
    constexpr int kEl = kv_element_bytes(KIND, 8);                // bytes of a lane's 8 elements
    Lane<D> at;
    if (!at.init(p)) return;
    const int s0 = at.unit * p.per, s1 = min(2 * p.KH, s0 + p.per);
    if (s0 >= 2 * p.KH) return;
    int pg0, room;
    const int pos = kv_len_of(p.page_indptr, p.last, at.b, p.page_size, &pg0, &room) - at.n + at.j;
    const bool ok = at.live && pos >= 0 && pos < room;
    const int page = ok ? pos / p.page_size : 0, slot = ok ? pos - page * p.page_size : 0;
    if (!ok) return;
    const unsigned char* from = p.cache + (int64_t)p.indices[pg0 + page] * p.g.page;
    const int64_t row = at.a0 + at.j;
#pragma unroll 4
    for (int s = s0; s < s1; ++s) {
        const bool v = s >= p.KH;
        const int h = s - (v ? p.KH : 0);
        const unsigned char* head = from + (v ? p.g.half : 0) + (int64_t)h * p.g.head;
        const unsigned char* el = head + (int64_t)slot * p.g.slot + at.c * kEl;
        u32x4 y;
        if constexpr (KIND == MD_KV_BF16) {
            y = *reinterpret_cast<const u32x4*>(el);
        } else if constexpr (KIND == MD_KV_MXFP4) {
            unsigned t[4];
            mx4_to_bf16(*reinterpret_cast<const unsigned*>(el), mx_scale(head[p.g.scales + slot * (D / 32) + (at.c >> 2)]), t);
            y = u32x4{t[0], t[1], t[2], t[3]};
        } else {
            const u32x2 x = *reinterpret_cast<const u32x2*>(el);
            const float scale = KIND == MD_KV_MXFP8 ? mx_scale(head[p.g.scales + slot * (D / 32) + (at.c >> 2)]) : 1.f;
            unsigned t[4];
            mx8_to_bf16(x[0], scale, t[0], t[1]);
            mx8_to_bf16(x[1], scale, t[2], t[3]);
            if constexpr (KIND == MD_KV_FP8_E4M3) {
                const float sc = v ? p.v_scale[h] : p.k_scale[h];
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const bf16x2 pk = {f32_to_bf16(__uint_as_float(t[w] << 16) * sc), f32_to_bf16(__uint_as_float(t[w] & 0xffff0000u) * sc)};
                    t[w] = __builtin_bit_cast(unsigned, pk);
                }
            }
            y = u32x4{t[0], t[1], t[2], t[3]};
        }
        *reinterpret_cast<u32x4*>((v ? p.v_out + row * p.vs : p.k_out + row * p.ks) + h * D + at.c * 8) = y;
    }
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// Rows to wavefronts: as many of a workgroup's along the rows as there are rows for, the others along the heads; heads one after another in a
// wavefront once every CU has sixteen of them.
dim3 rows_grid(RowsParams& p, int D, int B, int n_max, int slots) {
    const int rows = 64 / (D / 8), groups = (n_max + rows - 1) / rows;
    p.wr = groups >= 4 ? 4 : groups >= 2 ? 2 : 1;
    const int64_t waves = (int64_t)groups * B * slots;
    p.per = (int)std::min<int64_t>({std::max<int64_t>(waves / 4096, 1), 8, slots});
    const int units = (slots + p.per - 1) / p.per, each = 4 / p.wr;
    return dim3((groups + p.wr - 1) / p.wr, B, (units + each - 1) / each);
}

}  // namespace

int md_mx_append(const void* q, const void* k, const void* v, int64_t qs, int64_t ks, int64_t vs, void* q_out, const int32_t* indptr,
                 const int32_t* offsets, int B, int n_max, int H, int KH, int D, const float* cos_sin, int max_pos, void* cache,
                 const int32_t* indices, const int32_t* page_indptr, const int32_t* last, void* cache2, const int32_t* indices2,
                 const int32_t* page_indptr2, const int32_t* last2, int page_size, int kv_dtype, hipStream_t stream, const char* what) {
    const int kind = kv_dtype & MD_KV_DTYPE_MASK;
    MD_CHECK_ARG(kv_dtype & MD_KV_LAYOUT_HND, "%s: block-scaled pages are HND", what);
    MD_CHECK_ARG(B <= 65535 && n_max <= 1 << 30 && H >= 0 && page_size % 32 == 0 && page_size <= 65536,
                 "%s: bad shape B=%d n_max=%d H=%d page_size=%d (pages of multiples of 32 rows, to 65 536)", what, B, n_max, H, page_size);
    if (D != 64 && D != 128) {
        md_set_error("%s: head_dim %d of a block-scaled cache unsupported (64 or 128)", what, D);
        return MD_ERR_UNSUPPORTED;
    }
    RowsParams p = {};
    p.dropped = md_page_overflow_counter_device();
    if (!p.dropped) {
        md_set_error("%s: cannot resolve the dropped-row counter", what);
        return MD_ERR_LAUNCH;
    }
    p.q = (const bf16_t*)q;
    p.k = (const bf16_t*)k;
    p.v = (const bf16_t*)v;
    p.qs = qs;
    p.ks = ks;
    p.vs = vs;
    p.q_out = (bf16_t*)q_out;
    p.indptr = indptr;
    p.offsets = offsets;
    p.cos_sin = cos_sin;
    p.cache = (unsigned char*)cache;
    p.indices = indices;
    p.page_indptr = page_indptr;
    p.last = last;
    p.cache2 = (bf16_t*)cache2;
    p.indices2 = indices2;
    p.page_indptr2 = page_indptr2;
    p.last2 = last2;
    p.g = kv_pages(kind, KH, D, page_size, true);
    p.H = H;
    p.KH = KH;
    p.page_size = page_size;
    p.max_pos = max_pos;
    const dim3 grid = rows_grid(p, D, B, n_max, H + 2 * KH);
    const auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, p); };
    const bool fp4 = kind == MD_KV_MXFP4, turn = cos_sin != nullptr;
    if (D == 128)
        launch(fp4 ? turn ? mx_append_kernel<128, true, true> : mx_append_kernel<128, true, false>
                   : turn ? mx_append_kernel<128, false, true> : mx_append_kernel<128, false, false>);
    else
        launch(fp4 ? turn ? mx_append_kernel<64, true, true> : mx_append_kernel<64, true, false>
                   : turn ? mx_append_kernel<64, false, true> : mx_append_kernel<64, false, false>);
    MD_CHECK_LAUNCH(what);
    return MD_OK;
}

extern "C" size_t md_kv_row_bytes(int kv_dtype, int D) {
    const int kind = kv_dtype & MD_KV_DTYPE_MASK;
    return (D == 64 || D == 128) && kind <= MD_KV_MXFP4 ? kv_row_bytes(kind, D) : 0;
}

extern "C" int md_read_paged_kv(void* k_out, void* v_out, int64_t k_row_stride, int64_t v_row_stride, const int32_t* indptr, const void* cache,
                                const int32_t* page_indices, const int32_t* page_indptr, const int32_t* last_page_len, int B, int n_max, int KH,
                                int D, int page_size, int kv_dtype, const float* k_scale, const float* v_scale, md_stream_t stream) {
    MD_CHECK_ARG(k_out && v_out && indptr && cache && page_indices && page_indptr && last_page_len, "md_read_paged_kv: null pointer argument");
    MD_CHECK_ARG(B > 0 && B <= 65535 && n_max > 0 && n_max <= 1 << 30 && KH > 0 && page_size > 0 && page_size % 32 == 0 && page_size <= 65536,
                 "md_read_paged_kv: bad shape B=%d n_max=%d KH=%d page_size=%d (pages of multiples of 32 rows, to 65 536)", B, n_max, KH, page_size);
    if (D != 64 && D != 128) {
        md_set_error("md_read_paged_kv: head_dim %d unsupported (64 or 128)", D);
        return MD_ERR_UNSUPPORTED;
    }
    MD_CHECK_ARG((kv_dtype & ~(MD_KV_DTYPE_MASK | MD_KV_LAYOUT_HND)) == 0, "md_read_paged_kv: unknown kv_dtype flags");
    const bool hnd = (kv_dtype & MD_KV_LAYOUT_HND) != 0;
    const int kind = kv_dtype & MD_KV_DTYPE_MASK;
    MD_CHECK_ARG(kind <= MD_KV_MXFP4 && (kind != MD_KV_FP8_E4M3 || (k_scale && v_scale)),
                 "md_read_paged_kv: kv_dtype must be MD_KV_BF16, MD_KV_FP8_E4M3 (with per-head scales), MD_KV_MXFP8 or MD_KV_MXFP4");
    MD_CHECK_ARG(hnd || !kv_is_mx(kind), "md_read_paged_kv: block-scaled pages are HND");
    MD_CHECK_ARG(aligned16(k_out) && aligned16(v_out) && aligned16(cache) && k_row_stride % 8 == 0 && v_row_stride % 8 == 0,
                 "md_read_paged_kv: k_out/v_out/cache must be 16-byte aligned, row strides multiples of 8");
    RowsParams p = {};
    p.k_out = (bf16_t*)k_out;
    p.v_out = (bf16_t*)v_out;
    p.ks = k_row_stride;
    p.vs = v_row_stride;
    p.indptr = indptr;
    p.cache = (unsigned char*)const_cast<void*>(cache);
    p.indices = page_indices;
    p.page_indptr = page_indptr;
    p.last = last_page_len;
    p.k_scale = k_scale;
    p.v_scale = v_scale;
    p.g = kv_pages(kind, KH, D, page_size, hnd);
    p.KH = KH;
    p.page_size = page_size;
    const dim3 grid = rows_grid(p, D, B, n_max, 2 * KH);
    const auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, (hipStream_t)stream, p); };
    if (kind == MD_KV_BF16)
        launch(D == 128 ? read_kernel<128, MD_KV_BF16> : read_kernel<64, MD_KV_BF16>);
    else if (kind == MD_KV_FP8_E4M3)
        launch(D == 128 ? read_kernel<128, MD_KV_FP8_E4M3> : read_kernel<64, MD_KV_FP8_E4M3>);
    else if (kind == MD_KV_MXFP8)
        launch(D == 128 ? read_kernel<128, MD_KV_MXFP8> : read_kernel<64, MD_KV_MXFP8>);
    else
        launch(D == 128 ? read_kernel<128, MD_KV_MXFP4> : read_kernel<64, MD_KV_MXFP4>);
    MD_CHECK_LAUNCH("md_read_paged_kv");
    return MD_OK;
}

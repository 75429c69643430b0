// md_window_attn of more than 32 rows (query heads of a kv head x new tokens): a prompt's portion, bound by the matrix instructions.
//
// A workgroup of NW wavefronts, 32 query rows each, shares tiles of KT keys: read once, converted to bf16 once, into LDS images that two
// v_mfma_f32_32x32x16_bf16 products read, S^T = K Q^T and O^T = V^T P^T.  The accumulator registers of the first are the operand of the second as
// they lie, a query's statistics are in two lanes.  Images alternate, so that a tile costs one barrier: tile t + 2 overwrites tile t's behind
// the barrier of t + 1.  The workgroup walks the tiles that any of its rows sees; a wavefront leaves out those that none of its own does.
//
// Weights are exp2(score * scale - reference) in one fused operation, whose exponent is off by at most 2^-24 of the reference.  Beyond 2^12
// scores are rounded before the reference comes off them, so that the largest one's weight is 1 however large it is.
//
// Infinite values and NaN in tiles that hide a key from some row: as in winattn.hip, by all wavefronts together.
//
// 128 rows a request x 16 requests behind 16 032 keys (8-bit pages, 4 query heads of 128 on each of 8) take 550 to 557 us, 975 TFLOP/s: matrix cores and vector
// instructions each in 46 % of the cycles, mostly in turn, at 2.0 GHz (the power limit; a library product of 8 192^3 reaches 1 189).  Prompts of 2 x 4 133
// tokens with a window of 1 024 196 to 204 us, 610 TFLOP/s of the weights that count: a tenth more keys than a group's windows hold, and the first tile of each of
// four rounds of workgroups, one a CU (eight wavefronts of 256 registers, 137 KB of images).  Tiles of 32-key blocks (555 -> 610), masked and unmasked
// tiles in a body each (spills), two tiles in flight (bf16 to 1.5 times the time) and half of the wavefronts half a tile behind the others, so that
// one's products run beside the other's exponentials (545 -> 575 to 620), were slower.
#include "winattn.h"

#include <algorithm>

#ifndef MD_WIN_KIND
#error "MD_WIN_KIND: the cache's element type"
#endif

namespace {

template <int D, int KT>
__host__ __device__ constexpr int prompt_image_bytes() {
    return KT * (D * 2 + 16) + (KT / 32) * (D / 16) * kVSub;
}

template <int D, int NW, int KT, int KIND>
__global__ __launch_bounds__(64 * NW, D == 64 ? 4 : 2) void window_prompt_kernel(const WinParams p) {
    constexpr int EB = kv_element_bytes(KIND, D);
    constexpr bool MX = kv_is_mx(KIND);
    constexpr int KG = KT / 32, KS = D / 16, NB = D / 16, DB = D / 32, SB = D / 32;
    constexpr int CH = EB / 16, RPI = 64 / CH;                   // 16-byte pieces of a row, rows of a wavefront's load
    constexpr int NL = KT / RPI, NLW = (NL + NW - 1) / NW;        // loads of a tile, of a wavefront
    constexpr int PIECE = KIND == MD_KV_BF16 ? 8 : KIND == MD_KV_MXFP4 ? 32 : 16;      // elements of a piece
    constexpr int KROW = D * 2 + 16, K_BYTES = KT * KROW, VG = NB * kVSub, IMAGE = prompt_image_bytes<D, KT>();

    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];      // 2 images; [2][NW]: does an image have infinite values
    int* s_infinite = reinterpret_cast<int*>(smem + 2 * IMAGE);
    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lane = tid & 63;
    const int j = lane & 31, kh = lane >> 5;

    int sub;
    const int pair = win_pair(p, p.n_qgroups * p.nsplit, sub), split = sub % p.nsplit;
    const int qg = p.n_qgroups - 1 - sub / p.nsplit;             // the last rows, with the most keys, first
    const int b = pair / p.KH, kvh = pair % p.KH, g = p.group;
    const int q0 = p.qo_indptr[b], n_b = p.qo_indptr[b + 1] - q0, nrows = n_b * g;
    if (qg * NW * 32 >= nrows) return;
    int pg0, room;
    const int kv_len = min(kv_len_of(p.indptr, p.last, b, p.page_size, &pg0, &room), room);
    const int R = (qg * NW + wave) * 32 + j;
    const bool valid = R < nrows;
    const int qi = R / g, qr = R - qi * g;
    const int lim = valid ? kv_len - n_b + qi : -1, low = p.window > 0 ? lim - p.window : -1;
    // lo, hi: of the wavefront's first and last row; of the workgroup's
    const int first = qg * NW * 32, last = min(first + NW * 32, nrows) - 1, first_w = first + wave * 32, last_w = min(first_w + 32, nrows) - 1;
    const int lo_all = kv_len - n_b + first / g, hi_all = kv_len - n_b + last / g;
    const int lo = first_w <= last_w ? kv_len - n_b + first_w / g : 0x7fffffff, hi = first_w <= last_w ? kv_len - n_b + last_w / g : -1;
    const Tiles tiles(lo_all, min(hi_all + 1, kv_len), p.window, p.sinks, KT);
    const int per = (tiles.count + p.nsplit - 1) / p.nsplit, t_begin = split * per, t_end = min(tiles.count, t_begin + per);
    // does a tile that begins at `pos` hide a key from a row between two positions; does any of them see one
    auto hides = [&](int pos, int first, int last) {
        return pos + KT - 1 > first || (p.window > 0 && pos <= last - p.window && pos + KT - 1 >= p.sinks);
    };
    auto sees = [&](int pos) { return pos <= hi && (p.window <= 0 || pos + KT - 1 > lo - p.window || pos < p.sinks); };

    bf16x8 qf[KS];
    const float ksc = KIND == MD_KV_FP8_E4M3 ? p.k_scale[kvh] : 1.0f;
    const float sl2 = KIND == MD_KV_FP8_E4M3 ? size_of_scale(p.scale_log2, ksc) : p.scale_log2;
    f32x16 o[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[db][r] = 0.f;
    float m = kLowest, l = 0.f;

    // staging: wavefront w takes the loads w, w + NW ... of a tile
    const int wrow = lane / CH, wch = lane % CH;
    const unsigned goff = (unsigned)(wrow * p.g.slot + wch * 16);
    u32x4 kreg[NLW], vreg[NLW];
    unsigned kscale[NLW], vscale[NLW];
    PageCursor at(p, pg0, room);
    auto tile_base = [&](int pos) {
        at.seek(pos);
        return p.cache + at.id() * p.g.page + (int64_t)kvh * p.g.head;
    };
    auto load = [&](const unsigned char* head, int slot0, int s, u32x4& x, unsigned& scale) {
        const int first = (wave + NW * s) * RPI;
        x = *reinterpret_cast<const u32x4*>(head + (int64_t)(slot0 + first) * p.g.slot + goff);
        if constexpr (MX) scale = head[p.g.scales + (slot0 + first + wrow) * SB + wch * PIECE / 32];
    };
    auto issue = [&](int i) {
        const unsigned char* head = tile_base(tiles.at(i) * KT);
        const int slot0 = at.slot;
#pragma unroll
        for (int s = 0; s < NLW; ++s)
            if (wave + NW * s < NL) {
                load(head, slot0, s, kreg[s], kscale[s]);
                load(head + p.g.half, slot0, s, vreg[s], vscale[s]);
            }
    };
    constexpr int YD = PIECE / 2;
    auto convert = [&](const u32x4 x, unsigned scale_byte, unsigned (&y)[YD]) {
        const float scale = MX ? mx_scale(scale_byte) : 1.0f;
        if constexpr (KIND == MD_KV_BF16) {
#pragma unroll
            for (int w = 0; w < 4; ++w) y[w] = x[w];
        } else if constexpr (KIND == MD_KV_MXFP4) {
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                unsigned t[4];
                mx4_to_bf16(x[w], scale, t);
#pragma unroll
                for (int e = 0; e < 4; ++e) y[4 * w + e] = t[e];
            }
        } else {
#pragma unroll
            for (int w = 0; w < 4; ++w) mx8_to_bf16(x[w], scale, y[2 * w], y[2 * w + 1]);
        }
    };
    auto put_values = [&](unsigned char* img, int s, const unsigned (&y)[YD]) {
        const int row = wrow + (wave + NW * s) * RPI;
        unsigned char* at = img + K_BYTES + (row >> 5) * VG + (row & 31) * 32;
#pragma unroll
        for (int c = 0; c < PIECE / 8; ++c) {
            const int d8 = wch * (PIECE / 8) + c;                 // the piece's 8-element part in the row
            *reinterpret_cast<u32x4*>(at + (d8 >> 1) * kVSub + (d8 & 1) * 16) = u32x4{y[4 * c], y[4 * c + 1], y[4 * c + 2], y[4 * c + 3]};
        }
    };
    auto stage = [&](int i, unsigned char* img) {
        const bool some = hides(tiles.at(i) * KT, lo_all, hi_all);
        unsigned infinite = 0;
#pragma unroll
        for (int s = 0; s < NLW; ++s)
            if (wave + NW * s < NL) {
                unsigned y[YD];
                convert(kreg[s], kscale[s], y);
                unsigned char* at = img + (wrow + (wave + NW * s) * RPI) * KROW + wch * PIECE * 2;
#pragma unroll
                for (int c = 0; c < PIECE / 8; ++c) *reinterpret_cast<u32x4*>(at + c * 16) = u32x4{y[4 * c], y[4 * c + 1], y[4 * c + 2], y[4 * c + 3]};
                convert(vreg[s], vscale[s], y);
                if (some) {
#pragma unroll
                    for (int e = 0; e < YD; ++e) {
                        const unsigned n = nonfinite_halves(y[e]);
                        infinite |= n;
                        y[e] &= ~n;
                    }
                }
                put_values(img, s, y);
            }
        if (some) {
            const bool any = __builtin_amdgcn_ballot_w64(infinite != 0) != 0;
            if (lane == 0) s_infinite[(i & 1) * NW + wave] = any;
        }
    };
    // fragments.  Keys, lane (j, kh): row j, 16-byte piece 2 ks + kh.  Values: a 16-lane group reads [4 keys][16 d]; a pair of d blocks apart by
    // half of all, whose images begin in different halves of the banks
    const int kra = j * KROW + (kh << 4), lq = lane & 15;
    const int vra = K_BYTES + ((lane >> 4) & 1) * (NB / 2) * kVSub + (kh * 4 + (lq >> 2)) * 32 + (lq & 3) * 8;
    auto value_fragment = [&](const unsigned char* img, int kg, int s16, int db) {
        const unsigned char* at = img + kg * VG + db * kVSub + vra + s16 * 16 * 32;
        const bf16x4 a = lds_read_tr(at), c = lds_read_tr(at + 8 * 32);
        return __builtin_shufflevector(a, c, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    auto hidden = [&](int pos) { return pos > lim || (pos <= low && pos >= p.sinks); };

    auto compute = [&](int i, const unsigned char* img) __attribute__((always_inline)) {
        const int pos0 = tiles.at(i) * KT;
        f32x16 sc[KG];
#pragma unroll
        for (int kg = 0; kg < KG; ++kg)
#pragma unroll
            for (int r = 0; r < 16; ++r) sc[kg][r] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int kg = 0; kg < KG; ++kg)
                sc[kg] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(lds_read_b128(img + kra + kg * 32 * KROW + ks * 32), qf[ks], sc[kg], 0, 0, 0);
        if (hides(pos0, lo, hi)) {
            // a branch of the wavefront: volatile, or every tile would compare and select
#pragma unroll
            for (int kg = 0; kg < KG; ++kg)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    float v = hidden(pos0 + kg * 32 + (r & 3) + 8 * (r >> 2) + 4 * kh) ? -INFINITY : sc[kg][r];
                    asm volatile("" : "+v"(v));
                    sc[kg][r] = v;
                }
        }
        float mx = sc[0][0];
#pragma unroll
        for (int kg = 0; kg < KG; ++kg)
#pragma unroll
            for (int r = 0; r < 16; ++r) mx = fmaxf(mx, sc[kg][r]);
        mx = max_over_32(mx) * sl2;
        if (__builtin_amdgcn_ballot_w64(mx > m) != 0) {
            const float mnew = fmaxf(m, mx), alpha = __builtin_amdgcn_exp2f(m - mnew);
            m = mnew;
            l *= alpha;
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[db][r] *= alpha;
        }
        float times = sl2;
        if (__builtin_amdgcn_ballot_w64(fabsf(m) > 4096.f && m != kLowest) != 0) {
            times = 1.0f;
#pragma unroll
            for (int kg = 0; kg < KG; ++kg)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    float v = sc[kg][r] * sl2;
                    asm volatile("" : "+v"(v));
                    sc[kg][r] = v;
                }
        }
        const float mneg = -m;
        float ps = 0.f;
        bf16x8 pf[KG][2];
#pragma unroll
        for (int kg = 0; kg < KG; ++kg)
#pragma unroll
            for (int s16 = 0; s16 < 2; ++s16) {
                f32x8 w;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    w[e] = __builtin_amdgcn_exp2f(fmaf(sc[kg][s16 * 8 + e], times, mneg));
                    ps += w[e];
                }
                pf[kg][s16] = __builtin_convertvector(w, bf16x8);        // weights from 0 to 1, off by 2^-8 of themselves at most
            }
        l += ps;
#pragma unroll
        for (int kg = 0; kg < KG; ++kg)
#pragma unroll
            for (int s16 = 0; s16 < 2; ++s16)
#pragma unroll
                for (int db = 0; db < DB; ++db)
                    o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(value_fragment(img, kg, s16, db), pf[kg][s16], o[db], 0, 0, 0);
    };
    // infinite values and NaN of a tile to the rows that see them: by images of their signs in the values' place
    auto spread = [&](int i, unsigned char* img) __attribute__((always_inline)) {
        const int pos0 = tiles.at(i) * KT;
        const unsigned char* head = tile_base(pos0) + p.g.half;
        const int slot0 = at.slot;
#pragma unroll 1
        for (int negative = 0; negative < 2; ++negative) {
            __syncthreads();
#pragma unroll 1
            for (int s = 0; s < NLW; ++s)
                if (wave + NW * s < NL) {
                    u32x4 x;
                    unsigned scale = 0, y[YD];
                    load(head, slot0, s, x, scale);
                    convert(x, scale, y);
#pragma unroll
                    for (int e = 0; e < YD; ++e) y[e] = infinite_halves(y[e], negative != 0);
                    put_values(img, s, y);
                }
            __syncthreads();
            const float add = negative ? -INFINITY : INFINITY;
#pragma unroll
            for (int db = 0; db < DB; ++db) {
                f32x16 n;
#pragma unroll
                for (int r = 0; r < 16; ++r) n[r] = 0.f;
#pragma unroll
                for (int kg = 0; kg < KG; ++kg)
#pragma unroll
                    for (int s16 = 0; s16 < 2; ++s16) {
                        bf16x8 seen;
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const int r = s16 * 8 + e;
                            seen[e] = hidden(pos0 + kg * 32 + (r & 3) + 8 * (r >> 2) + 4 * kh) ? (bf16_t)0.f : (bf16_t)1.f;
                        }
                        n = __builtin_amdgcn_mfma_f32_32x32x16_bf16(value_fragment(img, kg, s16, db), seen, n, 0, 0, 0);
                    }
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (n[r] > 0.f) o[db][r] += add;
            }
        }
        __syncthreads();
    };

    if (t_begin < t_end) issue(t_begin);
    // behind the first tile's loads, which wait for the numbers of their pages
    {
        const bf16_t* qp = p.q + (int64_t)(q0 + qi) * p.q_row_stride + (kvh * g + qr) * D;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const bf16x8 z = {0, 0, 0, 0, 0, 0, 0, 0};
            qf[ks] = valid ? *reinterpret_cast<const bf16x8*>(qp + ks * 16 + kh * 8) : z;
            if constexpr (KIND == MD_KV_FP8_E4M3) qf[ks] = with_sign_of(ksc, qf[ks]);
        }
    }
    for (int i = t_begin; i < t_end; ++i) {
        unsigned char* img = smem + (i & 1) * IMAGE;
        const int pos0 = tiles.at(i) * KT;
        stage(i, img);
        if (i + 1 < t_end) issue(i + 1);
        __syncthreads();
        if (sees(pos0)) compute(i, img);
        if (hides(pos0, lo_all, hi_all)) {
            int any = 0;
#pragma unroll
            for (int w = 0; w < NW; ++w) any |= NL > w ? s_infinite[(i & 1) * NW + w] : 0;
            if (__builtin_amdgcn_readfirstlane(any)) spread(i, img);
        }
    }

    l += __shfl_xor(l, 32);
    if (p.nsplit > 1) {
        if (!valid) return;
        const int64_t slot = (((int64_t)pair * p.n_qgroups + qg) * p.nsplit + split) * (NW * 32) + wave * 32 + j;
        if (kh == 0) {
            p.ws_ml[slot * 2] = m;
            p.ws_ml[slot * 2 + 1] = l;
        }
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int rg = 0; rg < 4; ++rg)
                *reinterpret_cast<f32x4*>(p.ws_o + slot * D + ((db + (rg >> 1) * (NB / 2)) * 2 + (rg & 1)) * 8 + kh * 4) =
                    f32x4{o[db][rg * 4], o[db][rg * 4 + 1], o[db][rg * 4 + 2], o[db][rg * 4 + 3]};
        return;
    }
    // output rows through LDS: a store writes whole rows
    const float vsc = KIND == MD_KV_FP8_E4M3 ? p.v_scale[kvh] : 1.0f;
    const float inv = l == 0.f ? 0.f : vsc / l;
    __syncthreads();                                       // every wavefront is past the last image
    int ln = lane;
    asm volatile("" : "+v"(ln));                           // nothing below is computed, and kept, in front of the tiles
    const int oj = ln & 31, oR = (qg * NW + wave) * 32 + oj, oq = oR / g;
    const int64_t orow = oR < nrows ? (int64_t)(q0 + oq) * p.H + kvh * g + oR - oq * g : -1;
    unsigned char* mine = smem + wave * 32 * D * 2;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int rg = 0; rg < 4; ++rg) {
            f32x4 ov;
#pragma unroll
            for (int r = 0; r < 4; ++r) ov[r] = l == 0.f ? 0.f : o[db][rg * 4 + r] * inv;
            const int ch = (db + (rg >> 1) * (NB / 2)) * 2 + (rg & 1);
            *reinterpret_cast<bf16x4*>(mine + oj * D * 2 + lds_place<D / 8>(ch, oj) * 16 + (ln >> 5) * 8) = __builtin_convertvector(ov, bf16x4);
        }
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
        const int c = i * 64 + ln, r = c / (D / 8), ch = c % (D / 8);
        const int64_t row = __shfl(orow, r);
        const bf16x8 v = lds_read_b128(mine + r * D * 2 + lds_place<D / 8>(ch, r) * 16);
        if (row >= 0) *reinterpret_cast<bf16x8_a8*>(p.out + row * D + ch * 8) = v;
    }
}

template <int D, int NW, int KT>
int launch_prompt(const WinParams& p, int grid, hipStream_t st) {
    constexpr int lds = std::max(2 * prompt_image_bytes<D, KT>() + 2 * NW * 4, NW * 32 * D * 2);
    auto k = window_prompt_kernel<D, NW, KT, MD_WIN_KIND>;
    if constexpr (lds > 64 * 1024) {
        static MdPerDeviceOnce once;
        if (once.first()) {
            const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
            if (e != hipSuccess) {
                once.undo();
                md_set_error("md_window_attn: hipFuncSetAttribute(%d B LDS) failed: %s", lds, hipGetErrorString(e));
                return MD_ERR_LAUNCH;
            }
        }
    }
    hipLaunchKernelGGL(k, dim3(grid), dim3(64 * NW), lds, st, p);
    MD_CHECK_LAUNCH("md_window_attn(prompt)");
    return MD_OK;
}

}  // namespace

#define MD_WIN_CAT_(a, b) a##b
#define MD_WIN_CAT(a, b) MD_WIN_CAT_(a, b)

int MD_WIN_CAT(md_window_prompt_, MD_WIN_KIND)(const WinParams& p, int D, int nw, int grid, hipStream_t st) {
    const bool small = window_prompt_tile(D, nw, p.page_size) == 32;
    if (D == 128) {
        if (nw == 8) return small ? launch_prompt<128, 8, 32>(p, grid, st) : launch_prompt<128, 8, 128>(p, grid, st);
        return small ? launch_prompt<128, 4, 32>(p, grid, st) : launch_prompt<128, 4, 64>(p, grid, st);
    }
    if (nw == 8) return small ? launch_prompt<64, 8, 32>(p, grid, st) : launch_prompt<64, 8, 64>(p, grid, st);
    return small ? launch_prompt<64, 4, 32>(p, grid, st) : launch_prompt<64, 4, 64>(p, grid, st);
}

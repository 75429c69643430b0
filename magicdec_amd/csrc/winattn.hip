// md_window_attn: softmax attention of new tokens over paged K / V of any element type, over everything before them or over a sliding window
// and some first tokens.
//
// One wavefront owns a stream of 32-key tiles of one (request, kv head) and up to 32 query rows (query heads of the kv head x new tokens), as
// S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_16x16x32_bf16:
//   * the keys of a 16-key block come from memory as the matrix instruction's A operand: lane (row lq, quarter lc) loads the bytes of its own
//     row that it multiplies, whatever elements of the row they are -- the sum over the elements has any order, the queries are loaded in
//     the same.  No LDS, no transposition: 8- and 4-bit elements become bf16 in registers, times their block's scale in the conversion.
//   * the values have to be transposed: converted the same way, they go through a wavefront-private LDS image that ds_read_b64_tr_b16 reads.
//   * the scores of query lq lie in the lanes of its column, so that the softmax's statistics are per lane, and are the next product's
//     B operand as they lie.
// The scales of a tile's 32 keys and 32 values are one load of a wavefront (a lane a row) and go to the lanes that use them by ds_bpermute.
// The four wavefronts of a workgroup take a (request, kv head, row group)'s tiles in turn and merge through LDS; `nsplit` workgroups share
// its tiles where there are few of them, merged by a launch behind.
//
// What a mask hides may hold anything.  Scores are replaced, not added to.  Values count with weight 0, which is not enough for an infinity or
// a NaN: in tiles that hide a key from some row, such values are taken out of the image, and what rows that do see them get of them is
// added by itself (`spread`), from a second and third image of their signs.
//
// Long streams are bound by memory: 64 requests of 16 036 keys x 16 rows (8 heads of 128) take 330 us from 8-bit pages (2.2 GB, 6.6 TB/s; loads alone
// 328) and 184 from 4-bit ones (1.1 GB, 6.1 TB/s), vector instructions in 26 and 45 % of the cycles, the matrix
// cores in 8 and 16.  Short ones by the way through a workgroup, its page numbers, keys, sums and rows one behind the other: 64 requests that see 257 keys
// of 64 in bf16 11.5 us (34 MB), one of 32 065 keys 13 and 4 for the launch that joins its 32 parts.
#include "winattn.h"

#include <algorithm>

namespace {

template <int D, int QT, int KG>
__host__ __device__ constexpr int win_wave_lds() {
    const int image = KG * (D / 16) * kVSub, merge = QT * 16 * (D + 4) * 4 + QT * 128;
    return ((image > merge ? image : merge) + 255) / 256 * 256;
}

constexpr int kWaves = 4;

// KG: groups of 32 keys in a tile
template <int D, int QT, int KIND, int KG>
__global__ __launch_bounds__(64 * kWaves, 2) void window_attn_kernel(const WinParams p) {
    constexpr int KT = KG * 32, VG = (D / 16) * kVSub;
    constexpr int EB = kv_element_bytes(KIND, D);        // bytes of a row's elements
    constexpr bool MX = kv_is_mx(KIND);
    constexpr int KS = D / 32, NB = D / 16, SB = D / 32;  // matrix steps of a score, 16-d blocks, scales of a row
    // keys: a lane's loads of a row, their dwords, elements and matrix steps
    constexpr int KI = EB >= 64 ? EB / 64 : 1, KW = EB >= 64 ? 4 : EB / 16, EL = D / (4 * KI), SPL = EL / 8;
    // values: 16-byte pieces of a row, rows of a load, loads of a group
    constexpr int CH = EB / 16, RPI = 64 / CH, NL = 32 / RPI;
    // 8 neighbouring lanes write 16-byte halves of 32-byte rows: the upper half of the pieces begin with their second half, so that they
    // lie in different banks; in the d blocks from 4 on the halves are then the other way round (undone where rows are stored)
    constexpr bool SWAP = KIND != MD_KV_BF16 && D == 128;
    constexpr int WAVE_LDS = win_wave_lds<D, QT, KG>();
    // tiles in flight: as many as the registers hold
    constexpr int NS = KG * EB * QT > 256 || (QT == 2 && D == 128 && KIND != MD_KV_MXFP4) ? 1 : 2;

    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lane = tid & 63;
    const int lq = lane & 15, lc = lane >> 4;

    int sub;
    const int pair = win_pair(p, p.n_qgroups * p.nsplit, sub);
    const int qg = sub / p.nsplit, split = sub % p.nsplit;
    const int b = pair / p.KH, kvh = pair % p.KH;
    const int g = p.group;
    const int q0 = p.qo_indptr[b], n_b = p.qo_indptr[b + 1] - q0;
    int pg0, room;
    const int kv_len = min(kv_len_of(p.indptr, p.last, b, p.page_size, &pg0, &room), room);
    const int nrows = n_b * g;

    // a lane's query rows see up to lim, and of those up to low only the first tokens; lo, hi: the first and the last row's lim
    int lim[QT], low[QT];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
        const int R = (qg * QT + qt) * 16 + lq;
        lim[qt] = R < nrows ? kv_len - n_b + R / g : -1;
        low[qt] = p.window > 0 ? lim[qt] - p.window : -1;
    }
    const int first = qg * QT * 16, last = min(first + QT * 16, nrows) - 1;
    if (last < first) return;
    const int lo = kv_len - n_b + first / g, hi = kv_len - n_b + last / g;
    const int hi_low = p.window > 0 ? hi - p.window : -1;
    const Tiles tiles(lo, min(hi + 1, kv_len), p.window, p.sinks, KT);
    const int per = (tiles.count + p.nsplit - 1) / p.nsplit;
    const int t_begin = split * per, t_end = min(tiles.count, t_begin + per);

    const float ksc = KIND == MD_KV_FP8_E4M3 ? p.k_scale[kvh] : 1.0f;
    const float sl2 = KIND == MD_KV_FP8_E4M3 ? size_of_scale(p.scale_log2, ksc) : p.scale_log2;
    const float vsc = KIND == MD_KV_FP8_E4M3 ? p.v_scale[kvh] : 1.0f;
    f32x4 o[QT][NB];
    float m[QT], l[QT];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
        m[qt] = kLowest;
        l[qt] = 0.f;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) o[qt][nb] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    unsigned char* image = smem + wave * WAVE_LDS;
    const int wrow = lane / CH, wch = lane % CH;
    const bool swp = SWAP && wch >= CH / 2;
    const int vra = (lc * 4 + (lq >> 2)) * 32 + (lq & 3) * 8;       // + kg * VG + nb * kVSub, + 512 for the second 16 keys

    struct Staged {
        unsigned k[2 * KG][KI * KW];
        u32x4 v[KG][NL];
        unsigned scale[KG];
    };
    Staged st[NS];
    const unsigned koff = (unsigned)(lq * p.g.slot + lc * KW * 4), voff = (unsigned)(wrow * p.g.slot + wch * 16);
    const int64_t soff = (lane >= 32 ? p.g.half : 0) + (lane & 31) * SB;
    PageCursor at(p, pg0, room);
    auto tile_base = [&](int i) {
        at.seek(tiles.at(i) * KT);
        return p.cache + at.id() * p.g.page + (int64_t)kvh * p.g.head + (int64_t)at.slot * p.g.slot;
    };
    auto issue = [&](int i, Staged& s) __attribute__((always_inline)) {
        const unsigned char* base = tile_base(i);
#pragma unroll
        for (int kb = 0; kb < 2 * KG; ++kb)
#pragma unroll
            for (int k = 0; k < KI; ++k) {
                const unsigned char* from = base + (int64_t)kb * 16 * p.g.slot + koff + k * 64;
                if constexpr (KW == 4) {
                    const u32x4 x = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(from));
#pragma unroll
                    for (int e = 0; e < 4; ++e) s.k[kb][k * 4 + e] = x[e];
                } else {
                    const u32x2 x = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(from));
                    s.k[kb][0] = x[0];
                    s.k[kb][1] = x[1];
                }
            }
        if constexpr (MX) {
#pragma unroll
            for (int kg = 0; kg < KG; ++kg) {
                const unsigned char* from = base - (int64_t)at.slot * (EB - SB) + p.g.scales + kg * 32 * SB + soff;
                s.scale[kg] = SB == 4 ? *reinterpret_cast<const unsigned*>(from) : *reinterpret_cast<const unsigned short*>(from);
            }
        }
#pragma unroll
        for (int kg = 0; kg < KG; ++kg)
#pragma unroll
            for (int j = 0; j < NL; ++j)
                s.v[kg][j] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(base + p.g.half + (int64_t)(kg * 32 + j * RPI) * p.g.slot + voff));
    };
    auto scale_of = [&](unsigned scales, int row, int block) {       // row 0..31 keys, 32..63 values
        const unsigned u = (unsigned)__builtin_amdgcn_ds_bpermute(row * 4, (int)scales);
        return mx_scale((u >> (block * 8)) & 255u);
    };
    // a lane's 16 bytes of values as bf16 pairs, in the order of d
    constexpr int VD = KIND == MD_KV_BF16 ? 4 : KIND == MD_KV_MXFP4 ? 16 : 8;
    auto values = [&](const u32x4 x, float scale, unsigned (&y)[VD]) {
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
    auto put_values = [&](int kg, int j, const unsigned (&y)[VD]) {
        unsigned char* row = image + kg * VG + (wrow + j * RPI) * 32;
        if constexpr (KIND == MD_KV_BF16) {
            *reinterpret_cast<u32x4*>(row + (wch >> 1) * kVSub + (wch & 1) * 16) = u32x4{y[0], y[1], y[2], y[3]};
        } else {
            constexpr int SUBS = VD / 8;
#pragma unroll
            for (int s = 0; s < SUBS; ++s) {
                unsigned char* to = row + (wch * SUBS + s) * kVSub;
                *reinterpret_cast<u32x4*>(to + (swp ? 16 : 0)) = u32x4{y[8 * s], y[8 * s + 1], y[8 * s + 2], y[8 * s + 3]};
                *reinterpret_cast<u32x4*>(to + (swp ? 0 : 16)) = u32x4{y[8 * s + 4], y[8 * s + 5], y[8 * s + 6], y[8 * s + 7]};
            }
        }
    };
    constexpr int VB = KIND == MD_KV_MXFP4 ? 32 : 16;                // elements of a lane's 16 bytes
    // one wavefront's LDS operations run in order: the compiler has to keep them so, too
    auto in_order = [&] {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    };
    auto value_fragment = [&](int kg, int nb) {
        const unsigned char* from = image + kg * VG + nb * kVSub + vra;
        const bf16x4 a = lds_read_tr(from), c = lds_read_tr(from + 512);
        return __builtin_shufflevector(a, c, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    // infinite values and NaN of tile i go to the rows that see them
    auto spread = [&](int i, const unsigned (&hidden)[QT]) __attribute__((always_inline)) {
        const unsigned char* base = tile_base(i);
#pragma unroll 1
        for (int negative = 0; negative < 2; ++negative) {
            in_order();
#pragma unroll
            for (int kg = 0; kg < KG; ++kg)
#pragma unroll
                for (int j = 0; j < NL; ++j) {
                    const int row = kg * 32 + wrow + j * RPI;
                    const u32x4 x = *reinterpret_cast<const u32x4*>(base + p.g.half + (int64_t)(kg * 32 + j * RPI) * p.g.slot + voff);
                    float scale = 1.0f;
                    if constexpr (MX) scale = mx_scale(base[p.g.half - (int64_t)at.slot * (EB - SB) + p.g.scales + row * SB + wch * VB / 32]);
                    unsigned y[VD];
                    values(x, scale, y);
#pragma unroll
                    for (int e = 0; e < VD; ++e) y[e] = infinite_halves(y[e], negative != 0);
                    put_values(kg, j, y);
                }
            in_order();
            const float add = negative ? -INFINITY : INFINITY;
#pragma unroll
            for (int qt = 0; qt < QT; ++qt)
#pragma unroll
                for (int kg = 0; kg < KG; ++kg) {
                    bf16x8 seen;
#pragma unroll
                    for (int e = 0; e < 8; ++e) seen[e] = hidden[qt] >> (kg * 8 + e) & 1 ? (bf16_t)0.f : (bf16_t)1.f;
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
                        const f32x4 n = __builtin_amdgcn_mfma_f32_16x16x32_bf16(value_fragment(kg, nb), seen, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (n[r] > 0.f) o[qt][nb][r] += add;
                    }
                }
        }
        in_order();
    };

    bf16x8 qf[QT][KS];
    auto process = [&](auto more, int i, Staged& s) __attribute__((always_inline)) {
        const int t = tiles.at(i);
        const bool need_mask = t * KT + KT - 1 > lo || (t * KT <= hi_low && t * KT + KT - 1 >= p.sinks);
        bool infinite = false;
#pragma unroll
        for (int kg = 0; kg < KG; ++kg)
#pragma unroll
            for (int j = 0; j < NL; ++j) {
                unsigned y[VD];
                values(s.v[kg][j], MX ? scale_of(s.scale[kg], 32 + wrow + j * RPI, wch * VB / 32) : 1.0f, y);
                if (need_mask) {
#pragma unroll
                    for (int e = 0; e < VD; ++e) {
                        const unsigned n = nonfinite_halves(y[e]);
                        infinite |= n != 0;
                        y[e] &= ~n;
                    }
                }
                put_values(kg, j, y);
            }
        f32x4 sc[QT][2 * KG];
#pragma unroll
        for (int kb = 0; kb < 2 * KG; ++kb) {
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) sc[qt][kb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < KI; ++k) {
                // a lane's piece of a row is one block's, or a half of it
                const float scale = MX ? scale_of(s.scale[kb / 2], (kb & 1) * 16 + lq, EL == 32 ? lc : k * 2 + (lc >> 1)) : 1.0f;
#pragma unroll
                for (int h = 0; h < SPL; ++h) {
                    unsigned y[4];
                    if constexpr (KIND == MD_KV_BF16) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) y[e] = s.k[kb][k * 4 + e];
                    } else if constexpr (KIND == MD_KV_MXFP4) {
                        mx4_to_bf16(s.k[kb][k * KW + h], scale, y);
                    } else {
                        mx8_to_bf16(s.k[kb][k * KW + 2 * h], scale, y[0], y[1]);
                        mx8_to_bf16(s.k[kb][k * KW + 2 * h + 1], scale, y[2], y[3]);
                    }
                    const bf16x8 kf = __builtin_bit_cast(bf16x8, u32x4{y[0], y[1], y[2], y[3]});
#pragma unroll
                    for (int qt = 0; qt < QT; ++qt)
                        sc[qt][kb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[qt][k * SPL + h], sc[qt][kb], 0, 0, 0);
                }
            }
        }
        if constexpr (decltype(more)::value) {
            issue(i + NS * kWaves, s);
        } else {
            if (i + NS * kWaves < t_end) issue(i + NS * kWaves, s);
        }
        in_order();

        bf16x8 pf[QT][KG];
        unsigned hidden[QT];
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) {
            float v[8 * KG];
#pragma unroll
            for (int e = 0; e < 8 * KG; ++e) v[e] = sc[qt][e >> 2][e & 3];
            hidden[qt] = 0;
            if (need_mask) {
                // a branch of the wavefront: volatile, or every tile would compare and select
#pragma unroll
                for (int e = 0; e < 8 * KG; ++e) {
                    const int pos = t * KT + (e >> 2) * 16 + lc * 4 + (e & 3);
                    const bool out = pos > lim[qt] || (pos <= low[qt] && pos >= p.sinks);
                    float x = out ? -INFINITY : v[e];
                    asm volatile("" : "+v"(x));
                    v[e] = x;
                    hidden[qt] |= (unsigned)out << e;
                }
            }
            float mx = v[0];
#pragma unroll
            for (int e = 1; e < 8 * KG; ++e) mx = fmaxf(mx, v[e]);
            mx = max_over_32(max_over_16(mx)) * sl2;
            if (__builtin_amdgcn_ballot_w64(mx > m[qt]) != 0) {         // some row has a new reference
                const float mnew = fmaxf(m[qt], mx), alpha = __builtin_amdgcn_exp2f(m[qt] - mnew);
                m[qt] = mnew;
                l[qt] *= alpha;
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) o[qt][nb] *= alpha;
            }
            const float times = exponent_factor(m[qt], sl2, v);
            float ps = 0.f;
#pragma unroll
            for (int kg = 0; kg < KG; ++kg) {
                f32x8 w;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    w[e] = __builtin_amdgcn_exp2f(fmaf(v[kg * 8 + e], times, -m[qt]));
                    ps += w[e];
                }
                pf[qt][kg] = __builtin_convertvector(w, bf16x8);       // the matrix instruction's operand: weights from 0 to 1, off by 2^-8 of themselves
            }
            l[qt] += ps;
        }
#pragma unroll
        for (int kg = 0; kg < KG; ++kg)
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                const bf16x8 vf = value_fragment(kg, nb);
#pragma unroll
                for (int qt = 0; qt < QT; ++qt) o[qt][nb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[qt][kg], o[qt][nb], 0, 0, 0);
            }
        if (need_mask && __builtin_amdgcn_ballot_w64(infinite) != 0) spread(i, hidden);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
    };

    int i = t_begin + wave;
#pragma unroll
    for (int s = 0; s < NS; ++s)
        if (i + s * kWaves < t_end) issue(i + s * kWaves, st[s]);
    // the queries behind the first tiles' loads
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
        const int R = (qg * QT + qt) * 16 + lq;
        const int qi = R / g, r = R - qi * g;
        const bf16_t* qp = p.q + (int64_t)(q0 + qi) * p.q_row_stride + (kvh * g + r) * D;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const bf16x8 z = {0, 0, 0, 0, 0, 0, 0, 0};
            qf[qt][s] = R < nrows ? *reinterpret_cast<const bf16x8*>(qp + (s / SPL) * 4 * EL + lc * EL + (s % SPL) * 8) : z;
            if constexpr (KIND == MD_KV_FP8_E4M3) qf[qt][s] = with_sign_of(ksc, qf[qt][s]);
        }
    }
    // steady state: loads of the tile NS turns on are issued without a condition, so that waits are for the tile at hand alone
    for (; i + (2 * NS - 1) * kWaves < t_end; i += NS * kWaves) {
#pragma unroll
        for (int s = 0; s < NS; ++s) process(std::true_type{}, i + s * kWaves, st[s]);
    }
    for (; i < t_end; i += NS * kWaves) {
#pragma unroll
        for (int s = 0; s < NS; ++s)
            if (i + s * kWaves < t_end) process(std::false_type{}, i + s * kWaves, st[s]);
    }

#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
        l[qt] += __shfl_xor(l[qt], 16);
        l[qt] += __shfl_xor(l[qt], 32);
    }
    __syncthreads();
    // rows of sums, 4 numbers apart from whole banks: 16 lanes write and read different ones
    constexpr int ROWS = QT * 16, PITCH = D + 4;
    float* mo = reinterpret_cast<float*>(smem + wave * WAVE_LDS);
    float* mst = mo + ROWS * PITCH;
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
            *reinterpret_cast<f32x4*>(mo + (qt * 16 + lq) * PITCH + nb * 16 + ((SWAP && nb >= 4) ? (lc ^ 2) : lc) * 4) = o[qt][nb];
        if (lc == 0) {
            mst[(qt * 16 + lq) * 2] = m[qt];
            mst[(qt * 16 + lq) * 2 + 1] = l[qt];
        }
    }
    __syncthreads();
#pragma unroll
    for (int e = tid; e < ROWS * (D / 4); e += 64 * kWaves) {
        const int Rl = e / (D / 4), d = e % (D / 4) * 4, R = first + Rl;
        if (R > last) break;                                     // (rows ascend with e)
        float M = kLowest, L = 0.f;
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) M = fmaxf(M, reinterpret_cast<const float*>(smem + w * WAVE_LDS)[ROWS * PITCH + Rl * 2]);
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float* ow = reinterpret_cast<const float*>(smem + w * WAVE_LDS);
            const float a = __builtin_amdgcn_exp2f(ow[ROWS * PITCH + Rl * 2] - M);
            L += ow[ROWS * PITCH + Rl * 2 + 1] * a;
            acc += *reinterpret_cast<const f32x4*>(ow + Rl * PITCH + d) * a;
        }
        if (p.nsplit == 1) {
            const int qi = R / g;
            const float inv = L == 0.f ? 0.f : vsc / L;
            if (L == 0.f) acc = f32x4{0.f, 0.f, 0.f, 0.f};
            *reinterpret_cast<bf16x4*>(p.out + ((int64_t)(q0 + qi) * p.H + kvh * g + R - qi * g) * D + d) = __builtin_convertvector(acc * inv, bf16x4);
        } else {
            const int64_t slot = (((int64_t)pair * p.n_qgroups + qg) * p.nsplit + split) * ROWS + Rl;
            *reinterpret_cast<f32x4*>(p.ws_o + slot * D + d) = acc;
            if (d == 0) {
                p.ws_ml[slot * 2] = M;
                p.ws_ml[slot * 2 + 1] = L;
            }
        }
    }
}

// The splits of a row joined: D / 4 lanes a row, SG groups of them share its splits and meet through LDS.
template <int D, int SG>
__global__ __launch_bounds__(256) void window_merge_kernel(const WinParams p, int rows) {
    constexpr int VPR = D / 4, TPR = VPR * SG, RPB = 256 / TPR;
    __shared__ float s_ml[SG > 1 ? 512 : 1];
    __shared__ f32x4 s_o[SG > 1 ? 256 : 1];
    const int tid = threadIdx.x, v = tid % VPR, sg = tid / VPR % SG;
    const int64_t rowid = (int64_t)blockIdx.x * RPB + tid / TPR;
    const int Rl = (int)(rowid % rows), item = (int)(rowid / rows);
    const int pair = item / p.n_qgroups, qg = item % p.n_qgroups, R = qg * rows + Rl;
    int q0 = 0;
    bool live = pair < p.B * p.KH;
    if (live) {
        q0 = p.qo_indptr[pair / p.KH];
        live = R < (p.qo_indptr[pair / p.KH + 1] - q0) * p.group;
    }
    float M = kLowest, L = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    if (live) {
        for (int s0 = sg; s0 < p.nsplit; s0 += 8 * SG) {           // eight requested together: one wait
            float ms[8], ls[8];
            f32x4 os[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int s = s0 + u * SG;
                const int64_t slot = ((int64_t)item * p.nsplit + (s < p.nsplit ? s : s0)) * rows + Rl;
                ms[u] = p.ws_ml[slot * 2];
                ls[u] = p.ws_ml[slot * 2 + 1];
                os[u] = *reinterpret_cast<const f32x4*>(p.ws_o + slot * D + v * 4);
            }
            float mn = M;
#pragma unroll
            for (int u = 0; u < 8; ++u) mn = fmaxf(mn, ms[u]);
            const float a = __builtin_amdgcn_exp2f(M - mn);
            L *= a;
            acc *= a;
#pragma unroll
            for (int u = 0; u < 8; ++u)
                if (s0 + u * SG < p.nsplit) {
                    const float c = __builtin_amdgcn_exp2f(ms[u] - mn);
                    L += ls[u] * c;
                    acc += os[u] * c;
                }
            M = mn;
        }
    }
    if constexpr (SG > 1) {
        s_ml[tid * 2] = M;
        s_ml[tid * 2 + 1] = L;
        s_o[tid] = acc;
        __syncthreads();
        if (sg != 0) return;
        const float m0 = M;
#pragma unroll
        for (int u = 1; u < SG; ++u) M = fmaxf(M, s_ml[(tid + u * VPR) * 2]);
        const float a = __builtin_amdgcn_exp2f(m0 - M);
        L *= a;
        acc *= a;
#pragma unroll
        for (int u = 1; u < SG; ++u) {
            const float c = __builtin_amdgcn_exp2f(s_ml[(tid + u * VPR) * 2] - M);
            L += s_ml[(tid + u * VPR) * 2 + 1] * c;
            acc += s_o[tid + u * VPR] * c;
        }
    }
    if (!live) return;
    const int kvh = pair % p.KH, i = R / p.group;
    const float inv = L == 0.f ? 0.f : (p.v_scale ? p.v_scale[kvh] : 1.f) / L;
    if (L == 0.f) acc = f32x4{0.f, 0.f, 0.f, 0.f};
    *reinterpret_cast<bf16x4*>(p.out + ((int64_t)(q0 + i) * p.H + kvh * p.group + R - i * p.group) * D + v * 4) = __builtin_convertvector(acc * inv, bf16x4);
}

// How a call's rows and keys lie over workgroups
struct WinPlan {
    int nw;                 // wavefronts of a workgroup of winprompt.hip, 0: the kernel above
    int kg;                 // groups of 32 keys in its tiles
    int rows, n_qgroups, nsplit;
    size_t slots;
};

// What a way of laying out more than 32 rows a kv head is expected to take, in us: workgroups of `rows` rows walk their keys in steps of `unit`, in `parts`
// of them.  A step takes `tau` while a CU has one workgroup, and `full` for each of the most that one has; where it holds one at a time, each after the
// first begins with `next`.  A window's ends and its first tokens are steps of their own.  A second launch joins parts, whose sums are written and read
// back.  The numbers are fitted to 237 shapes, one request to 64 of 40 to 32 000 rows over 10 to 16 000 keys, in every way and number of parts: what this
// picks takes 2 to 3 % more than the best of them on average.
struct WinWay {
    int nw, rows, unit;
    double fixed, tau, full, next;
    double us(int64_t workgroups, int64_t keys, int edges, int64_t parts, double sums) const {
        const double steps = (double)(((keys + unit - 1) / unit + edges + parts - 1) / parts), most = (double)((workgroups + 255) / 256);
        return fixed + (most - 1) * next + steps * std::max(tau, full * most) + (parts > 1 ? 2.6 + sums * parts / 5e6 : 0.);
    }
};

int* g_report = nullptr;       // dev knob (md_debug_set_window_report)

// All in us, 8 kv heads unless said.  The bounds alone are known here, not the rows: one request's many choose the layout of all (63 requests of one token behind 16 032
// and one of 128 in 8 bits 1 439; in a call each 324 and 55).
WinPlan window_plan(int B, int n_max, int H, int KH, int D, int max_pages, int page_size, int kind, int window, int sinks) {
    WinPlan pl;
    const int64_t rows = (int64_t)n_max * (H / KH), pairs = (int64_t)B * KH;
    // keys that a group of rows looks at, at most
    const int64_t all = (int64_t)max_pages * page_size;
    const auto seen = [&](int64_t of) {
        const int64_t n = std::min<int64_t>(n_max, (of + H / KH - 1) / (H / KH) + 1);
        return window > 0 ? std::min<int64_t>(all, (int64_t)window + n + std::min<int64_t>(sinks, all)) : all;
    };
    pl.nw = 0;
    pl.rows = rows <= 16 ? 16 : 32;
    if (rows > 32) {
        // the kernel above, whose wavefronts share a group's keys, so that keys are read and unpacked for every 32 rows; 4 and 8 wavefronts of winprompt.hip,
        // which share them all
        const int bits = kind == MD_KV_BF16 ? 16 : kind == MD_KV_MXFP4 ? 4 : 8;
        const WinWay wide[3] = {{0, 32, 128, bits == 16 ? 6.7 : 8.2, bits == 4 ? 1.16 : 1.36, bits == 16 ? 2.2 : bits == 8 ? 1.37 : 1.06, 0},
                                {4, 128, 64, 7.7, 1.78, 1.27, 0}, {8, 256, 128, 10.8, 3.2, 3.2, 8}};
        const WinWay narrow[3] = {{0, 32, 128, 6.4, 0.9, bits == 16 ? 1.03 : bits == 8 ? 0.83 : 0.66, 0},
                                  {4, 128, 64, 6.8, 1.18, 0.77, 0}, {8, 256, 64, 8.1, 1.35, 1.05, 3}};
        const double sums = (double)(pairs * rows) * (D * 8 + 16);
        double least = 1e300;
        for (const WinWay& w : D == 64 ? narrow : wide) {
            const int64_t groups = pairs * ((rows + w.rows - 1) / w.rows), keys = seen(w.rows);
            const int edges = keys == all ? 0 : 1 + (sinks > 0);
            for (int parts : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32}) {
                if (parts > 1 && (keys < 128 * parts || groups * parts > 1024)) break;
                const double us = w.us(groups * parts, keys, edges, parts, sums);
                if (us < least) least = us, pl.nw = w.nw, pl.rows = w.rows, pl.nsplit = parts;
            }
        }
    }
    pl.n_qgroups = (int)((rows + pl.rows - 1) / pl.rows);
    const int64_t keys = seen(pl.rows), have = pairs * pl.n_qgroups;
    if (rows <= 32) {
        // Keys over several workgroups, of enough keys each to pay for the launch that joins them (3.5).  One a CU up to half as many (4 x 4 rows over 5 000
        // keys in bf16: 70 whole, 22 in 256, 25 in 512), two where 8- or 4-bit streams stay long (8 x 4 over 8 000 37 and 34).  Up to a workgroup a
        // CU three each where that is two a CU (130 over 8 000 keys of 64 in 4 bits 38 whole, 24; over 1 200 10.6 and 11.0), of 8- and 4-bit streams
        // two beyond (200 over 8 000 in 8 bits 89 and 82, in bf16 143 and 156).  More workgroups: three where streams are long and the last ones
        // would leave CUs behind (40 x 4 x 8 over 9 000 in bf16 311 whole, 242 in three; 48 x 4 x 8 337 and 289 in two)
        const int64_t stream = keys * 2 * kv_row_bytes(kind, D);
        const bool long_way = stream >= 700000, left = have * 100 < (have + 511) / 512 * 512 * 85;
        int64_t want;
        if (have <= 128)
            want = (kind != MD_KV_BF16 && keys * have >= 512000 ? 512 : 256) / have;
        else if (have <= 256)
            want = have * 3 <= 512 && keys >= 2048 ? 3 : kind != MD_KV_BF16 && keys >= 4096 ? 2 : 1;
        else
            want = !long_way || !left ? 1 : have <= 352 ? 3 : 2;
        pl.nsplit = (int)std::max<int64_t>(1, std::min<int64_t>({want, keys <= 512 ? 1 : keys / 128, 64}));
    }
    // 64 keys at a time where that spills nothing and the stream is long: 4-bit heads of 64, 64 requests of 16 036 keys x 16 rows 133 -> 114, of 1 000 12.9
    // -> 12.2; one request of 1 500 in eight parts 8.5 -> 9.9
    pl.kg = kind == MD_KV_MXFP4 && D == 64 && pl.rows == 16 && page_size % 64 == 0 && keys / pl.nsplit >= 1024 ? 2 : 1;
    pl.slots = pl.nsplit > 1 ? (size_t)have * pl.nsplit * pl.rows : 0;
    if (g_report) {
        const int report[5] = {pl.nw, pl.rows, pl.n_qgroups, pl.nsplit, pl.nw ? window_prompt_tile(D, pl.nw, page_size) : 32 * pl.kg};
        std::copy(report, report + 5, g_report);
    }
    return pl;
}

template <int D, int QT, int KIND, int KG>
int launch_window(const WinParams& p, int grid, hipStream_t st) {
    constexpr int lds = kWaves * win_wave_lds<D, QT, KG>();
    auto k = window_attn_kernel<D, QT, KIND, KG>;
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
    hipLaunchKernelGGL(k, dim3(grid), dim3(64 * kWaves), lds, st, p);
    MD_CHECK_LAUNCH("md_window_attn");
    return MD_OK;
}

template <int D, int KIND>
int launch_window_rows(const WinParams& p, const WinPlan& pl, int grid, hipStream_t st) {
    if constexpr (D == 64 && KIND == MD_KV_MXFP4)
        if (pl.kg == 2) return launch_window<D, 1, KIND, 2>(p, grid, st);
    return pl.rows == 16 ? launch_window<D, 1, KIND, 1>(p, grid, st) : launch_window<D, 2, KIND, 1>(p, grid, st);
}

template <int D>
int launch_window_kind(const WinParams& p, int kind, const WinPlan& pl, int grid, hipStream_t st) {
    switch (kind) {
        case MD_KV_BF16: return launch_window_rows<D, MD_KV_BF16>(p, pl, grid, st);
        case MD_KV_FP8_E4M3: return launch_window_rows<D, MD_KV_FP8_E4M3>(p, pl, grid, st);
        case MD_KV_MXFP8: return launch_window_rows<D, MD_KV_MXFP8>(p, pl, grid, st);
        default: return launch_window_rows<D, MD_KV_MXFP4>(p, pl, grid, st);
    }
}

int launch_window_prompt(const WinParams& p, int kind, int D, int nw, int grid, hipStream_t st) {
    switch (kind) {
        case MD_KV_BF16: return md_window_prompt_0(p, D, nw, grid, st);
        case MD_KV_FP8_E4M3: return md_window_prompt_1(p, D, nw, grid, st);
        case MD_KV_MXFP8: return md_window_prompt_2(p, D, nw, grid, st);
        default: return md_window_prompt_3(p, D, nw, grid, st);
    }
}

template <int D>
void launch_window_merge(const WinParams& p, int rows, hipStream_t st) {
    const int64_t threads = (int64_t)p.B * p.KH * p.n_qgroups * rows * (D / 4);
    const int sg = p.nsplit <= 8 ? 1 : 8;
    const dim3 grid((unsigned)((threads * sg + 255) / 256));
    if (sg == 1)
        hipLaunchKernelGGL((window_merge_kernel<D, 1>), grid, dim3(256), 0, st, p, rows);
    else
        hipLaunchKernelGGL((window_merge_kernel<D, 8>), grid, dim3(256), 0, st, p, rows);
}

bool window_shape_ok(int B, int n_max, int H, int KH, int max_pages, int page_size) {
    return B > 0 && n_max > 0 && KH > 0 && H > 0 && H % KH == 0 && max_pages > 0 && page_size > 0 && page_size % 32 == 0 && page_size <= 65536 &&
           (int64_t)max_pages * page_size < (1 << 30) && (int64_t)n_max * (H / KH) < (1 << 30);
}

}  // namespace

#ifdef MD_DEV_KNOBS   // include/magicdec_hip_dev.h: not part of the drop-in boundary
extern "C" void md_debug_set_window_report(int* report) { g_report = report; }
#endif

extern "C" size_t md_window_attn_workspace_bytes(int B, int n_max, int H, int KH, int D, int max_pages_per_req, int page_size, int kv_dtype,
                                                 int window, int sinks) {
    if (!window_shape_ok(B, n_max, H, KH, max_pages_per_req, page_size) || window < 0 || sinks < 0) return 0;
    return window_plan(B, n_max, H, KH, D, max_pages_per_req, page_size, kv_dtype & MD_KV_DTYPE_MASK, window, sinks).slots * ((size_t)D * 4 + 8) + 256;
}

extern "C" int md_window_attn(const void* q, int64_t q_row_stride, const void* cache, void* out, const int32_t* qo_indptr,
                              const int32_t* page_indices, const int32_t* page_indptr, const int32_t* last_page_len, int B, int n_max, int H,
                              int KH, int D, int page_size, int window, int sinks, float sm_scale, int max_pages_per_req, int kv_dtype,
                              const float* k_scale, const float* v_scale, void* workspace, size_t workspace_bytes, md_stream_t stream) {
    MD_CHECK_ARG(q && cache && out && qo_indptr && page_indices && page_indptr && last_page_len, "md_window_attn: null pointer argument");
    MD_CHECK_ARG(window_shape_ok(B, n_max, H, KH, max_pages_per_req, page_size),
                 "md_window_attn: bad shape B=%d n_max=%d H=%d KH=%d pages=%d page_size=%d (pages of multiples of 32 rows, to 65 536)", B, n_max, H, KH,
                 max_pages_per_req, page_size);
    if (D != 64 && D != 128) {
        md_set_error("md_window_attn: head_dim %d unsupported (64 or 128)", D);
        return MD_ERR_UNSUPPORTED;
    }
    MD_CHECK_ARG(window >= 0 && sinks >= 0, "md_window_attn: window %d and sinks %d must not be negative", window, sinks);
    MD_CHECK_ARG(sm_scale > 0.f, "md_window_attn: sm_scale must be > 0");
    MD_CHECK_ARG(q_row_stride % 8 == 0 && ((uintptr_t)q & 15) == 0 && ((uintptr_t)cache & 15) == 0 && ((uintptr_t)out & 7) == 0,
                 "md_window_attn: q/cache must be 16-byte aligned with a row stride multiple of 8, out 8-byte aligned");
    MD_CHECK_ARG((kv_dtype & ~(MD_KV_DTYPE_MASK | MD_KV_LAYOUT_HND)) == 0, "md_window_attn: unknown kv_dtype flags");
    const bool hnd = (kv_dtype & MD_KV_LAYOUT_HND) != 0;
    const int kind = kv_dtype & MD_KV_DTYPE_MASK;
    MD_CHECK_ARG(kind <= MD_KV_MXFP4 && (kind != MD_KV_FP8_E4M3 || (k_scale && v_scale)),
                 "md_window_attn: kv_dtype must be MD_KV_BF16, MD_KV_FP8_E4M3 (with per-head scales), MD_KV_MXFP8 or MD_KV_MXFP4");
    MD_CHECK_ARG(hnd || !kv_is_mx(kind), "md_window_attn: block-scaled pages are HND");

    const WinPlan pl = window_plan(B, n_max, H, KH, D, max_pages_per_req, page_size, kind, window, sinks);
    const size_t need = pl.slots * ((size_t)D * 4 + 8);
    if (pl.nsplit > 1 && !(workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0)) {
        md_set_error("md_window_attn: workspace too small or misaligned (%zu < %zu)", workspace_bytes, need);
        return MD_ERR_WORKSPACE;
    }
    const int64_t grid = (int64_t)B * KH * pl.n_qgroups * pl.nsplit;
    MD_CHECK_ARG(grid <= 0x7fffffff, "md_window_attn: too many rows for a grid");
    WinParams p = {};
    p.q = (const bf16_t*)q;
    p.cache = (const unsigned char*)cache;
    p.out = (bf16_t*)out;
    p.qo_indptr = qo_indptr;
    p.indices = page_indices;
    p.indptr = page_indptr;
    p.last = last_page_len;
    p.ws_o = (float*)workspace;
    p.ws_ml = p.ws_o + pl.slots * D;
    p.q_row_stride = q_row_stride;
    p.g = kv_pages(kind, KH, D, page_size, hnd);
    p.B = B;
    p.H = H;
    p.KH = KH;
    p.group = H / KH;
    p.page_size = page_size;
    p.nsplit = pl.nsplit;
    p.n_qgroups = pl.n_qgroups;
    p.window = std::min(window, 1 << 30);      // more than all, and positions less it stay in range
    p.sinks = std::min(sinks, 1 << 30);
    p.scale_log2 = sm_scale * 1.4426950408889634f;
    p.k_scale = kind == MD_KV_FP8_E4M3 ? k_scale : nullptr;
    p.v_scale = kind == MD_KV_FP8_E4M3 ? v_scale : nullptr;
    hipStream_t st = (hipStream_t)stream;
    const int rc = pl.nw ? launch_window_prompt(p, kind, D, pl.nw, (int)grid, st)
                   : D == 128 ? launch_window_kind<128>(p, kind, pl, (int)grid, st) : launch_window_kind<64>(p, kind, pl, (int)grid, st);
    if (rc != MD_OK) return rc;
    if (pl.nsplit > 1) {
        D == 128 ? launch_window_merge<128>(p, pl.rows, st) : launch_window_merge<64>(p, pl.rows, st);
        MD_CHECK_LAUNCH("md_window_attn(merge)");
    }
    return MD_OK;
}

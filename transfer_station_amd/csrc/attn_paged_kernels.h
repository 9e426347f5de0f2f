// attn_paged_kernels.h -- gfx950 kernels of the paged KV cache: attention over it (attn_paged), appending
// to it (attn_kv_append) and reading it back (attn_kv_read). Part of attn_kernels.hip.
//
// The cache: pages of 16 .. 256 tokens, K and V [pages][Hkv][page][D], in bf16, or in 4 bits as E2M1 codes
// (two to a byte, the even element low) with one E8M0 scale byte per 32 elements of a row. A sequence's
// pages are named by its row of the table. Every 16 keys that start at a multiple of 16 lie in one page,
// back to back, so the kernels address the cache in such blocks: one page id, one buffer descriptor of at
// most 16 rows whose range ends at the sequence's last key (keys past it arrive as zeros) and 32-bit
// offsets inside it, however large the cache. A page id outside the cache gives an empty range, and its
// keys are masked.
//
//   S = scale Q.K, optionally cap tanh(S / cap), minus slope |position - key|; softmax; O = P.V
//
// in fp32 but for the operands of the MFMAs: K, V, Q as they are (4-bit codes become bf16 exactly) and P
// rounded to bf16, as in attn_flash; O is rounded once, to bf16.
#ifndef ATTN_PAGED_KERNELS_H
#define ATTN_PAGED_KERNELS_H

#include "attn_device.h"
#include "attn_launch.h"
#include "attn_paged_cut.h"
#include "attn_paged_rule.h"

namespace {

typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
// Tables and lengths are read through the scalar cache: wave-uniform and not written by the kernel.
typedef const __attribute__((address_space(4))) int32_t const_i32;
__device__ __forceinline__ int scalar_i32(const int32_t *p, long i) {
    return ((const_i32 *)(uintptr_t)p)[i];
}

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// Eight 4-bit codes, times their scale, as eight bf16 values: exact, but for a scale so small or large
// that bf16 has no such value.
__device__ __forceinline__ u32x4 fp4_to_bf16(uint32_t w, float scale) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0);
    const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2);
    const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3);
    return u32x4{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b),
                 __builtin_bit_cast(uint32_t, c), __builtin_bit_cast(uint32_t, d)};
}
__device__ __forceinline__ float e8m0(uint32_t e) { return __builtin_bit_cast(float, e << 23); }

__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
    const bf16x2 r = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(uint32_t, r);
}

// Scores in units of log2 from raw dot products: each(f) applies f(score, offset of its key behind the first)
// to all of them, `first` is how far the row's position lies behind the first key. The tests are uniform, and
// outside the loops over the scores.
//   cap tanh(y), y = score / cap, as cap (1 - 2 / (2^x + 1)) with x = 2 log2(e) y: five instructions, off by up to
//   2^-20 of the cap, whatever the score is. Up to a cap of kCapNear that is a sixteenth of what P's rounding to bf16
//   does. Past it a |y| below a quarter takes cap y (1 - y^2 / 3 + 2 y^4 / 15 - ..), up to y^8 with the last term
//   spread over the others by a Chebyshev polynomial (2^-26 in all): off by a few 2^-24 of the score, so that a
//   cap far above the scores leaves them as they are. In w = 0.3287 y^2 the last coefficient is -1/2, an immediate.
//   Nine instructions more, behind a uniform branch: 512 tokens over 8192 keys 102 us with a cap of 30, 130 with one of
//   1000 (64 sequences of 4096 in bf16 164 with either, in 4 bits 57 and 63).
//   The distance is exact up to 2^24 tokens, and its absolute value free.
constexpr float kCapNear = 256.0f * 1.44269504088896341f; // log2(e) times a cap of 256
template <typename E>
__device__ __forceinline__ void modify_scores(const attn_paged_args &a, float slope, int first, E &&each) {
    auto capped = [&](float x) {
        return fmaf(-2.f * a.cap_out, __builtin_amdgcn_rcpf(fast_exp2(x) + 1.f), a.cap_out);
    };
    const int cap = __builtin_bit_cast(int, a.cap_out); // >= 0: ordered as integers, which the scalar unit compares
    if (cap > __builtin_bit_cast(int, kCapNear))
        each([&](float s, int) {
            const float x = s * a.cap_in, w = x * x * 0.0394809060f;
            const float p = fmaf(w, fmaf(w, fmaf(w, -0.5f, 0.427360013f), -0.351460313f), 0.346573590f);
            float far = capped(x);
            asm volatile("" : "+v"(far)); // a select: with a branch for each score D = 256 spills
            return fabsf(x) < 0.72134752f ? x * p * a.cap_out : far; // |y| = 1/4
        });
    else if (cap != 0)
        each([&](float s, int) { return capped(s * a.cap_in); });
    else
        each([&](float s, int) { return s * a.c; });
    if (a.slopes) {
        const float d = (float)first;
        each([&](float s, int off) { return fmaf(-slope, fabsf(d - (float)off), s); });
    }
}

__device__ __forceinline__ attn_seq seq_at(const attn_paged_args &a, int b) {
    return attn_seq_of(scalar_i32(a.q_start, b), scalar_i32(a.q_start, b + 1), scalar_i32(a.kv_len, b), a.T,
                       a.cols, a.lgp);
}

// Sum or maximum over the wave, in every lane.
template <bool MAX> __device__ __forceinline__ int wave_all(int x) {
    auto op = [](int p, int q) { return MAX ? max(p, q) : p + q; };
    x = op(x, __builtin_amdgcn_update_dpp(x, x, 0x128, 0xf, 0xf, false)); // row_ror:8, 4, 2, 1
    x = op(x, __builtin_amdgcn_update_dpp(x, x, 0x124, 0xf, 0xf, false));
    x = op(x, __builtin_amdgcn_update_dpp(x, x, 0x122, 0xf, 0xf, false));
    x = op(x, __builtin_amdgcn_update_dpp(x, x, 0x121, 0xf, 0xf, false));
    const auto p = __builtin_amdgcn_permlane16_swap((unsigned)x, (unsigned)x, false, false);
    x = op((int)p[0], (int)p[1]);
    const auto r = __builtin_amdgcn_permlane32_swap((unsigned)x, (unsigned)x, false, false);
    return op((int)r[0], (int)r[1]);
}

// x plus those of the lanes below (DPP row shifts, then the rows' last lanes broadcast to the rows behind).
__device__ __forceinline__ int wave_scan(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true); // row_shr:1, 2, 4, 8
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false); // row_bcast:15 into rows 1 and 3
    return x + __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false); // row_bcast:31 into rows 2 and 3
}

// The decode line (attn_quota) as a wave sees it, 64 sequences at a time: a kv head's units and the quota.
// One sequence needs no sum, and up to 64 are read once.
struct line {
    int total, quota;
    int n, sum; // of sequence `lane`: units, and units up to and with it
};
__device__ __forceinline__ int units_at(const attn_paged_args &a, int i) {
    if (i >= a.B)
        return 0;
    const attn_seq s = attn_seq_of(a.q_start[i], a.q_start[i + 1], a.kv_len[i], a.T, a.cols, a.lgp);
    return attn_units(s.n, s.kend);
}
__device__ __forceinline__ line line_at(const attn_paged_args &a, int lane) {
    line l;
    int most;
    if (a.B == 1) {
        const attn_seq s = seq_at(a, 0);
        l.n = l.sum = l.total = most = attn_units(s.n, s.kend);
    } else {
        l.n = units_at(a, lane);
        l.sum = wave_scan(l.n);
        l.total = __builtin_amdgcn_readlane(l.sum, 63);
        int m = l.n;
        for (int i0 = 64; i0 < a.B; i0 += 64) {
            const int n = units_at(a, i0 + lane);
            m = max(m, n);
            l.total += __builtin_amdgcn_readlane(wave_scan(n), 63);
        }
        most = uniform(wave_all<true>(m));
    }
    l.quota = uniform(attn_quota(l.total, most, a.Hkv, a.teams, a.nsplit));
    return l;
}
// The sequence that unit `at` of a kv head's line belongs to, and the units before that.
__device__ __forceinline__ int seq_of_unit(const attn_paged_args &a, const line &l, int lane, int at,
                                           int &before) {
    before = 0;
    if (a.B == 1)
        return 0;
    int n = l.n, sum = l.sum, base = 0;
    for (int i0 = 0;;) {
        const uint64_t past = __builtin_amdgcn_ballot_w64(base + sum > at);
        if (past != 0) {
            const int k = __builtin_ctzll(past);
            before = base + __builtin_amdgcn_readlane(sum - n, k);
            return i0 + k;
        }
        base += __builtin_amdgcn_readlane(sum, 63);
        i0 += 64;
        if (i0 >= a.B) // not reached for a unit of the line
            return 0;
        n = units_at(a, i0 + lane);
        sum = wave_scan(n);
    }
}

// N = 16 keys of the cache from key kb (a multiple of N): their rows' place, and how many of them there are (0
// where the page id is none, or past the sequence's end).
struct kv_block {
    int64_t row;
    int n;
};
// The id of the page that key kb's block is in, for kend >= 1. Its scalar load is issued a tile ahead: waited
// for where its rows are asked for, every tile began with its latency.
__device__ __forceinline__ int page_id(const attn_paged_args &a, const int32_t *table, int kb, int kend) {
    return scalar_i32(table, min(kb, kend - 1) >> a.lgp);
}
template <int N = 16>
__device__ __forceinline__ kv_block block_in(const attn_paged_args &a, int pg, int u, int kb, int kend) {
    const bool ok = attn_page_ok(pg, a.pages);
    return kv_block{attn_page_row(ok ? pg : 0, a.Hkv, u, kb, a.lgp), ok ? max(0, min(N, kend - kb)) : 0};
}

// b ? x : y of two values (of two array elements the operator itself would choose the address, and keep the
// array in memory).
__device__ __forceinline__ uint32_t pick(bool b, uint32_t x, uint32_t y) { return b ? x : y; }

template <bool NT> __device__ __forceinline__ u32x4 buf16(__amdgpu_buffer_rsrc_t r, uint32_t off) {
    return __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, NT ? kDmaNT : 0);
}

// What a sum of p changes by when the maximum that p is taken against rises from m0 to m1: p is 2^(s c - m c) with m c
// rounded, so the factor is between the rounded products. Taken from m0 - m1 it was off by their roundings, at
// scores of 2^20 by up to 9%.
__device__ __forceinline__ float rescale(float m0, float m1, float c) {
#pragma clang fp contract(off)
    const float a = m0 * c, b = m1 == kNegInf ? 0.f : m1 * c;
    return fast_exp2(a - b);
}

// A part's maximum as the merge is told it. There +inf says that the row is written and -inf that the part has
// nothing: an infinite score, and a part of NaN alone, go by finite ones, and their sums carry the NaN.
__device__ __forceinline__ float part_max(float m, float l) {
    uint32_t bits = __builtin_bit_cast(uint32_t, l);
    asm("" : "+v"(bits)); // as a comparison of floats, which the compiler makes of it, it would leave out NaN
    const bool lost = m == kNegInf && bits << 1 != 0;
    return lost ? 0.f : fminf(m, 3.402823466e38f);
}

// ------------------------------------------------------------------------------------------
// Few query rows per kv head. A workgroup takes its quota of the decode line (attn_quota) -- keys of one
// sequence and kv head after the other -- for one tile of 16 NRB rows (or, without teams, a whole sequence); a
// sequence's rows are its tokens' heads of the group, token by token. The four waves take interleaved tiles of 32
// keys (two blocks of 16), each with a softmax of its own:
//   S^T[key][row] = K . Q^T   (v_mfma_f32_16x16x32_bf16, K from memory straight into the operand)
//   O^T[d][row]  += V^T . P^T (V through a wave-private LDS tile and the transposed read)
// and merge in LDS at the end of each sequence. Tiles past the grid's (a sequence with more rows than max_q says)
// follow in the same workgroup.
//
// Bound by HBM: 64 sequences of 4096 keys, 8 kv heads, D = 128: bf16 163 us (6.6 TB/s), 4 bits 52.6 (5.4 TB/s, where
// the unpacking takes 11 instructions per MFMA); of 250 to 8192 keys 162 us for 1.02 GB. Equal quotas are why: with
// a workgroup per part of a sequence the same ragged batch took 198. They hold as long as the partial slots, one per
// row of T and part, allow as many parts: 512 sequences of 64 heads have two each, so that no quota is below the
// longest sequence, and with one of 32768 keys among 1000s they take 1004 us, 344 without it. One sequence of
// 32768, D = 256, 4 bits, is 14.4 us of latency: start, four units, the join.
// Past D = 128 a row tile is 16 rows and reads all keys for itself: 16 x 8 tokens over 2000 to 4000 keys, 32 heads on 8,
// at D = 256 bf16 114 us, 4 bits 47; at D = 128, where it is 32 rows, 46 and 28.
// ------------------------------------------------------------------------------------------
template <int DP, bool F4, int NRB, bool MOD, bool NTL>
__global__ __launch_bounds__(256, 2) void attn_paged_decode_kernel(const attn_paged_args a) {
    constexpr int VSTR = DP + 16; // elements of a V row in LDS: the eight rows of a pass on other banks
    constexpr int KN = DP / 32;   // MFMA steps along d
    constexpr int NV = DP / 16;   // bf16: 16-byte pieces of a V tile per lane
    // 4 bits: a lane's piece of a V row (PB bytes), lanes per row, rows per load, loads per tile
    constexpr int PB = DP == 64 ? 8 : 16, LPR = DP / 2 / PB, RPL = 64 / LPR, NV4 = 32 / RPL;
    constexpr int NSC = DP == 256 ? 2 : 1; // scales of a lane's share of a K row
    constexpr int VTILE = 32 * VSTR;
    __shared__ __attribute__((aligned(16))) uint16_t Vw[4 * VTILE];
    __shared__ float red_m[NRB][4][16], red_l[NRB][4][16];
    static_assert(4 * 16 * (DP + 4) * 4 <= 4 * VTILE * 2, "merge area must fit in the V tiles");

    const int tid = wi_id_x(), w = uniform(tid >> 6), lane = tid & 63;
    const int r16 = lane & 15, grp = lane >> 4;
    const int g = a.Hq / a.Hkv, D = a.D;
    const float c = MOD ? 1.f : a.c;
    const float lift = 8.f / c; // how far a score may pass the running maximum
    // This workgroup's row tile t0 and its place on the line: sequence b, kv head u, first unit `off` of the
    // sequence, `left` units in all. The workgroups of a team, and of neighbouring ones, share an XCD.
    const int L = uniform(xcd_remap(wg_id_x(), (a.teams ? a.teams : a.B * a.Hkv) * a.tps));
    const int team = uniform(L / a.tps), t0 = L - team * a.tps;
    int u, b, off = 0, left = 1, pos0 = 0;
    line ln = {0, 1, 0, 0};
    if (a.teams) {
        ln = line_at(a, lane);
        if ((int64_t)team * ln.quota >= (int64_t)ln.total * a.Hkv)
            return;
        pos0 = team * ln.quota;
        left = min(ln.quota, ln.total * a.Hkv - pos0);
        u = uniform(pos0 / ln.total);
        int before;
        b = uniform(seq_of_unit(a, ln, lane, pos0 - u * ln.total, before));
        off = pos0 - u * ln.total - before;
    } else {
        u = uniform(team / a.B);
        b = team - u * a.B;
    }
    uint16_t *vt = &Vw[w * VTILE];

    while (left > 0 && u < a.Hkv) {
        const attn_seq sq = seq_at(a, b);
        const int units = attn_units(sq.n, sq.kend), R = sq.n * g;
        const int take = a.teams ? min(left, units - off) : 1;
        attn_cover cover = {0, 1};
        if (a.teams) {
            cover = attn_cover_of(pos0 - off, max(units, 1), ln.quota);
            cover = attn_cover{uniform(cover.first), uniform(cover.live)};
        }
        const int live = cover.live, sp = team - cover.first;
        const int k0 = min(off * 128, sq.kend), k1 = a.teams ? min((off + take) * 128, sq.kend) : sq.kend;
        const int32_t *table = a.table + (int64_t)b * a.cols;
        for (int tile = t0; take > 0 && (int64_t)tile * 16 * NRB < R; tile += a.tps) {
            const int row0 = tile * 16 * NRB;
            bf16x8 qb[NRB][KN];
            int lim[NRB], pos[NRB];
            float m_run[NRB], l_run[NRB], slope[NRB];
            f32x4 o[NRB][DP / 16];
    #pragma unroll
            for (int i = 0; i < NRB; ++i) {
                const int row = row0 + 16 * i + r16;
                const bool valid = row < R;
                const int tok = valid ? row / g : 0, h = u * g + (valid ? row % g : 0);
                const uint16_t *q = a.q + (sq.q0 + tok) * a.q_tok + h * a.q_head;
    #pragma unroll
                for (int kk = 0; kk < KN; ++kk) {
                    const int col = F4 ? grp * (DP / 4) + kk * 8 : kk * 32 + grp * 8;
                    u32x4 x = zero4();
                    if (valid && col < D)
                        x = *reinterpret_cast<const u32x4 *>(q + col);
                    qb[i][kk] = as_bf16x8(x);
                }
                pos[i] = sq.len - sq.n + tok;
                lim[i] = a.causal ? min(pos[i], k1 - 1) : k1 - 1;
                slope[i] = MOD && a.slopes ? a.slopes[h] * 1.44269504088896341f : 0.f;
                m_run[i] = kNegInf;
                l_run[i] = 0.f;
    #pragma unroll
                for (int db = 0; db < DP / 16; ++db)
                    o[i][db] = f32x4{0.f, 0.f, 0.f, 0.f};
            }
            // Keys from the tile's last row's position on are hidden from it.
            const int kstop = a.causal ? min(k1, sq.len - sq.n + (min(row0 + 16 * NRB, R) - 1) / g + 1) : k1;

            struct frags {
                u32x4 k[F4 ? 1 : 2 * KN], v[F4 ? 1 : NV];
                uint32_t kw[F4 ? 2 * KN : 1], ksc[F4 ? 2 : 1];
                uint32_t vw[F4 ? NV4 * PB / 4 : 1], vsc[F4 ? NV4 : 1];
            };
            // The loads of the next tile are issued as soon as this one's have been used: V's once it is in LDS,
            // K's once the scores are there. K and V of a tile, Q and O do not fit 256 registers at DP = 256 in
            // bf16: there a tile's K is loaded at its start, and V once the scores have freed K's registers.
            constexpr bool kLate = DP == 256 && !F4;
            auto load_k = [&](const kv_block &b0, const kv_block &b1, frags &f) __attribute__((always_inline)) {
    #pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const kv_block &bl = t ? b1 : b0;
                    if constexpr (!F4) {
                        const uint32_t rb = (uint32_t)D * 2u; // bytes of a row
                        const auto kr = make_rsrc(a.k + bl.row * rb, bl.n * rb);
    #pragma unroll
                        for (int kk = 0; kk < KN; ++kk) {
                            const int col = kk * 32 + grp * 8;
                            f.k[t * KN + kk] = buf16<NTL>(kr, col < D ? r16 * rb + col * 2 : 0x80000000u);
                        }
                    } else {
                        constexpr int RB = DP / 2, SB = DP / 32; // bytes of a row's codes and scales
                        const auto kr = make_rsrc(a.k + bl.row * RB, bl.n * RB);
                        const auto sr = make_rsrc(a.ks + bl.row * SB, bl.n * SB);
                        if constexpr (DP == 64) {
                            const u32x2 x = __builtin_amdgcn_raw_buffer_load_b64(
                                kr, r16 * RB + grp * (RB / 4), 0, NTL ? kDmaNT : 0);
                            f.kw[t * KN] = x[0];
                            f.kw[t * KN + 1] = x[1];
                        } else {
    #pragma unroll
                            for (int j = 0; j < KN / 4; ++j) {
                                const u32x4 x = buf16<NTL>(kr, r16 * RB + grp * (RB / 4) + 16 * j);
    #pragma unroll
                                for (int i = 0; i < 4; ++i)
                                    f.kw[t * KN + 4 * j + i] = x[i];
                            }
                        }
                        if constexpr (NSC == 2)
                            f.ksc[t] = __builtin_amdgcn_raw_buffer_load_b16(sr, r16 * SB + grp * 2, 0, 0);
                        else
                            f.ksc[t] = __builtin_amdgcn_raw_buffer_load_b8(sr, r16 * SB + grp * SB / 4, 0, 0);
                    }
                }
            };
            auto load_v = [&](const kv_block &b0, const kv_block &b1, frags &f) __attribute__((always_inline)) {
                if constexpr (!F4) {
                    const uint32_t rb = (uint32_t)D * 2u;
                    const auto vr0 = make_rsrc(a.v + b0.row * rb, b0.n * rb);
                    const auto vr1 = make_rsrc(a.v + b1.row * rb, b1.n * rb);
                    const uint32_t v0 = (lane % (DP / 8)) * 8 < D
                                            ? (lane / (DP / 8)) * rb + (lane % (DP / 8)) * 16
                                            : 0x80000000u;
    #pragma unroll
                    for (int r = 0; r < NV; ++r)
                        f.v[r] = buf16<NTL>(r < NV / 2 ? vr0 : vr1, v0 + (r % (NV / 2)) * (512 / DP) * rb);
                } else {
                    constexpr int RB = DP / 2, SB = DP / 32;
    #pragma unroll
                    for (int r = 0; r < NV4; ++r) {
                        const kv_block &bl = r < NV4 / 2 ? b0 : b1;
                        const auto vr = make_rsrc(a.v + bl.row * RB, bl.n * RB);
                        const auto sr = make_rsrc(a.vs + bl.row * SB, bl.n * SB);
                        const int row = lane / LPR + r % (NV4 / 2) * RPL, piece = lane % LPR;
                        if constexpr (DP == 64) {
                            const u32x2 x = __builtin_amdgcn_raw_buffer_load_b64(
                                vr, row * RB + piece * PB, 0, NTL ? kDmaNT : 0);
                            f.vw[2 * r] = x[0];
                            f.vw[2 * r + 1] = x[1];
                        } else {
                            const u32x4 x = buf16<NTL>(vr, row * RB + piece * PB);
    #pragma unroll
                            for (int i = 0; i < 4; ++i)
                                f.vw[4 * r + i] = x[i];
                        }
                        f.vsc[r] = __builtin_amdgcn_raw_buffer_load_b8(sr, row * SB + piece * SB / LPR, 0, 0);
                    }
                }
            };
            // 4 bits: of the eight lanes that write together, which hold pieces of one row or two, several would
            // have their chunk j on the same banks; so it lies at j ^ swap of its piece.
            auto put_v = [&](const frags &f) __attribute__((always_inline)) {
                lds_wave_fence(); // the previous tile's transposed reads are complete
                if constexpr (!F4) {
    #pragma unroll
                    for (int r = 0; r < NV; ++r) {
                        const int at = lane + 64 * r;
                        *reinterpret_cast<u32x4 *>(&vt[at / (DP / 8) * VSTR + at % (DP / 8) * 8]) = f.v[r];
                    }
                } else {
    #pragma unroll
                    for (int r = 0; r < NV4; ++r) {
                        const int row = lane / LPR + r * RPL, piece = lane % LPR;
                        const int swap = DP == 64 ? row & 1 : piece >> 1;
                        const float sc = e8m0(f.vsc[r]);
#pragma unroll
                        for (int j = 0; j < PB / 4; ++j)
                            *reinterpret_cast<u32x4 *>(&vt[row * VSTR + piece * 2 * PB + 8 * (j ^ swap)]) =
                                fp4_to_bf16(f.vw[r * (PB / 4) + j], sc);
                    }
                }
            };
            auto compute = [&](int tb, const kv_block &b0, const kv_block &b1, const kv_block &n0,
                               const kv_block &n1, frags &f) __attribute__((always_inline)) {
                bf16x8 kf[2][KN], pk[NRB];
                f32x4 s[NRB][2];
    #pragma unroll
                for (int t = 0; t < 2; ++t)
    #pragma unroll
                    for (int kk = 0; kk < KN; ++kk) {
                        if constexpr (F4)
                            kf[t][kk] = as_bf16x8(fp4_to_bf16(
                                f.kw[t * KN + kk],
                                e8m0(NSC == 2 ? (f.ksc[t] >> (kk / 4 * 8)) & 0xff : f.ksc[t])));
                        else
                            kf[t][kk] = as_bf16x8(f.k[t * KN + kk]);
                    }
    #pragma unroll
                for (int i = 0; i < NRB; ++i)
    #pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        s[i][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    #pragma unroll
                        for (int kk = 0; kk < KN; ++kk)
                            s[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[t][kk], qb[i][kk], s[i][t], 0, 0, 0);
                    }
                __builtin_amdgcn_sched_barrier(0);
                if (kLate)
                    load_v(b0, b1, f);
                else
                    load_k(n0, n1, f);
    #pragma unroll
                for (int i = 0; i < NRB; ++i) {
                    // Register (t, j) of this lane holds key tb + 16t + 4grp + j for row r16.
                    if (MOD)
                        modify_scores(a, slope[i], pos[i] - tb - 4 * grp, [&](auto f) __attribute__((always_inline)) {
    #pragma unroll
                            for (int t = 0; t < 2; ++t)
    #pragma unroll
                                for (int j = 0; j < 4; ++j)
                                    s[i][t][j] = f(s[i][t][j], 16 * t + j);
                        });
                    float mx = kNegInf;
    #pragma unroll
                    for (int t = 0; t < 2; ++t)
    #pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int key = tb + 16 * t + 4 * grp + j;
                            if (key > lim[i] || (t ? b1.n : b0.n) == 0)
                                s[i][t][j] = kNegInf;
                            mx = fmaxf(mx, s[i][t][j]);
                        }
                    mx = max_xor32(max_xor16(mx));
                    if (__builtin_amdgcn_ballot_w64(mx > m_run[i] + lift) != 0) {
                        const float mnew = fmaxf(m_run[i], mx);
                        const float alpha = rescale(m_run[i], mnew, c);
                        m_run[i] = mnew;
                        l_run[i] *= alpha;
    #pragma unroll
                        for (int db = 0; db < DP / 16; ++db)
                            o[i][db] *= alpha;
                    }
                    const float mc = m_run[i] == kNegInf ? 0.f : m_run[i] * c;
                    float psum = 0.f;
    #pragma unroll
                    for (int t = 0; t < 2; ++t)
    #pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float p = fast_exp2(fmaf(s[i][t][j], c, -mc));
                            psum += p;
                            pk[i][4 * t + j] = (__bf16)p;
                        }
                    l_run[i] += psum;
                }
                if (kLate)
                    put_v(f);
                lds_wave_fence(); // this tile's V is in LDS before the transposed reads
                const uint16_t *vrow = &vt[(4 * grp + (r16 >> 2)) * VSTR];
                const int quad = F4 && DP == 64 ? (r16 & 3) ^ (r16 >> 1 & 2) : r16 & 3; // put_v's swap
                const uint16_t *const vb[2] = {vrow + 4 * quad, vrow + 4 * (quad ^ 2)};
#pragma unroll
                for (int db = 0; db < DP / 16; ++db) {
                    const uint16_t *y = F4 && DP > 64 ? vb[db >> 2 & 1] + (db ^ db >> 3) * 16 : vb[0] + db * 16;
                    const bf16x8 x = join_tr(lds_read_tr(y), lds_read_tr(y + 16 * VSTR));
    #pragma unroll
                    for (int i = 0; i < NRB; ++i)
                        o[i][db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, pk[i], o[i][db], 0, 0, 0);
                }
            };
            // Tiles in flight per wave: one and a half ahead of the one at work, or, with 4-bit rows, which are
            // short, two and a half.
            constexpr int AHEAD = F4 ? 2 : 1;
            int tb = k0 + 32 * w;
            if (tb < kstop) {
                frags f[AHEAD];
                kv_block b0[AHEAD], b1[AHEAD];
                int pg0[AHEAD], pg1[AHEAD], pn0, pn1;
    #pragma unroll
                for (int i = 0; i < AHEAD; ++i) {
                    pg0[i] = page_id(a, table, tb + 128 * i, k1);
                    pg1[i] = page_id(a, table, tb + 128 * i + 16, k1);
                }
                pn0 = page_id(a, table, tb + 128 * AHEAD, k1);
                pn1 = page_id(a, table, tb + 128 * AHEAD + 16, k1);
                // Blocks of the tile at t; past the last tile they are empty and their loads read nothing. No branch
                // goes around a load: a wait behind it would have to be for all of them.
                auto blocks = [&](int t, int p0, int p1, kv_block &x, kv_block &y) __attribute__((always_inline)) {
                    x = block_in(a, p0, u, t, k1);
                    y = block_in(a, p1, u, t + 16, k1);
                    if (t >= kstop)
                        x.n = y.n = 0;
                };
    #pragma unroll
                for (int i = 0; i < AHEAD; ++i) {
                    blocks(tb + 128 * i, pg0[i], pg1[i], b0[i], b1[i]);
                    if (!kLate) {
                        load_v(b0[i], b1[i], f[i]);
                        load_k(b0[i], b1[i], f[i]);
                    }
                }
                for (; tb < kstop; tb += 128 * AHEAD)
    #pragma unroll
                    for (int i = 0; i < AHEAD; ++i) {
                        const int t = tb + 128 * i, tn = t + 128 * AHEAD;
                        if (i > 0 && t >= kstop)
                            break;
                        kv_block n0, n1;
                        blocks(tn, pn0, pn1, n0, n1);
                        pn0 = page_id(a, table, tn + 128, k1);
                        pn1 = page_id(a, table, tn + 144, k1);
                        if (kLate) {
                            load_k(b0[i], b1[i], f[i]);
                        } else {
                            put_v(f[i]);
                            __builtin_amdgcn_sched_barrier(0);
                            load_v(n0, n1, f[i]);
                        }
                        compute(t, b0[i], b1[i], n0, n1, f[i]);
                        b0[i] = n0;
                        b1[i] = n1;
                    }
            }
    #pragma unroll
            for (int i = 0; i < NRB; ++i)
                l_run[i] = sum_xor32(sum_xor16(l_run[i]));

            // Merge the waves: O^T register (db, j) of this lane holds d = 16db + 4grp + j of row r16.
            float *om = reinterpret_cast<float *>(Vw); // [4][16][DP + 4]
            if (grp == 0)
    #pragma unroll
                for (int i = 0; i < NRB; ++i) {
                    red_m[i][w][r16] = m_run[i] * c; // in log2 units; -inf stays
                    red_l[i][w][r16] = l_run[i];
                }
    #pragma unroll
            for (int i = 0; i < NRB; ++i) {
                __syncthreads();
    #pragma unroll
                for (int db = 0; db < DP / 16; ++db)
                    *reinterpret_cast<f32x4 *>(&om[(w * 16 + r16) * (DP + 4) + db * 16 + 4 * grp]) = o[i][db];
                __syncthreads();
                const int rowb = row0 + 16 * i, nrow = min(16, R - rowb);
                for (int idx = tid; idx < nrow * (DP / 4); idx += 256) {
                    const int r = idx / (DP / 4), d = 4 * (idx % (DP / 4));
                    if (d >= D)
                        continue;
                    float mx = kNegInf;
    #pragma unroll
                    for (int ww = 0; ww < 4; ++ww)
                        mx = fmaxf(mx, red_m[i][ww][r]);
                    const float muse = mx == kNegInf ? 0.f : mx;
                    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
                    float lsum = 0.f;
    #pragma unroll
                    for (int ww = 0; ww < 4; ++ww) {
                        const float wgt = fast_exp2(red_m[i][ww][r] - muse);
                        const f32x4 x = *reinterpret_cast<const f32x4 *>(&om[(ww * 16 + r) * (DP + 4) + d]);
    #pragma unroll
                        for (int j = 0; j < 4; ++j)
                            acc[j] += wgt * x[j];
                        lsum += wgt * red_l[i][ww][r];
                    }
                    const int64_t tok = sq.q0 + (rowb + r) / g;
                    const int h = u * g + (rowb + r) % g;
                    const int64_t slot = (tok * a.Hq + h) * a.nsplit;
                    if (live == 1) {
                        const float inv = lsum > 0.f ? 1.0f / lsum : 0.f;
                        *reinterpret_cast<u32x2 *>(a.o + tok * a.o_tok + h * a.o_head + d) =
                            u32x2{bf16_pair(acc[0] * inv, acc[1] * inv), bf16_pair(acc[2] * inv, acc[3] * inv)};
                        if (d == 0 && a.nsplit > 1)
                            a.pm[slot] = -kNegInf; // the row is written
                    } else {
                        if (d == 0) {
                            a.pm[slot + sp] = part_max(mx, lsum);
                            a.pl[slot + sp] = lsum;
                        }
                        *reinterpret_cast<f32x4 *>(a.pacc + (slot + sp) * D + d) = acc;
                        if (sp == live - 1) // no parts behind the last
                            for (int s = live + d / 4; s < a.nsplit; s += D / 4)
                                a.pm[slot + s] = kNegInf;
                    }
                }
            }
            __syncthreads(); // the merge area is V tiles again
        }
        left -= take;
        pos0 += take;
        off = 0;
        if (++b == a.B) {
            b = 0;
            ++u;
        }
    }
}

// Joins the parts of each row: w_s = 2^(m_s - max m), O = sum w_s acc_s / sum w_s l_s. A workgroup takes
// 256 / (LP SG) rows of one sequence and kv head at a time: LP lanes of four columns each, SG groups of
// parts, NL loads of each thread on their way before the weights are known. The attention kernel says what
// a row has: +inf as the first m where it wrote the row itself, -inf behind the last part (whose acc is
// whatever it was: it gets no weight and is not multiplied). What bounds it is latency: the maxima, sums
// and columns of a row are all asked for at once, right behind the sequence's start. 2.8-4.7 us where nothing
// or little was cut, 4.3-5.1 for 16 rows of 65 parts at D = 256, 6.4-6.8 for 16384 rows of two parts.
constexpr int kPagedMaxSplit = ATTN_PAGED_MAX_PARTS;
template <int NL>
__global__ __launch_bounds__(256) void attn_paged_merge_kernel(const attn_paged_args a, int lglp, int lgsg,
                                                               int tpm) {
    __shared__ float wsh[ATTN_PAGED_MERGE_WEIGHTS]; // [rows][parts]
    __shared__ int nsh[32];                         // parts of each row; -1: written already
    __shared__ __attribute__((aligned(16))) f32x4 red[256];
    const int bu = uniform(wg_id_x() / tpm), t0 = wg_id_x() - bu * tpm;
    const int b = uniform(bu / a.Hkv), u = bu - b * a.Hkv;
    const int tid = wi_id_x(), lane = tid & 63;
    const attn_seq sq = seq_at(a, b);
    const int g = a.Hq / a.Hkv, rpw = 256 >> (lglp + lgsg), R = sq.n * g;
    auto slot_of = [&](int r) { // the first partial of row r
        return ((int64_t)(sq.q0 + r / g) * a.Hq + u * g + r % g) * a.nsplit;
    };
    const int rl = tid >> (lglp + lgsg), sg = (tid >> lglp) & ((1 << lgsg) - 1);
    const int d = 4 * (tid & ((1 << lglp) - 1));
    for (int r0 = t0 * rpw; r0 < R; r0 += tpm * rpw) {
        const int row = r0 + rl;
        const float *p = a.pacc + slot_of(min(row, R - 1)) * a.D + min(d, a.D - 4);
        f32x4 x[NL];
        auto load = [&](int s0) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < NL; ++i)
                x[i] = *reinterpret_cast<const f32x4 *>(
                    p + (int64_t)min(s0 + sg + (i << lgsg), a.nsplit - 1) * a.D);
        };
        load(0);
        // Weights: 16 lanes per row up to 16 parts, else a wave per row, which has NI parts per lane.
        auto weights = [&](auto N, bool all) __attribute__((always_inline)) {
            constexpr int NI = decltype(N)::value;
            const int lgs = all ? 6 : 4, sl = lane & ((1 << lgs) - 1);
            for (int r = tid >> lgs; r < rpw; r += 256 >> lgs) {
                const int64_t slot = slot_of(min(r0 + r, R - 1));
                float m[NI], l[NI], mx = kNegInf;
                int last = 0;
#pragma unroll
                for (int i = 0; i < NI; ++i) {
                    const int s = min(sl + 64 * i, a.nsplit - 1);
                    m[i] = a.pm[slot + s];
                    l[i] = a.pl[slot + s];
                }
                const float first = __builtin_bit_cast(
                    float, __builtin_amdgcn_ds_bpermute((lane & ~((1 << lgs) - 1)) * 4,
                                                        __builtin_bit_cast(int, m[0])));
#pragma unroll
                for (int i = 0; i < NI; ++i) {
                    if (sl + 64 * i >= a.nsplit)
                        m[i] = kNegInf;
                    if (m[i] > kNegInf)
                        last = sl + 64 * i + 1;
                    mx = fmaxf(mx, m[i]);
                }
                mx = seg_all<true>(mx, all);
                const float fl = seg_all<true>((float)last, all);
                const float muse = mx == kNegInf ? 0.f : mx;
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < NI; ++i) {
                    const bool none = m[i] == kNegInf;
                    m[i] = none ? 0.f : fast_exp2(m[i] - muse);
                    sum += none ? 0.f : m[i] * l[i];
                }
                sum = seg_all<false>(sum, all);
                const float inv = sum > 0.f ? 1.0f / sum : 0.f;
#pragma unroll
                for (int i = 0; i < NI; ++i)
                    if (sl + 64 * i < a.nsplit)
                        wsh[r * a.nsplit + sl + 64 * i] = m[i] * inv;
                if (sl == 0)
                    nsh[r] = first == -kNegInf ? -1 : (int)fl;
            }
        };
        if (a.nsplit <= 16)
            weights(std::integral_constant<int, 1>{}, false);
        else if (a.nsplit <= 64)
            weights(std::integral_constant<int, 1>{}, true);
        else
            weights(std::integral_constant<int, kPagedMaxSplit / 64>{}, true);
        __syncthreads();
        const int parts = nsh[rl];
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
        for (int s0 = 0;;) {
#pragma unroll
            for (int i = 0; i < NL; ++i) {
                const int s = s0 + sg + (i << lgsg);
                const float wgt = s < parts ? wsh[rl * a.nsplit + s] : 0.f;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    acc[j] += s < parts ? wgt * x[i][j] : 0.f;
            }
            s0 += NL << lgsg;
            if (s0 >= parts)
                break;
            load(s0);
        }
        if (lgsg > 0) {
            red[tid] = acc;
            __syncthreads();
        }
        if (sg == 0 && row < R && d < a.D && parts >= 0) {
            for (int k = 1; k < 1 << lgsg; ++k) {
                const f32x4 y = red[tid + (k << lglp)];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    acc[j] += y[j];
            }
            *reinterpret_cast<u32x2 *>(a.o + (int64_t)(sq.q0 + row / g) * a.o_tok +
                                       (u * g + row % g) * a.o_head + d) =
                u32x2{bf16_pair(acc[0], acc[1]), bf16_pair(acc[2], acc[3])};
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------------------------------------
// Many query rows per kv head. One workgroup of four waves per (sequence, kv head, part, tile of 128 rows, or
// 64 with KH = 2), tiles of KT keys staged in LDS, two of them: the next one's loads run beside this one's
//   S^T[key][row] = K . Q^T, O^T[d][row] += V^T . P^T   (v_mfma_f32_32x32x16_bf16)
// with the LDS layouts of attn_prefill_fast_kernel. KH = 1: a wave takes 32 rows and all keys of a tile;
// KH = 2: waves w and w + 2 take the same 32 rows and a half of each tile, joined through LDS at the end.
//   * bf16: LDS-DMA, a wave KT / 4 keys of each tile, block by block of 16 (or 8) with a descriptor each.
//   * 4 bits: a lane loads 32 codes of a row and their scale at the start of the tile before, and puts them into
//     LDS as bf16 at its end (two tiles ahead is no faster, and at DP = 256 its registers spill: 2 x 2048 causal,
//     32 heads 220 us, 166 with one).
// The running maximum is raised only where a lane's sum of p over a tile passes kPagedSum, so that O is rarely
// rescaled and most tiles look for no maximum.
//
// No unit is full; two waves per SIMD (three in 4 bits at D = 64) do not cover each other's waits. At D = 128 the matrix
// unit is at work in half of the SIMDs' cycles and the VALU issues in 39% (5.2 VALU and MFMA instructions per MFMA, 6.5
// with the unpacking), at D = 64 in 39 and 56%; a wave waits 28 to 33% of its time for data, barriers and LDS,
// and as long for its turn to issue. 32 heads on 8 kv heads, 2 x 4096 without a mask: D = 128 535 us (1028 TFLOP/s) in
// bf16 and 536 in 4 bits, 656 with a cap of 30, 621 with the distance; D = 64 316 and 301. 2 x 2048 causal: D = 32, 64,
// 80, 96, 128, 192 and 256 51, 57, 76, 78, 85, 138 and 151 (head dims between 64, 128 and 256 run at the next one's
// cost), 164 in 4 bits at 256. 512 tokens over 8192 keys 75 and the merge. LDS-DMA instead of registers in bf16: 614
// -> 526 at D = 128.
// ------------------------------------------------------------------------------------------
// Bound on a lane's sum of p over a tile against a maximum that may lie below the tile's: p costs no precision
// up to it, only exponent range.
constexpr float kPagedSum = 65536.0f;

constexpr int paged_tile_keys(int DP, bool F4) { return DP == 64 ? (F4 ? 64 : 128) : DP == 128 ? 64 : 32; }

template <int DP, bool F4, bool MOD, int KH, int NW>
__global__ __launch_bounds__(64 * NW, 8 / NW) void attn_paged_prefill_kernel(const attn_paged_args a) {
    constexpr int KT = paged_tile_keys(DP, F4) * NW / 4, KN = DP / 16, RWV = KT / NW; // rows a wave stages
    constexpr int PW = KT * DP / 512 / NW;                // 1 KB blocks of a bf16 tile per wave
    constexpr int NBK = RWV <= 16 ? 1 : RWV / 16;         // blocks of 16 keys per wave
    constexpr int AUX = KH == 2 && NW == 4 ? kDmaNT : 0;  // a sequence's only row tile: its keys are read once
    constexpr int NR = NW / KH, BQ = 32 * NR, KW = KT / KH, NT = KW / 32; // rows, keys of a wave
    constexpr int LB = RWV * DP / 2 / 64; // 4 bits: bytes of codes per lane (16, or 8 at DP = 64)
    static_assert(NT >= 1 && PW % NBK == 0 && (!F4 || (NBK == 1 && LB * 2 % 16 == 0)), "tile shape");
    // Each buffer is a variable of its own: the compiler tells LDS accesses apart by variable.
    __shared__ __attribute__((aligned(1024))) uint16_t Ks0[KT * DP], Ks1[KT * DP];
    __shared__ __attribute__((aligned(1024))) uint16_t Vs0[KT * DP], Vs1[KT * DP];
    __shared__ float kh_ml[KH > 1 ? 2 * NR * 64 : 1];

    const attn_place at = attn_place_of(wg_id_x(), a.B * a.Hkv * a.nsplit, a.tps, a.deal);
    if (at.group < 0)
        return;
    const int t0 = uniform(a.tps - 1 - at.tile); // heaviest first
    const int sp = uniform(at.group / (a.B * a.Hkv)), bu = at.group - sp * (a.B * a.Hkv);
    const int u = uniform(bu % a.Hkv), b = uniform(bu / a.Hkv);
    const int tid = wi_id_x(), w = uniform(tid >> 6), lane = tid & 63;
    const attn_seq sq = seq_at(a, b);
    // The divisions run on the vector unit: back into scalar registers, with all that follows from them.
    const attn_parts parts = attn_parts_of(sq.kend, a.share, a.nsplit);
    const int live = uniform(parts.live), kps = uniform(parts.kps);
    if (sp >= live)
        return;
    const int k0 = attn_part_start(sq.kend, kps, sp), k1 = attn_part_start(sq.kend, kps, sp + 1);
    const int32_t *table = a.table + (int64_t)b * a.cols;
    const int l32 = lane & 31, hi = lane >> 5, g16 = lane >> 4, i16 = lane & 15;
    const int wr = KH > 1 ? w % NR : w, kh = KH > 1 ? w / NR : 0;
    const int g = a.Hq / a.Hkv, R = sq.n * g, D = a.D;
    const float c = MOD ? 1.f : a.c;

    // Offsets of this lane's operand reads (elements): K row kperm, chunk 2kk + hi; V rows 8hi + i16 / 4
    // (+ 4), columns 16 (g16 & 1) + 4 (i16 & 3); and the wave's keys of the tile.
    const int kperm = (l32 & ~12) | ((l32 & 4) << 1) | ((l32 & 8) >> 1);
    const int kfo = (kperm >> 3) * 8 * DP + (kperm & 7) * 16 +
                    (((hi ^ kperm >> 3 ^ (F4 ? kperm >> 2 : 0)) & 1) * 8) + kh * KW * DP;
    const int vfo = hi * 8 * DP + (i16 >> 2) * 32 + (2 * (g16 & 1) + ((i16 & 3) >> 1)) * 8 + (i16 & 1) * 4 +
                    kh * KW * DP;

    // bf16: byte (w PW + p) 1024 + 16 lane of the tile's layout is row kr of the wave's rows.
    uint32_t kso[PW], vso[PW];
    if constexpr (!F4)
#pragma unroll
        for (int p = 0; p < PW; ++p) {
            const int x = (w * PW + p) * 1024 + 16 * lane;
            const int kg = x / (16 * DP), kw = x % (16 * DP);
            const int kr = kg * 8 + (kw % 256) / 32 - RWV * w;
            const int kc = 2 * (kw / 256) + (((kw % 32) / 16) ^ (kg & 1));
            kso[p] = kc * 8 < D ? (uint32_t)((kr & 15) * D * 2 + kc * 16) : 0x80000000u;
            const int vg = x / (8 * DP), vw = x % (8 * DP);
            const int vr = vg * 4 + (vw % 256) / 64 - RWV * w;
            const int vc = 4 * (vw / 256) + (vw % 64) / 16;
            vso[p] = vc * 8 < D ? (uint32_t)((vr & 15) * D * 2 + vc * 16) : 0x80000000u;
        }
    // Row and group of 32 (DP = 64: 16) codes that this lane loads of a 4-bit tile.
    const int srow = lane % RWV, sgrp = lane / RWV;
    struct stage {
        uint32_t k[F4 ? LB / 4 : 1], v[F4 ? LB / 4 : 1], ks, vs;
    };
    constexpr int RB = DP / 2, SB = DP / 32; // bytes of a row's codes and scales
    // The wave's rows of the tile from key kb: into LDS, or (4 bits) into registers.
    int pid[NBK]; // the pages of the wave's blocks of the next tile to load
    auto pages_of = [&](int kb) __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < NBK; ++h)
            pid[h] = page_id(a, table, kb + RWV * w + 16 * h, k1);
    };
    auto load = [&](int kb, [[maybe_unused]] int kstop, [[maybe_unused]] uint16_t *Kd,
                    [[maybe_unused]] uint16_t *Vd, [[maybe_unused]] stage &f) __attribute__((always_inline)) {
        if constexpr (!F4) {
            const uint32_t rb = (uint32_t)D * 2u;
#pragma unroll
            for (int h = 0; h < NBK; ++h) {
                const kv_block m = block_in<(RWV < 16 ? RWV : 16)>(a, pid[h], u, kb + RWV * w + 16 * h, k1);
                const auto kr = make_rsrc(a.k + m.row * rb, m.n * rb);
                const auto vr = make_rsrc(a.v + m.row * rb, m.n * rb);
#pragma unroll
                for (int p = h * PW / NBK; p < (h + 1) * PW / NBK; ++p)
                    dma16<0, AUX>(kr, Kd + (w * PW + p) * 512, kso[p]);
#pragma unroll
                for (int p = h * PW / NBK; p < (h + 1) * PW / NBK; ++p)
                    dma16<0, AUX>(vr, Vd + (w * PW + p) * 512, vso[p]);
            }
        } else {
            kv_block m = block_in<(RWV < 16 ? RWV : 16)>(a, pid[0], u, kb + RWV * w, k1);
            if (kb >= kstop) // nothing is read; no branch goes around the loads, whose waits would then be for all
                m.n = 0;
            const auto kr = make_rsrc(a.k + m.row * RB, m.n * RB), vr = make_rsrc(a.v + m.row * RB, m.n * RB);
            const auto ksr = make_rsrc(a.ks + m.row * SB, m.n * SB);
            const auto vsr = make_rsrc(a.vs + m.row * SB, m.n * SB);
            const uint32_t off = srow * RB + sgrp * LB, soff = srow * SB + sgrp * LB / 16;
            if constexpr (LB == 8) {
                const u32x2 x = __builtin_amdgcn_raw_buffer_load_b64(kr, off, 0, 0);
                const u32x2 y = __builtin_amdgcn_raw_buffer_load_b64(vr, off, 0, 0);
                f.k[0] = x[0], f.k[1] = x[1], f.v[0] = y[0], f.v[1] = y[1];
            } else {
                const u32x4 x = buf16<false>(kr, off), y = buf16<false>(vr, off);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    f.k[i] = x[i], f.v[i] = y[i];
            }
            f.ks = __builtin_amdgcn_raw_buffer_load_b8(ksr, soff, 0, 0);
            f.vs = __builtin_amdgcn_raw_buffer_load_b8(vsr, soff, 0, 0);
        }
    };
    // 4 bits: the lane's chunks of eight elements into the tile's layouts, eight lanes (rows) at a time over 128
    // bytes of banks. K: rows four apart swap the chunks of a pair. V: rows two apart start at another of
    // their chunks; four apart at DP = 64, where they have only two of them, and at DP = 256, where the second
    // exchange spills (2 x 2048 causal, 32 heads: 172 us with it, 166 without).
    auto put = [&](const stage &f, uint16_t *Kd, uint16_t *Vd) __attribute__((always_inline)) {
        constexpr int NC = LB / 4;
        const int r = RWV * w + srow, c0 = sgrp * NC;
        const float ksc = e8m0(f.ks), vsc = e8m0(f.vs);
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            const int cc = c0 + j;
            *reinterpret_cast<u32x4 *>(&Kd[(r >> 3) * 8 * DP + (cc >> 1) * 128 + (r & 7) * 16 +
                                           ((cc ^ r >> 3 ^ r >> 2) & 1) * 8]) = fp4_to_bf16(f.k[j], ksc);
        }
        const int rot = (DP == 128 ? srow >> 1 : srow >> 2) & (NC - 1);
        uint32_t x[NC], y[NC];
#pragma unroll
        for (int j = 0; j < NC; ++j)
            x[j] = pick(rot & 1, f.v[(j + 1) % NC], f.v[j]);
#pragma unroll
        for (int j = 0; j < NC; ++j)
            y[j] = pick(rot & 2, x[(j + 2) % NC], x[j]);
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            const int cc = c0 + ((j + rot) & (NC - 1));
            *reinterpret_cast<u32x4 *>(&Vd[(r >> 2) * 4 * DP + (cc >> 2) * 128 + (r & 3) * 32 + (cc & 3) * 8]) =
                fp4_to_bf16(y[j], vsc);
        }
    };
    // Whether any page of the part is none: looked for once, so that tiles need no look of their own.
    bool lost = false;
    if (k1 > k0)
        for (int x = (k0 >> a.lgp) + lane; x <= (k1 - 1) >> a.lgp; x += 64)
            lost |= !attn_page_ok(table[x], a.pages);
    const bool holes = __builtin_amdgcn_ballot_w64(lost) != 0;

    for (int tile = t0; (int64_t)tile * BQ < R; tile += a.tps) {
        const int row0 = tile * BQ, row = row0 + 32 * wr + l32;
        const bool valid = row < R;
        const int tok = valid ? row / g : 0, h = u * g + (valid ? row % g : 0);
        const uint16_t *q = a.q + (sq.q0 + tok) * a.q_tok + h * a.q_head;
        bf16x8 qb[KN];
#pragma unroll
        for (int kk = 0; kk < KN; ++kk) {
            const int col = kk * 16 + hi * 8;
            u32x4 x = zero4();
            if (valid && col < D)
                x = *reinterpret_cast<const u32x4 *>(q + col);
            qb[kk] = as_bf16x8(x);
        }
        const int p0 = sq.len - sq.n; // position of the sequence's first row
        const int pos = p0 + tok, lim = a.causal ? min(pos, k1 - 1) : k1 - 1;
        const float slope = MOD && a.slopes ? a.slopes[h] * 1.44269504088896341f : 0.f;
        // The wave's smallest and largest limits, and where the workgroup's tiles end.
        const int wfirst = row0 + 32 * wr, wlast = min(wfirst + 31, R - 1);
        const int wmin = uniform(a.causal ? min(p0 + min(wfirst, R - 1) / g, k1 - 1) : k1 - 1);
        const int wmax = uniform(wfirst >= R ? -1 : a.causal ? min(p0 + wlast / g, k1 - 1) : k1 - 1);
        const int kstop = uniform(a.causal ? min(k1, p0 + min(row0 + BQ - 1, R - 1) / g + 1) : k1);

        float m_run = kNegInf, l_run = 0.f;
        f32x16 o[DP / 32];
#pragma unroll
        for (int db = 0; db < DP / 32; ++db)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                o[db][i] = 0.f;

        // One tile from key kb, in the buffers Kb and Vb.
        auto compute = [&](int kb, const uint16_t *Kb, const uint16_t *Vb)
            __attribute__((always_inline)) {
            const int kw = kb + kh * KW; // the wave's first key
            if (kw > wmax)
                return;
            f32x16 s[NT];
            bf16x8 ka[2][KN];
            const uint16_t *kp = Kb + kfo;
#pragma unroll
            for (int kk = 0; kk < KN; ++kk)
                ka[0][kk] = as_bf16x8(*reinterpret_cast<const u32x4 *>(kp + kk * 128));
            __builtin_amdgcn_sched_group_barrier(0x100, KN, 0);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    s[t][i] = 0.f;
#pragma unroll
                for (int kk = 0; kk < KN; ++kk) {
                    s[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ka[t & 1][kk], qb[kk], s[t], 0, 0, 0);
                    if (t + 1 < NT)
                        ka[(t + 1) & 1][kk] = as_bf16x8(
                            *reinterpret_cast<const u32x4 *>(kp + (t + 1) * 32 * DP + kk * 128));
                }
#pragma unroll
                for (int kk = 0; kk < KN; ++kk) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    if (t + 1 < NT)
                        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                }
            }
            // Register i of sub-tile t: key kw + 32t + 16 (i / 8) + 8hi + i % 8.
            if (MOD)
                modify_scores(a, slope, pos - kw - 8 * hi, [&](auto f) __attribute__((always_inline)) {
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            s[t][i] = f(s[t][i], 32 * t + 16 * (i >> 3) + (i & 7));
                });
            if (holes || kw + KW - 1 > wmin) {
                // A block without a page hides its keys.
                uint32_t none = 0;
#pragma unroll
                for (int j = 0; holes && j < KW / 16; ++j)
                    none |= attn_page_ok(page_id(a, table, kw + 16 * j, k1), a.pages) ? 0u : 1u << j;
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (kw + 32 * t + 16 * (i >> 3) + 8 * hi + (i & 7) > lim ||
                            (none >> (2 * t + (i >> 3)) & 1))
                            s[t][i] = kNegInf;
            }
            bf16x8 pk[2 * NT];
            // p against the running maximum m as it is; a lane whose sum of them passes kPagedSum (or whose row
            // has no m yet) sends its wave to raise m to the tile's maximum and take p again.
            float psum;
            auto weigh = [&]() __attribute__((always_inline)) {
                const float mc = m_run == kNegInf ? 0.f : m_run * c;
                psum = 0.f;
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float p = fast_exp2(fmaf(s[t][i], c, -mc));
                        psum += p;
                        pk[2 * t + (i >> 3)][i & 7] = (__bf16)p;
                    }
            };
            weigh();
            if (__builtin_amdgcn_ballot_w64(!(psum <= kPagedSum) || m_run == kNegInf) != 0) {
                float mx = kNegInf;
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int i = 0; i < 16; i += 2)
                        mx = max3f(mx, s[t][i], s[t][i + 1]);
                const float mnew = fmaxf(m_run, max_xor32(mx));
                const float alpha = rescale(m_run, mnew, c);
                m_run = mnew;
                l_run *= alpha;
#pragma unroll
                for (int db = 0; db < DP / 32; ++db)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        o[db][i] *= alpha;
                weigh();
            }
            l_run += psum;
            const uint16_t *vp = Vb + vfo;
#pragma unroll
            for (int cc = 0; cc < 2 * NT; ++cc)
#pragma unroll
                for (int db = 0; db < DP / 32; ++db) {
                    const uint16_t *x = vp + cc * 16 * DP + db * 128;
                    o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                        join_tr(lds_read_tr(x), lds_read_tr(x + 4 * DP)), pk[cc], o[db], 0, 0, 0);
                }
        };
        auto wait_loads = [] { __builtin_amdgcn_s_waitcnt(waitcnt_vm(0)); };

        stage st;
        if (k0 < kstop) {
            pages_of(k0);
            load(k0, kstop, Ks0, Vs0, st);
            pages_of(k0 + KT);
            if constexpr (F4)
                put(st, Ks0, Vs0);
        }
        // Q has arrived as well: waited for at its first use, inside the loop, it would be waited for there on
        // every tile, together with the loads of the next ones.
        wait_loads();
        __syncthreads();
        // A tile in buffer Kb, Vb; the next one's rows are on their way meanwhile.
        auto step = [&](int kb, const uint16_t *Kb, const uint16_t *Vb, uint16_t *Kn, uint16_t *Vn)
            __attribute__((always_inline)) {
            if (F4 || kb + KT < kstop) // 4 bits: without a branch, see load
                load(kb + KT, kstop, Kn, Vn, st);
            pages_of(kb + 2 * KT);
            compute(kb, Kb, Vb);
            if constexpr (F4) {
                put(st, Kn, Vn);
            } else {
                wait_loads(); // this wave's part of the next tile has arrived
            }
            __syncthreads();
        };
        for (int kb = k0; kb < kstop; kb += 2 * KT) {
            step(kb, Ks0, Vs0, Ks1, Vs1);
            if (kb + KT < kstop)
                step(kb + KT, Ks1, Vs1, Ks0, Vs0);
        }
        l_run = sum_xor32(l_run);

        bool writes = valid;
        float m_log = m_run * c; // in log2 units; -inf stays
        if constexpr (KH > 1) {
            // Join the halves of the tiles: the second half's waves leave (m, l) and O in LDS.
            static_assert(KT * 4 >= 64 * NW, "O of the second half's waves fits two buffers");
            float *kho = reinterpret_cast<float *>(wr & 1 ? Vs0 : Ks0) + (wr >> 1) * DP * 32 + lane;
            if (kh == 1) {
                kh_ml[wr * 64 + lane] = m_log;
                kh_ml[NR * 64 + wr * 64 + lane] = l_run;
#pragma unroll
                for (int db = 0; db < DP / 32; ++db)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        kho[(db * 16 + i) * 64] = o[db][i];
            }
            __syncthreads();
            if (kh == 0) {
                const float m1 = kh_ml[wr * 64 + lane], l1 = kh_ml[NR * 64 + wr * 64 + lane];
                const float mm = fmaxf(m_log, m1);
                const float w0 = rescale(m_log, mm, 1.f), w1 = rescale(m1, mm, 1.f);
                l_run = w0 * l_run + w1 * l1;
                m_log = mm;
#pragma unroll
                for (int db = 0; db < DP / 32; ++db)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        o[db][i] = w0 * o[db][i] + w1 * kho[(db * 16 + i) * 64];
            }
            __syncthreads();
            writes = valid && kh == 0;
        }
        if (writes) {
            const int64_t orow = sq.q0 + tok;
            const int64_t slot = (orow * a.Hq + h) * a.nsplit;
            if (live == 1) {
                const float inv = l_run > 0.f ? 1.0f / l_run : 0.f;
                if (hi == 0 && a.nsplit > 1)
                    a.pm[slot] = -kNegInf; // the row is written
                uint16_t *dst = a.o + orow * a.o_tok + h * a.o_head;
#pragma unroll
                for (int db = 0; db < DP / 32; ++db)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int d = db * 32 + 8 * j + 4 * hi;
                        if (d < D)
                            *reinterpret_cast<u32x2 *>(dst + d) =
                                u32x2{bf16_pair(o[db][4 * j] * inv, o[db][4 * j + 1] * inv),
                                      bf16_pair(o[db][4 * j + 2] * inv, o[db][4 * j + 3] * inv)};
                    }
            } else {
                if (hi == 0) {
                    a.pm[slot + sp] = part_max(m_log, l_run);
                    a.pl[slot + sp] = l_run;
                    if (sp == live - 1) // no parts behind the last
                        for (int s = live; s < a.nsplit; ++s)
                            a.pm[slot + s] = kNegInf;
                }
                float *dst = a.pacc + (slot + sp) * D;
#pragma unroll
                for (int db = 0; db < DP / 32; ++db)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int d = db * 32 + 8 * j + 4 * hi;
                        if (d < D)
                            *reinterpret_cast<f32x4 *>(dst + d) =
                                f32x4{o[db][4 * j], o[db][4 * j + 1], o[db][4 * j + 2], o[db][4 * j + 3]};
                    }
            }
        }
    }
}

// ------------------------------------------------------------------------------------------
// Append. A workgroup takes one token at a time, its four waves two halves of q's heads, k and v. A lane holds
// the two eights of a head that rotate with each other ((x1, x2) -> (x1 c - x2 s, x2 c + x1 s), in fp32,
// products and sums rounded apart, the result once to bf16), the wave's lanes lie across several heads, and
// two of a lane's heads are in flight, so that the cosines and sines are read once per wave. K and V of the
// 4-bit cache go eight elements to a lane, four lanes to a group. HBM-bound: each element is read and
// written once, past the L2, whose copies the attention on other XCDs could not use. 12700 tokens of 32 + 2 x 8
// heads, D = 128, bf16: 56 us, 5.6 TB/s read and written, the rate of a copy (a wave per token 62.7); one token 2.4 us.
// The grid is max_q workgroups per sequence, which end at once where a sequence has fewer tokens: 512 single tokens take
// 4.3 us, with a prompt of 512 tokens among them 134.
// ------------------------------------------------------------------------------------------
__device__ __forceinline__ float lo_bf16(uint32_t x) { return __builtin_bit_cast(float, x << 16); }
__device__ __forceinline__ float hi_bf16(uint32_t x) {
    return __builtin_bit_cast(float, x & 0xffff0000u);
}
__device__ __forceinline__ void to_f32(u32x4 v, float *x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = lo_bf16(v[i]);
        x[2 * i + 1] = hi_bf16(v[i]);
    }
}
__device__ __forceinline__ u32x4 to_bf16(const float *x) {
    return u32x4{bf16_pair(x[0], x[1]), bf16_pair(x[2], x[3]), bf16_pair(x[4], x[5]),
                 bf16_pair(x[6], x[7])};
}

// max over each four consecutive lanes, in every one of them
__device__ __forceinline__ uint32_t quad_max(uint32_t x) {
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, 0xB1, 0xf, 0xf, false)); // 1,0,3,2
    return max(x, (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, 0x4E, 0xf, 0xf, false)); // 2,3,0,1
}

// Scale byte of a group whose largest magnitude has the fp32 bits amax: the smallest power of two 2^(e-127)
// under which that is at most 7, so that no element is further off than half of E2M1's widest step
// (between 4 and 6; 7 is held as 6), but within 2^-126 .. 2^125, so that scale and values are normal
// numbers (8 2^125 is no bf16 value). 255, E8M0's NaN, where the group is not finite.
__device__ __forceinline__ uint32_t e8m0_of(uint32_t amax) {
    if (amax >= 0x7f800000u)
        return 255u;
    const int e = (int)(amax >> 23) - 2 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
    return (uint32_t)min(max(e, 1), 252);
}

template <bool F4, bool PAIRS>
__global__ __launch_bounds__(256) void attn_kv_append_kernel(const attn_kv_args a) {
#pragma clang fp contract(off)
    const int b = uniform(wg_id_x() / a.tblk), tb = wg_id_x() - b * a.tblk;
    const attn_seq sq = attn_seq_of(scalar_i32(a.q_start, b), scalar_i32(a.q_start, b + 1),
                                    scalar_i32(a.kv_len, b), a.T, a.cols, a.lgp);
    const int lane = wi_id_x() & 63, w = uniform(wi_id_x() >> 6), D = a.D, half = a.rot / 2;
    const int32_t *table = a.table + (int64_t)b * a.cols;
    constexpr int U = 2; // heads of a lane in flight

    // This wave's heads: of q (waves 0 and 1), k (2) or v (3).
    const int h0 = w == 1 ? (a.Hq + 1) / 2 : 0;
    const int heads = w > 1 ? a.Hkv : w == 1 ? a.Hq - h0 : (a.Hq + 1) / 2;
    const int64_t tok_s = w < 2 ? a.q_tok : w == 2 ? a.k_tok : a.v_tok;
    const int64_t head_s = w < 2 ? a.q_head : w == 2 ? a.k_head : a.v_head;
    const uint16_t *src = w < 2 ? a.q : w == 2 ? a.k : a.v;
    uint8_t *const cache = w == 2 ? a.ck : a.cv, *const scales = w == 2 ? a.cks : a.cvs;
    if (heads == 0)
        return;

    // Sixteen elements of a head per lane: columns c0 .. + 7 and c1 .. + 7, which turn by the angles from r on;
    // or eight (k and v in 4 bits), columns c0 .. + 7, and the columns c1 .. + 7 that they turn with.
    const bool eight = F4 && w > 1;
    const int n = eight ? D / 8 : D / 16, hp = 64 / n, hl = lane / n, j = lane % n;
    const bool turn = w < 3 && (eight ? 8 : 16) * j < a.rot;
    int c0 = 16 * j, c1 = 16 * j + 8, r = 8 * j;
    bool low = true;
    if (eight) {
        low = PAIRS || 8 * j < half;
        c0 = 8 * j;
        c1 = !turn || PAIRS ? c0 : low ? c0 + half : c0 - half;
        r = PAIRS ? 4 * j : low ? c0 : c0 - half;
    } else if (turn && !PAIRS) {
        c0 = 8 * j;
        c1 = half + 8 * j;
    }

    for (int i = tb; i < sq.n; i += a.tblk) {
        // The rows are asked for before their place is known; a token without one is not stored.
        const int pos = sq.len - sq.n + i;
        const uint16_t *s = src + (sq.q0 + i) * tok_s + h0 * head_s;
        u32x4 x0[U], x1[U];
        auto load = [&](int h) __attribute__((always_inline)) {
#pragma unroll
            for (int e = 0; e < U; ++e) {
                const uint16_t *t = s + min(h + e * hp + hl, heads - 1) * head_s;
                x0[e] = *reinterpret_cast<const u32x4 *>(t + c0);
                x1[e] = *reinterpret_cast<const u32x4 *>(t + c1);
            }
        };
        load(0);
        const bool placed = pos >= 0 && (a.rot == 0 || pos < a.rope_rows);
        const int pg = scalar_i32(table, max(0, min(pos, sq.kend - 1)) >> a.lgp);
        float cs[8], sn[8];
        if (turn) {
            const float *cr = a.rope + (int64_t)(placed ? pos : 0) * a.rot + r;
#pragma unroll
            for (int e = 0; e < 8; e += 4) {
                if (PAIRS && eight && e == 4) // eight elements are four pairs
                    break;
                const f32x4 y0 = *reinterpret_cast<const f32x4 *>(cr + e);
                const f32x4 y1 = *reinterpret_cast<const f32x4 *>(cr + half + e);
#pragma unroll
                for (int f = 0; f < 4; ++f)
                    cs[e + f] = y0[f], sn[e + f] = y1[f];
            }
        }
        if (!placed || (w > 1 && (pos >= sq.kend || !attn_page_ok(pg, a.pages))))
            continue;
        const int64_t row = attn_page_row(pg, a.Hkv, 0, max(pos, 0), a.lgp);
        for (int h = 0;;) {
#pragma unroll
            for (int e = 0; e < U; ++e) {
                if (h + e * hp >= heads)
                    break;
                if (turn) {
                    float p[8], q[8], y0[8], y1[8];
                    to_f32(x0[e], p);
                    to_f32(x1[e], q);
                    if (PAIRS) { // neighbours; of sixteen elements eight pairs
#pragma unroll
                        for (int f = 0; f < 4; ++f) {
                            y0[2 * f] = p[2 * f] * cs[f] - p[2 * f + 1] * sn[f];
                            y0[2 * f + 1] = p[2 * f + 1] * cs[f] + p[2 * f] * sn[f];
                            if (!eight) {
                                y1[2 * f] = q[2 * f] * cs[4 + f] - q[2 * f + 1] * sn[4 + f];
                                y1[2 * f + 1] = q[2 * f + 1] * cs[4 + f] + q[2 * f] * sn[4 + f];
                            }
                        }
                    } else {
#pragma unroll
                        for (int f = 0; f < 8; ++f) {
                            const float m = q[f] * sn[f];
                            y0[f] = low ? p[f] * cs[f] - m : p[f] * cs[f] + m;
                            if (!eight)
                                y1[f] = q[f] * cs[f] + p[f] * sn[f];
                        }
                    }
                    x0[e] = to_bf16(y0);
                    if (!eight)
                        x1[e] = to_bf16(y1);
                }
                const int hh = h + e * hp + hl;
                if (eight) {
                    uint32_t am = 0;
#pragma unroll
                    for (int f = 0; f < 4; ++f)
                        am = max(am, max(x0[e][f] << 16 & 0x7fff0000u, x0[e][f] & 0x7fff0000u));
                    const uint32_t e8 = e8m0_of(quad_max(am));
                    const float sc = e8m0(e8);
                    uint32_t c = 0;
                    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, lo_bf16(x0[e][0]), hi_bf16(x0[e][0]), sc, 0);
                    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, lo_bf16(x0[e][1]), hi_bf16(x0[e][1]), sc, 1);
                    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, lo_bf16(x0[e][2]), hi_bf16(x0[e][2]), sc, 2);
                    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, lo_bf16(x0[e][3]), hi_bf16(x0[e][3]), sc, 3);
                    if (hh < heads) { // D is 64, 128 or 256: every lane has a head
                        const int64_t at = row + ((int64_t)hh << a.lgp);
                        *reinterpret_cast<uint32_t *>(cache + at * (D / 2) + 4 * j) = e8 == 255 ? 0u : c;
                        if (j % 4 == 0)
                            scales[at * (D / 32) + j / 4] = (uint8_t)e8;
                    }
                } else if (hl < hp && hh < heads) {
                    uint16_t *d = w < 2 ? a.q_out + (sq.q0 + i) * a.qo_tok + (h0 + hh) * a.qo_head
                                        : reinterpret_cast<uint16_t *>(cache) + (row + ((int64_t)hh << a.lgp)) * D;
                    __builtin_nontemporal_store(x0[e], reinterpret_cast<u32x4 *>(d + c0));
                    __builtin_nontemporal_store(x1[e], reinterpret_cast<u32x4 *>(d + c1));
                }
            }
            h += U * hp;
            if (h >= heads)
                break;
            load(h);
        }
    }
}

// Read back: a wave per token, eight elements of a head per lane, four heads of a lane in flight. A token
// without a place in the cache gives zeros. HBM-bound by what it writes, which goes past the L2: 32768 tokens
// of 8 heads from 4 bits 38.3 us through it, 28.4 past it; from bf16 48 (5.6 TB/s read and written).
template <bool F4>
__global__ __launch_bounds__(256) void attn_kv_read_kernel(const attn_kv_args a) {
    const int b = uniform(wg_id_x() / a.tblk), tb = wg_id_x() - b * a.tblk;
    const attn_seq sq = attn_seq_of(scalar_i32(a.q_start, b), scalar_i32(a.q_start, b + 1),
                                    scalar_i32(a.kv_len, b), a.T, a.cols, a.lgp);
    const int lane = wi_id_x() & 63, w = uniform(wi_id_x() >> 6), D = a.D;
    const int uh = D / 8, hp = 64 / uh, hl = lane / uh, j = lane % uh;
    const int32_t *table = a.table + (int64_t)b * a.cols;
    constexpr int U = 4;
    for (int i = tb * 4 + w; i < sq.n; i += a.tblk * 4) {
        const int pos = sq.len - sq.n + i;
        const int pg = pos >= 0 && pos < sq.kend ? scalar_i32(table, pos >> a.lgp) : -1;
        const bool ok = attn_page_ok(pg, a.pages);
        const int64_t row = attn_page_row(ok ? pg : 0, a.Hkv, 0, ok ? pos : 0, a.lgp);
        const int64_t tok = sq.q0 + i;
        auto rows = [&](const uint8_t *pages, const uint8_t *scales, uint16_t *dst, int64_t dhead)
            __attribute__((always_inline)) {
            const int64_t phead = (int64_t)(F4 ? D / 2 : 2 * D) << a.lgp;
            const uint8_t *src = pages + row * (F4 ? D / 2 : 2 * D);
            for (int h0 = 0; h0 < a.Hkv; h0 += U * hp) {
                u32x4 x[U];
                uint32_t sc[U];
#pragma unroll
                for (int e = 0; e < U; ++e) {
                    if (h0 + e * hp >= a.Hkv)
                        break;
                    const int h = min(h0 + e * hp + hl, a.Hkv - 1);
                    if constexpr (F4) {
                        x[e][0] = *reinterpret_cast<const uint32_t *>(src + h * phead + 4 * j);
                        sc[e] = scales[row * (D / 32) + h * (phead / 16) + j / 4];
                    } else {
                        x[e] = *reinterpret_cast<const u32x4 *>(src + h * phead + 16 * j);
                    }
                }
#pragma unroll
                for (int e = 0; e < U; ++e) {
                    if (h0 + e * hp >= a.Hkv)
                        break;
                    const int h = h0 + e * hp + hl;
                    u32x4 y = x[e];
                    if constexpr (F4)
                        y = fp4_to_bf16(x[e][0], e8m0(sc[e]));
                    if (hl < hp && h < a.Hkv)
                        __builtin_nontemporal_store(ok ? y : zero4(),
                                                    reinterpret_cast<u32x4 *>(dst + h * dhead + 8 * j));
                }
            }
        };
        rows(a.ck, a.cks, a.k_out + tok * a.k_tok, a.k_head);
        rows(a.cv, a.cvs, a.v_out + tok * a.v_tok, a.v_head);
    }
}

// ---- launchers -------------------------------------------------------------------------------
template <int DP, bool F4>
hipError_t launch_paged_d(const attn_paged_args &a, const attn_paged_cut &cut, hipStream_t st) {
    const dim3 grid((unsigned)cut.grid), block(256);
    const bool mod = a.cap_out != 0.f || a.slopes;
    return with_flag(mod, [&](auto M) {
        constexpr bool kM = decltype(M)::value;
        auto decode = [&](auto NB, auto NT) {
            constexpr int kN = decltype(NB)::value;
            constexpr bool kT = decltype(NT)::value;
            if (t_plan) {
                plan_note(grid, block, "attn_paged_decode_kernel<%d, %d, %d, %s, %s> teams=%d parts=%d", DP,
                          F4 ? 4 : 16, kN, tf(kM), tf(kT), a.teams, a.nsplit);
                return hipSuccess;
            }
            hipLaunchKernelGGL((attn_paged_decode_kernel<DP, F4, kN, kM, kT>), grid, block, 0, st, a);
            return hipGetLastError();
        };
        constexpr std::integral_constant<int, 1> one;
        constexpr std::integral_constant<int, 2> two;
        // Non-temporal where a row tile is the only one of its sequence, which at D <= 128 it always is.
        if constexpr (DP > 128) {
            if (cut.rows16 == 1)
                return with_flag(a.tps == 1, [&](auto NT) { return decode(one, NT); });
        } else {
            if (cut.rows16 == 1)
                return decode(one, std::true_type{});
            if (cut.rows16 == 2)
                return decode(two, std::true_type{});
        }
        auto prefill = [&](auto KHF, auto NWF) {
            constexpr int kK = decltype(KHF)::value, kW = decltype(NWF)::value;
            if (t_plan) {
                plan_note(grid, dim3(64 * kW), "attn_paged_prefill_kernel<%d, %d, %s, %d, %d> parts=%d share=%d",
                          DP, F4 ? 4 : 16, tf(kM), kK, kW, a.nsplit, a.share);
                return hipSuccess;
            }
            hipLaunchKernelGGL((attn_paged_prefill_kernel<DP, F4, kM, kK, kW>), grid, dim3(64 * kW), 0, st, a);
            return hipGetLastError();
        };
        constexpr std::integral_constant<int, 4> four;
        constexpr std::integral_constant<int, 8> eight;
        if constexpr (DP <= 128) {
            if (cut.rows16 == 4)
                return prefill(two, four);
            if (cut.halves)
                return prefill(two, eight);
        }
        return prefill(one, four);
    });
}

} // namespace

// The attention kernel that the cut names and, where it may leave parts, the merge.
extern "C" int attn_hip_launch_paged(const struct attn_paged_args *ap, const struct attn_paged_cut *cut, int bits,
                                     void *stream) {
    const attn_paged_args &a = *ap;
    const hipStream_t st = (hipStream_t)stream;
    if (cut->grid <= 0 || cut->grid > ATTN_PAGED_MAX_GRID || a.nsplit > kPagedMaxSplit ||
        (a.nsplit > 1 && (256 >> (cut->lglp + cut->lgsg)) * a.nsplit > ATTN_PAGED_MERGE_WEIGHTS))
        return (int)hipErrorInvalidValue;
    hipError_t e;
    if (bits == 4)
        e = a.D == 64    ? launch_paged_d<64, true>(a, *cut, st)
            : a.D == 128 ? launch_paged_d<128, true>(a, *cut, st)
                         : launch_paged_d<256, true>(a, *cut, st);
    else
        e = a.D <= 64    ? launch_paged_d<64, false>(a, *cut, st)
            : a.D <= 128 ? launch_paged_d<128, false>(a, *cut, st)
                         : launch_paged_d<256, false>(a, *cut, st);
    if (e != hipSuccess || a.nsplit == 1)
        return (int)e;
    const dim3 mgrid((unsigned)((long)a.B * a.Hkv * cut->merge_tiles));
    auto merge = [&](auto L) {
        constexpr int kL = decltype(L)::value;
        if (t_plan) {
            plan_note(mgrid, dim3(256), "attn_paged_merge_kernel<%d> rows=%d", kL,
                      256 >> (cut->lglp + cut->lgsg));
            return hipSuccess;
        }
        hipLaunchKernelGGL(attn_paged_merge_kernel<kL>, mgrid, dim3(256), 0, st, a, cut->lglp, cut->lgsg,
                           cut->merge_tiles);
        return hipGetLastError();
    };
    return (int)(cut->merge_loads == 2   ? merge(std::integral_constant<int, 2>{})
                 : cut->merge_loads == 4 ? merge(std::integral_constant<int, 4>{})
                                         : merge(std::integral_constant<int, 8>{}));
}

extern "C" int attn_hip_launch_kv_append(const struct attn_kv_args *ap, int bits, int pairs, void *stream) {
    const attn_kv_args &a = *ap;
    const long grid = (long)a.B * a.tblk;
    if (grid <= 0 || grid > ATTN_PAGED_MAX_GRID)
        return (int)hipErrorInvalidValue;
    return (int)with_flag(bits == 4, [&](auto F) {
        return with_flag(pairs != 0, [&](auto P) {
            hipLaunchKernelGGL((attn_kv_append_kernel<decltype(F)::value, decltype(P)::value>),
                               dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream, a);
            return hipGetLastError();
        });
    });
}

extern "C" int attn_hip_launch_kv_read(const struct attn_kv_args *ap, int bits, void *stream) {
    const attn_kv_args &a = *ap;
    const long grid = (long)a.B * a.tblk;
    if (grid <= 0 || grid > ATTN_PAGED_MAX_GRID)
        return (int)hipErrorInvalidValue;
    return (int)with_flag(bits == 4, [&](auto F) {
        hipLaunchKernelGGL((attn_kv_read_kernel<decltype(F)::value>), dim3((unsigned)grid), dim3(256), 0,
                           (hipStream_t)stream, a);
        return hipGetLastError();
    });
}

#endif

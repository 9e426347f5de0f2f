// attn_cross_kernels.h -- gfx950 kernels of cross attention over ragged batches: forward with the log-sum-exp of
// each row (attn_cross) and the gradients (attn_cross_grad). Part of attn_kernels.hip.
//
//   S = scale Q.K, lse = log sum exp S, P = exp(S - lse), O = P.V
//   delta = sum_d dO O, dS = P (dO.V - delta), dQ = scale dS.K, dK = scale dS^T.Q, dV = P^T.dO
//
// in fp32 but for the operands of the MFMAs: Q, K, V and dO as they are, P and dS rounded to bf16 (half a unit of
// 2^-8, as much as the outputs' own rounding), in the gradients of small calls in two parts (FINE, ATTN_CROSS_FINE);
// outputs are rounded once. Nothing is accumulated by atomics: each
// output has one workgroup, or parts that are added in order, so that a call gives the same bits every time.
//
// Tiles lie in LDS in one layout that serves both ways of reading them without bank conflicts: rows in groups of
// four, a group's rows in blocks of 64 bytes, and in a block the four 16-byte chunks in an order that the group picks
// (chunk ^ group mod 4).
//   * As a row operand (16 bytes of a row per lane, 32 rows): sixteen neighbouring rows lie on different banks.
//   * Transposed (ds_read_b64_tr_b16: 8 bytes per lane of four rows): a group's four rows are 256 bytes apart from none.
#ifndef ATTN_CROSS_KERNELS_H
#define ATTN_CROSS_KERNELS_H

#include "attn_cross_rule.h"
#include "attn_device.h"
#include "attn_launch.h"
#include "attn_line.h"

namespace {

__device__ __forceinline__ attn_range rows_of(const int32_t *start, const int32_t *second, int is_len, int b, int T) {
    const attn_range r = attn_range_of(scalar_i32(start, b), scalar_i32(second, b), is_len, T);
    return attn_range{uniform(r.at), uniform(r.n)};
}
__device__ __forceinline__ attn_range q_rows(const attn_cross_args &a, int b) {
    return rows_of(a.q_start, a.q_second, a.q_is_len, b, a.Tq);
}
__device__ __forceinline__ attn_range k_rows(const attn_cross_args &a, int b) {
    return rows_of(a.k_start, a.k_second, a.k_is_len, b, a.Tk);
}

// The sequence at place nth of the call's: as they come, or by falling length of the rows that a tile has to walk (its
// states, or with BY_Q its rows), so that no long one is left for the end: each lane counts how many are ahead of its own.
struct cross_seq {
    attn_range q, k;
};
template <bool BY_Q> __device__ __forceinline__ cross_seq seq_at(const attn_cross_args &a, int nth, int lane) {
    if (!a.by_length) {
        int q0 = scalar_i32(a.q_start, nth), q1 = scalar_i32(a.q_second, nth);
        int k0 = scalar_i32(a.k_start, nth), k1 = scalar_i32(a.k_second, nth);
        asm("" : "+s"(q0), "+s"(q1), "+s"(k0), "+s"(k1)); // asked for together
        return cross_seq{attn_range_of(q0, q1, a.q_is_len, a.Tq), attn_range_of(k0, k1, a.k_is_len, a.Tk)};
    }
    const int i = min(lane, a.B - 1);
    const attn_range q = attn_range_of(a.q_start[i], a.q_second[i], a.q_is_len, a.Tq);
    const attn_range k = attn_range_of(a.k_start[i], a.k_second[i], a.k_is_len, a.Tk);
    const int len = lane >= a.B ? -1 : BY_Q ? q.n : k.n; // the lanes past the last: behind all sequences
    int ahead = 0;
    for (int j = 0; j < a.B; ++j) {
        const int x = __builtin_amdgcn_readlane(len, j);
        ahead += x > len || (x == len && j < lane) ? 1 : 0;
    }
    const int b = __builtin_ctzll(__builtin_amdgcn_ballot_w64(ahead == nth));
    auto of = [&](attn_range r) {
        return attn_range{__builtin_amdgcn_readlane(r.at, b), __builtin_amdgcn_readlane(r.n, b)};
    };
    return cross_seq{of(q), of(k)};
}

__device__ __forceinline__ attn_cut part_of(int total, int share, int nsplit, int step) {
    if (nsplit == 1) // no divisions
        return attn_cut{1, max(total, 1)};
    const attn_cut c = attn_cut_of(total, share, nsplit, step);
    return attn_cut{uniform(c.live), uniform(c.per)};
}

constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.693147180559945309f;

// The log-sum-exp of a row from its maximum in units of log2 and its sum: -inf where there is nothing.
__device__ __forceinline__ float lse_of(float m, float l) { return (m + __builtin_amdgcn_logf(l)) * kLn2; }

__device__ __forceinline__ f32x16 mfma32(bf16x8 x, bf16x8 y, f32x16 z) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, y, z, 0, 0, 0);
}

// Element i of 16 as a matrix operand's: rounded to bf16, with FINE in two parts, the second what the first leaves (off by
// 2^-17 of the element).
template <bool FINE> __device__ __forceinline__ void split(float x, int i, bf16x8 *hi, bf16x8 *lo) {
    hi[i >> 3][i & 7] = (__bf16)x;
    if constexpr (FINE)
        lo[i >> 3][i & 7] = (__bf16)(x - (float)(__bf16)x);
}
template <bool FINE> __device__ __forceinline__ f32x16 mfma_fine(bf16x8 x, const bf16x8 &hi, const bf16x8 &lo, f32x16 z) {
    z = mfma32(x, hi, z);
    if constexpr (FINE)
        z = mfma32(x, lo, z);
    return z;
}

// Bytes from a row's first element to the end of `rows` rows, 0 where there are none.
__device__ __forceinline__ uint32_t row_bytes(int rows, attn_stride tok, int D) {
    return rows < 1 ? 0u : (uint32_t)(rows - 1) * (uint32_t)(tok.n * 2) + D * 2;
}

// ROWS rows of a token tensor into LDS by NW waves' LDS-DMA. A wave writes H KBs that hold whole groups of rows, of
// every NW H in turn, so that a lane's chunks, and with them its offsets, are the same in all turns but for the rows'
// distance. Columns past D, and rows past the last, lie outside the buffer and arrive as zeros.
template <int DP, int ROWS, int NW = 4> struct cross_stage {
    static constexpr int PW = ROWS * DP / (512 * NW), H = DP == 256 ? 2 : DP == 96 ? 3 : 1;
    static_assert(PW > 0 && PW % H == 0 && H * 512 % (4 * DP) == 0, "whole groups");
    uint32_t off[H];
    __device__ __forceinline__ void init(int w, int lane, attn_stride tok, int D) {
#pragma unroll
        for (int p = 0; p < H; ++p) {
            const int x = (w * H + p) * 1024 + 16 * lane;
            const int rg = x / (8 * DP), y = x % (8 * DP);
            const int r = rg * 4 + (y % 256) / 64, c = y / 256 * 4 + ((y % 64 / 16) ^ (rg & 3));
            off[p] = c * 8 < D ? (uint32_t)r * (uint32_t)(tok.n * 2) + c * 16 : 0x80000000u;
        }
    }
    // rows: how many there are from `first` on.
    __device__ __forceinline__ void load(const uint16_t *first, int rows, attn_stride tok, int D, uint16_t *lds,
                                         int w) const {
        const auto r = make_rsrc(first, row_bytes(min(rows, ROWS), tok, D));
#pragma unroll
        for (int p = 0; p < PW; ++p) {
            const uint32_t far = (uint32_t)(p / H * (NW * H * 512 / DP)) * (uint32_t)(tok.n * 2);
            dma16<0>(r, lds + (w * H + p % H + p / H * NW * H) * 512, opaque(off[p % H]) + far); // not held in registers
        }
    }
};

// A lane's places in such tiles, in elements.
template <int DP> struct cross_lane {
    int nat0, nat1, tr0, tr1;
    __device__ __forceinline__ explicit cross_lane(int lane) {
        const int l32 = lane & 31, hi = lane >> 5, g1 = lane >> 4 & 1, i16 = lane & 15, x = l32 >> 2 & 3;
        const int row = (l32 >> 2) * 4 * DP + (l32 & 3) * 32;
        nat0 = row + (hi ^ x) * 8;
        nat1 = row + (hi ^ x ^ 2) * 8;
        const int c = 2 * g1 + (i16 >> 1 & 1);
        const int tr = hi * 4 * DP + (i16 >> 2) * 32 + (i16 & 1) * 4;
        tr0 = tr + (c ^ hi) * 8;
        tr1 = tr + 8 * DP + (c ^ hi ^ 2) * 8;
    }
    // Row operand: lane l32 has row 32 t + l32, columns 16 kk + 8 hi .. + 7.
    __device__ __forceinline__ bf16x8 nat(const uint16_t *tile, int t, int kk) const {
        return as_bf16x8(
            *reinterpret_cast<const u32x4 *>(tile + (kk & 1 ? nat1 : nat0) + t * 32 * DP + (kk >> 1) * 128));
    }
    // Transposed: lane l32 has column 32 db + l32 of rows 16 c + 4 hi .. + 3 and 16 c + 8 + 4 hi .. + 3, the rows whose
    // scores registers 8 (c % 2) .. + 7 of a row operand's product hold.
    __device__ __forceinline__ bf16x8 tr(const uint16_t *tile, int c, int db) const {
        const uint16_t *x = tile + c * 16 * DP + db * 128;
        return join_tr(lds_read_tr(x + tr0), lds_read_tr(x + tr1));
    }
};

__device__ __forceinline__ void zero16(f32x16 &x) {
#pragma unroll
    for (int i = 0; i < 16; ++i)
        x[i] = 0.f;
}

// A lane's row of an output tile O^T (register 4 j + i of block db: column 32 db + 8 j + 4 hi + i), times f, to bf16 or
// as it is to fp32.
template <int DP>
__device__ __forceinline__ void put_row(const f32x16 *o, float f, uint16_t *dst, int hi, int D) {
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int d = db * 32 + 8 * j + 4 * hi;
            if (db * 32 + 16 * (j >> 1) < D) // D % 16 == 0: the same for all lanes
                *reinterpret_cast<u32x2 *>(dst + d) = u32x2{bf16_pair(o[db][4 * j] * f, o[db][4 * j + 1] * f),
                                                            bf16_pair(o[db][4 * j + 2] * f, o[db][4 * j + 3] * f)};
        }
}
template <int DP> __device__ __forceinline__ void put_part(const f32x16 *o, float *dst, int hi, int D) {
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int d = db * 32 + 8 * j + 4 * hi;
            if (db * 32 + 16 * (j >> 1) < D)
                *reinterpret_cast<f32x4 *>(dst + d) =
                    f32x4{o[db][4 * j], o[db][4 * j + 1], o[db][4 * j + 2], o[db][4 * j + 3]};
        }
}

// Keys of a tile, by the tile's width: two tiles of K and V in two buffers are 64 KB.
constexpr int cross_tile_keys(int DP) { return DP <= 128 ? 64 : 32; }
// A lane's sum of p over a tile up to which the running maximum may lie below the tile's.
constexpr float kCrossSum = 65536.0f;

// ------------------------------------------------------------------------------------------
// Forward, many rows per kv head. One workgroup of four waves per (sequence, kv head, part of its states, tile of 128
// rows): a sequence's rows are its tokens' heads of the group, token by token, 32 to a wave. Tiles of K and V go to LDS
// by LDS-DMA, the next one's beside the products of this one:
//   S^T[key][row] = K . Q^T, O^T[d][row] += V^T . P^T   (v_mfma_f32_32x32x16_bf16)
// The running maximum is raised only where a lane's sum of p over a tile passes kCrossSum.
// Bound by the matrix units and what feeds them: 2 x 4096 rows over 4096 states, 32 heads on 8, D = 128: 519 us, 1060 TFLOP/s
// where a library product of 8192^3 reaches 1279; the matrix units are at work in 54% of the cycles, the LDS in 27%. At
// D = 64 287 us (960 TFLOP/s; the exponentials weigh twice as much), 16 heads of 80 209, 2 x 2048 of 16 heads of 256 140. At
// 77 states (4 x 4096 rows, 10 heads of 64: 19 us) it is bound by the rows' way in and out, 43 MB, and by its start.
// ------------------------------------------------------------------------------------------
template <int DP> __global__ __launch_bounds__(256, DP <= 96 ? 3 : 2) void attn_cross_kernel(const attn_cross_args a) {
    constexpr int KT = cross_tile_keys(DP), KN = DP / 16, NT = KT / 32;
    // K's tile and V's behind it. Each buffer is a variable of its own: the compiler tells LDS accesses apart by
    // variable, and needs address registers for each.
    constexpr int VO = KT * DP;
    __shared__ __attribute__((aligned(1024))) uint16_t KV0[2 * VO], KV1[2 * VO];

    const attn_cross_place at = attn_cross_place_of(&a, wg_id_x());
    const int u = at.u, sp = at.sp;
    const int tid = wi_id_x(), w = uniform(tid >> 6), lane = tid & 63, l32 = lane & 31, hi = lane >> 5;
    const cross_seq seq = seq_at<false>(a, at.nth, lane);
    const attn_range qr = seq.q, kr = seq.k;
    const attn_cut cut = part_of(kr.n, a.share, a.nsplit, ATTN_CROSS_KEY_STEP);
    if (sp >= cut.live)
        return;
    const int k0 = min(sp * cut.per, kr.n), k1 = min(k0 + cut.per, kr.n);
    const int g = a.g, R = qr.n * g, D = a.D;
    const uint16_t *kp = a.k + kr.at * a.k_tok + u * a.k_head, *vp = a.v + kr.at * a.v_tok + u * a.v_head;
    const cross_lane<DP> ln(lane);
    cross_stage<DP, KT> ks, vs;
    ks.init(w, lane, a.k_tok, D);
    vs.init(w, lane, a.v_tok, D);
    auto load = [&](int kb, uint16_t *to) __attribute__((always_inline)) {
        ks.load(kp + kb * a.k_tok, k1 - kb, a.k_tok, D, to, w);
        vs.load(vp + kb * a.v_tok, k1 - kb, a.v_tok, D, to + VO, w);
    };
    auto wait_loads = [] { __builtin_amdgcn_s_waitcnt(waitcnt_vm(0)); };

    for (int tile = at.tile; (int64_t)tile * ATTN_CROSS_ROWS < R; tile += a.tps) {
        const int row = tile * ATTN_CROSS_ROWS + 32 * w + l32;
        const bool valid = row < R;
        const int tok = valid ? attn_div_by(row, a.by_g) : 0, h = u * g + (valid ? row - tok * g : 0);
        const uint16_t *q = a.q + (qr.at + tok) * a.q_tok + h * a.q_head; // without a row of its own: the first one's
        const bool idle = tile * ATTN_CROSS_ROWS + 32 * w >= R;           // the wave has no rows
        bf16x8 qb[KN];
#pragma unroll
        for (int kk = 0; kk < KN; ++kk)
            qb[kk] = as_bf16x8(kk * 16 < D ? *reinterpret_cast<const u32x4 *>(q + kk * 16 + hi * 8) : zero4());
        float m_run = kNegInf, l_run = 0.f;
        f32x16 o[DP / 32];
#pragma unroll
        for (int db = 0; db < DP / 32; ++db)
            zero16(o[db]);

        auto compute = [&](int kb, const uint16_t *kv) __attribute__((always_inline)) {
            if (idle)
                return;
            f32x16 s[NT];
            bf16x8 ka[2][KN];
#pragma unroll
            for (int kk = 0; kk < KN; ++kk)
                ka[0][kk] = ln.nat(kv, 0, kk);
            __builtin_amdgcn_sched_group_barrier(0x100, KN, 0);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                zero16(s[t]);
#pragma unroll
                for (int kk = 0; kk < KN; ++kk) {
                    s[t] = mfma32(ka[t & 1][kk], qb[kk], s[t]);
                    if (t + 1 < NT)
                        ka[(t + 1) & 1][kk] = ln.nat(kv, t + 1, kk);
                }
#pragma unroll
                for (int kk = 0; kk < KN; ++kk) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    if (t + 1 < NT)
                        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                }
            }
            // Register i of sub-tile t: key kb + 32 t + 8 (i / 4) + 4 hi + i % 4.
            if (kb + KT > k1)
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (kb + 32 * t + 8 * (i >> 2) + 4 * hi + (i & 3) >= k1)
                            s[t][i] = kNegInf;
            bf16x8 pk[2 * NT];
            float psum;
            // p against the running maximum; where there is none yet, or a lane's sum is too large, after it is raised.
            for (bool up = __builtin_amdgcn_ballot_w64(m_run == kNegInf) != 0;; up = true) {
                if (up) {
                    float mx = kNegInf;
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int i = 0; i < 16; i += 2)
                            mx = max3f(mx, s[t][i], s[t][i + 1]);
                    const float mnew = fmaxf(m_run, max_xor32(mx));
                    const float alpha = rescale(m_run, mnew, a.c);
                    m_run = mnew;
                    l_run *= alpha;
#pragma unroll
                    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            o[db][i] *= alpha;
                }
                const float mc = m_run == kNegInf ? 0.f : m_run * a.c;
                psum = 0.f;
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float p = fast_exp2(fmaf(s[t][i], a.c, -mc));
                        psum += p;
                        pk[2 * t + (i >> 3)][i & 7] = (__bf16)p;
                    }
                if (up || __builtin_amdgcn_ballot_w64(!(psum <= kCrossSum)) == 0)
                    break;
            }
            l_run += psum;
#pragma unroll
            for (int cc = 0; cc < 2 * NT; ++cc)
#pragma unroll
                for (int db = 0; db < DP / 32; ++db)
                    o[db] = mfma32(ln.tr(kv + VO, cc, db), pk[cc], o[db]);
        };
        if (k0 < k1)
            load(k0, KV0);
        wait_loads(); // for Q too
        __syncthreads();
        auto step = [&](int kb, const uint16_t *kv, uint16_t *next) __attribute__((always_inline)) {
            if (kb + KT < k1)
                load(kb + KT, next);
            compute(kb, kv);
            wait_loads(); // this wave's part of the next tile has arrived
            __syncthreads();
        };
        for (int kb = k0; kb < k1; kb += 2 * KT) {
            step(kb, KV0, KV1);
            if (kb + KT < k1)
                step(kb + KT, KV1, KV0);
        }
        l_run = sum_xor32(l_run);
        if (valid) {
            const float m_log = m_run * a.c;
            const int64_t slot = (int64_t)(qr.at + tok) * a.Hq + h;
            if (cut.live == 1) {
                put_row<DP>(o, l_run > 0.f ? 1.0f / l_run : 0.f, a.o + (qr.at + tok) * a.o_tok + h * a.o_head, hi, D);
                if (a.lse && hi == 0)
                    a.lse[slot] = lse_of(m_log, l_run);
            } else {
                if (hi == 0) {
                    a.pm[slot * a.nsplit + sp] = m_log;
                    a.pl[slot * a.nsplit + sp] = l_run;
                }
                put_part<DP>(o, a.pacc + (slot * a.nsplit + sp) * D, hi, D);
            }
        }
    }
}

// ------------------------------------------------------------------------------------------
// The decode line's units of a call (attn_line.h).
struct cross_units {
    static __device__ __forceinline__ int at(const attn_cross_args &a, int i) {
        if (i >= a.B)
            return 0;
        const attn_range q = attn_range_of(a.q_start[i], a.q_second[i], a.q_is_len, a.Tq);
        return attn_units(q.n, attn_range_of(a.k_start[i], a.k_second[i], a.k_is_len, a.Tk).n);
    }
    static __device__ __forceinline__ int one(const attn_cross_args &a) {
        return attn_units(q_rows(a, 0).n, k_rows(a, 0).n);
    }
    static __device__ __forceinline__ int heads(const attn_cross_args &a) { return a.Hkv_wg; }
};

// Forward, few rows per kv head (single tokens, beams): a workgroup of four waves takes 16 NRB rows over a part of the
// states, the waves interleaved tiles of 32 states, each with a softmax of its own:
//   S^T[key][row] = K . Q^T   (v_mfma_f32_16x16x32_bf16, K from memory straight into the operand)
//   O^T[d][row]  += V^T . P^T (V through a wave-private LDS tile and the transposed read)
// and joins them in LDS. NTL: K and V are read once, past the L2. NW = 1: the waves take a kv head each, whose
// rows are read 1 KB of neighbouring heads at a time (rows_cut has the rule). Bound by HBM:
// 64 tokens over 3277 to 8192 states of 8 heads of 128, 1.55 GB, 231 us (6.7 TB/s), 32 over 4096 at D = 256 161 us; by latency
// where there is less: 16 times five beams over 750 to 1500 states of 16 heads of 64, 72 MB, 22 us, one over 1500 6 us.
// ------------------------------------------------------------------------------------------
template <int DP, int NRB, bool NTL, int NW>
__global__ __launch_bounds__(256, 2) void attn_cross_rows_kernel(const attn_cross_args a) {
    constexpr int VSTR = DP + 16; // elements of a V row in LDS: the eight rows of a pass on other banks
    constexpr int KN = DP / 32, NV = DP / 16, VTILE = 32 * VSTR;
    // K and V of a tile, Q and O do not fit 256 registers at DP = 256: there V is loaded once the scores have freed K's
    // registers, and the next K once V is in LDS. (Left to itself the compiler asked for K one operand at a time.)
    constexpr bool kLate = DP == 256;
    __shared__ __attribute__((aligned(16))) uint16_t Vw[4 * VTILE];
    __shared__ float red_m[NRB][4][16], red_l[NRB][4][16];
    static_assert(16 * (DP + 4) * 4 <= VTILE * 2, "the area for joining must fit in the V tiles");

    const int tid = wi_id_x(), w = uniform(tid >> 6), lane = tid & 63;
    const int r16 = lane & 15, grp = lane >> 4;
    const int team = w / NW, wk = w % NW; // of the workgroup's kv heads, and of that one's waves
    const int g = a.g, D = a.D;
    const float c = a.c, lift = 8.f / c; // how far a score may pass the running maximum
    // This workgroup's row tile t0 and its place on the line: sequence b, group ug of kv heads, first unit `off` of the
    // sequence, `left` units in all. Neighbouring workgroups share an XCD.
    const int L = attn_xcd_order(wg_id_x(), a.wgs);
    const int at = attn_div_by(L, a.by_tps), t0 = L - at * a.tps;
    int ug, b, off = 0, left = 1, pos0 = 0;
    line ln = {0, 1, 0, 0};
    if (a.teams) {
        ln = line_at<cross_units>(a, lane);
        if ((int64_t)at * ln.quota >= (int64_t)ln.total * a.Hkv_wg)
            return;
        pos0 = at * ln.quota;
        left = min(ln.quota, ln.total * a.Hkv_wg - pos0);
        ug = uniform(pos0 / ln.total);
        int before;
        b = uniform(seq_of_unit<cross_units>(a, ln, lane, pos0 - ug * ln.total, before));
        off = pos0 - ug * ln.total - before;
    } else {
        ug = attn_div_by(at, a.by_B);
        b = at - ug * a.B;
    }
    const uint32_t kb2 = (uint32_t)a.k_tok.n * 2, vb2 = (uint32_t)a.v_tok.n * 2; // bytes from row to row
    uint16_t *vt = &Vw[w * VTILE];
    const uint32_t koff = grp * 8 < D ? r16 * kb2 + grp * 16 : 0x80000000u;
    const uint32_t voff = (lane % (DP / 8)) * 8 < D ? (lane / (DP / 8)) * vb2 + (lane % (DP / 8)) * 16 : 0x80000000u;

    while (left > 0 && ug < a.Hkv_wg) {
        const attn_range qr = q_rows(a, b), kr = k_rows(a, b);
        const int u = ug * (4 / NW) + team, R = qr.n * g, units = attn_units(qr.n, kr.n);
        const int take = a.teams ? min(left, units - off) : 1;
        attn_cover cover = {0, 1};
        if (a.teams) {
            cover = attn_cover_of(pos0 - off, max(units, 1), ln.quota);
            cover = attn_cover{uniform(cover.first), uniform(cover.live)};
        }
        const int live = cover.live, sp = at - cover.first;
        const int k0 = min(off * 128, kr.n), k1 = a.teams ? min((off + take) * 128, kr.n) : kr.n;
        const uint16_t *kp = a.k + kr.at * a.k_tok + u * a.k_head, *vp = a.v + kr.at * a.v_tok + u * a.v_head;
        for (int tile = t0; take > 0 && (int64_t)tile * 16 * NRB < R; tile += a.tps) {
            const int row0 = tile * 16 * NRB;
            bf16x8 qb[NRB][KN];
            float m_run[NRB], l_run[NRB];
            f32x4 o[NRB][DP / 16];
#pragma unroll
            for (int i = 0; i < NRB; ++i) {
                const int row = row0 + 16 * i + r16;
                const bool valid = row < R;
                const int tok = valid ? attn_div_by(row, a.by_g) : 0, h = u * g + (valid ? row - tok * g : 0);
                const uint16_t *q = a.q + (qr.at + tok) * a.q_tok + h * a.q_head;
#pragma unroll
                for (int kk = 0; kk < KN; ++kk) {
                    const int col = kk * 32 + grp * 8;
                    u32x4 x = zero4();
                    if (valid && col < D)
                        x = *reinterpret_cast<const u32x4 *>(q + col);
                    qb[i][kk] = as_bf16x8(x);
                }
                m_run[i] = kNegInf;
                l_run[i] = 0.f;
#pragma unroll
                for (int db = 0; db < DP / 16; ++db)
                    o[i][db] = f32x4{0.f, 0.f, 0.f, 0.f};
            }
            struct frags {
                u32x4 k[2 * KN], v[NV];
            };
            // Rows past the part's end, or tiles behind it, lie outside the buffer: nothing is read, zeros arrive.
            auto bytes = [&](int tb, uint32_t step) __attribute__((always_inline)) {
                const int n = min(k1 - tb, 32);
                return n > 0 ? (uint32_t)(n - 1) * step + D * 2 : 0u;
            };
            auto load_k = [&](int tb, frags &f) __attribute__((always_inline)) {
                const auto r = make_rsrc(kp + min(tb, k1) * a.k_tok, bytes(tb, kb2));
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int kk = 0; kk < KN; ++kk)
                        f.k[t * KN + kk] =
                            buf16<NTL>(r, kk * 32 + grp * 8 < D ? koff + 16 * t * kb2 + kk * 64 : 0x80000000u);
            };
            auto load_v = [&](int tb, frags &f) __attribute__((always_inline)) {
                const auto r = make_rsrc(vp + min(tb, k1) * a.v_tok, bytes(tb, vb2));
#pragma unroll
                for (int i = 0; i < NV; ++i)
                    f.v[i] = buf16<NTL>(r, voff + i * (512 / DP) * vb2);
            };
            auto put_v = [&](const frags &f) __attribute__((always_inline)) {
                lds_wave_fence(); // the previous tile's transposed reads are complete
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int x = lane + 64 * i;
                    *reinterpret_cast<u32x4 *>(&vt[x / (DP / 8) * VSTR + x % (DP / 8) * 8]) = f.v[i];
                }
            };
            auto compute = [&](int tb, frags &f) __attribute__((always_inline)) {
                bf16x8 pk[NRB];
                f32x4 s[NRB][2];
#pragma unroll
                for (int i = 0; i < NRB; ++i)
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        s[i][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int kk = 0; kk < KN; ++kk)
                            s[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(f.k[t * KN + kk]), qb[i][kk],
                                                                              s[i][t], 0, 0, 0);
                    }
                __builtin_amdgcn_sched_barrier(0);
                if (kLate)
                    load_v(tb, f);
                else
                    load_k(tb + 32 * NW, f);
#pragma unroll
                for (int i = 0; i < NRB; ++i) {
                    // Register (t, j) of this lane holds key tb + 16t + 4grp + j for row r16.
                    float mx = kNegInf;
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            if (tb + 16 * t + 4 * grp + j >= k1)
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
                if (kLate) {
                    put_v(f);
                    load_k(tb + 32 * NW, f);
                    __builtin_amdgcn_sched_barrier(0);
                }
                lds_wave_fence(); // this tile's V is in LDS before the transposed reads
                const uint16_t *vrow = &vt[(4 * grp + (r16 >> 2)) * VSTR + 4 * (r16 & 3)];
#pragma unroll
                for (int db = 0; db < DP / 16; ++db) {
                    const bf16x8 x = join_tr(lds_read_tr(vrow + db * 16), lds_read_tr(vrow + db * 16 + 16 * VSTR));
#pragma unroll
                    for (int i = 0; i < NRB; ++i)
                        o[i][db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, pk[i], o[i][db], 0, 0, 0);
                }
            };
            int tb = k0 + 32 * wk;
            if (tb < k1) {
                frags f;
                if (!kLate)
                    load_v(tb, f);
                load_k(tb, f);
                for (; tb < k1; tb += 32 * NW) {
                    if (!kLate) {
                        put_v(f);
                        __builtin_amdgcn_sched_barrier(0);
                        load_v(tb + 32 * NW, f);
                    }
                    compute(tb, f);
                }
            }
#pragma unroll
            for (int i = 0; i < NRB; ++i)
                l_run[i] = sum_xor32(sum_xor16(l_run[i]));

            // Join the waves: O^T register (db, j) of this lane holds d = 16db + 4grp + j of row r16.
            float *om = reinterpret_cast<float *>(Vw); // [NW][16][DP + 4]
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
                for (int idx = tid - 64 * NW * team; idx < nrow * (DP / 4); idx += 64 * NW) {
                    const int r = idx / (DP / 4), d = 4 * (idx % (DP / 4));
                    if (d >= D)
                        continue;
                    float mx = kNegInf;
#pragma unroll
                    for (int ww = 0; ww < NW; ++ww)
                        mx = fmaxf(mx, red_m[i][NW * team + ww][r]);
                    const float muse = mx == kNegInf ? 0.f : mx;
                    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
                    float lsum = 0.f;
#pragma unroll
                    for (int ww = 0; ww < NW; ++ww) {
                        const float wgt = fast_exp2(red_m[i][NW * team + ww][r] - muse);
                        const f32x4 x = *reinterpret_cast<const f32x4 *>(&om[((NW * team + ww) * 16 + r) * (DP + 4) + d]);
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            acc[j] += wgt * x[j];
                        lsum += wgt * red_l[i][NW * team + ww][r];
                    }
                    const int i_tok = attn_div_by(rowb + r, a.by_g), h = u * g + rowb + r - i_tok * g;
                    const int tok = qr.at + i_tok;
                    const int64_t slot = (int64_t)tok * a.Hq + h;
                    if (live == 1) {
                        const float inv = lsum > 0.f ? 1.0f / lsum : 0.f;
                        *reinterpret_cast<u32x2 *>(a.o + tok * a.o_tok + h * a.o_head + d) =
                            u32x2{bf16_pair(acc[0] * inv, acc[1] * inv), bf16_pair(acc[2] * inv, acc[3] * inv)};
                        if (a.lse && d == 0)
                            a.lse[slot] = lse_of(mx, lsum);
                    } else {
                        if (d == 0) {
                            a.pm[slot * a.nsplit + sp] = mx;
                            a.pl[slot * a.nsplit + sp] = lsum;
                        }
                        *reinterpret_cast<f32x4 *>(a.pacc + (slot * a.nsplit + sp) * D + d) = acc;
                    }
                }
            }
            __syncthreads(); // the area for joining is V tiles again
        }
        left -= take;
        pos0 += take;
        off = 0;
        if (++b == a.B) {
            b = 0;
            ++ug;
        }
    }
}

// Joins the parts of each row: w_s = 2^(m_s - max m), O = sum w_s acc_s / sum w_s l_s, lse the logarithm of the sum. A
// workgroup takes 256 / (LP SG) rows of one sequence at a time: LP = 2^lglp lanes of four columns each, SG groups of
// parts. What bounds it is latency: NP parts of a thread are asked for at once (3.6 to 4.8 us a launch).
template <int NP, int SG>
__global__ __launch_bounds__(256) void attn_cross_merge_kernel(const attn_cross_args a, int lglp, int tpm) {
    __shared__ __attribute__((aligned(16))) f32x4 accs[SG > 1 ? 256 : 1];
    __shared__ float ms[SG > 1 ? 256 : 1], ls[SG > 1 ? 256 : 1];
    const int b = uniform(wg_id_x() / tpm), t0 = wg_id_x() - b * tpm, tid = wi_id_x();
    const attn_range qr = q_rows(a, b), kr = k_rows(a, b);
    // The parts of a row: its sequence's, or those that the line's quotas make of it, which differ by the kv heads.
    int parts = 1, units = 1, before = 0;
    line ln = {0, 1, 0, 0};
    if (a.teams) {
        ln = line_at<cross_units>(a, tid & 63);
        before = units_before<cross_units>(a, ln, tid & 63, b);
        units = max(attn_units(qr.n, kr.n), 1);
    } else {
        parts = part_of(kr.n, a.share, a.nsplit, ATTN_CROSS_KEY_STEP).live;
        if (parts == 1)
            return; // written already
    }
    constexpr int kLgSG = SG == 1 ? 0 : 2;
    static_assert(1 << kLgSG == SG, "");
    const int R = qr.n * a.Hq, rpw = 256 >> (lglp + kLgSG), d = 4 * (tid & ((1 << lglp) - 1));
    const int rl = tid >> (lglp + kLgSG), sg = tid >> lglp & (SG - 1);
    for (int r0 = t0 * rpw; r0 < R; r0 += tpm * rpw) {
        const int row = r0 + rl, i_tok = attn_div_by(min(row, R - 1), a.by_hq), h = min(row, R - 1) - i_tok * a.Hq;
        const int64_t slot = (int64_t)qr.at * a.Hq + min(row, R - 1);
        if (a.teams)
            parts = attn_cover_of(attn_div_by(h, a.by_gwg) * ln.total + before, units, ln.quota).live;
        const float *pm = a.pm + slot * a.nsplit, *pl = a.pl + slot * a.nsplit;
        const float *p = a.pacc + slot * a.nsplit * a.D + min(d, a.D - 4);
        float mx = kNegInf, sum = 0.f;
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
        for (int s0 = sg; s0 < parts; s0 += NP * SG) {
            float m[NP], l[NP], top = mx;
            f32x4 x[NP];
#pragma unroll
            for (int i = 0; i < NP; ++i) { // parts behind the last: the last again, without weight
                const int s = min(s0 + SG * i, parts - 1);
                m[i] = pm[s];
                l[i] = pl[s];
                x[i] = *reinterpret_cast<const f32x4 *>(p + (int64_t)s * a.D);
            }
#pragma unroll
            for (int i = 0; i < NP; ++i)
                top = fmaxf(top, m[i]); // the last one may be another group's: any maximum not below its own serves
            const float use = top == kNegInf ? 0.f : top, old = fast_exp2(mx - use);
            mx = top;
            sum *= old;
            acc *= old;
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                const bool in = s0 + SG * i < parts;
                const float wgt = fast_exp2(m[i] - use);
                sum += in ? wgt * l[i] : 0.f;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    acc[j] += in ? wgt * x[i][j] : 0.f;
            }
        }
        if constexpr (SG > 1) {
            __syncthreads(); // what the turn before left has been read
            ms[tid] = mx;
            ls[tid] = sum;
            accs[tid] = acc;
            __syncthreads();
            if (sg == 0) {
#pragma unroll
                for (int k = 1; k < SG; ++k)
                    mx = fmaxf(mx, ms[tid + (k << lglp)]);
                const float all = mx == kNegInf ? 0.f : mx;
                sum = 0.f;
                acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < SG; ++k) {
                    const float wgt = fast_exp2(ms[tid + (k << lglp)] - all);
                    const f32x4 y = accs[tid + (k << lglp)];
                    sum += wgt * ls[tid + (k << lglp)];
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        acc[j] += wgt * y[j];
                }
            }
        }
        if (sg == 0 && row < R && d < a.D && parts > 1) { // one part: written already
            const float inv = sum > 0.f ? 1.0f / sum : 0.f;
            const int tok = qr.at + i_tok;
            *reinterpret_cast<u32x2 *>(a.o + tok * a.o_tok + h * a.o_head + d) =
                u32x2{bf16_pair(acc[0] * inv, acc[1] * inv), bf16_pair(acc[2] * inv, acc[3] * inv)};
            if (a.lse && d == 0)
                a.lse[slot] = lse_of(mx, sum);
        }
    }
}

// ------------------------------------------------------------------------------------------
// dQ. Laid out as the forward kernel: 32 rows of a wave keep Q and dO in registers, tiles of K and V pass through LDS:
//   S^T[key][row] = K . Q^T, dP^T[key][row] = V . dO^T, dQ^T[d][row] += K^T . dS^T
// K's tile is read both ways. delta = sum dO O is taken on the way in and left for the kernel of dK and dV. Where a
// sequence has up to 32 states it is sum P dP instead: O's rounding shifts all of a row's dS alike, and O is the larger beside
// V - O the fewer states there are (3 states: dQ off by 2.9e-3 in the norm, without 2.4e-3).
// Six products of the size of S where the forward has four: 724 us at its 4096 x 4096 (1139 TFLOP/s, matrix units 60%), D = 64
// 386, 16 heads of 80 285, 2 x 2048 of 16 heads of 256 263 (one wave per SIMD: Q, dO and dQ are 256 registers).
// ------------------------------------------------------------------------------------------
template <int DP, bool FINE>
__global__ __launch_bounds__(256, FINE ? 1 : DP == 64 ? 4 : DP == 96 ? 3 : DP == 128 ? 2 : 1) void attn_cross_dq_kernel(const attn_cross_args a) {
    constexpr int KT = cross_tile_keys(DP), KN = DP / 16, NT = KT / 32;
    constexpr int VO = KT * DP;
    __shared__ __attribute__((aligned(1024))) uint16_t KV0[2 * VO], KV1[2 * VO];

    const attn_cross_place at = attn_cross_place_of(&a, wg_id_x());
    const int u = at.u, sp = at.sp;
    const int tid = wi_id_x(), w = uniform(tid >> 6), lane = tid & 63, l32 = lane & 31, hi = lane >> 5;
    const cross_seq seq = seq_at<false>(a, at.nth, lane);
    const attn_range qr = seq.q, kr = seq.k;
    const attn_cut cut = part_of(kr.n, a.share, a.nsplit, ATTN_CROSS_KEY_STEP);
    if (sp >= cut.live)
        return;
    const int k0 = min(sp * cut.per, kr.n), k1 = min(k0 + cut.per, kr.n);
    const int g = a.g, R = qr.n * g, D = a.D;
    const uint16_t *kp = a.k + kr.at * a.k_tok + u * a.k_head, *vp = a.v + kr.at * a.v_tok + u * a.v_head;
    const cross_lane<DP> ln(lane);
    cross_stage<DP, KT> ks, vs;
    ks.init(w, lane, a.k_tok, D);
    vs.init(w, lane, a.v_tok, D);
    auto load = [&](int kb, uint16_t *to) __attribute__((always_inline)) {
        ks.load(kp + kb * a.k_tok, k1 - kb, a.k_tok, D, to, w);
        vs.load(vp + kb * a.v_tok, k1 - kb, a.v_tok, D, to + VO, w);
    };
    auto wait_loads = [] { __builtin_amdgcn_s_waitcnt(waitcnt_vm(0)); };

    for (int tile = at.tile; (int64_t)tile * ATTN_CROSS_ROWS < R; tile += a.tps) {
        const int row = tile * ATTN_CROSS_ROWS + 32 * w + l32;
        const bool valid = row < R, idle = tile * ATTN_CROSS_ROWS + 32 * w >= R;
        const int tok = valid ? attn_div_by(row, a.by_g) : 0, h = u * g + (valid ? row - tok * g : 0);
        const int64_t slot = (int64_t)(qr.at + tok) * a.Hq + h;
        bf16x8 qb[KN], gb[KN];
        float delta = 0.f;
        {
            const uint16_t *q = a.q + (qr.at + tok) * a.q_tok + h * a.q_head;
            const uint16_t *go = a.go + (qr.at + tok) * a.go_tok + h * a.go_head;
            const uint16_t *o = a.o + (qr.at + tok) * a.o_tok + h * a.o_head;
#pragma unroll
            for (int kk = 0; kk < KN; ++kk) {
                const int col = kk * 16 + hi * 8;
                u32x4 x = zero4(), y = zero4(), z = zero4();
                if (kk * 16 < D) {
                    x = *reinterpret_cast<const u32x4 *>(q + col);
                    y = *reinterpret_cast<const u32x4 *>(go + col);
                    z = *reinterpret_cast<const u32x4 *>(o + col);
                }
                qb[kk] = as_bf16x8(x);
                gb[kk] = as_bf16x8(y);
                const bf16x8 ob = as_bf16x8(z);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    delta = fmaf((float)gb[kk][i], (float)ob[i], delta);
            }
        }
        delta = sum_xor32(delta);
        const float lse2 = a.lse[slot] * kLog2e;
        f32x16 o[DP / 32];
#pragma unroll
        for (int db = 0; db < DP / 32; ++db)
            zero16(o[db]);

        auto products = [&](const uint16_t *kv, int t, f32x16 &s, f32x16 &dp) __attribute__((always_inline)) {
            zero16(s);
            zero16(dp);
#pragma unroll
            for (int kk = 0; kk < KN; ++kk)
                s = mfma32(ln.nat(kv, t, kk), qb[kk], s);
#pragma unroll
            for (int kk = 0; kk < KN; ++kk)
                dp = mfma32(ln.nat(kv + VO, t, kk), gb[kk], dp);
        };
        auto compute = [&](int kb, const uint16_t *kv) __attribute__((always_inline)) {
            if (idle)
                return;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                if (t > 0 && kb + 32 * t >= k1)
                    return;
                f32x16 s, dp;
                products(kv, t, s, dp);
                bf16x8 pk[2], lo[2];
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    dp[i] = fast_exp2(fmaf(s[i], a.c, -lse2)) * (dp[i] - delta);
                // Past the last key K and V are zeros, but exp(0 - lse) may be infinite.
                if (kb + 32 * t + 32 > k1)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (kb + 32 * t + 8 * (i >> 2) + 4 * hi + (i & 3) >= k1)
                            dp[i] = 0.f;
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    split<FINE>(dp[i], i, pk, lo);
#pragma unroll
                for (int cc = 0; cc < 2; ++cc)
#pragma unroll
                    for (int db = 0; db < DP / 32; ++db)
                        o[db] = mfma_fine<FINE>(ln.tr(kv, 2 * t + cc, db), pk[cc], lo[cc], o[db]);
            }
        };
        if (k0 < k1)
            load(k0, KV0);
        wait_loads();
        __syncthreads();
        if (kr.n <= 32 && k0 < k1 && !idle) {
            f32x16 s, dp;
            products(KV0, 0, s, dp);
            delta = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (8 * (i >> 2) + 4 * hi + (i & 3) < k1)
                    delta = fmaf(fast_exp2(fmaf(s[i], a.c, -lse2)), dp[i], delta);
            delta = sum_xor32(delta);
        }
        if (valid && sp == 0 && hi == 0)
            a.delta[slot] = delta;
        auto step = [&](int kb, const uint16_t *kv, uint16_t *next) __attribute__((always_inline)) {
            if (kb + KT < k1)
                load(kb + KT, next);
            compute(kb, kv);
            wait_loads();
            __syncthreads();
        };
        for (int kb = k0; kb < k1; kb += 2 * KT) {
            step(kb, KV0, KV1);
            if (kb + KT < k1)
                step(kb + KT, KV1, KV0);
        }
        if (valid) {
            if (cut.live == 1)
                put_row<DP>(o, a.scale, a.dq + (qr.at + tok) * a.dq_tok + h * a.dq_head, hi, D);
            else
                put_part<DP>(o, a.pacc + (slot * a.nsplit + sp) * D, hi, D);
        }
    }
}

// ------------------------------------------------------------------------------------------
// dK and dV. One workgroup per (sequence, kv head, part of its rows, tile of 128 states): 32 states of a wave keep K and V in
// registers, the rows of the group's heads, one head after the other, pass through LDS, Q and dO:
//   S[row][key] = Q . K^T, dP[row][key] = dO . V^T, dV^T[d][key] += dO^T . P, dK^T[d][key] += Q^T . dS
// Both tiles are read both ways. Two teams of four waves (TEAMS = 2) have the same states and take steps of 32 rows in turn;
// their sums are joined in LDS at the end.
// Eight products of that size: 997 us at 4096 x 4096 (1103 TFLOP/s, matrix units 53%; half of a wave's time goes in waits, for
// operands and at the barrier of each step, with all 256 registers in use), D = 64 594, 16 heads of 80 410. At D = 256 dK and
// dV are two launches (232 and 184 us for 2 x 2048 of 16 heads on 8): with both, accumulators go to memory, 578 us.
// ------------------------------------------------------------------------------------------
template <int DP, bool DK, bool DV, int TEAMS, bool FINE>
__global__ __launch_bounds__(256 * TEAMS, TEAMS > 1 || FINE ? 1 : DP == 64 ? 3 : DP <= 128 || !DK ? 2 : 1)
void attn_cross_dkv_kernel(const attn_cross_args a) {
    constexpr int QT = ATTN_CROSS_STEP, KN = DP / 16, KEYS = ATTN_CROSS_KEYS;
    constexpr int GO = QT * DP; // dO's tile behind Q's
    static_assert(QT == 32, "a step is one block of rows");
    __shared__ __attribute__((aligned(1024))) uint16_t QG0[TEAMS * 2 * GO], QG1[TEAMS * 2 * GO];
    __shared__ __attribute__((aligned(16))) float st0[TEAMS * 256], st1[TEAMS * 256]; // lse in log2 units, from 64 on delta

    const attn_cross_place at = attn_cross_place_of(&a, wg_id_x());
    const int u = at.u, sp = at.sp;
    const int tid = wi_id_x(), w = uniform(tid >> 6), lane = tid & 63, l32 = lane & 31, hi = lane >> 5;
    const int wk = w & 3, team = w >> 2;
    const cross_seq seq = seq_at<true>(a, at.nth, lane);
    const attn_range qr = seq.q, kr = seq.k;
    const int g = a.g, D = a.D;
    const int per_head = uniform((qr.n + QT - 1) / QT), steps = per_head * g; // of QT rows of one head
    const attn_cut cut = part_of(steps, a.share, a.nsplit, TEAMS);
    if (sp >= cut.live)
        return;
    const int t0 = min(sp * cut.per, steps), t1 = min(t0 + cut.per, steps);
    const cross_lane<DP> ln(lane);
    // At DP = 96 the tiles are 6 KB, three for each of two waves: the first two load Q's, the others dO's.
    constexpr int LW = DP == 96 ? 2 : 4;
    const bool second = LW == 2 && wk >= 2;
    cross_stage<DP, QT, LW> qs, gs;
    qs.init(wk % LW, lane, second ? a.go_tok : a.q_tok, D);
    if constexpr (LW == 4)
        gs.init(wk, lane, a.go_tok, D);
    auto wait_loads = [] { __builtin_amdgcn_s_waitcnt(waitcnt_vm(0)); };

    for (int tile = at.tile; (int64_t)tile * KEYS < kr.n; tile += a.tps) {
        // The wave's rows of K and V, by lane: what lies past the last state or past D is outside the buffer, zeros.
        bf16x8 kf[KN], vf[KN];
        {
            const int first = kr.at + tile * KEYS + 32 * wk;
            const int rows = min(32, kr.n - tile * KEYS - 32 * wk);
            const auto rk = make_rsrc(a.k + first * a.k_tok + u * a.k_head, row_bytes(rows, a.k_tok, D));
            const auto rv = make_rsrc(a.v + first * a.v_tok + u * a.v_head, row_bytes(rows, a.v_tok, D));
            const uint32_t ok = l32 * (uint32_t)(a.k_tok.n * 2) + hi * 16, ov = l32 * (uint32_t)(a.v_tok.n * 2) + hi * 16;
#pragma unroll
            for (int kk = 0; kk < KN; ++kk) {
                const bool in = kk * 16 < D; // D % 16 == 0
                kf[kk] = as_bf16x8(buf16<false>(rk, in ? ok + kk * 32 : 0x80000000u));
                if (DK)
                    vf[kk] = as_bf16x8(buf16<false>(rv, in ? ov + kk * 32 : 0x80000000u));
            }
        }
        f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
        for (int db = 0; db < DP / 32; ++db) {
            zero16(dk[db]);
            zero16(dv[db]);
        }
        // The step to load: head and step of it. Behind the part's last step come empty ones: nothing is read, and P
        // is 0, as it is past a head's last row: 2^(0 - inf). No branch goes around a step: there the
        // allocator copied accumulators to and fro, or to memory.
        const int from = max(min(t0 + team, t1 - 1), 0);
        int ls = t0 + team, lh = uniform(from / max(per_head, 1)), lt = from - lh * per_head;
        float st; // of one row of that step: lse (even waves) or delta
        auto load = [&](uint16_t *to) __attribute__((always_inline)) {
            const int h = u * g + lh, r0 = lt * QT, rows = ls < t1 ? min(qr.n - r0, QT) : 0;
            const int first = qr.at + r0;
            const uint16_t *q = a.q + first * a.q_tok + h * a.q_head, *go = a.go + first * a.go_tok + h * a.go_head;
            uint16_t *const place = to + team * 2 * GO;
            if constexpr (LW == 4) {
                qs.load(q, rows, a.q_tok, D, place, wk);
                gs.load(go, rows, a.go_tok, D, place + GO, wk);
            } else {
                qs.load(second ? go : q, rows, second ? a.go_tok : a.q_tok, D, place + (second ? GO : 0), wk % 2);
            }
            const int r = opaque(lane) & (QT - 1);
            const float *src = (w & 1 ? a.delta : a.lse) + (int64_t)first * a.Hq + h;
            const float x = src[max(min(r, rows - 1), 0) * a.Hq];
            st = w & 1 ? x : r < rows ? x * kLog2e : __builtin_inff();
            ls += TEAMS;
            // The last step's place stays: the empty ones name it. At D = 256 without a branch, with which registers spill
            // (2 x 2048 rows of 16 heads on 8 over as many states: dV 346 us, without 209); below it is faster with one
            // (32 heads on 8, 4096, D = 64: 672 and 736).
            if constexpr (DP > 128) {
                static_assert(TEAMS == 1, "one head further at most");
                lt += ls < t1 ? 1 : 0;
                const int over = lt == per_head ? 1 : 0;
                lh += over;
                lt -= over * per_head;
            } else if (ls < t1) {
                for (lt += TEAMS; lt >= per_head; lt -= per_head)
                    ++lh;
            }
        };
        auto compute = [&](const uint16_t *qg, const float *sb) __attribute__((always_inline)) {
            {
                constexpr int t = 0; // of the steps' rows one block
                f32x16 s, dp;
                zero16(s);
                zero16(dp);
#pragma unroll
                for (int kk = 0; kk < KN; ++kk)
                    s = mfma32(ln.nat(qg, t, kk), kf[kk], s);
#pragma unroll
                for (int kk = 0; DK && kk < KN; ++kk)
                    dp = mfma32(ln.nat(qg + GO, t, kk), vf[kk], dp);
                if constexpr (DP > 64) { // three operands on their way: more, and registers spill
                    constexpr int N = DK ? 2 * KN : KN;
                    __builtin_amdgcn_sched_group_barrier(0x100, 3, 0);
#pragma unroll
                    for (int x = 0; x < N - 3; ++x) {
                        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                    }
                    __builtin_amdgcn_sched_group_barrier(0x008, 3, 0);
                    __builtin_amdgcn_sched_barrier(0);
                }
                bf16x8 pk[2], dk8[2], plo[2], dlo[2];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const f32x4 l = *reinterpret_cast<const f32x4 *>(sb + 32 * t + 8 * j + 4 * hi);
                    const f32x4 e = *reinterpret_cast<const f32x4 *>(sb + 64 + 32 * t + 8 * j + 4 * hi);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float p = fast_exp2(fmaf(s[4 * j + i], a.c, -l[i]));
                        if constexpr (FINE) {
                            split<FINE>(p, 4 * j + i, pk, plo);
                            split<FINE>(p * (dp[4 * j + i] - e[i]), 4 * j + i, dk8, dlo);
                        } else {
                            pk[j >> 1][4 * (j & 1) + i] = (__bf16)p;
                            dk8[j >> 1][4 * (j & 1) + i] = (__bf16)(p * (dp[4 * j + i] - e[i]));
                        }
                    }
                }
#pragma unroll
                for (int cc = 0; cc < 2; ++cc)
#pragma unroll
                    for (int db = 0; db < DP / 32; ++db) {
                        if (DV)
                            dv[db] = mfma32(ln.tr(qg + GO, 2 * t + cc, db), pk[cc], dv[db]);
                        if constexpr (DV && FINE)
                            dv[db] = mfma32(ln.tr(qg + GO, 2 * t + cc, db), plo[cc], dv[db]);
                        if (DK)
                            dk[db] = mfma32(ln.tr(qg, 2 * t + cc, db), dk8[cc], dk[db]);
                        if constexpr (DK && FINE)
                            dk[db] = mfma32(ln.tr(qg, 2 * t + cc, db), dlo[cc], dk[db]);
                    }
            }
        };
        if (t0 < t1) {
            load(QG0);
            st0[tid] = st;
            wait_loads();
            __syncthreads();
            auto step = [&](const uint16_t *qg, const float *sb, uint16_t *next, float *sn) __attribute__((always_inline)) {
                load(next);
                compute(qg + team * 2 * GO, sb + team * 256);
                wait_loads();
                sn[tid] = st;
                __syncthreads();
            };
            for (int i = t0; i < t1; i += 2 * TEAMS) {
                step(QG0, st0, QG1, st1);
                step(QG1, st1, QG0, st0);
            }
        }
        if constexpr (TEAMS > 1) {
            // The second team leaves its sums in the tiles' place: 4 waves x DP 128 bytes in two buffers of DP 256.
            float *const place = reinterpret_cast<float *>(wk & 2 ? QG1 : QG0) + (wk & 1) * (DP * 32) + lane;
            auto join = [&](f32x16 *x) __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; team == 1 && i < DP / 2; ++i)
                    place[i * 64] = x[i / 16][i % 16];
                __syncthreads();
#pragma unroll
                for (int i = 0; team == 0 && i < DP / 2; ++i)
                    x[i / 16][i % 16] += place[i * 64];
                __syncthreads();
            };
            join(dk);
            join(dv);
        }
        // Taken from the lane anew, so that nothing of it is held through the loop.
        const int ln2 = opaque(lane), hi2 = ln2 >> 5, key = tile * KEYS + 32 * wk + (ln2 & 31);
        const int tok = kr.at + key;
        if (team == 0 && key < kr.n) {
            if (cut.live == 1) {
                if (DK)
                    put_row<DP>(dk, a.scale, a.dk + tok * a.dk_tok + u * a.dk_head, hi2, D);
                if (DV)
                    put_row<DP>(dv, 1.f, a.dv + tok * a.dv_tok + u * a.dv_head, hi2, D);
            } else {
                float *dst = a.pacc + (((int64_t)tok * a.Hkv + u) * a.nsplit + sp) * 2 * D;
                if (DK)
                    put_part<DP>(dk, dst, hi2, D);
                if (DV)
                    put_part<DP>(dv, dst + D, hi2, D);
            }
        }
    }
}

// Adds the parts of dQ's rows (KV = false), or of dK's and dV's, in order. 256 / LP rows of one sequence at a time. 5 to 8 us.
template <bool KV>
__global__ __launch_bounds__(256) void attn_cross_sum_kernel(const attn_cross_args a, int lglp, int tpm) {
    const int b = uniform(wg_id_x() / tpm), t0 = wg_id_x() - b * tpm, tid = wi_id_x();
    const attn_range qr = q_rows(a, b), kr = k_rows(a, b);
    const int g = a.g, H = KV ? a.Hkv : a.Hq, W = KV ? 2 * a.D : a.D; // floats of a row's part
    const attn_cut cut = KV ? part_of((qr.n + ATTN_CROSS_STEP - 1) / ATTN_CROSS_STEP * g, a.share, a.nsplit, a.row_teams)
                            : part_of(kr.n, a.share, a.nsplit, ATTN_CROSS_KEY_STEP);
    if (cut.live == 1)
        return; // written already
    const int first = KV ? kr.at : qr.at;
    const int R = (KV ? kr.n : qr.n) * H, rpw = 256 >> lglp, d = 4 * (tid & ((1 << lglp) - 1));
    for (int row = t0 * rpw + (tid >> lglp); row < R; row += tpm * rpw) {
        if (d >= W)
            continue;
        const float *p = a.pacc + ((int64_t)first * H + row) * a.nsplit * W + d;
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int s = 0; s < cut.live; ++s) {
            const f32x4 x = *reinterpret_cast<const f32x4 *>(p + (int64_t)s * W);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                acc[j] += x[j];
        }
        const int i_tok = attn_div_by(row, KV ? a.by_heads : a.by_hq), h = row - i_tok * H;
        const int tok = first + i_tok;
        const bool v = KV && d >= a.D;
        const float f = v ? 1.f : a.scale;
        uint16_t *dst = !KV ? a.dq + tok * a.dq_tok + h * a.dq_head + d
                        : v ? a.dv + tok * a.dv_tok + h * a.dv_head + d - a.D
                            : a.dk + tok * a.dk_tok + h * a.dk_head + d;
        *reinterpret_cast<u32x2 *>(dst) = u32x2{bf16_pair(acc[0] * f, acc[1] * f), bf16_pair(acc[2] * f, acc[3] * f)};
    }
}

// ---- launchers -------------------------------------------------------------------------------
// Calls f(std::integral_constant<int, DP>{}) with the tile width for head dim D. 96 for what is above 64: eight sequences of
// up to 1000 rows and 1500 states, 16 heads, D = 80, forward and gradients 281 us, in tiles of 128 340.
template <typename F> hipError_t with_width(int D, F &&f) {
    return D <= 64    ? f(std::integral_constant<int, 64>{})
           : D <= 96  ? f(std::integral_constant<int, 96>{})
           : D <= 128 ? f(std::integral_constant<int, 128>{})
                      : f(std::integral_constant<int, 256>{});
}

// log2 of the lanes that rows of n floats take, four each: at most the workgroup.
int lg_lanes(int n) {
    int lg = 2;
    while (4 << lg < n)
        ++lg;
    return lg;
}

bool cross_grid_ok(const attn_cross_args &a, const attn_cross_cut &cut) {
    return cut.grid > 0 && cut.grid <= ATTN_CROSS_MAX_GRID && a.nsplit >= 1 && a.nsplit <= ATTN_CROSS_MAX_PARTS &&
           a.tps >= 1;
}

// Workgroups per sequence that look over `rows` rows at rpw a time, not above 2^18 in all.
int cross_sum_tiles(int B, int64_t rows, int rpw) {
    const int64_t t = (rows + rpw - 1) / rpw, most = (1 << 18) / B;
    return (int)(t < 1 || most < 1 ? 1 : t < most ? t : most);
}

} // namespace

extern "C" int attn_hip_launch_cross(const struct attn_cross_args *ap, const struct attn_cross_cut *cut, int max_q,
                                     void *stream) {
    const attn_cross_args &a = *ap;
    const hipStream_t st = (hipStream_t)stream;
    if (!cross_grid_ok(a, *cut))
        return (int)hipErrorInvalidValue;
    const dim3 grid((unsigned)cut->grid), block(256);
    const hipError_t e = with_width(a.D, [&](auto W) {
        constexpr int DP = decltype(W)::value;
        auto rows = [&](auto NB, auto NT, auto NWF) {
            constexpr int kN = decltype(NB)::value, kW = decltype(NWF)::value, RP = DP == 96 ? 128 : DP; // bound by HBM
            constexpr bool kT = decltype(NT)::value;
            if (t_plan) {
                plan_note(grid, block, "attn_cross_rows_kernel<%d, %d, %s, %d> parts=%d share=%d", RP, kN, tf(kT),
                          kW, a.nsplit, a.share);
                return hipSuccess;
            }
            hipLaunchKernelGGL((attn_cross_rows_kernel<RP, kN, kT, kW>), grid, block, 0, st, a);
            return hipGetLastError();
        };
        constexpr std::integral_constant<int, 1> one;
        constexpr std::integral_constant<int, 2> two;
        constexpr std::integral_constant<int, 4> four;
        // Past the L2 where a row tile is the only one of its sequence, which up to D = 128 it always is.
        if constexpr (DP > 128) {
            if (cut->rows16 == 1)
                return with_flag(a.tps == 1, [&](auto NT) {
                    return cut->quads ? rows(one, NT, one) : rows(one, NT, four);
                });
        } else {
            if (cut->rows16 == 1)
                return cut->quads ? rows(one, std::true_type{}, one) : rows(one, std::true_type{}, four);
            if (cut->rows16 == 2)
                return cut->quads ? rows(two, std::true_type{}, one) : rows(two, std::true_type{}, four);
        }
        if (t_plan) {
            plan_note(grid, block, "attn_cross_kernel<%d> parts=%d share=%d", DP, a.nsplit, a.share);
            return hipSuccess;
        }
        hipLaunchKernelGGL((attn_cross_kernel<DP>), grid, block, 0, st, a);
        return hipGetLastError();
    });
    if (e != hipSuccess || a.nsplit == 1)
        return (int)e;
    const int lglp = lg_lanes(a.D);
    auto merge = [&](auto N, auto G) {
        constexpr int kN = decltype(N)::value, kG = decltype(G)::value;
        const int tpm = cross_sum_tiles(a.B, (int64_t)max_q * a.Hq, (256 >> lglp) / kG);
        const dim3 mgrid((unsigned)(a.B * tpm));
        if (t_plan) {
            plan_note(mgrid, block, "attn_cross_merge_kernel<%d, %d>", kN, kG);
            return hipSuccess;
        }
        hipLaunchKernelGGL((attn_cross_merge_kernel<kN, kG>), mgrid, block, 0, st, a, lglp, tpm);
        return hipGetLastError();
    };
    constexpr std::integral_constant<int, 1> one;
    constexpr std::integral_constant<int, 4> four;
    constexpr std::integral_constant<int, 16> sixteen;
    return (int)(cut->parts <= 4 ? merge(four, one) : cut->parts <= 16 ? merge(sixteen, one) : merge(sixteen, four));
}

// One of the two gradient kernels and, where it may leave parts, their sum. kv: dK and dV, after dQ.
extern "C" int attn_hip_launch_cross_grad(const struct attn_cross_args *ap, const struct attn_cross_cut *cut, int kv,
                                          int most, void *stream) {
    const attn_cross_args &a = *ap;
    const hipStream_t st = (hipStream_t)stream;
    if (!cross_grid_ok(a, *cut))
        return (int)hipErrorInvalidValue;
    const dim3 grid((unsigned)cut->grid), block(256);
    const hipError_t e = with_width(a.D, [&](auto W) {
        constexpr int DP = decltype(W)::value;
        if (!kv)
            return with_flag(cut->fine, [&](auto F) {
                constexpr bool kF = decltype(F)::value;
                if (t_plan) {
                    plan_note(grid, block, "attn_cross_dq_kernel<%d, %s> parts=%d share=%d", DP, tf(kF), a.nsplit, a.share);
                    return hipSuccess;
                }
                hipLaunchKernelGGL((attn_cross_dq_kernel<DP, kF>), grid, block, 0, st, a);
                return hipGetLastError();
            });
        auto dkv = [&](auto K, auto V, auto T, auto F) {
            constexpr bool kK = decltype(K)::value, kV = decltype(V)::value, kF = decltype(F)::value;
            constexpr int kT = decltype(T)::value;
            if (t_plan) {
                plan_note(grid, dim3(256 * kT), "attn_cross_dkv_kernel<%d, %s, %s, %d, %s> parts=%d share=%d", DP, tf(kK),
                          tf(kV), kT, tf(kF), a.nsplit, a.share);
                return hipSuccess;
            }
            hipLaunchKernelGGL((attn_cross_dkv_kernel<DP, kK, kV, kT, kF>), grid, dim3(256 * kT), 0, st, a);
            return hipGetLastError();
        };
        constexpr std::true_type yes;
        constexpr std::false_type no;
        constexpr std::integral_constant<int, 1> one;
        constexpr std::integral_constant<int, 2> two;
        if (cut->row_teams == 2) {
            if constexpr (DP <= 128)
                return dkv(yes, yes, two, no);
            return hipErrorInvalidValue;
        }
        return with_flag(cut->fine, [&](auto F) {
            if constexpr (DP > 128) {
                const hipError_t x = dkv(yes, no, one, F);
                return x != hipSuccess ? x : dkv(no, yes, one, F);
            } else {
                return dkv(yes, yes, one, F);
            }
        });
    });
    if (e != hipSuccess || a.nsplit == 1)
        return (int)e;
    const int lglp = lg_lanes(kv ? 2 * a.D : a.D);
    const int tpm = cross_sum_tiles(a.B, (int64_t)most * (kv ? a.Hkv : a.Hq), 256 >> lglp);
    const dim3 sgrid((unsigned)(a.B * tpm));
    if (t_plan) {
        plan_note(sgrid, block, "attn_cross_sum_kernel<%s>", tf(kv));
        return (int)hipSuccess;
    }
    if (kv)
        hipLaunchKernelGGL(attn_cross_sum_kernel<true>, sgrid, block, 0, st, a, lglp, tpm);
    else
        hipLaunchKernelGGL(attn_cross_sum_kernel<false>, sgrid, block, 0, st, a, lglp, tpm);
    return (int)hipGetLastError();
}

#endif

/* attn_paged_cut.h -- what the paged kernels are given, and how the host layer cuts a call into workgroups.
 * Lengths of sequences lie in device memory, so the cut goes by the caller's bounds (max_q, max_kv); the
 * kernels go by the lengths, and serve sequences past the bounds too. */
#ifndef ATTN_PAGED_CUT_H
#define ATTN_PAGED_CUT_H

#include <stdint.h>

#include "attn_decode_rule.h"
#include "attn_paged_rule.h"

/* What the attention kernels are given. */
struct attn_paged_args {
    const uint16_t *q;
    uint16_t *o;
    int64_t q_tok, q_head, o_tok, o_head; /* strides in elements */
    const uint8_t *k, *v, *ks, *vs;       /* the cache's pages and, in 4 bits, their scales */
    const int32_t *table, *kv_len, *q_start;
    const float *slopes;
    float *pm, *pl, *pacc; /* partials of split calls, one slot per (token, head, part) */
    int32_t B, T, Hq, Hkv, D, cols, pages, lgp, causal;
    float c;                  /* scale log2(e) */
    float cap_in, cap_out;    /* softcap: 2 log2(e) scale / cap and cap log2(e); cap_out = 0 without */
    int32_t tps, nsplit; /* row tiles per sequence, parts of a sequence at most */
    int32_t teams;       /* decode: see attn_quota; 0: a workgroup takes a whole sequence */
    int32_t deal, share; /* prefill: see attn_place_of, attn_parts_of */
};

/* What the append and read kernels are given. */
struct attn_kv_args {
    const uint16_t *q, *k, *v;       /* append: the new rows */
    uint16_t *q_out, *k_out, *v_out; /* where rows go: append's rotated q, read's K and V */
    int64_t q_tok, q_head, qo_tok, qo_head, k_tok, k_head, v_tok, v_head;
    uint8_t *ck, *cv, *cks, *cvs;
    const int32_t *table, *kv_len, *q_start;
    const float *rope;
    int32_t B, T, Hq, Hkv, D, cols, pages, lgp, rope_rows, rot;
    int32_t tblk; /* workgroups per sequence */
};

#define ATTN_PAGED_DECODE_WG 512 /* workgroups of a decode call: two per CU */
#define ATTN_PAGED_MAX_PARTS 256
#define ATTN_PAGED_MAX_GRID 0xffffffL
#define ATTN_PAGED_MERGE_WEIGHTS 2048 /* rows x parts that a workgroup of the merge holds the weights of */

/* rows16: row blocks of 16 per workgroup, 1 or 2 (the decode kernel), 4 or 8 (the prefill kernel); rpw: rows
 * that a workgroup of the merge takes at a time, 0 without one (lglp, lgsg: log2 of its lanes per row and
 * of its groups of parts). */
struct attn_paged_cut {
    int rows16, tps, nsplit, teams, deal, share;
    int64_t grid;
    int lglp, lgsg, merge_tiles, merge_loads;
    int halves; /* prefill: eight waves on key halves instead of four */
};

static inline struct attn_paged_cut attn_paged_cut_of(int B, int Hkv, int g, int T, int max_q, int max_kv,
                                                      int D, int bits, int causal) {
    if (max_kv > 1 << 30) /* what a row of the table can hold */
        max_kv = 1 << 30;
    const int64_t rows = (int64_t)(max_q < T ? max_q : T) * g;
    const int rows16 = rows <= 16 ? 1 : rows > 64 ? 8 : D > 128 ? 1 : rows <= 32 ? 2 : 4;
    const int64_t seqs = (int64_t)B * Hkv;
    int64_t tps = (rows + 16 * rows16 - 1) / (16 * rows16);
    if (tps * seqs > ATTN_PAGED_MAX_GRID / 16) /* workgroups go on to further tiles */
        tps = ATTN_PAGED_MAX_GRID / 16 / seqs > 1 ? ATTN_PAGED_MAX_GRID / 16 / seqs : 1;
    const int64_t cap = ATTN_SLOTS / ((int64_t)T * Hkv * g);
    const int64_t units = ((int64_t)max_kv + 127) / 128;
    struct attn_paged_cut c = {rows16, (int)tps, 1, 0, 1, 1 << 30, 0, 0, 0, 0, 8, 0};
    int64_t likely = 1; /* parts of a sequence */
    if (rows16 <= 2) {
        /* Two workgroups per CU, but one at head dims past 128 in bf16 (us, 512 -> 256 workgroups: 32 sequences
         * of 4096 keys 177 -> 170, one of 32768 33.5 -> 31), and in 4 bits where they would have less than four
         * units each (one of 32768 22.0 -> 20.4; 32 of 4096 stay at 57, 71 with 256). */
        const int one = D > 128 && (bits == 16 || seqs * units < 2048);
        int64_t teams = ((one ? ATTN_PAGED_DECODE_WG / 2 : ATTN_PAGED_DECODE_WG) + tps - 1) / tps;
        if (teams > seqs * units)
            teams = seqs * units;
        if (cap >= 2) {
            c.teams = (int)teams;
            const int64_t most = units + 1 > ATTN_PAGED_MAX_PARTS ? ATTN_PAGED_MAX_PARTS : units + 1;
            c.nsplit = (int)(cap > most ? most : cap);
            likely = teams / seqs + 1;
        }
        c.grid = (c.teams ? c.teams : seqs) * tps;
    } else {
        /* Eight waves on key halves, one workgroup per CU (256 of them), where there is at most a round of
         * them, or two of a causal prompt's tiles, whose lengths differ. Four waves, two workgroups per
         * CU, otherwise. us at D = 128, 32 heads on 8 kv heads, four waves -> key halves: 512 tokens over
         * 8192 keys 85 -> 79, 128 over 4096 30.6 -> 26.7, prompts of 1200 35.7 -> 30.2 and 2048 55.4 -> 52.2;
         * kept at four: 1200 over 8192 (300 tiles) 204 and 224, 4096 over 4096 147 and 162. */
        const int64_t w = seqs * tps;
        c.halves = rows16 == 8 && D <= 128 &&
                   (w <= 256 || (w <= 512 && causal && max_kv / 2 <= max_q));
        int64_t ns = 1;
        if (!c.halves) {
            ns = (512 + w - 1) / w;
        } else if (w <= 256) {
            /* The parts that take the least time: rounds of a tile over its part's keys (us at 4.3 TFLOP/s per
             * CU), and for each part its rows written and read again (6 TB/s). */
            double best = 0;
            for (int64_t n = 1; n <= 16 && (n == 1 || n * 256 <= max_kv); ++n) {
                const double t = (double)((w * n + 255) / 256) / (double)n * 128 * max_kv * D * 4 / 4.3e6 +
                                 (n > 1 ? 4 + (double)n * (double)seqs * (double)rows * D * 8 / 6e6 : 0);
                if (n == 1 || t < best)
                    best = t, ns = n;
            }
        }
        ns = ns > units ? units : ns;
        ns = ns > cap ? cap : ns;
        ns = ns > ATTN_PAGED_MAX_PARTS ? ATTN_PAGED_MAX_PARTS : ns;
        if (ns >= 2) {
            c.nsplit = (int)ns;
            c.share = (int)((((int64_t)max_kv + ns - 1) / ns + 127) / 128 * 128);
        }
        const int64_t groups = seqs * c.nsplit;
        while (c.deal < 8 && c.deal < tps && groups < 64 && groups * c.deal % 8 != 0)
            c.deal *= 2;
        c.grid = attn_place_grid(groups, c.tps, c.deal);
        likely = c.nsplit;
    }
    if (c.nsplit > 1) {
        /* Lanes of four columns each; groups of parts until a thread has eight loads or fewer, or the
         * workgroup is one row's. */
        c.lglp = 3;
        while ((4 << c.lglp) < D)
            ++c.lglp;
        while (c.lglp + c.lgsg < 8 && (8 << c.lgsg) < likely)
            ++c.lgsg;
        while (c.lglp + c.lgsg < 8 && (2 << c.lgsg) <= likely && seqs * rows << (c.lglp + c.lgsg) < 65536)
            ++c.lgsg;
        /* Loads of a thread in flight. us, four parts with eight loads and with four: 16 x 8 tokens of 64 heads
         * 50.0 and 48.4, 200 tokens over 3000 29.7 and 28.2; three parts with two and with four: 300 over 8192
         * 56.3 and 57.1. */
        c.merge_loads = likely <= 3 << c.lgsg ? 2 : likely <= 4 << c.lgsg ? 4 : 8;
        const int64_t rpw = 256 >> (c.lglp + c.lgsg);
        if (c.nsplit > ATTN_PAGED_MERGE_WEIGHTS / rpw)
            c.nsplit = (int)(ATTN_PAGED_MERGE_WEIGHTS / rpw);
        int64_t tiles = (rows + rpw - 1) / rpw;
        if (tiles * seqs > ATTN_PAGED_MAX_GRID)
            tiles = ATTN_PAGED_MAX_GRID / seqs;
        c.merge_tiles = (int)tiles;
    }
    return c;
}

/* Append and read: workgroups per sequence, of tpw tokens each (append one, read one per wave). */
static inline int attn_kv_blocks(int B, int T, int max_q, int tpw) {
    const int64_t n = ((int64_t)(max_q < T ? max_q : T) + tpw - 1) / tpw;
    return (int)(n * B > ATTN_PAGED_MAX_GRID ? ATTN_PAGED_MAX_GRID / B : n);
}

#endif

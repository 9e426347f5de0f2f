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
};

static inline struct attn_paged_cut attn_paged_cut_of(int B, int Hkv, int g, int T, int max_q, int max_kv,
                                                      int D) {
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
    struct attn_paged_cut c = {rows16, (int)tps, 1, 0, 1, 1 << 30, 0, 0, 0, 0, 8};
    int64_t likely = 1; /* parts of a sequence */
    if (rows16 <= 2) {
        int64_t teams = (ATTN_PAGED_DECODE_WG + tps - 1) / tps;
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
        int64_t ns = (512 + seqs * tps - 1) / (seqs * tps);
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
        c.merge_loads = likely <= 3 << c.lgsg ? 2 : 8;
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

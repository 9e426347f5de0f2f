/* attn_paged_cut.h -- what the paged kernels are given, and how the host layer cuts a call into workgroups.
 * Lengths of sequences lie in device memory, so the cut goes by the caller's bounds (max_q, max_kv); the
 * kernels go by the lengths, and serve sequences past the bounds too. */
#ifndef ATTN_PAGED_CUT_H
#define ATTN_PAGED_CUT_H

#include <stdint.h>

#include "attn_decode_rule.h"

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
    int32_t tps, nsplit, kps; /* row tiles per sequence, parts, keys per part */
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
    int32_t tblk, ublk, tpw; /* token blocks per sequence, blocks of 256 units, tokens per block */
};

#define ATTN_PAGED_MAX_PARTS 256
#define ATTN_PAGED_MAX_GRID 0xffffffL

/* rows16: row blocks of 16 per workgroup, 1 or 2 (the decode kernel) or 8 (the prefill kernel). */
struct attn_paged_cut {
    int rows16, tps, nsplit, kps;
};

static inline struct attn_paged_cut attn_paged_cut_of(int B, int Hkv, int g, int T, int max_q, int max_kv,
                                                      int D) {
    if (max_kv > 1 << 30) /* what a row of the table can hold */
        max_kv = 1 << 30;
    const int64_t rows = (int64_t)(max_q < T ? max_q : T) * g;
    const int rows16 = rows <= 16 ? 1 : rows > 64 ? 8 : D <= 128 ? 2 : 1;
    int64_t tps = (rows + 16 * rows16 - 1) / (16 * rows16);
    const int64_t seqs = (int64_t)B * Hkv;
    if (tps * seqs > ATTN_PAGED_MAX_GRID) /* workgroups go on to further tiles */
        tps = ATTN_PAGED_MAX_GRID / seqs > 1 ? ATTN_PAGED_MAX_GRID / seqs : 1;
    const int64_t wgs = seqs * tps;
    const int64_t cap = ATTN_SLOTS / ((int64_t)T * Hkv * g);
    const int64_t by_len = ((int64_t)max_kv + 127) / 128;
    int64_t ns = (ATTN_DECODE_TARGET_WG + wgs - 1) / wgs;
    if (ns > by_len)
        ns = by_len;
    if (ns > cap)
        ns = cap;
    if (ns > ATTN_PAGED_MAX_PARTS)
        ns = ATTN_PAGED_MAX_PARTS;
    if (ns < 2)
        ns = 1;
    int64_t kps = ((int64_t)max_kv + ns - 1) / ns;
    kps = (kps + 127) / 128 * 128;
    struct attn_paged_cut c = {rows16, (int)tps, (int)(((int64_t)max_kv + kps - 1) / kps), (int)kps};
    return c;
}

struct attn_kv_cut {
    int tblk, ublk, tpw;
};

/* Tokens per workgroup: one while that leaves a grid of at most 2048 workgroups, else up to 8. */
static inline struct attn_kv_cut attn_kv_cut_of(int B, int T, int max_q, int64_t units) {
    const int64_t ublk = (units + 255) / 256;
    const int64_t mq = max_q < T ? max_q : T;
    int64_t tpw = 1;
    while (tpw < 8 && (mq + tpw - 1) / tpw * ublk * B > 2048)
        tpw *= 2;
    int64_t tblk = (mq + tpw - 1) / tpw;
    if (tblk * ublk * B > ATTN_PAGED_MAX_GRID)
        tblk = ATTN_PAGED_MAX_GRID / (ublk * B) > 1 ? ATTN_PAGED_MAX_GRID / (ublk * B) : 1;
    struct attn_kv_cut c = {(int)tblk, (int)ublk, (int)tpw};
    return c;
}

#endif

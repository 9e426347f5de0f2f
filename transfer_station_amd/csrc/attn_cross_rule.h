/* attn_cross_rule.h -- cross attention's arguments, index arithmetic and how a call is cut. The kernels and the
 * host layer share it, and its arithmetic holds no pointer, so that the CPU tests run it with every kind of bad
 * start and length. */
#ifndef ATTN_CROSS_RULE_H
#define ATTN_CROSS_RULE_H

#include "attn_paged_rule.h"

/* A sequence's rows of a token tensor of T rows: at .. at + n - 1. Starts and lengths come from device memory:
 * whatever they are, at >= 0, n >= 0 and at + n <= T. */
struct attn_range {
    int at, n;
};

ATTN_HD struct attn_range attn_range_of(int start, int second, int is_len, int T) {
    struct attn_range r;
    r.at = start < 0 ? 0 : (start > T ? T : start);
    if (is_len) {
        r.n = second < 0 ? 0 : (second > T - r.at ? T - r.at : second);
    } else {
        const int end = second < r.at ? r.at : (second > T ? T : second);
        r.n = end - r.at;
    }
    return r;
}

/* `total` units (keys, or tiles of rows) in as many parts of `share` units as it takes, at most nsplit: all of `per`
 * units (a multiple of `step`) but the last, which ends at total. One part where there is nothing. */
struct attn_cut {
    int live, per;
};

ATTN_HD struct attn_cut attn_cut_of(int total, int share, int nsplit, int step) {
    int n = total / share + (total % share != 0);
    n = n < 1 ? 1 : (n > nsplit ? nsplit : n);
    int per = total / n + (total % n != 0);
    per = per < 1 ? step : (per + step - 1) / step * step;
    struct attn_cut c = {total / per + (total % per != 0), per};
    if (c.live < 1)
        c.live = 1;
    return c;
}

#define ATTN_CROSS_ROWS 128     /* rows of a tile: four waves of 32 */
#define ATTN_CROSS_KEYS 128     /* states of a tile of the kernel of dK and dV: four waves of 32 */
#define ATTN_CROSS_KEY_STEP 128 /* parts of the states are multiples of this */
#define ATTN_CROSS_MAX_PARTS 64
#define ATTN_CROSS_MAX_GRID 0x7fffffffL
/* Floats of partial gradients that a call of attn_cross_grad may take (128 MB). */
#define ATTN_CROSS_GRAD_FLOATS (1L << 25)

/* Rows of a step of the kernel of dK and dV. */
ATTN_HD int attn_cross_step_rows(int D) { return D <= 64 ? 64 : 32; }

/* What one launch looks like: row (or state) tiles per group and its parts, and how the groups are dealt to the XCDs
 * (attn_place_of). */
struct attn_cross_cut {
    int tps, nsplit, share, deal;
    int rows16; /* blocks of 16 rows per workgroup of the kernel for few rows, 0: tiles of 128 */
    long grid;
};

struct attn_cross_args {
    const uint16_t *q, *k, *v, *go; /* go: dO */
    uint16_t *o, *dq, *dk, *dv;
    float *lse, *delta; /* [Tq][Hq] */
    int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head, o_tok, o_head, go_tok, go_head;
    int64_t dq_tok, dq_head, dk_tok, dk_head, dv_tok, dv_head;
    const int32_t *q_start, *q_second, *k_start, *k_second; /* second: lengths, or the next starts */
    int q_is_len, k_is_len;
    int B, Tq, Tk, Hq, Hkv, D;
    float c, scale; /* scale log2(e), scale */
    int tps, nsplit, share, deal;
    float *pm, *pl, *pacc; /* partial maxima, sums and rows; of gradients: rows in pacc */
};

#endif

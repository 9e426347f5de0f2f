/* attn_cross_rule.h -- cross attention's arguments, index arithmetic and how a call is cut. The kernels and the
 * host layer share it, and its arithmetic holds no pointer, so that the CPU tests run it with every kind of bad
 * start and length. */
#ifndef ATTN_CROSS_RULE_H
#define ATTN_CROSS_RULE_H

#include "attn_div.h"
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
#define ATTN_CROSS_TEAMS 256 /* of the kernel for few rows: a workgroup per CU */
#define ATTN_CROSS_MAX_GRID 0xffffffL /* workgroups of 256 threads: a launch has less than 2^32 work-items */
/* Floats of partial gradients that a call of attn_cross_grad may take (128 MB). */
#define ATTN_CROSS_GRAD_FLOATS (1L << 25)

#define ATTN_CROSS_STEP 32 /* rows of a step of the kernel of dK and dV */

/* Calls of up to this many scores (heads, rows and states as the call bounds them) take P and dS of the gradients in two bf16
 * parts each, which makes their products as good as fp32's: dQ, dK and dV are off by their own rounding, 1.7e-3 in the norm,
 * not by 2.4e-3, which single rows and heads pass by a fifth. They wait more than they compute: 512 rows over 512 states, 16
 * heads of 64 48.5 -> 50.6 us, 8 x 100 over 100 of 128 46.9 -> 45.6, 37 over 50 16.5 -> 17.5; but 4 x 200 over 300 of 96,
 * 2^22 scores, 54 -> 61. */
#define ATTN_CROSS_FINE (1L << 21)

/* Launches of 2 to 64 sequences (a wave's lanes), of more workgroups than run at once, start the longest first: eight
 * prompts of 210 to 700 tokens over 2000 to 4001 states 226 -> 216 us, the step of eight by up to 1000 and 1500 268 ->
 * 245. Tiles that walk few rows are over before it pays (77 states: 3 us lost of 73). */
#define ATTN_CROSS_RANKED 64
#define ATTN_CROSS_AT_ONCE 512
#define ATTN_CROSS_LONG 512

/* What one launch looks like: row (or state) tiles of a sequence and kv head, its parts, and their share of units. */
struct attn_cross_cut {
    int tps, nsplit, share;
    int rows16; /* blocks of 16 rows per workgroup of the kernel for few rows, 0: tiles of 128 */
    int quads;  /* that kernel's form for four kv heads of a workgroup, a wave each */
    int parts;  /* of a sequence of the call's bounds, about */
    int teams;  /* that kernel: teams of the decode line, 0: whole sequences */
    int row_teams; /* the kernel of dK and dV: teams of four waves that share a tile of states */
    int fine;      /* gradients: P and dS in two parts */
    long grid;
};

/* Elements from row to row, at most ATTN_TOKEN_MAX. Its product with a row's number has 64 bits. */
struct attn_stride {
    int32_t n;
};
#ifdef __cplusplus
ATTN_HD int64_t operator*(int row, attn_stride s) { return (int64_t)row * s.n; }
#endif

struct attn_cross_args {
    const uint16_t *q, *k, *v, *go; /* go: dO */
    uint16_t *o, *dq, *dk, *dv;
    float *lse, *delta; /* [Tq][Hq] */
    int64_t q_head, k_head, v_head, o_head, go_head, dq_head, dk_head, dv_head;
    struct attn_stride q_tok, k_tok, v_tok, o_tok, go_tok, dq_tok, dk_tok, dv_tok;
    const int32_t *q_start, *q_second, *k_start, *k_second; /* second: lengths, or the next starts */
    int q_is_len, k_is_len;
    int B, Tq, Tk, Hq, Hkv, g, D; /* g = Hq / Hkv */
    float c, scale; /* scale log2(e), scale */
    int tps, nsplit, share, wgs;
    int teams, Hkv_wg; /* few rows: teams of the decode line, groups of kv heads */
    int row_teams;     /* dK and dV */
    int by_length;     /* the tile kernels' sequences come longest first */
    struct attn_div by_tps, by_B, by_heads, by_bh, by_hq, by_g, by_gwg; /* tps, B, Hkv, B Hkv, Hq, g, heads of a group of kv heads */
    float *pm, *pl, *pacc; /* partial maxima, sums and rows; of gradients: rows in pacc */
};

/* Place i of n neighbouring places, cut into one run of them for each of the eight XCDs, to which hardware ids are dealt
 * in turn. */
ATTN_HD int attn_xcd_order(int wg, int n) {
    const int per = n >> 3, rem = n & 7, x = wg & 7;
    return (x < rem ? x * (per + 1) : rem * (per + 1) + (x - rem) * per) + (wg >> 3);
}

/* Where a workgroup of the tile kernels is. A sequence's tiles of a kv head and part read the same rows, and share an XCD's
 * L2; these groups, in the order [part][place of the sequence][kv head], are dealt to the XCDs in turn, so that each
 * has some of every length, and the first sequences' of all heads first. The last groups, fewer than eight, are cut. */
struct attn_cross_place {
    int nth, u, sp, tile; /* nth: the sequence's place among the call's */
};
ATTN_HD struct attn_cross_place attn_cross_place_of(const struct attn_cross_args *a, int wg) {
    const int whole = attn_div_by(a->wgs, a->by_tps) & ~7, dealt = whole * a->tps;
    const int in = wg < dealt, at = in ? wg >> 3 : attn_xcd_order(wg - dealt, a->wgs - dealt);
    const int k = attn_div_by(at, a->by_tps);
    int group = in ? k * 8 + (wg & 7) : whole + k;
    struct attn_cross_place p;
    p.tile = at - k * a->tps;
    p.sp = attn_div_by(group, a->by_bh);
    group -= p.sp * a->B * a->Hkv;
    p.nth = attn_div_by(group, a->by_heads);
    p.u = group - p.nth * a->Hkv;
    return p;
}

#endif

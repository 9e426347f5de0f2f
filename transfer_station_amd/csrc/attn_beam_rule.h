/* attn_beam_rule.h -- arguments and sizes of the beam search's kernels, shared by the kernels and the host layer. */
#ifndef ATTN_BEAM_RULE_H
#define ATTN_BEAM_RULE_H

#include <stdint.h>

#include "attn_div.h"
#include "attn_paged_rule.h"

/* Logits of `size` bytes that a wave takes at a time: 4 KB. */
#define ATTN_BEAM_STEP(size) ((int)(4096 / (size)))

/* A row of logits is looked through in chunks, one workgroup of four waves each, `steps` steps to a wave. A chunk leaves
 * its K best and its maximum and sum of exponentials. Short chunks, of one step, where the rows are too few to fill the
 * GPU with longer ones; else four workgroups per CU: 512 rows of 128256 in bf16 38.9 us, with six 42.0, with eight 43.9 (a
 * longer piece of a row has fewer logits that pass its threshold). */
#define ATTN_BEAM_FILL 1024 /* workgroups */
struct attn_beam_cut {
    int chunks, steps;
};
ATTN_HD struct attn_beam_cut attn_beam_cut_of(int64_t rows, int V, int size) {
    const int64_t most = (V + 4 * ATTN_BEAM_STEP(size) - 1) / (4 * ATTN_BEAM_STEP(size)); /* chunks of one step */
    int64_t chunks = (ATTN_BEAM_FILL + rows - 1) / rows;
    chunks = chunks < most ? chunks : most;
    const int64_t steps = (most + chunks - 1) / chunks;
    struct attn_beam_cut c = {(int)((most + steps - 1) / steps), (int)steps};
    return c;
}

/* The second launch takes the chunks' lists of K in segments, of whose first logits a thread holds up to eight. */
#define ATTN_BEAM_HELD 2048
ATTN_HD int attn_beam_segment(int lists, int K) {
    int seg = 1;
    while (seg < K && (int64_t)lists * ((K + seg - 1) / seg) > ATTN_BEAM_HELD)
        ++seg;
    return seg;
}

struct attn_beam_args {
    const void *logits;
    int64_t row; /* elements from row to row */
    const float *scores;
    const uint8_t *done;
    int done_token;
    int B, beams, V, K, chunks, steps;
    int seg, segments; /* logits of a segment, segments of an entry */
    struct attn_div by_lists, by_chunks, by_K; /* beams * chunks, chunks, K */
    uint64_t *keys; /* [rows][chunks][K], largest first */
    float *ms;      /* [rows][chunks][2]: m, the largest logit, and the sum of exp(x - m) */
    float *score;   /* [B][K] */
    int32_t *token, *parent;
};

#define ATTN_REORDER_GRID 0xffffff /* workgroups of 256 threads: a launch has less than 2^32 work-items */

struct attn_reorder_args {
    uint8_t *k, *v, *ks, *vs;
    int32_t *table;
    const int32_t *kv_len, *parent;
    int first, groups; /* of this launch */
    int beams, cols, pages, lgp, Hkv;
    int row, srow;             /* bytes of a row's elements and scales, in one of K and V */
    int data_wgs, scale_wgs;   /* workgroups per group for each of K and V */
    int table_wgs;
};

/* Workgroups of a group. */
ATTN_HD int attn_reorder_wgs(const struct attn_reorder_args *a) {
    return 2 * (a->data_wgs + a->scale_wgs) + a->table_wgs;
}

/* The parent of a group's member i, as a member of the group: itself where the entry names no other one. */
ATTN_HD int attn_parent_of(int entry, int first, int i, int beams) {
    const int64_t p = (int64_t)entry - first;
    return p >= 0 && p < beams ? (int)p : i;
}

#endif

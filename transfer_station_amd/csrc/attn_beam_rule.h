/* attn_beam_rule.h -- arguments and sizes of the beam search's kernels, shared by the kernels and the host layer. */
#ifndef ATTN_BEAM_RULE_H
#define ATTN_BEAM_RULE_H

#include <stdint.h>

#include "attn_paged_rule.h"

/* A row of logits is looked through in chunks, one workgroup of 256 threads each: 8192 elements, or 2048 where the
 * rows are too few to fill the GPU with those. A chunk leaves its K best and its maximum and sum of exponentials. */
#define ATTN_BEAM_CHUNK 8192
#define ATTN_BEAM_CHUNK_SMALL 2048
#define ATTN_BEAM_FILL 1024 /* workgroups */

ATTN_HD int attn_beam_chunk_of(int64_t rows, int V) {
    return rows * ((V + ATTN_BEAM_CHUNK - 1) / ATTN_BEAM_CHUNK) < ATTN_BEAM_FILL ? ATTN_BEAM_CHUNK_SMALL
                                                                               : ATTN_BEAM_CHUNK;
}

struct attn_beam_args {
    const void *logits;
    int64_t row; /* elements from row to row */
    const float *scores;
    const uint8_t *done;
    int done_token;
    int B, beams, V, K, chunks;
    uint64_t *keys; /* [rows][chunks][K], largest first */
    float *ms;      /* [rows][chunks][2]: maximum, sum of exp(x - maximum) */
    float *score;   /* [B][K] */
    int32_t *token, *parent;
};

struct attn_reorder_args {
    uint8_t *k, *v, *ks, *vs;
    int32_t *table;
    const int32_t *kv_len, *parent;
    int groups, beams, cols, pages, lgp, Hkv;
    int row, srow;             /* bytes of a row's elements and scales, in one of K and V */
    int data_wgs, scale_wgs;   /* workgroups per group for each of K and V */
    int table_wgs;
};

/* The parent of a group's member i, as a member of the group: itself where the entry names no other one. */
ATTN_HD int attn_parent_of(int entry, int first, int i, int beams) {
    const int64_t p = (int64_t)entry - first;
    return p >= 0 && p < beams ? (int)p : i;
}

#endif

/* attn_beam.c -- C host layer of beam search: attn_beam_select and attn_kv_reorder.
 *
 * Checks the arguments (a bad one aborts with a message, as in attn_flash) and launches on the calling thread's
 * stream. Device memory is not read here.
 */
#define __HIP_PLATFORM_AMD__ 1
#include "attn_flash.h"

#include "attn_beam_rule.h"

#include <hip/hip_runtime_api.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

int attn_hip_launch_beam(const struct attn_beam_args *a, int bits, void *stream);
int attn_hip_launch_reorder(const struct attn_reorder_args *a, void *stream);

static void beam_fail(const char *who, const char *what) {
    fprintf(stderr, "%s: %s\n", who, what);
    abort();
}

static void beam_hip_check(int err, const char *who) {
    if (err != 0) {
        fprintf(stderr, "%s: HIP error %d (%s)\n", who, err, hipGetErrorString((hipError_t)err));
        abort();
    }
}

static int misaligned(const void *p, size_t to) { return !p || (uintptr_t)p % to != 0; }

/* Everything but the outputs; how the rows are cut. */
static struct attn_beam_cut beam_check(const char *who, const struct attn_beams *c) {
    if (!c)
        beam_fail(who, "the beams must be non-NULL");
    if (c->bits != 16 && c->bits != 32)
        beam_fail(who, "bits must be 16 (bf16 logits) or 32 (fp32)");
    if (c->B < 1 || c->beams < 1 || c->beams > ATTN_BEAMS_MAX || c->K < 1 || c->K > ATTN_BEAM_K_MAX || c->V < 1 ||
        c->V > ATTN_BEAM_V_MAX)
        beam_fail(who, "need B >= 1, beams in [1, 256], K in [1, 64] and V in [1, 2^20]");
    if ((int64_t)c->B * c->beams > 1 << 20)
        beam_fail(who, "need B * beams <= 2^20");
    if (misaligned(c->logits, c->bits / 8) || c->row < c->V)
        beam_fail(who, "logits must be a device pointer aligned to its elements, row at least V");
    if (misaligned(c->scores, 4))
        beam_fail(who, "scores must be a device pointer to B * beams floats");
    if (c->done && (c->done_token < 0 || c->done_token >= c->V))
        beam_fail(who, "done_token must be in [0, V)");
    return attn_beam_cut_of((int64_t)c->B * c->beams, c->V, c->bits / 8);
}

static size_t keys_bytes(const struct attn_beams *c, int chunks) {
    return (size_t)c->B * c->beams * chunks * c->K * sizeof(uint64_t);
}

size_t attn_beam_scratch_bytes(const struct attn_beams *c) {
    const struct attn_beam_cut cut = beam_check("attn_beam_scratch_bytes", c);
    return keys_bytes(c, cut.chunks) + (size_t)c->B * c->beams * cut.chunks * 2 * sizeof(float);
}

void attn_beam_select(const struct attn_beams *c, float *score, int32_t *token, int32_t *parent, void *scratch) {
    static const char *who = "attn_beam_select";
    const struct attn_beam_cut cut = beam_check(who, c);
    if (misaligned(score, 4) || misaligned(token, 4) || misaligned(parent, 4))
        beam_fail(who, "score, token and parent must be device pointers to B * K values");
    if (score == c->scores || token == parent || (void *)score == (void *)token || (void *)score == (void *)parent)
        beam_fail(who, "score, token, parent and scores must be four arrays");
    if (misaligned(scratch, ATTN_SCRATCH_ALIGN))
        beam_fail(who, "scratch must be non-NULL and ATTN_SCRATCH_ALIGN-aligned");
    struct attn_beam_args a;
    memset(&a, 0, sizeof a);
    a.logits = c->logits, a.row = c->row, a.scores = c->scores, a.done = c->done, a.done_token = c->done_token;
    a.B = c->B, a.beams = c->beams, a.V = c->V, a.K = c->K, a.chunks = cut.chunks, a.steps = cut.steps;
    a.seg = attn_beam_segment(c->beams * cut.chunks, c->K);
    a.segments = c->beams * cut.chunks * ((c->K + a.seg - 1) / a.seg);
    a.by_lists = attn_div_of(c->beams * cut.chunks), a.by_chunks = attn_div_of(cut.chunks), a.by_K = attn_div_of(c->K);
    a.keys = (uint64_t *)scratch;
    a.ms = (float *)((char *)scratch + keys_bytes(c, a.chunks));
    a.score = score, a.token = token, a.parent = parent;
    beam_hip_check(attn_hip_launch_beam(&a, c->bits, attn_flash_get_stream()), who);
}

void attn_kv_reorder(const struct attn_kv_cache *c, const int32_t *parent, int beams, int tables) {
    static const char *who = "attn_kv_reorder";
    if (!c)
        beam_fail(who, "the cache must be non-NULL");
    if (c->bits != ATTN_KV_BF16 && c->bits != ATTN_KV_FP4)
        beam_fail(who, "bits must be ATTN_KV_BF16 (16) or ATTN_KV_FP4 (4)");
    if (c->bits == ATTN_KV_BF16 ? c->D < 16 || c->D > ATTN_D_MAX || c->D % 16 != 0
                                : c->D != 64 && c->D != 128 && c->D != 256)
        beam_fail(who, "a bf16 cache needs D % 16 == 0 and D in [16, 256], a 4-bit one D of 64, 128 or 256");
    if (c->page < ATTN_KV_PAGE_MIN || c->page > ATTN_KV_PAGE_MAX || (c->page & (c->page - 1)) != 0)
        beam_fail(who, "page must be a power of two in [16, 256]");
    if (c->B < 1 || c->Hkv < 1 || c->pages < 1 || c->table_cols < 1 || (int64_t)c->B * c->Hkv > 1 << 20 ||
        (int64_t)c->table_cols * c->page > 1 << 30)
        beam_fail(who, "need B, Hkv, pages and table_cols of at least 1, B * Hkv <= 2^20 and rows of 2^30 tokens at "
                       "most");
    if (beams < 1 || beams > ATTN_REORDER_MAX || c->B % beams != 0)
        beam_fail(who, "need beams in [1, 32] and B % beams == 0");
    if (misaligned(c->k, 16) || misaligned(c->v, 16) ||
        (c->bits == ATTN_KV_FP4 && (misaligned(c->k_scale, 16) || misaligned(c->v_scale, 16))))
        beam_fail(who, "k and v, and a 4-bit cache's scales, must be 16-byte aligned device pointers");
    if (misaligned(c->table, 4) || misaligned(c->kv_len, 4) || misaligned(parent, 4))
        beam_fail(who, "table, kv_len and parent must be device pointers to int32");
    if ((int64_t)c->Hkv * c->page * c->D > 1 << 29)
        beam_fail(who, "a page of all heads has at most 2^29 elements");
    struct attn_reorder_args a;
    memset(&a, 0, sizeof a);
    a.k = c->k, a.v = c->v, a.ks = c->k_scale, a.vs = c->v_scale;
    a.table = (int32_t *)(uintptr_t)c->table; /* the one call that writes it */
    a.kv_len = c->kv_len, a.parent = parent;
    a.beams = beams, a.cols = c->table_cols, a.pages = c->pages, a.Hkv = c->Hkv;
    while (1 << a.lgp < c->page)
        ++a.lgp;
    a.row = c->bits == ATTN_KV_FP4 ? c->D / 2 : 2 * c->D;
    a.srow = c->bits == ATTN_KV_FP4 ? c->D / 32 : 0;
    a.data_wgs = (c->Hkv * ((a.row << a.lgp) / 16) + 255) / 256;
    a.scale_wgs = (c->Hkv * ((a.srow << a.lgp) / 16) + 255) / 256;
    a.table_wgs = !tables ? 0 : c->table_cols <= 4096 ? (c->table_cols + 255) / 256 : 16;
    /* Groups past what one launch has workgroups for take further launches. A group has 2^19 workgroups and some at most:
     * a page of all heads has at most 2^29 elements. */
    const int groups = c->B / beams, most = ATTN_REORDER_GRID / attn_reorder_wgs(&a);
    for (a.first = 0; a.first < groups; a.first += a.groups) {
        a.groups = groups - a.first < most ? groups - a.first : most;
        beam_hip_check(attn_hip_launch_reorder(&a, attn_flash_get_stream()), who);
    }
}

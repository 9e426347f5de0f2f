/* attn_cross.c -- C host layer of cross attention: attn_cross, attn_cross_grad and their workspaces.
 *
 * Checks the arguments (a bad one aborts with a message, as in attn_flash), cuts the work and launches it on the
 * calling thread's stream. Starts and lengths lie in device memory and are not read here: the kernels hold every use
 * of them inside its tensor (attn_cross_rule.h).
 */
#define __HIP_PLATFORM_AMD__ 1
#include "attn_flash.h"

#include "attn_cross_rule.h"
#include "attn_decode_rule.h"

#include <hip/hip_runtime_api.h>
#include <math.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

int attn_hip_launch_cross(const struct attn_cross_args *a, const struct attn_cross_cut *cut, int max_q, void *stream);
int attn_hip_launch_cross_grad(const struct attn_cross_args *a, const struct attn_cross_cut *cut, int kv, int most,
                               void *stream);
void attn_hip_plan_begin(char *buf, size_t len);
long attn_hip_plan_end(void);

static void cross_fail(const char *who, const char *what) {
    fprintf(stderr, "%s: %s\n", who, what);
    abort();
}

static void cross_hip_check(int err, const char *who) {
    if (err != 0) {
        fprintf(stderr, "%s: HIP error %d (%s)\n", who, err, hipGetErrorString((hipError_t)err));
        abort();
    }
}

static int misaligned(const void *p, size_t to) { return !p || (uintptr_t)p % to != 0; }

static int bound_of(const struct attn_spans *s) { return s->max < s->T ? s->max : s->T; }

static void cross_check_spans(const char *who, const char *what, const struct attn_spans *s) {
    if (misaligned(s->start, 4) || (s->len && misaligned(s->len, 4)) || s->T < 1 || s->T > 1 << 30 || s->max < 1) {
        fprintf(stderr, "%s: %s needs device pointers to int32, T in [1, 2^30] and max >= 1\n", who, what);
        abort();
    }
}

static void cross_check_call(const char *who, const struct attn_cross_call *c) {
    if (!c)
        cross_fail(who, "the call must be non-NULL");
    if (c->D < 16 || c->D > ATTN_D_MAX || c->D % 16 != 0)
        cross_fail(who, "need D % 16 == 0 and D in [16, 256]");
    if (c->B < 1 || c->Hkv < 1 || c->Hq < 1 || c->Hq % c->Hkv != 0)
        cross_fail(who, "need B >= 1, Hkv >= 1, Hq >= 1 and Hq % Hkv == 0");
    if ((int64_t)c->B * c->Hkv > 1 << 20)
        cross_fail(who, "need B * Hkv <= 2^20");
    cross_check_spans(who, "q", &c->q);
    cross_check_spans(who, "k", &c->k);
    if ((int64_t)c->q.T * c->Hq > 1 << 30 || (int64_t)c->k.T * c->Hkv > 1 << 30)
        cross_fail(who, "need q.T * Hq <= 2^30 and k.T * Hkv <= 2^30");
    if (!(c->scale == 0.f || (c->scale >= 1e-6f && c->scale <= 1e6f)))
        cross_fail(who, "scale must be 0 (1/sqrt(D)) or in [1e-6, 1e6]");
    if ((int64_t)c->B * c->Hkv * ((int64_t)bound_of(&c->q) * (c->Hq / c->Hkv) / 16 + 8) > 1 << 30 ||
        (int64_t)c->B * c->Hkv * ((int64_t)c->k.T / ATTN_CROSS_KEYS + 8) > 1 << 30)
        cross_fail(who, "B, the heads, q.max and k.T ask for too many tiles");
}

static void cross_check_rows(const char *who, const char *what, const struct attn_rows *r, int D) {
    if (!r || misaligned(r->data, 16) || r->head < 0 || r->token % 8 != 0 || r->head % 8 != 0 || r->token < D ||
        r->token > ATTN_TOKEN_MAX) {
        fprintf(stderr,
                "%s: %s needs a 16-byte aligned device pointer, strides that are multiples of 8 and a token stride in "
                "[D, 2^22]\n",
                who, what);
        abort();
    }
}

/* What a call writes: heads of one row must not share elements. */
static void cross_check_out(const char *who, const char *what, const struct attn_rows *r, int D, int heads) {
    cross_check_rows(who, what, r, D);
    if (heads > 1 && r->head < D) {
        fprintf(stderr, "%s: the heads of %s must not overlap\n", who, what);
        abort();
    }
}

static int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

/* Tiles of a sequence and kv head that the launch has workgroups for; these go on to any that are left (tile += tps). */
static int tiles_at_once(int64_t groups, int64_t tiles) {
    const int64_t most = ATTN_CROSS_MAX_GRID / groups; /* 15 and more: groups <= 2^20 */
    return (int)(tiles < most ? tiles : most);
}

/* Parts so that `base` workgroups become up to `target`, which run at once, each of `least` units or more of `total`. */
static struct attn_cross_cut cross_cut(int64_t groups, int tps, int64_t total, int64_t least, int64_t target,
                                       int64_t most, int step) {
    struct attn_cross_cut cut;
    memset(&cut, 0, sizeof cut);
    const int64_t base = groups * tps;
    int64_t n = target / base, by_len = total / least;
    n = n < by_len ? n : by_len;
    n = n < most ? n : most;
    n = n < ATTN_CROSS_MAX_PARTS ? n : ATTN_CROSS_MAX_PARTS;
    n = n < 2 ? 1 : n;
    cut.share = (int)(ceil_div(ceil_div(total, n), step) * step);
    cut.nsplit = cut.parts = (int)n;
    cut.tps = tps;
    cut.grid = (long)(base * n);
    return cut;
}

/* Few rows of a kv head (up to 32: single tokens, beams) have a kernel of their own, and its workgroups equal shares of
 * all sequences' states (attn_quota), whatever sequences they cut, where there is enough to share: a merge costs 4 us.
 * Measured, whole sequences -> shares (of 256 workgroups; with 512 they were slower): 64 sequences of up to 8192 states,
 * 8 kv heads, D = 128, 306 -> 268 us; 16 inputs' beams over up to 1500 states, 16 heads, D = 64, 22 -> 27.
 * Four kv heads in a workgroup, a wave each, read 1 KB of neighbouring heads of a row at a time, not 256 bytes. Against four
 * waves per head: the 64 sequences 268 -> 237, 32 of 4096 at D = 256 175 -> 167; one sequence of 32768 states, whose waves
 * then have four times the parts, 31 -> 48, the beams 22 -> 25. */
static struct attn_cross_cut rows_cut(const struct attn_cross_call *c, int64_t R, int64_t slots) {
    struct attn_cross_cut cut;
    memset(&cut, 0, sizeof cut);
    const int64_t groups = (int64_t)c->B * c->Hkv, keys = bound_of(&c->k), bytes = groups * keys * c->D * 4;
    cut.rows16 = R > 16 && c->D <= 128 ? 2 : 1;
    cut.quads = c->Hkv % 4 == 0 && bytes >= ATTN_CROSS_TEAMS * (2L << 20);
    cut.tps = (int)ceil_div(R, 16 * cut.rows16);
    cut.nsplit = (int)(slots < ATTN_CROSS_MAX_PARTS ? slots : ATTN_CROSS_MAX_PARTS);
    cut.share = 1;
    const int64_t lines = groups / (cut.quads ? 4 : 1), units = ceil_div(keys, 128) * lines;
    int64_t teams = ceil_div(ATTN_CROSS_TEAMS, cut.tps);
    teams = teams < units ? teams : units;
    if (cut.nsplit < 2 || teams < 2 || (lines * cut.tps >= ATTN_CROSS_TEAMS && bytes < ATTN_CROSS_TEAMS * (1L << 20))) {
        cut.nsplit = 1;
        teams = 0;
    }
    cut.teams = (int)teams;
    cut.parts = (int)(teams ? ceil_div(teams, lines) + 1 : 1);
    cut.grid = (long)((teams ? teams : lines) * cut.tps);
    return cut;
}

static struct attn_cross_cut forward_cut(const struct attn_cross_call *c) {
    const int64_t R = (int64_t)bound_of(&c->q) * (c->Hq / c->Hkv);
    const int64_t slots = ATTN_SLOTS / ((int64_t)c->q.T * c->Hq);
    if (R <= 32)
        return rows_cut(c, R, slots);
    const int64_t groups = (int64_t)c->B * c->Hkv;
    return cross_cut(groups, tiles_at_once(groups, ceil_div(R, ATTN_CROSS_ROWS)), bound_of(&c->k), 256, 512, slots,
                     ATTN_CROSS_KEY_STEP);
}

static int is_fine(const struct attn_cross_call *c) {
    const int64_t rows = (int64_t)c->B * c->Hq * bound_of(&c->q); /* the product with the states may pass 64 bits */
    return rows <= ATTN_CROSS_FINE && rows * bound_of(&c->k) <= ATTN_CROSS_FINE;
}

static struct attn_cross_cut dq_cut(const struct attn_cross_call *c) {
    const int64_t R = (int64_t)bound_of(&c->q) * (c->Hq / c->Hkv), groups = (int64_t)c->B * c->Hkv;
    struct attn_cross_cut cut =
        cross_cut(groups, tiles_at_once(groups, ceil_div(R, ATTN_CROSS_ROWS)), bound_of(&c->k), 256,
                  c->D <= 128 ? 512 : 256, ATTN_CROSS_GRAD_FLOATS / ((int64_t)c->q.T * c->Hq * c->D), ATTN_CROSS_KEY_STEP);
    cut.fine = is_fine(c);
    return cut;
}

/* Where tiles of states are no more than the CUs and each has rows enough, eight waves share one, as two teams that take its
 * rows in turn: partial gradients cost 8 D bytes per state and part, written and read again. One team -> two: 4096 rows of
 * 40 heads over 77 states, D = 64, 31.5 -> 28.4 us with their sum; 1500 of 16 heads on 4 over 300, D = 128, 42 -> 39; 37
 * rows of 24 heads over 50 states, which keep one, 6.0 -> 8.0. Calls that take P and dS in two parts have one team, and the
 * parts of two: both gradient kernels of 32 single rows of 64 heads on 8 over 128 states, D = 64, 22.6 us (with the parts of
 * one team 38.2; 19.8 with two teams, and P and dS in one part), 4 x 2048 rows of 10 heads over 20 37.6 (36.4, 32.5). */
static struct attn_cross_cut dkv_cut(const struct attn_cross_call *c) {
    const int64_t groups = (int64_t)c->B * c->Hkv, tps = ceil_div(bound_of(&c->k), ATTN_CROSS_KEYS);
    const int64_t steps = ceil_div(bound_of(&c->q), ATTN_CROSS_STEP) * (c->Hq / c->Hkv);
    const int fine = is_fine(c), shared = c->D <= 128 && groups * tps <= 256 && groups * tps * steps >= 2048;
    const int row_teams = shared && !fine ? 2 : 1;
    struct attn_cross_cut cut =
        cross_cut(groups, tiles_at_once(groups, tps), steps, shared ? 4 : 2, shared || c->D > 128 ? 256 : 512,
                  ATTN_CROSS_GRAD_FLOATS / ((int64_t)c->k.T * c->Hkv * c->D * 2), row_teams);
    cut.row_teams = row_teams;
    cut.fine = fine;
    return cut;
}

size_t attn_cross_scratch_bytes(const struct attn_cross_call *c) {
    cross_check_call("attn_cross_scratch_bytes", c);
    return attn_flash_scratch_bytes(c->D, ATTN_BK_DEFAULT);
}

static size_t delta_bytes(const struct attn_cross_call *c) {
    return ((size_t)c->q.T * c->Hq * sizeof(float) + 255) / 256 * 256;
}

size_t attn_cross_grad_scratch_bytes(const struct attn_cross_call *c) {
    cross_check_call("attn_cross_grad_scratch_bytes", c);
    const struct attn_cross_cut dq = dq_cut(c), dkv = dkv_cut(c);
    const size_t q = dq.nsplit > 1 ? (size_t)dq.nsplit * c->q.T * c->Hq * c->D : 0;
    const size_t kv = dkv.nsplit > 1 ? (size_t)dkv.nsplit * c->k.T * c->Hkv * c->D * 2 : 0;
    return delta_bytes(c) + (q > kv ? q : kv) * sizeof(float);
}

static struct attn_cross_args cross_args(const struct attn_cross_call *c) {
    struct attn_cross_args a;
    memset(&a, 0, sizeof a);
    a.scale = c->scale != 0.f ? c->scale : (float)(1.0 / sqrt((double)c->D));
    a.c = (float)((c->scale != 0.f ? (double)c->scale : 1.0 / sqrt((double)c->D)) * 1.4426950408889634);
    a.q_start = c->q.start, a.k_start = c->k.start;
    a.q_is_len = c->q.len != NULL, a.k_is_len = c->k.len != NULL;
    a.q_second = c->q.len ? c->q.len : c->q.start + 1;
    a.k_second = c->k.len ? c->k.len : c->k.start + 1;
    a.B = c->B, a.Tq = c->q.T, a.Tk = c->k.T, a.Hq = c->Hq, a.Hkv = c->Hkv, a.g = c->Hq / c->Hkv, a.D = c->D;
    return a;
}

/* walk: how many rows, at most, a tile of this launch walks. */
static void set_cut(struct attn_cross_args *a, const struct attn_cross_cut *cut, int walk) {
    a->tps = cut->tps, a->nsplit = cut->nsplit, a->share = cut->share, a->wgs = (int)cut->grid;
    a->teams = cut->teams, a->row_teams = cut->row_teams, a->Hkv_wg = cut->quads ? a->Hkv / 4 : a->Hkv;
    a->by_tps = attn_div_of(a->tps), a->by_B = attn_div_of(a->B), a->by_heads = attn_div_of(a->Hkv);
    a->by_bh = attn_div_of(a->B * a->Hkv);
    a->by_length = a->B > 1 && a->B <= ATTN_CROSS_RANKED && cut->grid > ATTN_CROSS_AT_ONCE && walk >= ATTN_CROSS_LONG;
    a->by_hq = attn_div_of(a->Hq), a->by_g = attn_div_of(a->g), a->by_gwg = attn_div_of(a->Hq / a->Hkv_wg);
}

static void cross_run(const char *who, const struct attn_cross_call *c, const struct attn_rows *q,
                      const struct attn_rows *k, const struct attn_rows *v, const struct attn_rows *o, float *lse,
                      void *scratch) {
    struct attn_cross_args a = cross_args(c);
    const struct attn_cross_cut cut = forward_cut(c);
    set_cut(&a, &cut, bound_of(&c->k));
    a.q = (const uint16_t *)q->data, a.q_tok.n = (int32_t)q->token, a.q_head = q->head;
    a.k = (const uint16_t *)k->data, a.k_tok.n = (int32_t)k->token, a.k_head = k->head;
    a.v = (const uint16_t *)v->data, a.v_tok.n = (int32_t)v->token, a.v_head = v->head;
    a.o = (uint16_t *)o->data, a.o_tok.n = (int32_t)o->token, a.o_head = o->head;
    a.lse = lse;
    /* the scratch of attn_flash: m, l and acc[D] of ATTN_SLOTS partials, each on 256 bytes */
    a.pm = (float *)scratch;
    a.pl = a.pm + ATTN_SLOTS;
    a.pacc = a.pl + ATTN_SLOTS;
    cross_hip_check(attn_hip_launch_cross(&a, &cut, bound_of(&c->q), attn_flash_get_stream()), who);
}

void attn_cross(const struct attn_cross_call *c, const struct attn_rows *q, const struct attn_rows *k,
                const struct attn_rows *v, const struct attn_rows *o, float *lse, void *scratch) {
    static const char *who = "attn_cross";
    cross_check_call(who, c);
    cross_check_rows(who, "q", q, c->D);
    cross_check_rows(who, "k", k, c->D);
    cross_check_rows(who, "v", v, c->D);
    cross_check_out(who, "o", o, c->D, c->Hq);
    if (o->data == q->data || o->data == k->data || o->data == v->data)
        cross_fail(who, "o must not be q, k or v");
    if (lse && misaligned(lse, 4))
        cross_fail(who, "lse must be NULL or a device pointer to floats");
    if (misaligned(scratch, ATTN_SCRATCH_ALIGN))
        cross_fail(who, "scratch must be non-NULL and ATTN_SCRATCH_ALIGN-aligned");
    cross_run(who, c, q, k, v, o, lse, scratch);
}

static void grad_run(const char *who, const struct attn_cross_call *c, const struct attn_rows *const *in,
                     const float *lse, const struct attn_rows *const *out, void *scratch) {
    struct attn_cross_args a = cross_args(c);
    a.q = (const uint16_t *)in[0]->data, a.q_tok.n = (int32_t)in[0]->token, a.q_head = in[0]->head;
    a.k = (const uint16_t *)in[1]->data, a.k_tok.n = (int32_t)in[1]->token, a.k_head = in[1]->head;
    a.v = (const uint16_t *)in[2]->data, a.v_tok.n = (int32_t)in[2]->token, a.v_head = in[2]->head;
    a.o = (uint16_t *)in[3]->data, a.o_tok.n = (int32_t)in[3]->token, a.o_head = in[3]->head; /* read */
    a.go = (const uint16_t *)in[4]->data, a.go_tok.n = (int32_t)in[4]->token, a.go_head = in[4]->head;
    a.dq = (uint16_t *)out[0]->data, a.dq_tok.n = (int32_t)out[0]->token, a.dq_head = out[0]->head;
    a.dk = (uint16_t *)out[1]->data, a.dk_tok.n = (int32_t)out[1]->token, a.dk_head = out[1]->head;
    a.dv = (uint16_t *)out[2]->data, a.dv_tok.n = (int32_t)out[2]->token, a.dv_head = out[2]->head;
    a.lse = (float *)(uintptr_t)lse; /* read */
    a.delta = (float *)scratch;
    a.pacc = (float *)((char *)scratch + delta_bytes(c));
    const struct attn_cross_cut dq = dq_cut(c), dkv = dkv_cut(c);
    set_cut(&a, &dq, bound_of(&c->k));
    cross_hip_check(attn_hip_launch_cross_grad(&a, &dq, 0, bound_of(&c->q), attn_flash_get_stream()), who);
    set_cut(&a, &dkv, bound_of(&c->q));
    cross_hip_check(attn_hip_launch_cross_grad(&a, &dkv, 1, bound_of(&c->k), attn_flash_get_stream()), who);
}

void attn_cross_grad(const struct attn_cross_call *c, const struct attn_rows *q, const struct attn_rows *k,
                     const struct attn_rows *v, const struct attn_rows *o, const float *lse,
                     const struct attn_rows *d_o, const struct attn_rows *dq, const struct attn_rows *dk,
                     const struct attn_rows *dv, void *scratch) {
    static const char *who = "attn_cross_grad";
    static const char *const names[] = {"q", "k", "v", "o", "d_o", "dq", "dk", "dv"};
    const struct attn_rows *const all[] = {q, k, v, o, d_o, dq, dk, dv};
    cross_check_call(who, c);
    for (int i = 0; i < 5; ++i)
        cross_check_rows(who, names[i], all[i], c->D);
    for (int i = 5; i < 8; ++i)
        cross_check_out(who, names[i], all[i], c->D, i == 5 ? c->Hq : c->Hkv);
    for (int i = 5; i < 8; ++i)
        for (int j = 0; j < i; ++j)
            if (all[i]->data == all[j]->data)
                cross_fail(who, "dq, dk and dv must be none of the other tensors");
    if (misaligned(lse, 4))
        cross_fail(who, "lse must be a device pointer to floats");
    if (misaligned(scratch, ATTN_SCRATCH_ALIGN))
        cross_fail(who, "scratch must be non-NULL and ATTN_SCRATCH_ALIGN-aligned");
    grad_run(who, c, all, lse, all + 5, scratch);
}

int attn_cross_plan(const struct attn_cross_call *c, int grad, char *buf, size_t len) {
    static const char *who = "attn_cross_plan";
    const struct attn_rows r = {(void *)(uintptr_t)256, 256, 256};
    const struct attn_rows *const all[] = {&r, &r, &r, &r, &r, &r, &r, &r};
    cross_check_call(who, c);
    if (!buf || len == 0)
        cross_fail(who, "buf must be non-NULL and len above 0");
    attn_hip_plan_begin(buf, len);
    if (grad)
        grad_run(who, c, all, (const float *)r.data, all, r.data);
    else
        cross_run(who, c, &r, &r, &r, &r, NULL, r.data);
    const long n = attn_hip_plan_end();
    return n < 0 || n > 0x7fffffffL ? -1 : (int)n;
}

/* attn_paged.c -- C host layer of the paged KV cache: attn_paged, attn_kv_append and attn_kv_read.
 *
 * Checks the arguments (a bad one aborts with a message, as in attn_flash), cuts the work and launches it
 * on the calling thread's stream. What lies in device memory -- the table, the lengths, the starts -- is
 * not read here: the kernels hold every use of it inside its tensor (attn_paged_rule.h).
 */
#define __HIP_PLATFORM_AMD__ 1
#include "attn_flash.h"

#include "attn_decode_rule.h"
#include "attn_paged_cut.h"
#include "attn_paged_rule.h"

#include <hip/hip_runtime_api.h>
#include <math.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

int attn_hip_launch_paged(const struct attn_paged_args *a, const struct attn_paged_cut *cut, int bits,
                          void *stream);
int attn_hip_launch_kv_append(const struct attn_kv_args *a, int bits, int pairs, void *stream);
int attn_hip_launch_kv_read(const struct attn_kv_args *a, int bits, void *stream);
void attn_hip_plan_begin(char *buf, size_t len);
long attn_hip_plan_end(void);

static void paged_fail(const char *who, const char *what) {
    fprintf(stderr, "%s: %s\n", who, what);
    abort();
}

static void paged_hip_check(int err, const char *who) {
    if (err != 0) {
        fprintf(stderr, "%s: HIP error %d (%s)\n", who, err, hipGetErrorString((hipError_t)err));
        abort();
    }
}

static int misaligned(const void *p, size_t to) { return !p || (uintptr_t)p % to != 0; }

/* The cache's description; returns log2(page). */
static int paged_check_cache(const char *who, const struct attn_kv_cache *c, int T) {
    if (!c)
        paged_fail(who, "the cache must be non-NULL");
    if (c->bits != ATTN_KV_BF16 && c->bits != ATTN_KV_FP4)
        paged_fail(who, "bits must be ATTN_KV_BF16 (16) or ATTN_KV_FP4 (4)");
    if (c->bits == ATTN_KV_BF16 && (c->D < 16 || c->D > ATTN_D_MAX || c->D % 16 != 0))
        paged_fail(who, "a bf16 cache needs D % 16 == 0 and D in [16, 256]");
    if (c->bits == ATTN_KV_FP4 && c->D != 64 && c->D != 128 && c->D != 256)
        paged_fail(who, "a 4-bit cache needs D of 64, 128 or 256");
    if (c->page < ATTN_KV_PAGE_MIN || c->page > ATTN_KV_PAGE_MAX || (c->page & (c->page - 1)) != 0)
        paged_fail(who, "page must be a power of two in [16, 256]");
    if (c->B < 1 || c->Hkv < 1 || c->pages < 1 || c->table_cols < 1)
        paged_fail(who, "need B >= 1, Hkv >= 1, pages >= 1 and table_cols >= 1");
    if ((int64_t)c->B * c->Hkv > 1 << 20)
        paged_fail(who, "need B * Hkv <= 2^20");
    if ((int64_t)c->table_cols * c->page > 1 << 30)
        paged_fail(who, "a table row holds at most 2^30 tokens");
    if (((int64_t)c->table_cols * c->page + 127) / 128 * c->B * c->Hkv > 0x7fffffff)
        paged_fail(who, "B * Hkv table rows hold at most 2^38 tokens");
    if (T < 1 || T > 1 << 30)
        paged_fail(who, "need T in [1, 2^30]");
    if (misaligned(c->k, 16) || misaligned(c->v, 16))
        paged_fail(who, "k and v must be 16-byte aligned device pointers");
    if (c->bits == ATTN_KV_FP4 && (misaligned(c->k_scale, 16) || misaligned(c->v_scale, 16)))
        paged_fail(who, "a 4-bit cache's k_scale and v_scale must be 16-byte aligned device pointers");
    if (misaligned(c->table, 4) || misaligned(c->kv_len, 4) || misaligned(c->q_start, 4))
        paged_fail(who, "table, kv_len and q_start must be device pointers to int32");
    int lgp = 4;
    while (1 << lgp < c->page)
        ++lgp;
    return lgp;
}

static void paged_check_rows(const char *who, const char *what, const struct attn_rows *r) {
    if (!r || misaligned(r->data, 16) || r->token < 0 || r->head < 0 || r->token % 8 != 0 ||
        r->head % 8 != 0) {
        fprintf(stderr,
                "%s: %s needs a 16-byte aligned device pointer and strides that are multiples of 8\n", who,
                what);
        abort();
    }
}

static void paged_check_heads(const char *who, const struct attn_kv_cache *c, int T, int Hq) {
    if (Hq < 1 || Hq % c->Hkv != 0)
        paged_fail(who, "need Hq >= 1 and Hq % Hkv == 0");
    if ((int64_t)T * Hq > 1 << 30)
        paged_fail(who, "need T * Hq <= 2^30");
}

/* Everything attn_paged checks but the tensors. */
static void paged_check_call(const char *who, const struct attn_kv_cache *c, int T, int Hq,
                             const struct attn_scores *sc, int max_q, int max_kv) {
    paged_check_cache(who, c, T);
    paged_check_heads(who, c, T, Hq);
    if (max_q < 1 || max_kv < 1)
        paged_fail(who, "need max_q >= 1 and max_kv >= 1");
    if (sc) {
        if (!(sc->scale == 0.f || (sc->scale >= 1e-6f && sc->scale <= 1e6f)))
            paged_fail(who, "scale must be 0 (1/sqrt(D)) or in [1e-6, 1e6]");
        if (!(sc->softcap == 0.f || (sc->softcap >= 1e-3f && sc->softcap <= 1e6f)))
            paged_fail(who, "softcap must be 0 (none) or in [1e-3, 1e6]");
        if (sc->slopes && misaligned(sc->slopes, 4))
            paged_fail(who, "slopes must be a device pointer to Hq floats");
    }
}

static void paged_run(const char *who, const struct attn_kv_cache *c, const struct attn_rows *q,
                      const struct attn_rows *o, int T, int Hq, int causal, const struct attn_scores *sc,
                      int max_q, int max_kv, void *scratch) {
    const double log2e = 1.4426950408889634;
    const double scale = sc && sc->scale != 0.f ? sc->scale : 1.0 / sqrt((double)c->D);
    struct attn_paged_args a;
    memset(&a, 0, sizeof a);
    a.q = (const uint16_t *)q->data;
    a.o = (uint16_t *)o->data;
    a.q_tok = q->token, a.q_head = q->head, a.o_tok = o->token, a.o_head = o->head;
    a.k = c->k, a.v = c->v, a.ks = c->k_scale, a.vs = c->v_scale;
    a.table = c->table, a.kv_len = c->kv_len, a.q_start = c->q_start;
    a.slopes = sc ? sc->slopes : NULL;
    a.B = c->B, a.T = T, a.Hq = Hq, a.Hkv = c->Hkv, a.D = c->D;
    a.cols = c->table_cols, a.pages = c->pages, a.causal = causal ? 1 : 0;
    while (16 << a.lgp < c->page)
        ++a.lgp;
    a.lgp += 4;
    a.c = (float)(scale * log2e);
    if (sc && sc->softcap != 0.f) {
        a.cap_in = (float)(2.0 * log2e * scale / sc->softcap);
        a.cap_out = (float)(sc->softcap * log2e);
    }
    if (max_kv > c->table_cols * c->page)
        max_kv = c->table_cols * c->page;
    const struct attn_paged_cut cut =
        attn_paged_cut_of(c->B, c->Hkv, Hq / c->Hkv, T, max_q, max_kv, c->D, c->bits, causal != 0);
    a.tps = cut.tps, a.nsplit = cut.nsplit, a.teams = cut.teams, a.deal = cut.deal, a.share = cut.share;
    /* the scratch of attn_flash: m, l and acc[D] of ATTN_SLOTS partials, each on 256 bytes */
    a.pm = (float *)scratch;
    a.pl = a.pm + ATTN_SLOTS;
    a.pacc = a.pl + ATTN_SLOTS;
    paged_hip_check(attn_hip_launch_paged(&a, &cut, c->bits, attn_flash_get_stream()), who);
}

void attn_paged(const struct attn_kv_cache *c, const struct attn_rows *q, const struct attn_rows *o, int T,
                int Hq, int causal, const struct attn_scores *sc, int max_q, int max_kv, void *scratch) {
    static const char *who = "attn_paged";
    paged_check_call(who, c, T, Hq, sc, max_q, max_kv);
    paged_check_rows(who, "q", q);
    paged_check_rows(who, "o", o);
    if (misaligned(scratch, ATTN_SCRATCH_ALIGN))
        paged_fail(who, "scratch must be non-NULL and ATTN_SCRATCH_ALIGN-aligned");
    if (o->data == q->data)
        paged_fail(who, "o must not be q");
    paged_run(who, c, q, o, T, Hq, causal, sc, max_q, max_kv, scratch);
}

int attn_paged_plan(const struct attn_kv_cache *c, int T, int Hq, int causal, const struct attn_scores *sc,
                    int max_q, int max_kv, char *buf, size_t len) {
    static const char *who = "attn_paged_plan";
    const struct attn_rows r = {(void *)(uintptr_t)256, 8, 8};
    paged_check_call(who, c, T, Hq, sc, max_q, max_kv);
    if (!buf || len == 0)
        paged_fail(who, "buf must be non-NULL and len above 0");
    attn_hip_plan_begin(buf, len);
    paged_run(who, c, &r, &r, T, Hq, causal, sc, max_q, max_kv, r.data);
    const long n = attn_hip_plan_end();
    return n < 0 || n > 0x7fffffffL ? -1 : (int)n;
}

/* What append and read share. */
static struct attn_kv_args kv_args(const struct attn_kv_cache *c, int lgp, int T, int max_q, int tpw,
                                   const struct attn_rows *k, const struct attn_rows *v) {
    struct attn_kv_args a;
    memset(&a, 0, sizeof a);
    a.k_tok = k->token, a.k_head = k->head, a.v_tok = v->token, a.v_head = v->head;
    a.ck = c->k, a.cv = c->v, a.cks = c->k_scale, a.cvs = c->v_scale;
    a.table = c->table, a.kv_len = c->kv_len, a.q_start = c->q_start;
    a.B = c->B, a.T = T, a.Hkv = c->Hkv, a.D = c->D;
    a.cols = c->table_cols, a.pages = c->pages, a.lgp = lgp;
    a.tblk = attn_kv_blocks(c->B, T, max_q, tpw);
    return a;
}

void attn_kv_append(const struct attn_kv_cache *c, const struct attn_rows *q, const struct attn_rows *q_out,
                    const struct attn_rows *k, const struct attn_rows *v, int T, int Hq, const float *rope,
                    int rope_rows, int rot, int pairs, int max_q) {
    static const char *who = "attn_kv_append";
    const int lgp = paged_check_cache(who, c, T);
    if (q) {
        paged_check_heads(who, c, T, Hq);
        paged_check_rows(who, "q", q);
        paged_check_rows(who, "q_out", q_out);
        if (q_out->data == q->data && (q_out->token != q->token || q_out->head != q->head))
            paged_fail(who, "q_out at q's address needs q's strides");
    } else if (q_out) {
        paged_fail(who, "q_out without q");
    }
    paged_check_rows(who, "k", k);
    paged_check_rows(who, "v", v);
    if (rot < 0 || rot > c->D || rot % 16 != 0)
        paged_fail(who, "rot must be a multiple of 16 in [0, D]");
    if (rot > 0 && (misaligned(rope, 16) || rope_rows < 1))
        paged_fail(who, "rope must be a 16-byte aligned device pointer to rope_rows >= 1 rows");
    if (max_q < 1)
        paged_fail(who, "need max_q >= 1");
    struct attn_kv_args a = kv_args(c, lgp, T, max_q, 1, k, v);
    if (q) {
        a.q = (const uint16_t *)q->data, a.q_out = (uint16_t *)q_out->data;
        a.q_tok = q->token, a.q_head = q->head, a.qo_tok = q_out->token, a.qo_head = q_out->head;
        a.Hq = Hq;
    }
    a.k = (const uint16_t *)k->data, a.v = (const uint16_t *)v->data;
    a.rope = rope, a.rope_rows = rope_rows, a.rot = rot;
    paged_hip_check(attn_hip_launch_kv_append(&a, c->bits, pairs != 0, attn_flash_get_stream()), who);
}

void attn_kv_read(const struct attn_kv_cache *c, const struct attn_rows *k, const struct attn_rows *v, int T,
                  int max_q) {
    static const char *who = "attn_kv_read";
    const int lgp = paged_check_cache(who, c, T);
    paged_check_rows(who, "k", k);
    paged_check_rows(who, "v", v);
    if (max_q < 1)
        paged_fail(who, "need max_q >= 1");
    struct attn_kv_args a = kv_args(c, lgp, T, max_q, 4, k, v);
    a.k_out = (uint16_t *)k->data, a.v_out = (uint16_t *)v->data;
    paged_hip_check(attn_hip_launch_kv_read(&a, c->bits, attn_flash_get_stream()), who);
}

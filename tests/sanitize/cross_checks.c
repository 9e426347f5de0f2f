/* cross_checks.c -- CPU-only sanitizer driver for cross attention's and beam search's host code (built and run by
 * tests/test_cross_host.py with -fsanitize=address,undefined).
 *
 * It runs the index arithmetic that the kernels use (attn_cross_rule.h) over bad starts and lengths, and the real host
 * layers (attn_cross.c, attn_beam.c) with stand-in launchers that walk the launch's workgroups with the kernels' own
 * arithmetic: every row (or state) and every unit of work of each sequence has to be taken exactly once, every row's
 * parts have to be written once, and what they write of the workspace goes into memory of exactly the size that the
 * library asks for. Prints "CROSS_CHECKS OK" and exits 0 when every check passes.
 */
#include "attn_beam_rule.h"
#include "attn_cross_rule.h"
#include "attn_decode_rule.h"
#include "attn_flash.h"

#include <hip/hip_runtime_api.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

static int failures, cut_calls, line_calls, team_calls;
#define CHECK(cond, ...)                                                                           \
    do {                                                                                           \
        if (!(cond)) {                                                                             \
            if (++failures < 20) {                                                                 \
                printf("FAIL %s:%d: ", __FILE__, __LINE__);                                        \
                printf(__VA_ARGS__);                                                               \
                printf("\n");                                                                      \
            }                                                                                      \
        }                                                                                          \
    } while (0)

const char *hipGetErrorString(hipError_t e) {
    (void)e;
    return "stand-in";
}
void attn_hip_plan_begin(char *buf, size_t len) { (void)buf, (void)len; }
long attn_hip_plan_end(void) { return 0; }
void *attn_flash_get_stream(void) { return NULL; }
size_t attn_flash_scratch_bytes(int D, int bk) {
    (void)bk;
    return sizeof(float) * ATTN_SLOTS * (size_t)(D + 2);
}

static uint64_t rng_state = 7;
static uint32_t rnd(void) {
    rng_state = rng_state * 6364136223846793005u + 1442695040888963407u;
    return (uint32_t)(rng_state >> 33);
}
static int pick(int lo, int hi) { return lo + (int)(rnd() % (uint32_t)(hi - lo + 1)); }

static struct attn_range q_of(const struct attn_cross_args *a, int b) {
    return attn_range_of(a->q_start[b], a->q_second[b], a->q_is_len, a->Tq);
}
static struct attn_range k_of(const struct attn_cross_args *a, int b) {
    return attn_range_of(a->k_start[b], a->k_second[b], a->k_is_len, a->Tk);
}

/* What the walk counts, by (sequence, row of a kv head's group or state, kv head): units of work that it took. */
struct seen {
    int64_t *work;  /* keys of a row, or steps of a state */
    int *parts;     /* written */
};

static struct attn_cut part_of(int total, int share, int nsplit, int step) {
    const struct attn_cut one = {1, total > 1 ? total : 1};
    return nsplit == 1 ? one : attn_cut_of(total, share, nsplit, step);
}

/* A partial row of `width` floats, and in the forward's workspace its maximum and sum. */
static void write_part(const struct attn_cross_args *a, int64_t slot, int width, int ml) {
    if (ml) {
        a->pm[slot] = 1.f;
        a->pl[slot] = 1.f;
    }
    a->pacc[slot * width] = 1.f;
    a->pacc[slot * width + width - 1] = 1.f;
}

/* One launch of tiles. kv: dK and dV, else rows over states. */
static void walk_tiles(const struct attn_cross_args *a, const struct attn_cross_cut *cut, int rows_wg, int kv, int ml) {
    ++cut_calls;
    for (int b0 = 0; b0 < a->B; ++b0)
        for (int u0 = 0; u0 < a->Hkv; ++u0) {
            const struct attn_range q = q_of(a, b0), k = k_of(a, b0);
            const int g = a->g, items = kv ? k.n : q.n * g;
            const int steps = (q.n + ATTN_CROSS_STEP - 1) / ATTN_CROSS_STEP * g, units = kv ? steps : k.n;
            const struct attn_cut c = part_of(units, a->share, a->nsplit, kv ? a->row_teams : ATTN_CROSS_KEY_STEP);
            CHECK(c.live >= 1 && c.live <= a->nsplit, "%d of %d parts", c.live, a->nsplit);
            int64_t *work = calloc((size_t)items + 1, sizeof *work);
            int *parts = calloc((size_t)items + 1, sizeof *parts);
            for (int wg = 0; wg < cut->grid; ++wg) {
                const struct attn_cross_place p = attn_cross_place_of(a, wg);
                CHECK(p.nth >= 0 && p.nth < a->B && p.u >= 0 && p.u < a->Hkv && p.sp >= 0 && p.sp < a->nsplit && p.tile >= 0 &&
                          p.tile < a->tps, "place of %d", wg);
                if (p.nth != b0 || p.u != u0 || p.sp >= c.live)
                    continue;
                const int t0 = p.sp * c.per < units ? p.sp * c.per : units;
                const int t1 = t0 + c.per < units ? t0 + c.per : units;
                for (int tile = p.tile; (int64_t)tile * rows_wg < items; tile += a->tps)
                    for (int r = tile * rows_wg; r < items && r < (tile + 1) * rows_wg; ++r) {
                        work[r] += t1 - t0;
                        ++parts[r];
                        if (c.live > 1) {
                            const int64_t tok = kv ? k.at + r : q.at + r / g;
                            const int64_t slot = kv ? tok * a->Hkv + u0 : tok * a->Hq + u0 * g + r % g;
                            write_part(a, slot * a->nsplit + p.sp, kv ? 2 * a->D : a->D, ml);
                        }
                    }
            }
            for (int r = 0; r < items; ++r)
                CHECK(work[r] == units && parts[r] == c.live, "%d: %lld of %d units, %d of %d parts", r,
                      (long long)work[r], units, parts[r], c.live);
            free(work);
            free(parts);
        }
}

static void walk_line(const struct attn_cross_args *a, const struct attn_cross_cut *cut) {
    const int rows_wg = 16 * cut->rows16, heads = a->Hkv / a->Hkv_wg, g = a->g;
    int total = 0, most = 0;
    line_calls += a->teams > 0;
    for (int b = 0; b < a->B; ++b) {
        const int n = attn_units(q_of(a, b).n, k_of(a, b).n);
        total += n;
        most = n > most ? n : most;
    }
    const int quota = a->teams ? attn_quota(total, most, a->Hkv_wg, a->teams, a->nsplit) : 1;
    int64_t *work = calloc((size_t)a->Tq * a->Hq, sizeof *work);
    int *parts = calloc((size_t)a->Tq * a->Hq, sizeof *parts);
    for (int wg = 0; wg < cut->grid; ++wg) {
        const int L = attn_xcd_order(wg, a->wgs), at = attn_div_by(L, a->by_tps), t0 = L - at * a->tps;
        int ug, b, off = 0, left = 1, pos0 = 0;
        if (a->teams) {
            if ((int64_t)at * quota >= (int64_t)total * a->Hkv_wg)
                continue;
            pos0 = at * quota;
            left = quota < total * a->Hkv_wg - pos0 ? quota : total * a->Hkv_wg - pos0;
            ug = pos0 / total;
            int before = 0;
            for (b = 0; before + attn_units(q_of(a, b).n, k_of(a, b).n) <= pos0 - ug * total; ++b)
                before += attn_units(q_of(a, b).n, k_of(a, b).n);
            off = pos0 - ug * total - before;
        } else {
            ug = attn_div_by(at, a->by_B);
            b = at - ug * a->B;
        }
        while (left > 0 && ug < a->Hkv_wg) {
            const struct attn_range q = q_of(a, b), k = k_of(a, b);
            const int R = q.n * g, units = attn_units(q.n, k.n);
            const int take = a->teams ? (left < units - off ? left : units - off) : 1;
            struct attn_cover cover = {0, 1};
            if (a->teams)
                cover = attn_cover_of(pos0 - off, units > 1 ? units : 1, quota);
            const int sp = at - cover.first;
            const int k0 = off * 128 < k.n ? off * 128 : k.n;
            const int k1 = a->teams && (off + take) * 128 < k.n ? (off + take) * 128 : k.n;
            for (int tile = t0; take > 0 && (int64_t)tile * rows_wg < R; tile += a->tps)
                for (int r = tile * rows_wg; r < R && r < (tile + 1) * rows_wg; ++r)
                    for (int x = 0; x < heads; ++x) {
                        const int tok = attn_div_by(r, a->by_g), h = (ug * heads + x) * g + r - tok * g;
                        const int64_t slot = (int64_t)(q.at + tok) * a->Hq + h;
                        work[slot] += k1 - k0;
                        ++parts[slot];
                        CHECK(!a->teams || (sp >= 0 && sp < cover.live && cover.live <= a->nsplit), "part %d of %d", sp, cover.live);
                        if (cover.live > 1)
                            write_part(a, slot * a->nsplit + sp, a->D, 1);
                    }
            left -= take;
            pos0 += take;
            off = 0;
            if (++b == a->B)
                b = 0, ++ug;
        }
    }
    for (int b = 0, before = 0; b < a->B; ++b) { /* what the merge expects */
        const struct attn_range q = q_of(a, b), k = k_of(a, b);
        const int units = attn_units(q.n, k.n);
        for (int r = 0; r < q.n * a->Hq; ++r) {
            const int tok = attn_div_by(r, a->by_hq), h = r - tok * a->Hq;
            const int64_t slot = (int64_t)q.at * a->Hq + r;
            const int live = a->teams ? attn_cover_of(attn_div_by(h, a->by_gwg) * total + before, units > 1 ? units : 1,
                                                      quota).live
                                      : 1;
            CHECK(tok == r / a->Hq, "row %d", r);
            CHECK(work[slot] == k.n && parts[slot] == live, "sequence %d row %d: %lld of %d keys, %d of %d parts", b, r,
                  (long long)work[slot], k.n, parts[slot], live);
        }
        before += units;
    }
    free(work);
    free(parts);
}

static int overlapping; /* rows of sequences that overlap: only bounds are checked */

int attn_hip_launch_cross(const struct attn_cross_args *a, const struct attn_cross_cut *cut, int max_q, void *stream) {
    (void)max_q, (void)stream;
    CHECK((int64_t)a->Tq * a->Hq * a->nsplit <= ATTN_SLOTS || a->nsplit == 1, "slots");
    if (overlapping)
        return 0;
    if (cut->rows16)
        walk_line(a, cut);
    else
        walk_tiles(a, cut, ATTN_CROSS_ROWS, 0, 1);
    return 0;
}

int attn_hip_launch_cross_grad(const struct attn_cross_args *a, const struct attn_cross_cut *cut, int kv, int most,
                               void *stream) {
    (void)most, (void)stream;
    a->delta[0] = 1.f;
    a->delta[(int64_t)a->Tq * a->Hq - 1] = 1.f;
    if (a->nsplit > 1) { /* the last part of the last row, whoever has it */
        const int64_t rows = kv ? (int64_t)a->Tk * a->Hkv : (int64_t)a->Tq * a->Hq;
        write_part(a, rows * a->nsplit - 1, kv ? 2 * a->D : a->D, 0);
    }
    team_calls += kv && a->row_teams > 1;
    if (!overlapping)
        walk_tiles(a, cut, kv ? ATTN_CROSS_KEYS : ATTN_CROSS_ROWS, kv, 0);
    return 0;
}

static void test_division(void) {
    for (int i = 0; i < 200000; ++i) {
        const int d = i < 3000 ? i + 1 : pick(1, i % 3 ? 100000 : 0x7fffffff);
        const struct attn_div x = attn_div_of(d);
        const int n[] = {0, 1, d - 1, d, d < 0x40000000 ? 2 * d - 1 : d, pick(0, 0x7ffffffe), 0x7fffffff,
                         (int)(0x7fffffffu / (uint32_t)d * (uint32_t)d), (int)(0x7fffffffu / (uint32_t)d * (uint32_t)d) - 1};
        for (unsigned j = 0; j < sizeof n / sizeof n[0]; ++j)
            CHECK(attn_div_by(n[j], x) == n[j] / d, "%d / %d", n[j], d);
    }
}

static void test_ranges(void) {
    const int bad[] = {-2147483647 - 1, -1, 0, 1, 5, 99, 100, 101, 2147483647};
    for (int s = 0; s < 9; ++s)
        for (int e = 0; e < 9; ++e)
            for (int l = 0; l < 2; ++l) {
                const struct attn_range r = attn_range_of(bad[s], bad[e], l, 100);
                CHECK(r.at >= 0 && r.n >= 0 && r.at + r.n <= 100, "%d %d", bad[s], bad[e]);
            }
    for (int i = 0; i < 20000; ++i) {
        const int total = pick(0, i & 1 ? 0x40000000 : 5000), share = pick(1, 3000), nsplit = pick(1, 64), step = pick(1, 128);
        const struct attn_cut c = attn_cut_of(total, share, nsplit, step);
        CHECK(c.live >= 1 && c.live <= nsplit && c.per % step == 0 && (int64_t)c.live * c.per >= total &&
                  (total == 0 || (int64_t)(c.live - 1) * c.per < total), "%d %d %d %d", total, share, nsplit, step);
    }
    for (int n = 1; n < 300; ++n) {
        char hit[300] = {0};
        for (int wg = 0; wg < n; ++wg)
            ++hit[attn_xcd_order(wg, n)];
        for (int i = 0; i < n; ++i)
            CHECK(hit[i] == 1, "place %d of %d", i, n);
    }
}

static void test_calls(void) {
    const int dims[] = {16, 32, 64, 80, 128, 144, 256};
    for (int i = 0; i < 260; ++i) {
        struct attn_cross_call c;
        memset(&c, 0, sizeof c);
        const int few = i % 2;
        c.D = dims[pick(0, 6)];
        c.B = pick(1, i % 7 == 0 ? 90 : 5);
        c.Hkv = i % 3 ? pick(1, 3) : 4 * pick(1, 2);
        c.Hq = c.Hkv * pick(1, few ? 3 : 6);
        int32_t *arr[4];
        for (int j = 0; j < 4; ++j)
            arr[j] = calloc((size_t)c.B + 1, sizeof(int32_t));
        overlapping = i % 5 == 0;
        const int mq = few ? pick(1, 6) : pick(1, i % 6 == 0 ? 4000 : 200), mk = pick(1, i % 11 == 0 ? 40000 : 900), padded = pick(0, 1);
        struct attn_spans *s[] = {&c.q, &c.k};
        for (int j = 0; j < 2; ++j) {
            int at = pick(0, 2);
            const int most = j ? mk : mq;
            for (int b = 0; b <= c.B; ++b) {
                const int n = pick(0, 4) ? pick(0, most) : b == 0 ? most : 0;
                arr[2 * j][b] = at;
                arr[2 * j + 1][b] = n;
                at += b < c.B ? (padded ? most : n) : 0;
                if (overlapping)
                    arr[2 * j][b] = (int32_t)(rnd() << 1) / (pick(0, 1) ? 1 : 100000), arr[2 * j + 1][b] = (int32_t)rnd() - 5;
            }
            s[j]->start = arr[2 * j];
            s[j]->len = padded ? arr[2 * j + 1] : NULL;
            s[j]->T = at + pick(1, 4);
            s[j]->max = pick(0, 2) ? most : pick(1, 2 * most); /* bounds may be wrong */
        }
        struct attn_rows r[8];
        static char base[8][16] __attribute__((aligned(16)));
        for (int j = 0; j < 8; ++j)
            r[j] = (struct attn_rows){base[j], 256, 256};
        const size_t sb = attn_cross_scratch_bytes(&c), gb = attn_cross_grad_scratch_bytes(&c);
        char *scratch = aligned_alloc(64, (sb + 63) / 64 * 64), *grad = aligned_alloc(64, (gb + 63) / 64 * 64);
        attn_cross(&c, &r[0], &r[1], &r[2], &r[3], (float *)base[4], scratch);
        attn_cross_grad(&c, &r[0], &r[1], &r[2], &r[3], (float *)base[4], &r[4], &r[5], &r[6], &r[7], grad);
        free(scratch);
        free(grad);
        for (int j = 0; j < 4; ++j)
            free(arr[j]);
    }
    /* Numbers at the limits: no overflow, no launch beyond them. */
    static const int32_t zeros[1 << 12];
    const int cases[][7] = {/* B, Hq, Hkv, D, q.T, k.T, max */
                            {1, 1, 1, 256, 1 << 30, 1 << 30, 1 << 30}, {1 << 10, 1 << 10, 1 << 10, 64, 1 << 20, 1 << 10, 1},
                            {1, 1 << 20, 1 << 20, 16, 1 << 10, 1 << 10, 5}, {1, 1 << 20, 1, 16, 1 << 10, 1 << 30, 1 << 10}};
    overlapping = 1;
    for (unsigned i = 0; i < sizeof cases / sizeof cases[0]; ++i) {
        struct attn_cross_call c = {{zeros, zeros, cases[i][4], cases[i][6]}, {zeros, zeros, cases[i][5], cases[i][6]},
                                    cases[i][0], cases[i][1], cases[i][2], cases[i][3], 0.f};
        CHECK(attn_cross_grad_scratch_bytes(&c) >= 4ull * c.q.T * c.Hq &&
                  attn_cross_grad_scratch_bytes(&c) <= 4ull * c.q.T * c.Hq + 256 + (4ull << 25), "case %u", i);
    }
}

/* ---- beam search ----------------------------------------------------------------------------- */
static int64_t beam_calls;
int attn_hip_launch_beam(const struct attn_beam_args *a, int bits, void *stream) {
    (void)stream;
    ++beam_calls;
    const int64_t rows = (int64_t)a->B * a->beams;
    CHECK(a->chunks >= 1 && a->steps >= 1 && (int64_t)a->chunks * a->steps * 4 * ATTN_BEAM_STEP(bits / 8) >= a->V &&
              (int64_t)(a->chunks - 1) * a->steps * 4 * ATTN_BEAM_STEP(bits / 8) < a->V && rows * a->chunks <= 0x7fffffff,
          "%d chunks of %d steps for %d", a->chunks, a->steps, a->V);
    /* each logit of an entry's lists belongs to one segment, and a thread holds all that are its */
    const int lists = a->beams * a->chunks;
    int seen = 0;
    for (int s = 0; s < a->segments; ++s) {
        const int sub = attn_div_by(s, a->by_lists), n = a->K - sub * a->seg;
        CHECK(sub == s / lists && n > 0, "segment %d", s);
        seen += n < a->seg ? n : a->seg;
    }
    CHECK(seen == lists * a->K && a->segments <= ATTN_BEAM_HELD, "%d of %d logits in %d segments", seen, lists * a->K, a->segments);
    a->keys[0] = 1, a->keys[rows * a->chunks * a->K - 1] = 1;
    a->ms[0] = 1.f, a->ms[rows * a->chunks * 2 - 1] = 1.f;
    return 0;
}
static int64_t reorder_calls;
int attn_hip_launch_reorder(const struct attn_reorder_args *a, void *stream) {
    (void)stream;
    ++reorder_calls;
    CHECK((int64_t)a->data_wgs * 256 * 16 >= (int64_t)a->Hkv * (a->row << a->lgp) &&
              (int64_t)a->scale_wgs * 256 * 16 >= (int64_t)a->Hkv * (a->srow << a->lgp) && a->groups >= 1, "workgroups");
    return 0;
}

static void test_beams(void) {
    static char base[64] __attribute__((aligned(64)));
    for (int i = 0; i < 300; ++i) {
        struct attn_beams c;
        memset(&c, 0, sizeof c);
        c.bits = i % 2 ? 16 : 32;
        c.B = pick(1, i % 3 ? 8 : 300), c.beams = pick(1, i % 5 ? 16 : 256), c.K = pick(1, 64);
        c.V = i % 4 ? pick(1, 70000) : pick(1, 1 << 20);
        c.row = c.V + pick(0, 5);
        c.logits = base, c.scores = (const float *)(base + 16);
        const size_t n = attn_beam_scratch_bytes(&c);
        if (n > (256u << 20))
            continue;
        /* sizes are multiples of 8: the block ends where the workspace does */
        char *s = aligned_alloc(64, (n + 63) / 64 * 64);
        attn_beam_select(&c, (float *)base, (int32_t *)(base + 4), (int32_t *)(base + 8), s);
        free(s);
    }
    for (int page = 16; page <= 256; page *= 2)
        for (int bits = 4; bits <= 16; bits += 12) {
            struct attn_kv_cache c = {.k = base, .v = base, .k_scale = base, .v_scale = base, .table = (int32_t *)base,
                                      .kv_len = (int32_t *)base, .q_start = NULL, .B = 12, .table_cols = 5000, .pages = 9,
                                      .page = page, .Hkv = pick(1, 9), .D = 64, .bits = bits};
            attn_kv_reorder(&c, (int32_t *)base, 4, 1);
            attn_kv_reorder(&c, (int32_t *)base, 12, 0);
        }
    for (int i = 0; i < 4000; ++i) {
        const int beams = pick(1, 32), first = pick(0, 1000), j = pick(0, beams - 1);
        const int entry = i % 3 ? first + pick(-3, beams + 3) : (int)(rnd() << 1);
        const int p = attn_parent_of(entry, first, j, beams);
        CHECK(p >= 0 && p < beams && (p == entry - first || p == j), "%d", entry);
    }
    CHECK(attn_parent_of(-2147483647 - 1, 0x7fffffff, 3, 32) == 3 && attn_parent_of(0x7fffffff, 0, 3, 32) == 3, "far entries");
}

int main(void) {
    test_division();
    test_ranges();
    test_calls();
    test_beams();
    CHECK(cut_calls > 100 && line_calls > 20 && team_calls > 5 && beam_calls > 100 && reorder_calls > 10,
          "%d %d %d %lld %lld calls", cut_calls, line_calls, team_calls, (long long)beam_calls, (long long)reorder_calls);
    if (failures)
        return 1;
    printf("CROSS_CHECKS OK: %d cut launches, %d lines, %d of two teams\n", cut_calls, line_calls, team_calls);
    return 0;
}

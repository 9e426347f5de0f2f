/* paged_checks.c -- CPU-only sanitizer driver for the paged cache's host code (built and run by
 * tests/test_paged_host.py with -fsanitize=address,undefined).
 *
 * It runs the index arithmetic that the kernels use (attn_paged_rule.h) over bad tables, lengths and starts
 * and walks, on host memory of exactly the tensors' sizes, every row of the token tensors, entry of the
 * table and row of the cache that a kernel's workgroups would touch: an index outside a tensor is a heap
 * overflow. The real host layer (attn_paged.c) runs with stand-in launchers that check its cut and write
 * every partial slot a kernel could write into a scratch of exactly attn_flash_scratch_bytes(D, bk).
 * Prints "PAGED_CHECKS OK" and exits 0 when every check passes.
 */
#include "attn_flash.h"
#include "attn_paged_cut.h"
#include "attn_paged_rule.h"

#include <hip/hip_runtime_api.h>
#include <limits.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

static int failures;
#define CHECK(cond, ...)                                                                           \
    do {                                                                                           \
        if (!(cond)) {                                                                             \
            failures++;                                                                            \
            printf("FAIL %s:%d: ", __FILE__, __LINE__);                                            \
            printf(__VA_ARGS__);                                                                   \
            printf("\n");                                                                          \
        }                                                                                          \
    } while (0)

static uint32_t rng_state = 12345;
static uint32_t rnd(void) { return rng_state = rng_state * 1664525u + 1013904223u, rng_state >> 8; }
static int pick_int(int lo, int hi) { return lo + (int)(rnd() % (uint32_t)(hi - lo + 1)); }

const char *hipGetErrorString(hipError_t e) {
    (void)e;
    return "stand-in";
}
static int stream_token;
void *attn_flash_get_stream(void) { return &stream_token; }
void attn_hip_plan_begin(char *buf, size_t len) {
    (void)len;
    buf[0] = '\0';
}
static int plan_ended;
long attn_hip_plan_end(void) {
    plan_ended++;
    return 0;
}

/* ---- what the attention kernels touch ------------------------------------------------------ */
static float *scratch_base;
static size_t scratch_len;

static void touch_slot(const struct attn_paged_args *a, int64_t slot, char *seen) {
    if (!scratch_base)
        return;
    a->pm[slot] = 1.f;
    a->pl[slot] = 1.f;
    memset(a->pacc + slot * a->D, 0x3f, sizeof(float) * (size_t)a->D);
    if (seen)
        seen[slot]++;
}

/* One pass over the grid of attn_hip_launch_paged, with the kernels' own arithmetic: the rows they write,
 * the table entries they read, the blocks of 16 keys they address. */
static char *token_seen; /* [T], or NULL: only the cut is checked */
static char *cache_rows; /* [pages * Hkv * page] */
static void touch_keys(const struct attn_paged_args *a, int b, int u, int k0, int k1) {
    for (int kb = k0; kb < k1; kb += 16) {
        const int pg = a->table[(int64_t)b * a->cols + ((kb < k1 - 1 ? kb : k1 - 1) >> a->lgp)];
        if (!attn_page_ok(pg, a->pages))
            continue;
        const int64_t row = attn_page_row(pg, a->Hkv, u, kb, a->lgp);
        const int n = k1 - kb < 16 ? k1 - kb : 16;
        for (int i = 0; i < n; ++i)
            cache_rows[row + i] = 1;
    }
}

static struct attn_seq seq_of(const struct attn_paged_args *a, int b) {
    return attn_seq_of(a->q_start[b], a->q_start[b + 1], a->kv_len[b], a->T, a->cols, a->lgp);
}

int attn_hip_launch_paged(const struct attn_paged_args *a, const struct attn_paged_cut *cut, int bits,
                          void *stream) {
    const int rows16 = cut->rows16;
    const int64_t seqs = (int64_t)a->B * a->Hkv;
    CHECK(stream == &stream_token && (bits == 4 || bits == 16), "launch");
    CHECK(rows16 == 1 || rows16 == 2 || rows16 == 4 || rows16 == 8, "rows16 %d", rows16);
    CHECK(a->D <= 128 || rows16 == 1 || rows16 == 8, "%d row blocks at D = %d", rows16, a->D);
    CHECK(a->tps >= 1 && a->nsplit >= 1 && a->nsplit <= ATTN_PAGED_MAX_PARTS, "cut");
    CHECK(cut->grid >= 1 && cut->grid <= ATTN_PAGED_MAX_GRID, "grid %lld", (long long)cut->grid);
    CHECK(a->nsplit == 1 || (int64_t)a->T * a->Hq * a->nsplit <= ATTN_SLOTS, "slots");
    CHECK(a->teams == 0 || a->nsplit >= 2, "teams without parts");
    if (a->nsplit > 1) {
        CHECK((256 >> (cut->lglp + cut->lgsg)) * a->nsplit <= ATTN_PAGED_MERGE_WEIGHTS, "merge weights");
        CHECK(cut->lglp + cut->lgsg <= 8 && 4 << cut->lglp >= a->D, "merge lanes");
        CHECK(cut->merge_tiles >= 1 && seqs * cut->merge_tiles <= ATTN_PAGED_MAX_GRID, "merge grid");
    }
    if (a->nsplit > 1 && scratch_base)
        touch_slot(a, (int64_t)a->T * a->Hq * a->nsplit - 1, NULL);
    if (!token_seen)
        return 0;
    const int g = a->Hq / a->Hkv;
    int64_t keys_seen = 0, keys_want = 0;
    for (int b = 0; b < a->B; ++b) {
        const struct attn_seq s = seq_of(a, b);
        CHECK(s.q0 >= 0 && s.n >= 0 && s.q0 + s.n <= a->T && s.len >= 0, "sequence");
        CHECK(s.kend >= 0 && s.kend <= (int64_t)a->cols << a->lgp && s.kend <= s.len, "kend");
        if (s.n > 0)
            keys_want += (int64_t)s.kend * a->Hkv;
        for (int t0 = 0; t0 < a->tps; ++t0)
            for (int tile = t0; (int64_t)tile * 16 * rows16 < s.n * g; tile += a->tps)
                for (int r = tile * 16 * rows16; r < (tile + 1) * 16 * rows16 && r < s.n * g; ++r)
                    token_seen[s.q0 + r / g]++;
    }
    if (rows16 >= 4) {
        const int64_t groups = seqs * a->nsplit;
        CHECK(a->share >= 128 && cut->grid >= groups * a->tps, "prefill grid");
        char *placed = calloc((size_t)(groups * a->tps), 1);
        for (int wg = 0; wg < cut->grid; ++wg) {
            const struct attn_place p = attn_place_of(wg, (int)groups, a->tps, a->deal);
            if (p.group >= 0)
                placed[(int64_t)p.group * a->tps + p.tile]++;
        }
        for (int64_t i = 0; i < groups * a->tps; ++i)
            CHECK(placed[i] == 1, "tile %lld placed %d times", (long long)i, placed[i]);
        free(placed);
        for (int b = 0; b < a->B; ++b) {
            const struct attn_seq s = seq_of(a, b);
            const struct attn_parts parts = attn_parts_of(s.kend, a->share, a->nsplit);
            CHECK(parts.live >= 1 && parts.live <= a->nsplit, "live");
            for (int sp = 0; sp < parts.live; ++sp) {
                const int k0 = attn_part_start(s.kend, parts.kps, sp);
                const int k1 = attn_part_start(s.kend, parts.kps, sp + 1);
                CHECK(k0 % 128 == 0 && k0 <= k1 && k1 <= s.kend, "part %d: %d %d", sp, k0, k1);
                CHECK(sp + 1 < parts.live || k1 == s.kend, "last part");
                if (s.n > 0)
                    keys_seen += (int64_t)(k1 - k0) * a->Hkv;
                for (int u = 0; u < a->Hkv; ++u)
                    touch_keys(a, b, u, k0, k1);
            }
        }
    } else if (a->teams == 0) {
        CHECK(cut->grid == seqs * a->tps, "whole grid");
        keys_seen = keys_want;
    } else {
        CHECK(cut->grid == (int64_t)a->teams * a->tps, "team grid");
        int total = 0, most = 0;
        for (int b = 0; b < a->B; ++b) {
            const struct attn_seq s = seq_of(a, b);
            const int n = attn_units(s.n, s.kend);
            total += n;
            most = n > most ? n : most;
        }
        const int q = attn_quota(total, most, a->Hkv, a->teams, a->nsplit);
        CHECK((int64_t)q * a->teams >= (int64_t)total * a->Hkv, "the teams cover the line");
        int *part_seen = calloc((size_t)seqs * a->nsplit, sizeof(int));
        for (int team = 0; team < a->teams; ++team) {
            if ((int64_t)team * q >= (int64_t)total * a->Hkv)
                continue;
            int pos = team * q, left = q < total * a->Hkv - pos ? q : total * a->Hkv - pos;
            int u = pos / total, b = 0, off = pos - u * total;
            for (;; ++b) {
                const struct attn_seq s = seq_of(a, b);
                const int n = attn_units(s.n, s.kend);
                if (off < n)
                    break;
                off -= n;
            }
            while (left > 0 && u < a->Hkv) {
                const struct attn_seq s = seq_of(a, b);
                const int units = attn_units(s.n, s.kend), take = left < units - off ? left : units - off;
                if (take > 0) {
                    const struct attn_cover c = attn_cover_of(pos - off, units, q);
                    const int sp = team - c.first;
                    CHECK(c.live <= a->nsplit && sp >= 0 && sp < c.live, "part %d of %d (%d)", sp, c.live,
                          a->nsplit);
                    part_seen[((int64_t)b * a->Hkv + u) * a->nsplit + sp]++;
                    const int k0 = off * 128 < s.kend ? off * 128 : s.kend;
                    const int k1 = (off + take) * 128 < s.kend ? (off + take) * 128 : s.kend;
                    keys_seen += k1 - k0;
                    touch_keys(a, b, u, k0, k1);
                }
                left -= take, pos += take, off = 0;
                if (++b == a->B)
                    b = 0, ++u;
            }
            CHECK(left == 0, "the line ends before the quota");
        }
        for (int b = 0, before = 0; b < a->B; ++b) { /* what the merge will read */
            const struct attn_seq s = seq_of(a, b);
            const int units = attn_units(s.n, s.kend);
            for (int u = 0; u < a->Hkv && units; ++u) {
                const struct attn_cover c = attn_cover_of(u * total + before, units, q);
                for (int sp = 0; sp < a->nsplit; ++sp)
                    CHECK(part_seen[((int64_t)b * a->Hkv + u) * a->nsplit + sp] == (sp < c.live),
                          "part %d of sequence %d head %d", sp, b, u);
            }
            before += units;
        }
        free(part_seen);
    }
    CHECK(keys_seen == keys_want, "every key once: %lld %lld", (long long)keys_seen, (long long)keys_want);
    return 0;
}

static char *row_seen;
static int walk_kv(const struct attn_kv_args *a, int tpw) {
    CHECK((int64_t)a->B * a->tblk <= ATTN_PAGED_MAX_GRID && a->tblk >= 1, "kv grid");
    if (!row_seen)
        return 0;
    for (int b = 0; b < a->B; ++b) {
        const struct attn_seq s =
            attn_seq_of(a->q_start[b], a->q_start[b + 1], a->kv_len[b], a->T, a->cols, a->lgp);
        for (int tb = 0; tb < a->tblk; ++tb)
            for (int w = 0; w < tpw; ++w)
                for (int i = tb * tpw + w; i < s.n; i += a->tblk * tpw) {
                    row_seen[s.q0 + i]++;
                    const int pos = s.len - s.n + i;
                    if (pos < 0 || pos >= s.kend)
                        continue;
                    const int pg = a->table[(int64_t)b * a->cols + (pos >> a->lgp)];
                    if (attn_page_ok(pg, a->pages))
                        for (int u = 0; u < a->Hkv; ++u)
                            cache_rows[attn_page_row(pg, a->Hkv, u, pos, a->lgp)] = 1;
                }
    }
    return 0;
}
int attn_hip_launch_kv_append(const struct attn_kv_args *a, int bits, int pairs, void *stream) {
    (void)pairs;
    CHECK(stream == &stream_token, "stream");
    (void)bits;
    return walk_kv(a, 1);
}
int attn_hip_launch_kv_read(const struct attn_kv_args *a, int bits, void *stream) {
    (void)bits;
    CHECK(stream == &stream_token, "stream");
    return walk_kv(a, 4);
}

static int bad_int(int sane) {
    switch (rnd() % 8) {
    case 0:
        return INT_MIN;
    case 1:
        return INT_MAX;
    case 2:
        return -pick_int(1, 100);
    case 3:
        return sane + pick_int(1, 100000);
    default:
        return sane;
    }
}

/* Random calls, a third of whose device values are nonsense. */
static void walk(void) {
    static const int pages_of[] = {16, 32, 64, 128, 256};
    for (int it = 0; it < 4000; ++it) {
        const int B = pick_int(1, 6), T = pick_int(1, 300), cols = pick_int(1, 12), Hkv = pick_int(1, 3);
        const int g = pick_int(1, 9), pages = pick_int(1, 40), page = pages_of[rnd() % 5];
        const int D = 16 * pick_int(1, 16), nonsense = rnd() % 3 == 0;
        int32_t *table = malloc(sizeof(int32_t) * (size_t)B * cols), *kv = malloc(sizeof(int32_t) * (size_t)B);
        int32_t *start = malloc(sizeof(int32_t) * (size_t)(B + 1));
        token_seen = calloc((size_t)T, 1);
        row_seen = calloc((size_t)T, 1);
        cache_rows = malloc((size_t)pages * Hkv * page);
        for (int i = 0; i < B * cols; ++i)
            table[i] = nonsense ? bad_int(pick_int(0, pages - 1)) : pick_int(0, pages - 1);
        start[0] = 0;
        for (int b = 0; b < B; ++b) {
            start[b + 1] = start[b] + (T - start[b] > 0 ? pick_int(0, T - start[b]) : 0);
            kv[b] = pick_int(0, cols * page);
        }
        if (nonsense)
            for (int b = 0; b < B; ++b)
                start[b + 1] = bad_int(start[b + 1]), kv[b] = bad_int(kv[b]);
        struct attn_kv_cache c = {(void *)4096, (void *)4096, NULL, NULL, table, kv,  start, B,
                                  cols,         pages,        page, Hkv,  D,     ATTN_KV_BF16};
        const struct attn_rows r = {(void *)4096, 8, 8}, o = {(void *)8192, 8, 8};
        const size_t len = 8u * ATTN_SLOTS + 4u * ATTN_SLOTS * (size_t)D;
        if (it % 50 == 0) { /* the partials of the largest slot */
            scratch_len = len;
            scratch_base = aligned_alloc(256, (len + 255) / 256 * 256);
        }
        attn_paged(&c, &r, &o, T, g * Hkv, (int)(rnd() % 2), NULL, pick_int(1, 400), pick_int(1, 5000),
                   scratch_base ? (void *)scratch_base : (void *)4096);
        free(scratch_base);
        scratch_base = NULL;
        attn_kv_read(&c, &r, &r, T, pick_int(1, 400));
        if (!nonsense)
            for (int t = 0; t < T; ++t) {
                const int mine = t < start[B];
                CHECK(token_seen[t] == (mine ? g : 0), "token %d of %d: %d", t, T, token_seen[t]);
                CHECK(row_seen[t] == mine, "row %d", t);
            }
        free(table), free(kv), free(start), free(token_seen), free(row_seen), free(cache_rows);
        token_seen = row_seen = NULL;
    }
}

/* The cut at the ends of its ranges: only its own invariants. */
static void cuts(void) {
    const int kends[] = {0, 1, 127, 128, 129, 5000, 1 << 20, (1 << 30) - 1, 1 << 30};
    for (int i = 0; i < 9; ++i)
        for (int sh = 128; sh > 0 && sh <= 1 << 29; sh *= 2)
            for (int ns = 1; ns <= ATTN_PAGED_MAX_PARTS; ns = ns * 3 / 2 + 1) {
                const struct attn_parts p = attn_parts_of(kends[i], sh, ns);
                CHECK(p.live >= 1 && p.live <= ns && p.kps % 128 == 0 && p.kps > 0, "parts");
                CHECK(attn_part_start(kends[i], p.kps, p.live) == kends[i], "parts cover");
                CHECK(p.live == 1 || attn_part_start(kends[i], p.kps, p.live - 1) < kends[i], "no empty part");
            }
    static int32_t one[2];
    const int bs[] = {1, 3, 64, 8192}, ts[] = {1, 64, 4096, 1 << 20, 1 << 30};
    const int qs[] = {1, 2, 17, 4096, INT_MAX}, ks[] = {1, 127, 129, 8192, 1 << 20, INT_MAX};
    const int hs[] = {1, 8, 128}, gs[] = {1, 4, 16}, ds[] = {16, 128, 256};
    for (unsigned i = 0; i < 4 * 5 * 5 * 6 * 3 * 3 * 3; ++i) {
        unsigned x = i;
        const int B = bs[x % 4], T = ts[(x /= 4) % 5], q = qs[(x /= 5) % 5], k = ks[(x /= 5) % 6];
        const int Hkv = hs[(x /= 6) % 3], g = gs[(x /= 3) % 3], D = ds[(x /= 3) % 3];
        if ((int64_t)T * Hkv * g > 1 << 30)
            continue;
        struct attn_kv_cache c = {(void *)4096, (void *)4096, NULL, NULL, one, one, one, B,
                                  1 << 9,       1000,         256,  Hkv,  D,   ATTN_KV_BF16};
        const struct attn_rows r = {(void *)4096, 8, 8};
        char buf[64];
        attn_paged_plan(&c, T, g * Hkv, 1, NULL, q, k, buf, sizeof buf);
        attn_kv_append(&c, &r, &r, &r, &r, T, g * Hkv, (const float *)4096, 1, 16, 0, q);
        attn_kv_read(&c, &r, &r, T, q);
    }
    CHECK(plan_ended > 1000, "plans");
}

int main(void) {
    walk();
    cuts();
    if (failures)
        return 1;
    printf("PAGED_CHECKS OK\n");
    return 0;
}

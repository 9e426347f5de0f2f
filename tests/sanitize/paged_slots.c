/* paged_slots.c -- CPU-only sanitizer driver for the scratch of paged attention (built and run by
 * tests/test_paged_slots.py with -fsanitize=address,undefined).
 *
 * The real host layers (attn_paged.c, attn_flash.c) cut calls of all kinds; a stand-in launcher then writes what the
 * kernels and the merge touch of the scratch -- m, l and acc of every part of every row, sequence by sequence, as the
 * cut says -- into memory of exactly attn_flash_scratch_bytes(D, bk): a slot outside it is a heap overflow, and one
 * that two rows or parts share is reported. Prints "PAGED_SLOTS OK" and exits 0 when every check passes.
 */
#include "attn_flash.h"
#include "attn_paged_cut.h"
#include "attn_paged_rule.h"

#include <hip/hip_runtime_api.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

static int failures, split_calls, full_calls;
#define CHECK(cond, ...)                                                                           \
    do {                                                                                           \
        if (!(cond)) {                                                                             \
            failures++;                                                                            \
            printf("FAIL %s:%d: ", __FILE__, __LINE__);                                            \
            printf(__VA_ARGS__);                                                                   \
            printf("\n");                                                                          \
        }                                                                                          \
    } while (0)

/* ---- what the host layers call -------------------------------------------------------------- */
const char *hipGetErrorString(hipError_t e) {
    (void)e;
    return "stand-in";
}
hipError_t hipEventCreate(hipEvent_t *ev) {
    *ev = NULL;
    return hipSuccess;
}
hipError_t hipEventRecord(hipEvent_t ev, hipStream_t st) {
    (void)ev, (void)st;
    return hipSuccess;
}
hipError_t hipEventSynchronize(hipEvent_t ev) {
    (void)ev;
    return hipSuccess;
}
hipError_t hipEventElapsedTime(float *ms, hipEvent_t a, hipEvent_t b) {
    (void)a, (void)b;
    *ms = 0.f;
    return hipSuccess;
}
static int unused(void) { /* the dense kernels and the append: not called here */
    CHECK(0, "another launcher");
    return 1;
}
int attn_hip_launch_prefill(void) { return unused(); }
int attn_hip_launch_decode(void) { return unused(); }
int attn_hip_launch_merge(void) { return unused(); }
int attn_hip_launch_pack_v(void) { return unused(); }
int attn_hip_static_scratch(void) { return unused(); }
int attn_hip_launch_kv_append(void) { return unused(); }
int attn_hip_launch_kv_read(void) { return unused(); }
int attn_hip_device_cus(void) { return 256; }
void attn_hip_plan_begin(char *buf, size_t len) { (void)buf, (void)len; }
long attn_hip_plan_end(void) { return 0; }

static struct attn_seq seq_of(const struct attn_paged_args *a, int b) {
    return attn_seq_of(a->q_start[b], a->q_start[b + 1], a->kv_len[b], a->T, a->cols, a->lgp);
}

/* Every part of every row of sequence b and kv head u, written where the kernels write it. */
static void write_parts(const struct attn_paged_args *a, int b, int u, int live, unsigned char *seen) {
    const struct attn_seq s = seq_of(a, b);
    const int g = a->Hq / a->Hkv;
    for (int r = 0; r < s.n * g; ++r) {
        const int64_t slot = ((int64_t)(s.q0 + r / g) * a->Hq + u * g + r % g) * a->nsplit;
        for (int sp = 0; sp < a->nsplit; ++sp) {
            a->pm[slot + sp] = (float)sp; /* parts behind the last are marked */
            if (sp >= live)
                continue;
            CHECK(!seen[slot + sp], "slot %lld twice", (long long)(slot + sp));
            seen[slot + sp] = 1;
            a->pl[slot + sp] = 1.f;
            for (int d = 0; d < a->D; ++d)
                a->pacc[(slot + sp) * a->D + d] = (float)slot;
        }
    }
}

int attn_hip_launch_paged(const struct attn_paged_args *a, const struct attn_paged_cut *cut, int bits,
                          void *stream) {
    (void)bits, (void)stream;
    if (a->nsplit == 1)
        return 0;
    ++split_calls;
    unsigned char *seen = calloc(ATTN_SLOTS, 1);
    int total = 0, most = 0;
    for (int b = 0; b < a->B; ++b) {
        const struct attn_seq s = seq_of(a, b);
        const int n = attn_units(s.n, s.kend);
        total += n;
        most = n > most ? n : most;
    }
    const int decode = cut->rows16 <= 2;
    CHECK(!decode || a->teams > 0, "parts without teams");
    const int quota = decode ? attn_quota(total, most, a->Hkv, a->teams, a->nsplit) : 1;
    for (int u = 0; u < a->Hkv; ++u)
        for (int b = 0, before = 0; b < a->B; ++b) {
            const struct attn_seq s = seq_of(a, b);
            const int units = attn_units(s.n, s.kend);
            if (units == 0)
                continue;
            const int live = decode ? attn_cover_of(u * total + before, units, quota).live
                                    : attn_parts_of(s.kend, a->share, a->nsplit).live;
            CHECK(live >= 1 && live <= a->nsplit, "%d of %d parts", live, a->nsplit);
            write_parts(a, b, u, live, seen);
            before += units;
        }
    /* What the sequences did not reach is in bounds too: T is the call's, not theirs. */
    const int64_t last = (int64_t)a->T * a->Hq * a->nsplit - 1;
    CHECK(last < ATTN_SLOTS, "%lld slots", (long long)last + 1);
    full_calls += last == ATTN_SLOTS - 1;
    a->pl[last] = 1.f;
    a->pacc[last * a->D + a->D - 1] = 1.f;
    free(seen);
    return 0;
}

static uint32_t rng_state = 99;
static int pick(int lo, int hi) {
    rng_state = rng_state * 1664525u + 1013904223u;
    return lo + (int)((rng_state >> 8) % (uint32_t)(hi - lo + 1));
}

static void call(int B, int T, int Hkv, int g, int D, int cols, const int32_t *start, const int32_t *kv, int bk,
                 int causal, int max_q, int max_kv) {
    int32_t *table = calloc((size_t)B * cols, sizeof *table);
    const struct attn_kv_cache c = {(void *)4096, (void *)4096, NULL, NULL, table, kv, start, B, cols,
                                    3,            32,           Hkv,  D,    ATTN_KV_BF16};
    const struct attn_rows r = {(void *)4096, 8, 8}, o = {(void *)8192, 8, 8};
    const size_t len = attn_flash_scratch_bytes(D, bk);
    CHECK(len % 256 == 0, "scratch of %zu bytes", len);
    char *scratch = aligned_alloc(ATTN_SCRATCH_ALIGN, len);
    attn_paged(&c, &r, &o, T, g * Hkv, causal, NULL, max_q, max_kv, scratch);
    free(scratch), free(table);
}

int main(void) {
    for (int it = 0; it < 300; ++it) {
        const int B = pick(1, 40), Hkv = pick(1, 4), g = pick(1, 8), D = 16 * pick(1, 16);
        const int q = it % 4 == 0 ? 1 : it % 4 == 1 ? pick(1, 12) : pick(1, 300), cols = pick(1, 200);
        int32_t kv[40], start[41];
        start[0] = 0;
        for (int b = 0; b < B; ++b) {
            start[b + 1] = start[b] + (pick(0, 4) ? pick(1, q) : 0);
            kv[b] = pick(0, cols * 32 + 40);
        }
        call(B, start[B] + pick(1, 9), Hkv, g, D, cols, start, kv, 16 << pick(0, 8), pick(0, 1), pick(1, 2 * q),
             pick(1, cols * 40));
    }
    /* Rows times parts that fill the scratch to its last slot: single tokens, drafts and chunks. */
    for (int lg = 0; lg <= 15; ++lg)
        for (int which = 0; which < 9; ++which) {
            const int Hkv = which % 3 == 2 ? 8 : 1, g = which % 3 == 0 ? 1 : 4, D = which < 3 ? 64 : which < 6 ? 128 : 256;
            if (1 << lg < Hkv * g)
                continue;
            const int T = (1 << lg) / (Hkv * g), n = T < 70 ? T : 70;
            const int32_t kv[2] = {60000, 3000}, start[3] = {0, T - n, T};
            for (int mq = 1; mq <= 64; mq *= 8)
                call(2, T, Hkv, g, D, 2048, start, kv, 128, 1, mq, 65536);
        }
    CHECK(full_calls > 20, "%d calls fill the scratch", full_calls);
    CHECK(split_calls > 150, "%d calls with parts", split_calls);
    if (failures)
        return 1;
    printf("PAGED_SLOTS OK\n");
    return 0;
}

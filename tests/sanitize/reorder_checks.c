/* reorder_checks.c -- CPU-only sanitizer driver for attn_kv_reorder's launches (built and run by
 * tests/test_launch_limits.py): each has less than 2^32 work-items, and together they take every group once, for any
 * number of sequences and any page that the call allows. Prints "REORDER_CHECKS OK" and exits 0 when every check passes.
 */
#include "attn_beam_rule.h"
#include "attn_flash.h"

#include <hip/hip_runtime_api.h>
#include <stdio.h>

static int failures, launches;
static int64_t taken;
#define CHECK(cond, ...)                                                                           \
    do {                                                                                           \
        if (!(cond) && ++failures < 20) {                                                          \
            printf("FAIL %s:%d: ", __FILE__, __LINE__);                                            \
            printf(__VA_ARGS__);                                                                   \
            printf("\n");                                                                          \
        }                                                                                          \
    } while (0)

const char *hipGetErrorString(hipError_t e) {
    (void)e;
    return "stand-in";
}
void *attn_flash_get_stream(void) { return NULL; }
int attn_hip_launch_beam(const struct attn_beam_args *a, int bits, void *stream) {
    (void)a, (void)bits, (void)stream;
    return 0;
}
int attn_hip_launch_reorder(const struct attn_reorder_args *a, void *stream) {
    (void)stream;
    ++launches;
    const int64_t wgs = (int64_t)a->groups * (2 * ((int64_t)a->data_wgs + a->scale_wgs) + a->table_wgs);
    CHECK(a->groups >= 1 && wgs >= 1 && wgs * 256 < (int64_t)1 << 32, "%d groups, %lld workgroups", a->groups, (long long)wgs);
    CHECK(a->first == taken, "from group %d, %lld taken", a->first, (long long)taken);
    taken += a->groups;
    return 0;
}

int main(void) {
    static char base[64] __attribute__((aligned(64)));
    for (int bits = 4; bits <= 16; bits += 12)
        for (int D = 64; D <= 256; D *= 2)
            for (int page = 16; page <= 256; page *= 4)
                for (int Hkv = 1; Hkv <= 1 << 13; Hkv *= 4)
                    for (int beams = 1; beams <= 32; beams += 31)
                        for (int near = 0; near < 2; ++near) {
                            const int B = (1 << 20) / Hkv - near * beams;
                            if (B < 1 || (int64_t)Hkv * page * D > 1 << 29 || B % beams != 0)
                                continue;
                            struct attn_kv_cache c = {.k = base, .v = base, .k_scale = base, .v_scale = base,
                                                      .table = (int32_t *)base, .kv_len = (int32_t *)base, .B = B,
                                                      .table_cols = 5000, .pages = 9, .page = page, .Hkv = Hkv, .D = D,
                                                      .bits = bits};
                            for (int tables = 0; tables < 2; ++tables) {
                                taken = 0;
                                attn_kv_reorder(&c, (int32_t *)base, beams, tables);
                                CHECK(taken == B / beams, "%lld of %d groups", (long long)taken, B / beams);
                            }
                        }
    /* the largest page of all heads: 2^29 elements */
    struct attn_kv_cache c = {.k = base, .v = base, .table = (int32_t *)base, .kv_len = (int32_t *)base, .B = 128,
                              .table_cols = 1, .pages = 1, .page = 256, .Hkv = 1 << 13, .D = 256, .bits = 16};
    taken = 0;
    attn_kv_reorder(&c, (int32_t *)base, 1, 1);
    CHECK(taken == 128, "%lld of 128 groups", (long long)taken);
    if (failures)
        return 1;
    printf("REORDER_CHECKS OK: %d launches\n", launches);
    return 0;
}

/* attn_paged_rule.h -- the paged cache's index arithmetic and how a paged call is cut. The kernels and
 * the host layer share it, and it holds no pointer, so that the CPU tests run it with every kind of bad
 * table, length and start. */
#ifndef ATTN_PAGED_RULE_H
#define ATTN_PAGED_RULE_H

#include <stdint.h>

#ifdef __HIPCC__
#define ATTN_HD __host__ __device__ static inline
#else
#define ATTN_HD static inline
#endif

/* One sequence of a call: its rows q0 .. q0 + n - 1 of the token tensors, its length with them (row i is
 * position len - n + i) and how many keys its row of the table can hold of it. Starts and lengths come
 * from device memory: whatever they are, q0 >= 0, n >= 0, q0 + n <= T and 0 <= kend <= cols << lgp. */
struct attn_seq {
    int q0, n, len, kend;
};

ATTN_HD struct attn_seq attn_seq_of(int start, int end, int kv_len, int T, int cols, int lgp) {
    struct attn_seq s;
    s.q0 = start < 0 ? 0 : (start > T ? T : start);
    const int q1 = end < s.q0 ? s.q0 : (end > T ? T : end);
    s.n = q1 - s.q0;
    s.len = kv_len < 0 ? 0 : kv_len;
    const int64_t cap = (int64_t)cols << lgp;
    s.kend = s.len > cap ? (int)cap : s.len;
    return s;
}

/* A page id names a page of the cache. */
ATTN_HD int attn_page_ok(int pg, int pages) { return (uint32_t)pg < (uint32_t)pages; }

/* Row of the cache ([pages][Hkv][page]) that holds key `key` of kv head u in page pg. */
ATTN_HD int64_t attn_page_row(int pg, int Hkv, int u, int key, int lgp) {
    return ((((int64_t)pg * Hkv + u) << lgp) + (key & ((1 << lgp) - 1)));
}

/* Parts of a sequence's keys that its workgroups share: kps keys each, the last one all that is left. */
ATTN_HD int attn_live_parts(int kend, int kps, int nsplit) {
    const int p = kend / kps + (kend % kps != 0);
    return p < 1 ? 1 : (p > nsplit ? nsplit : p);
}

/* Where part sp starts, and where it ends. */
ATTN_HD int attn_part_start(int kend, int kps, int sp) {
    const int64_t k = (int64_t)kps * sp;
    return k > kend ? kend : (int)k;
}
ATTN_HD int attn_part_end(int kend, int kps, int nsplit, int sp) {
    return sp == nsplit - 1 ? kend : attn_part_start(kend, kps, sp + 1);
}

#endif

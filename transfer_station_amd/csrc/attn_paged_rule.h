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

/* Prefill: a sequence's keys in as many parts of `share` keys as it takes, at most nsplit, all of kps keys
 * but the last; one workgroup each per kv head and row tile. */
struct attn_parts {
    int live, kps;
};

ATTN_HD struct attn_parts attn_parts_of(int kend, int share, int nsplit) {
    int n = kend / share + (kend % share != 0);
    n = n < 1 ? 1 : (n > nsplit ? nsplit : n);
    int kps = kend / n + (kend % n != 0);
    kps = kps < 1 ? 128 : (kps + 127) / 128 * 128;
    struct attn_parts p = {kend / kps + (kend % kps != 0), kps};
    if (p.live < 1)
        p.live = 1;
    return p;
}

/* Where part sp starts; the end of the last one is start(live) = kend. */
ATTN_HD int attn_part_start(int kend, int kps, int sp) {
    const int64_t k = (int64_t)kps * sp;
    return k > kend ? kend : (int)k;
}

/* Decode: the keys of all sequences, in units of 128, lie one sequence after the other on a line, once per
 * kv head, and each team of workgroups (one per row tile) takes `quota` units of that line, whatever
 * sequences they belong to: all workgroups read as much, and start and end together. A sequence that a
 * quota's end cuts is joined by the merge kernel. A sequence without keys has one empty unit, so that
 * its rows are written; one without rows has none. */
ATTN_HD int attn_units(int n, int kend) { return n < 1 ? 0 : kend < 1 ? 1 : (kend + 127) >> 7; }

/* The quota: the line over the teams, and enough that no sequence (of max_units at most) is cut into
 * more than nsplit parts. total: units of one kv head; total * Hkv < 2^31. */
ATTN_HD int attn_quota(int total, int max_units, int Hkv, int teams, int nsplit) {
    const int line = total * Hkv;
    int q = line / teams + (line % teams != 0);
    const int least = max_units / (nsplit - 1) + (max_units % (nsplit - 1) != 0);
    q = q < least ? least : q;
    return q < 1 ? 1 : q;
}

/* The parts of the sequence at units [at, at + units) of the line: those of teams first .. first + live - 1. */
struct attn_cover {
    int first, live;
};
ATTN_HD struct attn_cover attn_cover_of(int at, int units, int quota) {
    struct attn_cover c = {at / quota, 0};
    c.live = (at + units - 1) / quota - c.first + 1;
    return c;
}

/* The workgroup's place in the work: the XCDs (hardware ids are dealt to the eight of them in turn) take
 * whole groups of row tiles -- one kv head's keys of one sequence and part -- so that these share the
 * XCD's L2 copy of them, group by group in turn, so that sequences of unequal length leave no XCD idle.
 * Groups whose number is no multiple of 8 are dealt in `deal` pieces, every deal-th tile each. */
struct attn_place {
    int group, tile; /* group -1: none */
};
ATTN_HD struct attn_place attn_place_of(int wg, int groups, int tps, int deal) {
    const int tpp = (tps + deal - 1) / deal; /* tiles per piece */
    const int i = wg >> 3, slot = i / tpp;
    const int piece = (wg & 7) + 8 * slot;
    struct attn_place p = {piece / deal, piece % deal + deal * (i - slot * tpp)};
    if (p.group >= groups || p.tile >= tps)
        p.group = -1;
    return p;
}
ATTN_HD int64_t attn_place_grid(int64_t groups, int tps, int deal) {
    return (groups * deal + 7) / 8 * 8 * ((tps + deal - 1) / deal);
}

#endif

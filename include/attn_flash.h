/* attn_flash.h -- C ABI of the MI355X (gfx950) bf16 flash-attention forward.
 *
 * Drop-in for the C entry points of the reference's AArch64 kernel
 * (liujiang833/transfer_station, flash.c). Same names and parameter lists; the
 * differences are deliberate and listed here:
 *   - Q, K, V, O and scratch are DEVICE pointers (hipMalloc'd or equivalent).
 *   - Work is stream-ordered on the calling thread's stream (attn_flash_set_stream,
 *     default: the null stream). O is valid once that stream has synchronised. When
 *     `tm` is non-NULL the call synchronises itself and O is valid on return, as in
 *     the reference.
 *   - Validation aborts (stderr message, then abort()) on an invalid bk exactly like
 *     the reference, and additionally on Hq%Hkv != 0, Hkv < 1, Sq < 1, Sk < 1,
 *     D outside [1, ATTN_D_MAX], a NULL or misaligned scratch, and HIP errors.
 *   - The scratch keeps the reference's contract (caller-owned, size depends only on
 *     (D, bk), monotone in bk, the kernel allocates nothing and keeps no state) but its
 *     content is the GPU's: split-K partials (m, l, acc[D]), 65536 slots, for the decode
 *     path and for prefills too small to fill the GPU, whose key ranges are split (34 MB at
 *     D = 128).
 *   - bk is validated and sizes the scratch but does not pick the key tile: the GPU's
 *     tile (32, 64 or 128 keys) follows from the other arguments, so O is bit-identical at
 *     every bk. The reference's result is bk-invariant within its tolerance.
 *
 * Layouts (row-major, bf16 stored as uint16_t bits, O fp32):
 *   Q, O [Hq][Sq][D];  K, V [Hkv][Sk][D];  V^T when v_prepacked=1: [Hkv][D][Sk].
 *   A batch folds into the head axes: call with Hq' = B*Hq and Hkv' = B*Hkv.
 */
#ifndef ATTN_FLASH_H
#define ATTN_FLASH_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Key-block bounds and default (flash.c:132-134). bk must be a power of two in
 * [ATTN_BK_MIN, ATTN_BK_MAX]; anything else aborts. */
#define ATTN_BK_MIN 16
#define ATTN_BK_MAX 4096
#define ATTN_BK_DEFAULT 128

/* Required scratch alignment in bytes (flash.c:607). hipMalloc already returns
 * 256-byte aligned memory. */
#define ATTN_SCRATCH_ALIGN 64

/* Largest head dimension the compiled kernels accept (the reference has no bound). */
#define ATTN_D_MAX 256

/* Optional per-call timing (flash.c:704-706). The GPU kernel is one fused launch, so the
 * whole kernel time (HIP events, seconds) is ADDED to qxk; packv, softmax and sxv are
 * left unchanged (no per-phase split is fabricated). */
struct attn_times {
    double packv, qxk, softmax, sxv;
};

/* Bytes of device scratch attn_flash() needs for this head_dim and key-block size
 * (replaces flash.c:679 attn_flash_scratch_bytes). Depends only on (D, bk), never on
 * Sq/Sk; non-decreasing in bk. Aborts on an invalid bk (flash.c:641-647) or D. */
size_t attn_flash_scratch_bytes(int D, int bk);

/* Largest power-of-two bk in [16, 4096] whose modelled per-key-block working set,
 * double-buffered, fits l2_bytes (spec: README.md:138-140,359-436 of the reference;
 * the function is absent from the shipped flash.c). Pure host function. */
int attn_flash_pick_bk(int D, size_t l2_bytes);

/* The attention forward (replaces flash.c:727-729 attn_flash).
 *   O[h][i][:] = softmax_j(scale * Q[h][i]·K[kv][j]) · V[kv][j][:], kv = h / (Hq/Hkv),
 *   scale = 1/sqrtf(D); causal masks keys j > Sk-Sq+i (bottom-right aligned); a row with
 *   no admissible key is written as zeros. P is rounded to bf16 (RNE) before P·V; the
 *   softmax denominator sums the unrounded fp32 p. */
void attn_flash(const uint16_t *Q, const uint16_t *K, const uint16_t *V, float *O, int Hq,
                int Hkv, int Sq, int Sk, int D, int causal, int bk, void *scratch,
                int v_prepacked, struct attn_times *tm);

/* Separate V -> V^T operator: Vp[kv][d][k] = V[kv][k][d] (replaces flash.c:715-718
 * pack_v_full). Device pointers, stream-ordered like attn_flash. */
void pack_v_full(const uint16_t *V, uint16_t *Vp, int Hkv, int Sk, int D);

/* Allocation-free variant of attn_flash. No counterpart in the reference: it is for callers
 * that cannot allocate device memory or own a scratch (code under HIP graph capture, tight
 * serving loops, harnesses that forbid hipMalloc). Same arguments and semantics as attn_flash,
 * without scratch and tm; the split-K partials go to a static device array of
 * ATTN_NOALLOC_SCRATCH_BYTES that the library holds on every GPU it runs on until the process
 * ends (the layout of attn_flash's scratch at D = ATTN_NOALLOC_D_MAX, so the kernels, the splits
 * and the output are those of attn_flash). It calls no hipMalloc, hipFree or other allocating
 * routine. D above ATTN_NOALLOC_D_MAX is rejected (stderr message, then abort), as is everything
 * attn_flash rejects. Every call on one GPU shares that GPU's array: calls that overlap on one
 * GPU (other streams, other threads) race and must be serialised by the caller. */
#define ATTN_NOALLOC_D_MAX 128
#define ATTN_NOALLOC_SCRATCH_BYTES 34078720u /* = attn_flash_scratch_bytes(128, any bk) */
void attn_flash_noalloc(const uint16_t *Q, const uint16_t *K, const uint16_t *V, float *O, int Hq,
                        int Hkv, int Sq, int Sk, int D, int causal, int bk, int v_prepacked);

/* Kernel plan of an attn_flash call (no counterpart in the reference: introspection for tests
 * and integrators, who can see which kernels a shape takes on the current device). Runs
 * attn_flash's host-side choice for these arguments and, instead of launching, writes one line
 * per kernel the call would launch -- "name<template arguments> [notes] grid=x block=n" -- into
 * buf, NUL-terminated. Returns the length written, or -1 when buf is too small. Reads and writes
 * no device memory; the argument checks are attn_flash's (tensors and scratch aside). */
int attn_flash_plan(int Hq, int Hkv, int Sq, int Sk, int D, int causal, int bk, int v_prepacked,
                    char *buf, size_t len);

/* ---- The paged KV cache ------------------------------------------------------------------------
 * No counterpart in the reference (one call there is one dense problem): a cache that grows token by
 * token, shared by sequences of all lengths, and attention over it. Work is stream-ordered on the calling
 * thread's stream like attn_flash's; nothing is allocated and no device memory is read on the host, so
 * every call may be captured into a graph and replayed with other lengths, tables and rows.
 *
 * The cache holds `pages` pages of `page` tokens, K and V alike:
 *   bits 16: bf16 [pages][Hkv][page][D], D % 16 == 0, 16 <= D <= 256
 *   bits 4:  E2M1 codes [pages][Hkv][page][D/2] bytes, the even element in the low half, and one E8M0 scale
 *            byte e per 32 elements, [pages][Hkv][page][D/32]: an element is its code's value (0, 0.5, 1,
 *            1.5, 2, 3, 4, 6, the high bit negates) times 2^(e-127) as a bf16 number, infinite past its range
 *            (which takes an e of 253 or 254), or NaN where e is 255. D is 64, 128 or 256.
 * Sequence b holds kv_len[b] tokens, token p in page table[b * table_cols + p / page]. The tokens of a call
 * are rows of token tensors: sequence b's n_b = q_start[b+1] - q_start[b] of them are rows q_start[b] on,
 * and the last n_b of its kv_len[b] tokens (row i is position kv_len[b] - n_b + i). Rows of no sequence are
 * left as they are; kv_len counts a call's own tokens. Limits: B * Hkv <= 2^20, T * Hq <= 2^30, and table rows
 * for at most 2^38 tokens over all sequences and kv heads.
 *
 * table, kv_len and q_start lie in device memory and may hold anything: an entry of the table outside
 * [0, pages) names no page (its keys are hidden from attention, its tokens are not appended, read back as
 * zeros); of a length past what a row of the table holds only so many keys are seen, and a start is cut to
 * [0, T]. Starts are meant to rise: a sequence that ends before its start has no rows, and a row that two
 * sequences claim may hold neither's answer.
 * Pages may be shared between sequences that read them; a page that a call appends to belongs to one
 * sequence, and no call of another stream reads it meanwhile.
 *
 * max_q and max_kv are the caller's bounds of n_b and kv_len[b], and T of the rows. They choose kernels and cut
 * the work; a sequence that passes max_q or max_kv is served all the same, only slower. Two costs of loose bounds:
 *   - Every sequence is cut as if it had max_q rows. Single tokens beside a prompt go through the prompt's tiles in
 *     attn_paged, and attn_kv_append launches B * max_q workgroups, attn_kv_read a quarter. Such a step is faster as
 *     two calls on parts of the same arrays, the single tokens' rows first: theirs with T ending at their last row, the
 *     prompts' with table + b * table_cols, kv_len + b and q_start + b.
 *   - The scratch holds 65536 partial rows, so a sequence's keys are split into 65536 / (T * Hq) parts at most, and
 *     not at all with T * Hq above 32768: T far above the rows in use leaves one long sequence to few workgroups.
 */
#define ATTN_KV_BF16 16
#define ATTN_KV_FP4 4
#define ATTN_KV_PAGE_MIN 16 /* a page is a power of two of tokens */
#define ATTN_KV_PAGE_MAX 256

struct attn_kv_cache {
    void *k, *v;              /* device, 16-byte aligned */
    void *k_scale, *v_scale;  /* bits 4: device, 16-byte aligned */
    const int32_t *table;     /* device, [B][table_cols] */
    const int32_t *kv_len;    /* device, [B] */
    const int32_t *q_start;   /* device, [B + 1] */
    int32_t B, table_cols;    /* table_cols * page <= 2^30 */
    int32_t pages, page, Hkv, D, bits;
};

/* A token tensor [T][heads][D], bf16: 16-byte aligned, strides in elements, multiples of 8. */
struct attn_rows {
    void *data;
    int64_t token, head;
};

/* What attn_paged does to scores: scale * q.k (scale 0: 1/sqrt(D)); then, with softcap > 0,
 * softcap * tanh(score / softcap); then, with slopes (device, [Hq]), minus slopes[h] * |position - key|. */
struct attn_scores {
    float scale, softcap;
    const float *slopes;
};

/* Writes a call's K and V rows into the cache, K with its position's rotation, and the rotated Q to q_out
 * (q_out may be q, with its strides, and else overlaps none of the rows; q and q_out may both be NULL). The
 * first `rot` elements of a head turn (a multiple of 16; 0: none), in pairs (i, i + rot/2), or with `pairs`
 * (2i, 2i + 1): (x1, x2) -> (x1 c - x2 s, x2 c + x1 s) in fp32, rounded once to bf16, with c and s from row p of
 * rope [rope_rows][rot], cosines in its first half,
 * for position p. In 4 bits the rounded rows are quantised: a group's scale is the smallest power of two in
 * [2^-126, 2^125] under which its largest element is at most 7, elements round to nearest, ties to even; a
 * group with a NaN or an infinity reads as NaN. Tokens whose position is below 0 or has no row in rope are
 * skipped, q's rows too. */
void attn_kv_append(const struct attn_kv_cache *c, const struct attn_rows *q, const struct attn_rows *q_out,
                    const struct attn_rows *k, const struct attn_rows *v, int T, int Hq, const float *rope,
                    int rope_rows, int rot, int pairs, int max_q);

/* The inverse: a call's rows of the cache to k and v, bf16 (with token = D and head = n D the dense layout
 * that attn_flash takes). Reads every token of a sequence where n_b = kv_len[b]. */
void attn_kv_read(const struct attn_kv_cache *c, const struct attn_rows *k, const struct attn_rows *v, int T,
                  int max_q);

/* Attention of a call's rows over their sequences' caches, o in bf16: row i of sequence b sees keys
 * j < kv_len[b], and with causal j <= its position; kv = h / (Hq/Hkv). A row that sees none is written as
 * zeros. P is rounded to bf16 before P.V, as in attn_flash, and as there a NaN or an infinity in V reaches
 * the rows of its key tile that do not see it. P.V is summed before the division by the row's sum: elements of
 * V past 2^86 may overflow on the way. Scores past 2^30, whose rounding to fp32 is coarser than exp can take, give
 * rows without a meaning. o must not be q or overlap it. scores may be NULL (1/sqrt(D)).
 * scratch is an attn_flash scratch of this D (attn_flash_scratch_bytes); calls that may overlap need one
 * each. */
void attn_paged(const struct attn_kv_cache *c, const struct attn_rows *q, const struct attn_rows *o, int T,
                int Hq, int causal, const struct attn_scores *scores, int max_q, int max_kv, void *scratch);

/* The kernels that call would launch, as attn_flash_plan gives them; nothing is launched or read. */
int attn_paged_plan(const struct attn_kv_cache *c, int T, int Hq, int causal,
                    const struct attn_scores *scores, int max_q, int max_kv, char *buf, size_t len);

/* Stream selection for the calling thread (no counterpart in the reference, which has
 * no device). `stream` is a hipStream_t; NULL selects the null stream. */
void attn_flash_set_stream(void *stream);
void *attn_flash_get_stream(void);

#ifdef __cplusplus
}
#endif

#endif /* ATTN_FLASH_H */

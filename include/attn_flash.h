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

/* ---- Cross attention -----------------------------------------------------------------------------
 * No counterpart in the reference. The attention of an encoder-decoder model's rows to its encoder's states, for training
 * and serving: each sequence's rows (a prompt, a target text, a single token, the beams of one input) attend to all of its
 * states, whose number is another. There is no causal mask, so the gradients are those of cross attention and of an encoder's
 * own attention, not of a decoder's. Batches are ragged: packed one sequence behind the other, or padded. Work is
 * stream-ordered on the calling thread's stream, nothing is allocated and no device memory is read on the host, so
 * that every call may be captured into a graph and replayed with other lengths.
 */
/* Rows of each sequence in a token tensor of T rows: from start[b] on, len[b] of them, or, with len NULL, up to
 * start[b + 1]. start ([B], or [B + 1] with len NULL) and len ([B]) lie in device memory and may hold anything: a start
 * is cut to [0, T], and a sequence to the rows behind it. max is the caller's bound of a sequence's rows. It chooses
 * kernels and cuts the work; a sequence that passes it is served all the same, only slower. */
struct attn_spans {
    const int32_t *start, *len;
    int32_t T, max;
};

/* D % 16 == 0, 16 <= D <= 256; scale 0: 1/sqrt(D). Limits: B * Hkv <= 2^20, q.T * Hq and k.T * Hkv <= 2^30, and, as any
 * sequence may claim all states, B * Hkv * (k.T / 128 + 8) and B * (Hq * q.max / 16 + 8 Hkv) <= 2^30. The token strides of
 * all tensors of a call are in [D, ATTN_TOKEN_MAX] elements. */
#define ATTN_TOKEN_MAX 4194304 /* 2^22 */
struct attn_cross_call {
    struct attn_spans q, k;
    int32_t B, Hq, Hkv, D;
    float scale;
};

/* O[t][h] = sum_j P_j V[j][kv], P = softmax_j(scale * Q[t][h].K[j][kv]) over the states j of row t's sequence,
 * kv = h / (Hq/Hkv), in bf16; lse[t * Hq + h] = log sum_j exp(scale * Q.K), natural, in fp32 (lse may be NULL). A row
 * whose sequence has no states gets zeros and -inf; rows of no sequence are left as they are. Sequences may share
 * states (their spans may overlap), not rows. With few rows (up to 32 per kv head) each reads them from memory for itself;
 * as the rows of one sequence they read them once. P is rounded to bf16 before P.V, as in attn_flash; P.V is summed before the
 * division by the row's sum: elements of V past 2^86 may overflow on the way. States that no sequence names are not read,
 * whatever they hold. o must not overlap q, k or v, nor its heads each other.
 * scratch: attn_cross_scratch_bytes(c) bytes, ATTN_SCRATCH_ALIGN-aligned; calls that may overlap need one each. */
size_t attn_cross_scratch_bytes(const struct attn_cross_call *c);
void attn_cross(const struct attn_cross_call *c, const struct attn_rows *q, const struct attn_rows *k,
                const struct attn_rows *v, const struct attn_rows *o, float *lse, void *scratch);

/* The gradients of q, k and v, in bf16, from that of o (d_o) and what the forward call left in o and lse. dK and dV are
 * summed over the heads of a group. P and dS are rounded to bf16 before their products, in calls of up to 2^21 scores
 * (B Hq q.max k.max) in two parts, to 16 bits. States of a sequence without rows get zeros; rows and states of no sequence are
 * left as they are. Here sequences may share neither rows nor states: what two of them claim may hold neither's gradient. A NaN
 * or an infinity in a sequence's tensors may reach all of its gradients, from states of probability 0 too. dq, dk and dv must
 * overlap none of the other tensors. Sums have a fixed order: the same call gives the same bits.
 * scratch: attn_cross_grad_scratch_bytes(c) bytes: 4 q.T Hq, and, where few sequences leave the GPU unfilled, up to 128
 * MB of partial gradients. */
size_t attn_cross_grad_scratch_bytes(const struct attn_cross_call *c);
void attn_cross_grad(const struct attn_cross_call *c, const struct attn_rows *q, const struct attn_rows *k,
                     const struct attn_rows *v, const struct attn_rows *o, const float *lse,
                     const struct attn_rows *d_o, const struct attn_rows *dq, const struct attn_rows *dk,
                     const struct attn_rows *dv, void *scratch);

/* The kernels that attn_cross (or, with grad, attn_cross_grad) would launch, as attn_flash_plan gives them; nothing is
 * launched or read. */
int attn_cross_plan(const struct attn_cross_call *c, int grad, char *buf, size_t len);

/* ---- Beam search ---------------------------------------------------------------------------------
 * No counterpart in the reference. One step of a beam search over the paged cache: choose the continuations that go
 * on, and let the cache's sequences follow them. Stream-ordered, nothing allocated, capturable like the calls above.
 */
#define ATTN_BEAMS_MAX 256
#define ATTN_BEAM_K_MAX 64
#define ATTN_BEAM_V_MAX 1048576 /* 2^20 */
#define ATTN_REORDER_MAX 32

/* The beams of B batch entries: row b * beams + i of logits (bits 16: bf16, 32: fp32; `row` elements from row to row, at
 * any alignment of an element) are beam i's over V tokens, scores[b * beams + i] is what it has reached. done (bytes, or
 * NULL) marks beams that are complete. All device memory, but for the numbers. */
struct attn_beams {
    const void *logits;
    int64_t row;
    const float *scores;
    const uint8_t *done;
    int32_t bits, B, beams, V, K, done_token;
};

/* The K best continuations of each entry, best first: score = (x - log sum exp x) + scores, token and parent, the row
 * (b * beams + i) that it continues; [B][K] each. Ties go to the lowest beam, of its own to the largest logit, then the
 * lowest token. A done beam's only continuation is done_token, at its score; a logit of -inf is none, and a beam whose
 * score is not finite, or that has a NaN or +inf among its logits, has none. Where an entry has fewer than K, the rest is
 * score -inf, token -1 and the entry's first row. The sums of exponentials are taken in fp32, all else in fp64, as
 * (x - m) - log sum exp(x - m) with the beam's largest logit m, so that logits of any size keep their differences, and the
 * score is rounded once. A finite logit is a candidate however low: of a beam whose V logits are all the type's lowest
 * value each scores -log V. Two kinds of rows are slow, since what passes has to be searched for bit by bit: those most of
 * whose logits are one finite value (masked with the lowest value, not with -inf), and large K over many tokens: of 1024 beams
 * and more in all, K of 64 from some 32000 tokens on in bf16, 48 from 65536, 32 from 128000, 24 from 262144, in fp32 from half as
 * many; of fewer beams rows are cut, and may be as much longer.
 * scratch: attn_beam_scratch_bytes(c) bytes, ATTN_SCRATCH_ALIGN-aligned; calls that may overlap need one each. */
size_t attn_beam_scratch_bytes(const struct attn_beams *c);
void attn_beam_select(const struct attn_beams *c, float *score, int32_t *token, int32_t *parent, void *scratch);

/* The cache's sequences lie in groups of `beams` neighbours; sequence b continues parent[b] (device, [B], rows as
 * attn_beam_select gives them: members of b's group; any other entry means b itself). beams is at most ATTN_REORDER_MAX:
 * of a wider search, which attn_beam_select serves, the sequences are the caller's to move. All members of a group hold as many
 * tokens as its first one's kv_len says. Their full pages are shared: with tables, the entries of the parent's row of
 * the table for them replace b's, in place (the one call that writes the table). The tokens of the last, partly filled page
 * are copied into b's own page of that column, with what the 16 bytes at their end hold besides; members must not share
 * that page. A cache per layer that shares one table is reordered by a call per layer, `tables` set in one of them, in any
 * order. An entry of the table outside the cache is not followed: its tokens are not copied. q_start is not used. */
void attn_kv_reorder(const struct attn_kv_cache *c, const int32_t *parent, int beams, int tables);

/* Stream selection for the calling thread (no counterpart in the reference, which has
 * no device). `stream` is a hipStream_t; NULL selects the null stream. */
void attn_flash_set_stream(void *stream);
void *attn_flash_get_stream(void);

#ifdef __cplusplus
}
#endif

#endif /* ATTN_FLASH_H */

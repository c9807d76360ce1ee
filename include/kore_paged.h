/* kore_paged.h - a KV cache of pages for several sequences at once, and the
 * attention that reads it, on an MI355X (gfx950).
 *
 * kore's cache is one contiguous fp32 array for one sequence (Engine::kcache /
 * vcache, kore.cpp:1260; here kore_attn_t), and its server takes one session at
 * a time (kore.cpp:2512, 2600).  Here a pool of pages, each page_size positions
 * of every kv-head of a layer, is shared by any number of sequences; a table of
 * page numbers says where the positions of a sequence lie.  One call appends,
 * or attends, the new rows of all sequences of a batch: one row each in a decode
 * step, chunks of prompts, or both beside each other.
 *
 *   kore_paged_append_dev   rotates the new rows' q and k (kore_rope.h), rounds k
 *                           and v to the cache's type and stores them
 *   kore_paged_attend_dev   out = softmax(scale q K^T) V of each row over the
 *                           positions of its sequence up to its own
 *
 * Pool layout, in elements: [layer][page][kv_head][slot][head_dim], K and V each
 * in an array of its own.  Position p of sequence s is slot p % page_size of page
 * pages[s][p / page_size].
 *
 * The batch (device arrays, read when the call runs, so that a captured graph
 * can be replayed with other contents):
 *   rows q_start[s] .. q_start[s+1] - 1 of q, k, v and out are the new rows of
 *   sequence s (none, where the two are equal); q_start is ascending and within
 *   0 .. n_tok.  kv_len[s] counts the positions of the sequence with the new
 *   rows, so that row i of n has the position kv_len[s] - n + i.
 *   Rows that belong to no sequence (behind q_start[n_seq]) are left as they are.
 *   A page number outside 0 .. n_pages - 1 (say -1) is no page, and nothing past
 *   the table's pages_stride entries is: positions there are not stored, and not
 *   attended.  A row with nothing to attend gets zeros, and so does one whose
 *   attended scores are all -infinity.
 *   At most 2^23 rows, 2^27 rows x heads, 2^16 sequences and 2^22 sequences x
 *   kv-heads a call.
 *   With a q_start that is not ascending the rows of out (q_out, the slots stored)
 *   hold nothing of use; nothing else is written, and nothing outside the buffers
 *   is read.
 * Values of positions that a row does not attend (later ones, those before its
 * window, slots behind the sequence's end) do not reach it, infinities and NaN
 * included.  Of those that it attends, an infinity of V whose score is over
 * -infinity makes its dim of the row infinite, however small the weight (NaN: with
 * both signs, or a NaN); one whose score is -infinity does nothing.  A row with a
 * score of NaN or +infinity is NaN.  What a row gets whose q is not finite is not
 * said; no other row notices.  Pages may be shared by sequences as long as no two
 * rows of one append go to the same slot.
 *
 * Arithmetic: products of the cache's values with q and with the softmax's
 * weights are summed in fp32, and the result is rounded once to the rows' type.
 * What fp32 rows hold of a value on the way:
 *   batches of few rows (16-row tiles) over an fp32 cache: all 24 bits;
 *   over a bf16 cache: 24 bits of q and of the weights (three bf16 parts);
 *   over an fp16 cache: 22 bits of q, relative to its row's largest, and of the
 *   weights (two fp16 parts);
 *   chunks over an fp32 cache: 22 bits of q and of K, relative to their rows'
 *   largest, 24 of V and of the weights.
 * fp16 and bf16 rows hold q as it is; their weights are two parts of the type in
 * 16-row tiles and one, rounded to the type, in chunks (many new rows of a
 * sequence).  A sum is split over workgroups by a rule on the whole batch, in a
 * fixed order: the same call gives the same bits, another batch around a
 * sequence may differ in the last ones.
 *
 * Conventions are those of kore_attn.h: 0 or a negative KORE_PAGED_E_* code,
 * nothing throws, kore_paged_last_error() has the text; one thread at a time per
 * handle.  Append and attend allocate and synchronise nothing, so that they can
 * be captured into a HIP graph.  Part of libkore_paged.so. */
#ifndef KORE_PAGED_H
#define KORE_PAGED_H

#include "kore_rope.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct kore_paged *kore_paged_t;

typedef struct kore_paged_config {
    int n_layer, n_pages;
    int page_size;               /* positions of a page: 16, 32, 64, 128 or 256 */
    int n_head, n_head_kv;       /* n_head a multiple of n_head_kv */
    int head_dim;                /* a multiple of 8, up to 256 */
    int cache_type;              /* KORE_PAGED_F32, _F16 or _BF16 */
    kore_rope_config rope;       /* of append; rot_dim 0: rows are stored as given */
    void *k_pool, *v_pool;       /* device memory of the caller (16-byte aligned, kept by them while the handle
                                    lives), or both NULL: the handle allocates the pools, zeroed */
} kore_paged_config;

typedef struct kore_paged_batch {
    int n_seq, n_tok;            /* sequences; rows of q, k, v and out */
    const int *q_start;          /* device [n_seq + 1] */
    const int *kv_len;           /* device [n_seq] */
    const int *pages;            /* device [n_seq][pages_stride] */
    int pages_stride;            /* entries of a sequence's row of the table; 2^30 positions at most */
    int max_q;                   /* the most new rows that a sequence has, or 0 (unknown): picks the kernel, any
                                    value gives the same result but for rounding */
} kore_paged_batch;

/* A cache on the current HIP device. */
KORE_PAGED_API int kore_paged_create(kore_paged_t *out, const kore_paged_config *cfg);
KORE_PAGED_API void kore_paged_destroy(kore_paged_t h);

/* Appends the batch's rows to one layer.  k, v: [n_tok][n_head_kv * head_dim] of
 * `type`, row i at k + i * k_stride elements.  q (or NULL): [n_tok][n_head *
 * head_dim], rotated into q_out (which may be q itself with the same stride;
 * buffers do not overlap otherwise).  type: KORE_PAGED_F32, or the cache's type.
 * Device pointers aligned to an element, on the handle's device; enqueued on
 * `stream` (a hipStream_t; NULL: the handle's own stream, which is ordered with
 * the null stream). */
KORE_PAGED_API int kore_paged_append_dev(kore_paged_t h, int layer, const kore_paged_batch *b, int type, const void *k,
                                         int64_t k_stride, const void *v, int64_t v_stride, const void *q,
                                         int64_t q_stride, void *q_out, int64_t q_out_stride, void *stream);

/* Attention of the batch's rows over one layer.  q (rotated): [n_tok][n_head *
 * head_dim] of `type` (KORE_PAGED_F32, or the cache's type), out likewise (it may
 * be q itself with the same stride; they do not overlap otherwise); head j reads
 * kv-head j / (n_head / n_head_kv).  scale: 0 for 1 / sqrt(head_dim), or 1e-30 ..
 * 1e30.
 * window 0: a row at position p attends 0 .. p; window w > 0: the last w of
 * those.  Partial sums of a split go to `workspace` (device,
 * kore_paged_workspace_bytes() bytes, 16-byte aligned) or, where it is NULL, to
 * the handle's own: calls that may overlap (on two streams, in two graphs) each
 * need one of their own.  Same pointer and stream rules as the append. */
KORE_PAGED_API int kore_paged_attend_dev(kore_paged_t h, int layer, const kore_paged_batch *b, int type, const void *q,
                                         int64_t q_stride, void *out, int64_t out_stride, float scale, int window,
                                         void *workspace, void *stream);

/* Bytes of an attention workspace of this handle, for any batch. */
KORE_PAGED_API size_t kore_paged_workspace_bytes(kore_paged_t h);

typedef struct kore_paged_info {
    kore_paged_config config;    /* rope.freq_factors is NULL; the pools are those in use */
    int device, num_cu;
    size_t pool_bytes;           /* of K and of V, each */
    void *stream;                /* the handle's own hipStream_t */
} kore_paged_info;
KORE_PAGED_API int kore_paged_get_info(kore_paged_t h, kore_paged_info *info);

/* Wait for the handle's own stream. */
KORE_PAGED_API int kore_paged_sync(kore_paged_t h);

/* Text of the last failure on this handle (or of the last failed create when h
 * is NULL, per thread).  Never NULL. */
KORE_PAGED_API const char *kore_paged_last_error(kore_paged_t h);

#ifdef __cplusplus
}
#endif
#endif

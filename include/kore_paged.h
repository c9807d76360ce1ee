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
 * sequence; trees by a rule of their own, below).  A sum is split over workgroups by a rule on the whole batch, in a
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

/* ---- steps of drafted tokens -------------------------------------------------
 *
 * A server that drafts lets a sequence's new rows be a tree: several guesses at the
 * next tokens, checked at once.  The calls below make a step's tables on the
 * device (plan), store its rows by them (append_rows, with the norms of models that
 * have them), attend the tree (attend_tree) and keep its accepted path (keep), so
 * that a step needs nothing of the host but the drafted tokens and can be captured:
 *     plan (held -> kv_len) ... layers ... keep (kv_len -> held). */

/* What a step's tables are made of: the requests, and the pages that are free.
 * All arrays are device memory, ints aligned to 4 bytes, slot and mask to 8. */
typedef struct kore_paged_plan {
    int n_seq, n_tok;            /* sequences; rows that the step's buffers hold */
    const int *n_new;            /* [n_seq] new rows of each sequence, 0 or more */
    const int *kv_held;          /* [n_seq] positions that each holds */
    int *kv_len;                 /* [n_seq] out: with the new rows (may be kv_held) */
    int *pages;                  /* [n_seq][pages_stride]: entries that the new rows need are added */
    int pages_stride;
    const int *free_pages;       /* [n_pages]: the first n_free[0] are free, the last of them taken first */
    const int *n_free;           /* [1] */
    int *n_free_out;             /* [1] out: less those taken (may be n_free) */
    const int *parent;           /* [n_tok], or NULL: rows one behind the other.  Entry of a sequence's i-th new row: the
                                    row, 0 .. i - 1 of the same, that it follows, or -1 (what is held; so is any other) */
    int *q_start;                /* [n_seq + 1] out: the batch's */
    int *pos;                    /* [n_tok] out: each row's position, kv_held and its depth in the tree; -1: no row */
    int64_t *slot;               /* [n_tok] out: where it is stored, page * page_size + slot of it; -1: nowhere */
    uint64_t *mask;              /* [n_tok][mask_words] out with parent, else NULL: bit j % 64 of word j / 64 is set where
                                    the j-th new row of the sequence is the row itself or before it in the tree (in `window`) */
    int mask_words;              /* 1 .. 16 with parent, else 0 */
    int *status;                 /* [1] out */
    int window;                  /* with parent: rows this many positions or more before a row are not in its mask; 0: all
                                    before it are (layers of several windows: a plan for each, not in place, alike but for mask) */
} kore_paged_plan;

/* Makes the step's tables.  Sequence s gets rows q_start[s] .. and, where they pass
 * the pages that it holds, new ones: the pages of all sequences, one after the
 * other, are taken from the end of the free ones.  The i-th new row lies at position
 * kv_held + i of the sequence's pages, whatever its depth.
 * status 0: done.  Over 0: so many pages are missing; -1: a request is malformed (a
 * negative number, more positions than the table's row, more rows than n_tok or
 * than the mask's bits, an n_free outside 0 .. n_pages).  Then nothing is taken:
 * kv_len is kv_held, n_free_out is n_free, pages are as they were, and q_start, pos,
 * slot and mask are those of a step without rows, which the other calls take.
 * A page that the table names is taken to be the sequence's own behind its full
 * ones: rows go into the last, where it has room.  At most 2^16 sequences and 2^23
 * rows.  Without sequences their arrays and free_pages may be NULL, without rows
 * pos and slot.  But for the pairs named above no two arrays overlap.  Pointers on
 * the handle's device; stream as in the append. */
KORE_PAGED_API int kore_paged_plan_dev(kore_paged_t h, const kore_paged_plan *p, void *stream);

/* Rows as a plan leaves them, and the norms of their heads. */
typedef struct kore_paged_rows {
    int n_tok;
    const int *pos;              /* device [n_tok]: turned to this position; negative: the row is left as it is */
    const int64_t *slot;         /* device [n_tok]: page * page_size + slot; outside the pool: not stored */
    const float *q_norm, *k_norm;/* device, head_dim weights each, or NULL: that one is turned only */
    float norm_eps;              /* over 0 where there is a norm */
} kore_paged_rows;

/* kore_paged_append_dev by the rows' own positions and slots: q and k normalised
 * as by kore_rope_norm_dev, turned, rounded and stored (q into q_out), v rounded
 * and stored.  No two rows have the same slot.  Everything else as there. */
KORE_PAGED_API int kore_paged_append_rows_dev(kore_paged_t h, int layer, const kore_paged_rows *r, int type, const void *k,
                                              int64_t k_stride, const void *v, int64_t v_stride, const void *q,
                                              int64_t q_stride, void *q_out, int64_t q_out_stride, void *stream);

/* Which of its sequence's new rows a row attends. */
typedef struct kore_paged_tree {
    const uint64_t *mask;        /* device [n_tok][mask_words], aligned to 8 bytes: bit j % 64 of word j / 64 of a row is
                                    the j-th new row of its sequence */
    int mask_words;              /* 1 .. 16; new rows past the mask's bits are not attended */
    const int *pos;              /* device [n_tok] positions of the rows; NULL allowed without a window */
} kore_paged_tree;

/* kore_paged_attend_dev for new rows that are a tree, or any set: a row of a
 * sequence with n of them attends the kv_len - n positions before them, in a
 * window w those over pos - w alone (pos is taken within kv_len - n .. kv_len - 1),
 * and of the new ones those that its mask names, itself only if it does; the
 * window does not touch these, so that a model's window is also its plan's.
 * Whether a step takes 16-row tiles or chunks goes by its rows and by the positions
 * that pages_stride and the window allow (not by kv_len, which is the device's), and
 * with it what is rounded on the way (above): a few rows suffice where the table is
 * wide.  Everything else as there. */
KORE_PAGED_API int kore_paged_attend_tree_dev(kore_paged_t h, int layer, const kore_paged_batch *b, const kore_paged_tree *t,
                                              int type, const void *q, int64_t q_stride, void *out, int64_t out_stride,
                                              float scale, int window, void *workspace, void *stream);

/* What is kept of a step's rows.  Device memory, ints aligned to 4 bytes. */
typedef struct kore_paged_keep {
    int n_seq, n_tok;
    const int *q_start;          /* [n_seq + 1] of the step */
    const int *n_keep;           /* [n_seq]: so many of the sequence's n new rows (over n: all); negative: the sequence ends */
    const int *rows;             /* [n_tok]: entries from q_start[s] on, ascending: which of them, 0 .. n - 1; or NULL: the
                                    first ones */
    const int *kv_len;           /* [n_seq], with the step's rows */
    int *kv_out;                 /* [n_seq] out: with those kept (may be kv_len); 0 for a sequence that ends */
    const int *pages;            /* [n_seq][pages_stride] */
    int pages_stride;
    int *free_pages;             /* [n_pages], with n_free and n_free_out; or all NULL: no page is given back */
    const int *n_free;           /* [1] */
    int *n_free_out;             /* [1] out (may be n_free) */
} kore_paged_keep;

/* Moves the kept rows' K and V in every layer so that the i-th lies behind what the
 * sequence held before the step and the i - 1 before it, and gives the pages that no
 * position needs any more back: each sequence's, in the table's order, to the end
 * of the free ones.  The table keeps its entries.  Entries of it that are no page are
 * not given back, nor pages past n_pages free ones.  A sequence that ends gives all
 * its pages back (so it must share none).  Entries of `rows` outside 0 .. n - 1 move
 * nothing; entries that do not ascend leave nothing of use in the rows kept.  At most
 * 2^16 sequences.  But for the pairs named above no two arrays overlap.  Pointers on
 * the handle's device; stream as in the append. */
KORE_PAGED_API int kore_paged_keep_dev(kore_paged_t h, const kore_paged_keep *k, void *stream);

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

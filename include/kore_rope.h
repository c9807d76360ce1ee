/* kore_rope.h - rotary positions of rows of heads on an MI355X (gfx950), beyond
 * the one form kore has (NEOX pairs over the whole head, unscaled,
 * kore.cpp:1374-1385): two pair layouts, a part of the head, and scaled
 * frequencies for contexts past the trained one.
 *
 * A plan holds the frequencies.  Pair i of rot_dim / 2 turns by
 *     pos * f_i,   f_i = base^(-2 i / rot_dim), scaled as below,
 * where f_i is computed in double and rounded to float, as kore's inv_freq
 * (kore.cpp:1337-1339); the angle, its cosine and sine are computed in double,
 * multiplied by the plan's magnitude m and rounded to float.  Then
 *     y0 = x0 c - x1 s,   y1 = x0 s + x1 c
 * with every product and sum rounded to float (kore.cpp:1379-1382), and the
 * result rounded once to the row's type.  The dims from rot_dim on are copied.
 *
 * Scaling:
 *   LINEAR   f_i / factor.
 *   YARN     with corr(b) = rot_dim ln(orig_ctx / (2 pi b)) / (2 ln base),
 *            lo = max(floor(corr(beta_fast)), 0),
 *            hi = min(ceil(corr(beta_slow)), rot_dim - 1) and
 *            g_i = clamp((i - lo) / max(hi - lo, 0.001), 0, 1):
 *            f_i (1 - g_i) + g_i f_i / factor, and m = 0.1 ln(factor) + 1.
 * freq_factors (host, rot_dim / 2 floats, or NULL) then divides f_i by its
 * entry, as a GGUF file's rope_freqs tensor is applied.  No f_i may pass 2^20.
 *
 * Conventions are those of kore_attn.h: 0 or a negative code, nothing throws,
 * kore_rope_last_error() has the text.  Part of libkore_paged.so. */
#ifndef KORE_ROPE_H
#define KORE_ROPE_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#ifndef KORE_PAGED_API
#if defined(__GNUC__)
#define KORE_PAGED_API __attribute__((visibility("default")))
#else
#define KORE_PAGED_API
#endif
#endif

enum {
    KORE_PAGED_OK = 0,
    KORE_PAGED_E_INVALID = -1,     /* null pointer, bad size, type, stride or layer  */
    KORE_PAGED_E_UNSUPPORTED = -3, /* a geometry with no kernel                      */
    KORE_PAGED_E_HIP = -4,         /* HIP runtime failure (no device, launch)        */
    KORE_PAGED_E_NOMEM = -5        /* device or host allocation failed               */
};

/* Element types of rows and caches. */
enum { KORE_PAGED_F32 = 0, KORE_PAGED_F16 = 1, KORE_PAGED_BF16 = 2 };

enum { KORE_ROPE_HALF = 0,         /* pairs (i, i + rot_dim / 2): kore's NEOX form */
       KORE_ROPE_INTERLEAVED = 1   /* pairs (2 i, 2 i + 1) */ };
enum { KORE_ROPE_NONE = 0, KORE_ROPE_LINEAR = 1, KORE_ROPE_YARN = 2 };

typedef struct kore_rope_config {
    int rot_dim;                /* rotated dims of a head, even, 2..512 */
    int layout;                 /* KORE_ROPE_HALF or KORE_ROPE_INTERLEAVED */
    float base;                 /* > 0; > 1 for YARN */
    int scaling;                /* KORE_ROPE_NONE, _LINEAR or _YARN */
    float factor;               /* LINEAR: > 0; YARN: >= 1 */
    int orig_ctx;               /* YARN: the trained context */
    float beta_fast, beta_slow; /* YARN: 0 = 32 and 1 */
    float magnitude;            /* m; 0 = 1, and 0.1 ln(factor) + 1 for YARN */
    const float *freq_factors;  /* host, rot_dim / 2 floats > 0, or NULL; copied */
} kore_rope_config;

typedef struct kore_rope *kore_rope_t;

/* A plan on the current HIP device (its frequencies; a stream of its own). */
KORE_PAGED_API int kore_rope_create(kore_rope_t *out, const kore_rope_config *cfg);
KORE_PAGED_API void kore_rope_destroy(kore_rope_t r);

/* n_tok rows (up to 2^23) of n_head heads of head_dim values (head_dim even, >=
 * rot_dim, at most 1024): out = the rows of x turned to the positions pos (device, n_tok
 * ints >= 0).  Row i of x starts at x + i * x_stride elements (out likewise);
 * within a row the heads are contiguous.  out may be x itself (with the same
 * stride); otherwise the two do not overlap.  transpose != 0 turns the other
 * way (c, -s): the gradient of the forward call, and, divided by m^2, its
 * inverse.  Device pointers, aligned to an element; enqueued on `stream` (a
 * hipStream_t; NULL: the plan's own stream, which is ordered with the null
 * stream) and asynchronous.  n_tok = 0 does nothing.  The call allocates
 * nothing and keeps no state: any number may overlap. */
KORE_PAGED_API int kore_rope_apply_dev(kore_rope_t r, int type, int n_tok, int n_head, int head_dim, const void *x,
                                       int64_t x_stride, const int *pos, void *out, int64_t out_stride,
                                       int transpose, void *stream);

/* The plan's rot_dim / 2 frequencies (host copy) and m. */
KORE_PAGED_API int kore_rope_get_freqs(kore_rope_t r, float *freqs, float *magnitude);

/* Wait for the plan's own stream. */
KORE_PAGED_API int kore_rope_sync(kore_rope_t r);

/* Text of the last failure on this plan (or of the last failed create when r is
 * NULL, per thread).  Never NULL. */
KORE_PAGED_API const char *kore_rope_last_error(kore_rope_t r);

#ifdef __cplusplus
}
#endif
#endif

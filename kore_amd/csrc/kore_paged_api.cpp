// kore_paged_api.cpp - host side of libkore_paged.so (C++20): rotary plans and
// paged caches, the checks of their arguments, and the launches.
#include "kore_paged.h"
#include "kore_paged_kernels.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <new>
#include <vector>

using namespace kore_paged_gpu;

namespace {

constexpr int kErrBytes = 512;
thread_local char g_create_error[kErrBytes] = "";

// Makes a device current for a call and gives the caller's back.
class OnDevice {
  public:
    explicit OnDevice(int device) {
        err_ = hipGetDevice(&before_);
        if (err_ == hipSuccess && before_ != device) {
            err_ = hipSetDevice(device);
            changed_ = err_ == hipSuccess;
        }
    }
    ~OnDevice() {
        if (changed_) (void)hipSetDevice(before_);
    }
    OnDevice(const OnDevice &) = delete;
    OnDevice &operator=(const OnDevice &) = delete;
    hipError_t error() const { return err_; }

  private:
    int before_ = 0;
    bool changed_ = false;
    hipError_t err_ = hipSuccess;
};

int vfail(char *where, int code, const char *fmt, va_list ap) {
    vsnprintf(where, kErrBytes, fmt, ap);
    return code;
}

}  // namespace

struct kore_rope {
    kore_rope_config cfg{};
    int device = 0;
    hipStream_t stream = nullptr;
    std::vector<float> freq;
    float *d_freq = nullptr;
    double size = 1.0;
    char err[kErrBytes] = "";

    Turn turn() const { return Turn{d_freq, size, cfg.rot_dim, cfg.layout == KORE_ROPE_INTERLEAVED}; }
};

struct kore_paged {
    kore_paged_config cfg{};
    int device = 0, num_cu = 0, page_shift = 0;
    hipStream_t stream = nullptr;
    kore_rope_t rope = nullptr;         // NULL: rows are stored as given
    void *k_pool = nullptr, *v_pool = nullptr;
    bool own_pools = false;
    float *part = nullptr;
    size_t part_bytes = 0;
    char err[kErrBytes] = "";

    size_t layer_elems() const {
        return (size_t)cfg.n_pages * cfg.n_head_kv * cfg.page_size * cfg.head_dim;
    }
    size_t pool_bytes() const { return layer_elems() * cfg.n_layer * type_bytes(cfg.cache_type); }
};

namespace {

template <class H>
int fail(H *h, int code, const char *fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vfail(h ? h->err : g_create_error, code, fmt, ap);
    va_end(ap);
    return code;
}

#define FAIL0(code, ...) fail((kore_rope *)nullptr, code, __VA_ARGS__)
#define HIP_TRY(h, expr)                                                                               \
    do {                                                                                               \
        hipError_t e_ = (expr);                                                                        \
        if (e_ != hipSuccess) return fail((h), KORE_PAGED_E_HIP, "%s: %s", #expr, hipGetErrorString(e_)); \
    } while (0)

constexpr double kMaxFreq = 0x1p20;   // to which the kernels' angles are exact

bool type_ok(int t) { return t == KORE_PAGED_F32 || t == KORE_PAGED_F16 || t == KORE_PAGED_BF16; }

// The frequencies of the header's formulas, in double, and m.
class Freqs {
  public:
    explicit Freqs(const kore_rope_config &c) : c_(c), size_(c.magnitude > 0 ? (double)c.magnitude : 1.0) {
        if (c.scaling != KORE_ROPE_YARN) return;
        const auto corr = [&](double beta) {
            return c.rot_dim * std::log(c.orig_ctx / (beta * 2 * M_PI)) / (2 * std::log((double)c.base));
        };
        lo_ = std::max(std::floor(corr(c.beta_fast > 0 ? c.beta_fast : 32.0)), 0.0);
        hi_ = std::min(std::ceil(corr(c.beta_slow > 0 ? c.beta_slow : 1.0)), (double)c.rot_dim - 1);
        if (!(c.magnitude > 0)) size_ = 0.1 * std::log((double)c.factor) + 1.0;
    }
    double of(int i) const {
        double f = std::pow((double)c_.base, -2.0 * i / c_.rot_dim);   // kore.cpp:1339
        if (c_.scaling == KORE_ROPE_LINEAR) f /= c_.factor;
        if (c_.scaling == KORE_ROPE_YARN) {
            const double g = std::clamp((i - lo_) / std::max(hi_ - lo_, 0.001), 0.0, 1.0);
            f = f / c_.factor * g + f * (1 - g);
        }
        return c_.freq_factors ? f / c_.freq_factors[i] : f;
    }
    double size() const { return size_; }

  private:
    const kore_rope_config &c_;
    double size_, lo_ = 0, hi_ = 0;
};

int check_rope(const kore_rope_config &c) {
    if (c.rot_dim < 2 || c.rot_dim % 2 != 0 || c.rot_dim > kMaxRot)
        return FAIL0(KORE_PAGED_E_INVALID, "rot_dim %d is not even within 2..%d", c.rot_dim, kMaxRot);
    if (c.layout != KORE_ROPE_HALF && c.layout != KORE_ROPE_INTERLEAVED)
        return FAIL0(KORE_PAGED_E_INVALID, "unknown rotary layout %d", c.layout);
    if (!(c.base > 0) || !std::isfinite(c.base))
        return FAIL0(KORE_PAGED_E_INVALID, "rotary base must be positive and finite");
    if (c.scaling < KORE_ROPE_NONE || c.scaling > KORE_ROPE_YARN)
        return FAIL0(KORE_PAGED_E_INVALID, "unknown rotary scaling %d", c.scaling);
    if (c.scaling == KORE_ROPE_LINEAR && (!(c.factor > 0) || !std::isfinite(c.factor)))
        return FAIL0(KORE_PAGED_E_INVALID, "linear scaling needs a positive factor");
    if (c.scaling == KORE_ROPE_YARN) {
        if (!(c.factor >= 1) || !std::isfinite(c.factor))
            return FAIL0(KORE_PAGED_E_INVALID, "YaRN scaling needs a factor of 1 or more");
        if (!(c.base > 1)) return FAIL0(KORE_PAGED_E_INVALID, "YaRN scaling needs a base over 1");
        if (c.orig_ctx <= 0) return FAIL0(KORE_PAGED_E_INVALID, "YaRN scaling needs orig_ctx");
        if (!(c.beta_fast >= 0) || !(c.beta_slow >= 0) || !std::isfinite(c.beta_fast) || !std::isfinite(c.beta_slow))
            return FAIL0(KORE_PAGED_E_INVALID, "beta_fast and beta_slow must be finite, 0 or more");
    }
    if (!(c.magnitude >= 0) || !std::isfinite(c.magnitude))
        return FAIL0(KORE_PAGED_E_INVALID, "magnitude must be finite, 0 or more");
    if (c.freq_factors)
        for (int i = 0; i < c.rot_dim / 2; ++i)
            if (!(c.freq_factors[i] > 0) || !std::isfinite(c.freq_factors[i]))
                return FAIL0(KORE_PAGED_E_INVALID, "freq_factors[%d] is not positive and finite", i);
    const Freqs f(c);
    for (int i = 0; i < c.rot_dim / 2; ++i)
        if (!(f.of(i) <= kMaxFreq)) return FAIL0(KORE_PAGED_E_INVALID, "frequency %d is over 2^20", i);
    return KORE_PAGED_OK;
}

void release(kore_rope *r) {
    if (!r) return;
    {
        OnDevice on(r->device);
        if (r->stream) (void)hipStreamSynchronize(r->stream);
        if (r->d_freq) (void)hipFree(r->d_freq);   // waits for the device's work
        if (r->stream) (void)hipStreamDestroy(r->stream);
    }
    delete r;
}

void release(kore_paged *h) {
    if (!h) return;
    {
        OnDevice on(h->device);
        if (h->stream) (void)hipStreamSynchronize(h->stream);
        if (h->own_pools && h->k_pool) (void)hipFree(h->k_pool);
        if (h->own_pools && h->v_pool) (void)hipFree(h->v_pool);
        if (h->part) (void)hipFree(h->part);
        if (h->stream) (void)hipStreamDestroy(h->stream);
    }
    release(h->rope);
    delete h;
}

template <class H>
int on_device(H *h, const OnDevice &on) {
    if (on.error() != hipSuccess) return fail(h, KORE_PAGED_E_HIP, "hipSetDevice: %s", hipGetErrorString(on.error()));
    return KORE_PAGED_OK;
}

// A row's stride, of n values.
template <class H>
int check_stride(H *h, const char *what, int64_t stride, int64_t n, int n_tok) {
    if (stride < n) return fail(h, KORE_PAGED_E_INVALID, "%s stride %lld is under a row's %lld values", what,
                                (long long)stride, (long long)n);
    if (stride > (int64_t)1 << 40 || (n_tok > 0 && stride > ((int64_t)1 << 59) / n_tok))
        return fail(h, KORE_PAGED_E_INVALID, "%s stride %lld is too large", what, (long long)stride);
    return KORE_PAGED_OK;
}

template <class H>
int check_aligned(H *h, const char *what, const void *p, int type) {
    if ((uintptr_t)p % (size_t)type_bytes(type))
        return fail(h, KORE_PAGED_E_INVALID, "%s is not aligned to an element", what);
    return KORE_PAGED_OK;
}

// x's rows and y's, [n_tok] of xn and yn values: no byte in common.
template <class H>
int check_apart(H *h, const char *what, const void *x, int64_t xs, int64_t xn, const void *y, int64_t ys, int64_t yn, int n_tok,
                int type) {
    const uintptr_t size = (uintptr_t)type_bytes(type), x0 = (uintptr_t)x, y0 = (uintptr_t)y;
    const uintptr_t x1 = x0 + ((uintptr_t)(n_tok - 1) * xs + xn) * size, y1 = y0 + ((uintptr_t)(n_tok - 1) * ys + yn) * size;
    if (x0 < y1 && y0 < x1) {
        // rows that lie between each other (two parts of one wide row) share no byte
        const bool first = x0 < y0;
        const uintptr_t step = (uintptr_t)xs * size, d = (first ? y0 - x0 : x0 - y0) % step;
        const uintptr_t w = (uintptr_t)(first ? xn : yn) * size, next = (uintptr_t)(first ? yn : xn) * size;
        if (xs != ys || d < w || d + next > step) return fail(h, KORE_PAGED_E_INVALID, "%s rows overlap", what);
    }
    return KORE_PAGED_OK;
}

// Input rows and output rows of n values: the same buffer with the same stride, or no byte in common.
template <class H>
int check_overlap(H *h, const void *x, int64_t xs, const void *y, int64_t ys, int64_t n, int n_tok, int type) {
    if (x == y && xs == ys) return KORE_PAGED_OK;
    return check_apart(h, "input and output", x, xs, n, y, ys, n, n_tok, type);
}

int check_batch(kore_paged *h, int layer, const kore_paged_batch *b, int type) {
    if (!b) return fail(h, KORE_PAGED_E_INVALID, "null batch");
    if (layer < 0 || layer >= h->cfg.n_layer)
        return fail(h, KORE_PAGED_E_INVALID, "layer %d outside [0, %d)", layer, h->cfg.n_layer);
    if (!type_ok(type)) return fail(h, KORE_PAGED_E_INVALID, "unknown type %d", type);
    if (type != KORE_PAGED_F32 && type != h->cfg.cache_type)
        return fail(h, KORE_PAGED_E_INVALID, "rows of type %d with a cache of type %d (rows are fp32 or of the cache's type)",
                    type, h->cfg.cache_type);
    if (b->n_seq < 0 || b->n_tok < 0 || b->max_q < 0)
        return fail(h, KORE_PAGED_E_INVALID, "negative n_seq, n_tok or max_q");
    if (b->n_seq == 0 || b->n_tok == 0) return KORE_PAGED_OK;
    if (!b->q_start || !b->kv_len || !b->pages) return fail(h, KORE_PAGED_E_INVALID, "null q_start, kv_len or pages");
    if (b->pages_stride <= 0 || b->pages_stride > kMaxKeys / h->cfg.page_size)
        return fail(h, KORE_PAGED_E_INVALID, "pages_stride %d outside 1..%d", b->pages_stride, kMaxKeys / h->cfg.page_size);
    if (b->n_seq > kMaxSeq)
        return fail(h, KORE_PAGED_E_UNSUPPORTED, "n_seq %d is too large (over %d)", b->n_seq, kMaxSeq);
    if (b->n_tok > kMaxRows || (int64_t)b->n_tok * h->cfg.n_head > kMaxRowHeads ||
        (int64_t)b->n_seq * h->cfg.n_head_kv > kMaxSeqHeads)
        return fail(h, KORE_PAGED_E_UNSUPPORTED, "n_tok %d x %d heads or n_seq %d x %d kv-heads is too large", b->n_tok,
                    h->cfg.n_head, b->n_seq, h->cfg.n_head_kv);
    return KORE_PAGED_OK;
}

Batch device_batch(const kore_paged_batch *b) {
    return Batch{b->q_start, b->kv_len, b->pages, b->n_seq, b->n_tok, b->pages_stride};
}

template <class H>
hipStream_t pick_stream(H *h, void *stream) {
    return stream ? (hipStream_t)stream : h->stream;
}

}  // namespace

extern "C" {

int kore_rope_create(kore_rope_t *out, const kore_rope_config *cfg) {
    if (!out) return FAIL0(KORE_PAGED_E_INVALID, "null handle pointer");
    *out = nullptr;
    if (!cfg) return FAIL0(KORE_PAGED_E_INVALID, "null config");
    if (int rc = check_rope(*cfg)) return rc;
    kore_rope *r = new (std::nothrow) kore_rope;
    if (!r) return FAIL0(KORE_PAGED_E_NOMEM, "out of host memory");
    try {
        const Freqs f(*cfg);
        r->size = f.size();
        for (int i = 0; i < cfg->rot_dim / 2; ++i) r->freq.push_back((float)f.of(i));
    } catch (const std::exception &) {
        delete r;
        return FAIL0(KORE_PAGED_E_NOMEM, "out of host memory");
    }
    r->cfg = *cfg;
    r->cfg.freq_factors = nullptr;
    const size_t bytes = r->freq.size() * sizeof(float);
    const char *what = "hipGetDevice";
    hipError_t e = hipGetDevice(&r->device);
    if (e == hipSuccess) { what = "hipStreamCreate"; e = hipStreamCreate(&r->stream); }
    if (e == hipSuccess) { what = "hipMalloc"; e = hipMalloc(&r->d_freq, bytes); }
    if (e == hipSuccess) { what = "hipMemcpy"; e = hipMemcpy(r->d_freq, r->freq.data(), bytes, hipMemcpyHostToDevice); }
    if (e != hipSuccess) {
        const int rc = FAIL0(KORE_PAGED_E_HIP, "%s: %s", what, hipGetErrorString(e));
        release(r);
        return rc;
    }
    *out = r;
    return KORE_PAGED_OK;
}

void kore_rope_destroy(kore_rope_t r) { release(r); }

int kore_rope_apply_dev(kore_rope_t r, int type, int n_tok, int n_head, int head_dim, const void *x, int64_t x_stride,
                        const int *pos, void *out, int64_t out_stride, int transpose, void *stream) {
    if (!r) return FAIL0(KORE_PAGED_E_INVALID, "null handle");
    if (!type_ok(type)) return fail(r, KORE_PAGED_E_INVALID, "unknown type %d", type);
    if (n_tok < 0 || n_head <= 0) return fail(r, KORE_PAGED_E_INVALID, "bad n_tok %d or n_head %d", n_tok, n_head);
    if (head_dim < r->cfg.rot_dim || head_dim % 2 != 0)
        return fail(r, KORE_PAGED_E_INVALID, "head_dim %d is odd or under rot_dim %d", head_dim, r->cfg.rot_dim);
    if (n_tok > kMaxRows) return fail(r, KORE_PAGED_E_UNSUPPORTED, "n_tok %d is over %d", n_tok, kMaxRows);
    if (head_dim > kMaxRopeHeadDim)
        return fail(r, KORE_PAGED_E_UNSUPPORTED, "head_dim %d over %d", head_dim, kMaxRopeHeadDim);
    if ((int64_t)n_head * head_dim > 1 << 24)
        return fail(r, KORE_PAGED_E_UNSUPPORTED, "%d heads of %d are too large a row", n_head, head_dim);
    const int64_t n = (int64_t)n_head * head_dim;
    if (int rc = check_stride(r, "x", x_stride, n, n_tok)) return rc;
    if (int rc = check_stride(r, "out", out_stride, n, n_tok)) return rc;
    if (n_tok == 0) return KORE_PAGED_OK;
    if (!x || !out || !pos) return fail(r, KORE_PAGED_E_INVALID, "null buffer");
    if (int rc = check_aligned(r, "x", x, type)) return rc;
    if (int rc = check_aligned(r, "out", out, type)) return rc;
    if (int rc = check_overlap(r, x, x_stride, out, out_stride, n, n_tok, type)) return rc;
    OnDevice on(r->device);
    if (int rc = on_device(r, on)) return rc;
    const RopeArgs a{r->turn(), x, out, pos, x_stride, out_stride, n_tok, n_head, head_dim, transpose ? -1 : 1, type};
    HIP_TRY(r, launch_rope(a, pick_stream(r, stream)));
    return KORE_PAGED_OK;
}

int kore_rope_get_freqs(kore_rope_t r, float *freqs, float *magnitude) {
    if (!r) return FAIL0(KORE_PAGED_E_INVALID, "null handle");
    if (!freqs || !magnitude) return fail(r, KORE_PAGED_E_INVALID, "null buffer");
    std::copy(r->freq.begin(), r->freq.end(), freqs);
    *magnitude = (float)r->size;
    return KORE_PAGED_OK;
}

int kore_rope_sync(kore_rope_t r) {
    if (!r) return FAIL0(KORE_PAGED_E_INVALID, "null handle");
    OnDevice on(r->device);
    if (int rc = on_device(r, on)) return rc;
    HIP_TRY(r, hipStreamSynchronize(r->stream));
    return KORE_PAGED_OK;
}

const char *kore_rope_last_error(kore_rope_t r) { return r ? r->err : g_create_error; }

int kore_paged_create(kore_paged_t *out, const kore_paged_config *cfg) {
    if (!out) return FAIL0(KORE_PAGED_E_INVALID, "null handle pointer");
    *out = nullptr;
    if (!cfg) return FAIL0(KORE_PAGED_E_INVALID, "null config");
    const kore_paged_config &c = *cfg;
    if (c.n_layer <= 0 || c.n_pages <= 0 || c.n_head <= 0 || c.n_head_kv <= 0 || c.head_dim <= 0)
        return FAIL0(KORE_PAGED_E_INVALID, "non-positive geometry");
    if (c.n_head % c.n_head_kv != 0)
        return FAIL0(KORE_PAGED_E_INVALID, "n_head %d not a multiple of n_head_kv %d", c.n_head, c.n_head_kv);
    if (c.page_size != 16 && c.page_size != 32 && c.page_size != 64 && c.page_size != 128 && c.page_size != 256)
        return FAIL0(KORE_PAGED_E_INVALID, "page_size %d is not 16, 32, 64, 128 or 256", c.page_size);
    if (!type_ok(c.cache_type)) return FAIL0(KORE_PAGED_E_INVALID, "unknown cache type %d", c.cache_type);
    if (c.head_dim % 8 != 0 || c.head_dim > kMaxHeadDim)
        return FAIL0(KORE_PAGED_E_UNSUPPORTED, "no gfx950 kernel for head_dim %d (supported: multiples of 8 up to %d)",
                     c.head_dim, kMaxHeadDim);
    if ((double)c.n_head_kv * c.page_size * c.head_dim * type_bytes(c.cache_type) >= 4294967296.0)
        return FAIL0(KORE_PAGED_E_UNSUPPORTED, "a page of one layer takes 4 GiB or more");
    if (c.n_head > 1 << 16) return FAIL0(KORE_PAGED_E_UNSUPPORTED, "n_head %d is too large", c.n_head);
    if ((c.k_pool == nullptr) != (c.v_pool == nullptr)) return FAIL0(KORE_PAGED_E_INVALID, "one pool of two is given");
    if ((uintptr_t)c.k_pool % 16 || (uintptr_t)c.v_pool % 16)
        return FAIL0(KORE_PAGED_E_INVALID, "a pool is not 16-byte aligned");
    if ((double)c.n_layer * c.n_pages * c.n_head_kv * c.page_size * c.head_dim > 1e15)
        return FAIL0(KORE_PAGED_E_INVALID, "cache size overflows");
    if (c.rope.rot_dim != 0) {
        if (int rc = check_rope(c.rope)) return rc;
        if (c.rope.rot_dim > c.head_dim)
            return FAIL0(KORE_PAGED_E_INVALID, "rot_dim %d over head_dim %d", c.rope.rot_dim, c.head_dim);
    }
    kore_paged *h = new (std::nothrow) kore_paged;
    if (!h) return FAIL0(KORE_PAGED_E_NOMEM, "out of host memory");
    h->cfg = c;
    h->cfg.rope.freq_factors = nullptr;
    while (1 << h->page_shift < c.page_size) ++h->page_shift;
    const auto bail = [&](hipError_t e, const char *what) {
        const int rc = FAIL0(e == hipErrorOutOfMemory ? KORE_PAGED_E_NOMEM : KORE_PAGED_E_HIP, "%s: %s", what,
                             hipGetErrorString(e));
        release(h);
        return rc;
    };
    hipError_t e = hipGetDevice(&h->device);
    if (e != hipSuccess) return bail(e, "hipGetDevice");
    if ((e = hipDeviceGetAttribute(&h->num_cu, hipDeviceAttributeMultiprocessorCount, h->device)) != hipSuccess)
        return bail(e, "hipDeviceGetAttribute");
    if ((e = hipStreamCreate(&h->stream)) != hipSuccess) return bail(e, "hipStreamCreate");
    if (c.rope.rot_dim != 0)
        if (int rc = kore_rope_create(&h->rope, &c.rope)) {
            release(h);
            return rc;
        }
    h->k_pool = c.k_pool;
    h->v_pool = c.v_pool;
    if (!c.k_pool) {
        h->own_pools = true;
        if ((e = hipMalloc(&h->k_pool, h->pool_bytes())) != hipSuccess) return bail(e, "K pool allocation");
        if ((e = hipMalloc(&h->v_pool, h->pool_bytes())) != hipSuccess) return bail(e, "V pool allocation");
        if ((e = hipMemsetAsync(h->k_pool, 0, h->pool_bytes(), h->stream)) != hipSuccess) return bail(e, "hipMemset");
        if ((e = hipMemsetAsync(h->v_pool, 0, h->pool_bytes(), h->stream)) != hipSuccess) return bail(e, "hipMemset");
        if ((e = hipStreamSynchronize(h->stream)) != hipSuccess) return bail(e, "hipStreamSynchronize");
    }
    h->part_bytes = attend_workspace_bytes(c.head_dim, h->num_cu);
    if ((e = hipMalloc(&h->part, h->part_bytes)) != hipSuccess) return bail(e, "workspace allocation");
    h->cfg.k_pool = h->k_pool;
    h->cfg.v_pool = h->v_pool;
    *out = h;
    return KORE_PAGED_OK;
}

void kore_paged_destroy(kore_paged_t h) { release(h); }

int kore_paged_append_dev(kore_paged_t h, int layer, const kore_paged_batch *b, int type, const void *k,
                          int64_t k_stride, const void *v, int64_t v_stride, const void *q, int64_t q_stride,
                          void *q_out, int64_t q_out_stride, void *stream) {
    if (!h) return FAIL0(KORE_PAGED_E_INVALID, "null handle");
    if (int rc = check_batch(h, layer, b, type)) return rc;
    const kore_paged_config &c = h->cfg;
    const int64_t kvd = (int64_t)c.n_head_kv * c.head_dim, E = (int64_t)c.n_head * c.head_dim;
    if (int rc = check_stride(h, "k", k_stride, kvd, b->n_tok)) return rc;
    if (int rc = check_stride(h, "v", v_stride, kvd, b->n_tok)) return rc;
    if (b->n_seq == 0 || b->n_tok == 0) return KORE_PAGED_OK;
    if (!k || !v) return fail(h, KORE_PAGED_E_INVALID, "null buffer");
    if ((q == nullptr) != (q_out == nullptr)) return fail(h, KORE_PAGED_E_INVALID, "q without q_out, or q_out without q");
    if (int rc = check_aligned(h, "k", k, type)) return rc;
    if (int rc = check_aligned(h, "v", v, type)) return rc;
    if (q) {
        if (int rc = check_stride(h, "q", q_stride, E, b->n_tok)) return rc;
        if (int rc = check_stride(h, "q_out", q_out_stride, E, b->n_tok)) return rc;
        if (int rc = check_aligned(h, "q", q, type)) return rc;
        if (int rc = check_aligned(h, "q_out", q_out, type)) return rc;
        if (int rc = check_overlap(h, q, q_stride, q_out, q_out_stride, E, b->n_tok, type)) return rc;
        if (int rc = check_apart(h, "k and q_out", k, k_stride, kvd, q_out, q_out_stride, E, b->n_tok, type)) return rc;
        if (int rc = check_apart(h, "v and q_out", v, v_stride, kvd, q_out, q_out_stride, E, b->n_tok, type)) return rc;
    }
    OnDevice on(h->device);
    if (int rc = on_device(h, on)) return rc;
    AppendArgs a{};
    if (h->rope) a.turn = h->rope->turn();
    a.b = device_batch(b);
    a.k = k;
    a.v = v;
    a.q = q;
    a.q_out = q_out;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.q_stride = q ? q_stride : 0;
    a.q_out_stride = q ? q_out_stride : 0;
    const size_t at = (size_t)layer * h->layer_elems() * type_bytes(c.cache_type);
    a.k_pool = (char *)h->k_pool + at;
    a.v_pool = (char *)h->v_pool + at;
    a.n_pages = c.n_pages;
    a.page_shift = h->page_shift;
    a.n_head = c.n_head;
    a.n_head_kv = c.n_head_kv;
    a.hd = c.head_dim;
    a.type = type;
    a.cache_type = c.cache_type;
    HIP_TRY(h, launch_append(a, pick_stream(h, stream)));
    return KORE_PAGED_OK;
}

int kore_paged_attend_dev(kore_paged_t h, int layer, const kore_paged_batch *b, int type, const void *q,
                          int64_t q_stride, void *out, int64_t out_stride, float scale, int window, void *workspace,
                          void *stream) {
    if (!h) return FAIL0(KORE_PAGED_E_INVALID, "null handle");
    if (int rc = check_batch(h, layer, b, type)) return rc;
    const kore_paged_config &c = h->cfg;
    const int64_t E = (int64_t)c.n_head * c.head_dim;
    if (int rc = check_stride(h, "q", q_stride, E, b->n_tok)) return rc;
    if (int rc = check_stride(h, "out", out_stride, E, b->n_tok)) return rc;
    if (window < 0) return fail(h, KORE_PAGED_E_INVALID, "negative window");
    if (scale != 0 && !(scale >= 1e-30f && scale <= 1e30f))
        return fail(h, KORE_PAGED_E_INVALID, "scale is neither 0 nor within 1e-30 .. 1e30");
    if ((uintptr_t)workspace % 16) return fail(h, KORE_PAGED_E_INVALID, "the workspace is not 16-byte aligned");
    if (b->n_seq == 0 || b->n_tok == 0) return KORE_PAGED_OK;
    if (!q || !out) return fail(h, KORE_PAGED_E_INVALID, "null buffer");
    if (int rc = check_aligned(h, "q", q, type)) return rc;
    if (int rc = check_aligned(h, "out", out, type)) return rc;
    if (int rc = check_overlap(h, q, q_stride, out, out_stride, E, b->n_tok, type)) return rc;
    OnDevice on(h->device);
    if (int rc = on_device(h, on)) return rc;
    AttendArgs a{};
    a.b = device_batch(b);
    a.q = q;
    a.out = out;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    const size_t at = (size_t)layer * h->layer_elems() * type_bytes(c.cache_type);
    a.k_pool = (const char *)h->k_pool + at;
    a.v_pool = (const char *)h->v_pool + at;
    a.n_pages = c.n_pages;
    a.page_shift = h->page_shift;
    a.n_head = c.n_head;
    a.n_head_kv = c.n_head_kv;
    a.hd = c.head_dim;
    a.window = window ? window : INT_MAX;
    a.scale = scale > 0 ? scale : (float)(1.0 / std::sqrt((double)c.head_dim));
    a.type = type;
    a.cache_type = c.cache_type;
    a.max_q = b->max_q;
    a.num_cu = h->num_cu;
    a.part = workspace ? (float *)workspace : h->part;
    HIP_TRY(h, launch_attend(a, pick_stream(h, stream)));
    return KORE_PAGED_OK;
}

size_t kore_paged_workspace_bytes(kore_paged_t h) { return h ? h->part_bytes : 0; }

int kore_paged_get_info(kore_paged_t h, kore_paged_info *info) {
    if (!h) return FAIL0(KORE_PAGED_E_INVALID, "null handle");
    if (!info) return fail(h, KORE_PAGED_E_INVALID, "null info");
    info->config = h->cfg;
    info->device = h->device;
    info->num_cu = h->num_cu;
    info->pool_bytes = h->pool_bytes();
    info->stream = (void *)h->stream;
    return KORE_PAGED_OK;
}

int kore_paged_sync(kore_paged_t h) {
    if (!h) return FAIL0(KORE_PAGED_E_INVALID, "null handle");
    OnDevice on(h->device);
    if (int rc = on_device(h, on)) return rc;
    HIP_TRY(h, hipStreamSynchronize(h->stream));
    return KORE_PAGED_OK;
}

const char *kore_paged_last_error(kore_paged_t h) { return h ? h->err : g_create_error; }

}  // extern "C"

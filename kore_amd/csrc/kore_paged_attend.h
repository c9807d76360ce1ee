// kore_paged_attend.h - what the paged-attention kernels share: how the work of
// a batch is cut into workgroups, the 16-bit parts of fp32 values, the online
// softmax.  Internal to libkore_paged.so.
//
// The work.  The new rows of a sequence and the n_head / n_head_kv = rep q-heads
// of a kv-head are one list, row r being token r / rep and head r % rep, cut into
// tiles of a kernel's TILE rows: every q-head of a tile reads the same K and V.
// A tile's keys are cut into splits of len keys, the same len for the whole
// batch, and a workgroup takes one (sequence, tile, split, kv-head).  What a
// sequence has is read from device memory, so every workgroup finds its place
// itself: its waves scan the sequences 64 at a time.
#pragma once

#include "kore_paged_device.h"

namespace kore_paged_gpu {

// Division by a number that a launch fixes: with 2^(s - 1) < d <= 2^s and m =
// floor(2^(31 + s) / d) + 1, x m / 2^(31 + s) exceeds x / d by less than 1 / d for
// 0 <= x < 2^31, so its whole part is the quotient.
struct Divisor {
    unsigned m;
    int shift;
    __host__ __device__ int of(int x) const { return (int)((unsigned long long)(unsigned)x * m >> shift); }
};
inline Divisor divisor(int d) {
    int s = 0;
    while ((1LL << s) < d) ++s;
    return Divisor{(unsigned)((1ULL << (31 + s)) / (unsigned)d + 1), 31 + s};
}

// How a launch cuts its work; every field is the host's.
struct Cut {
    int rep;         // q-heads of a kv-head
    Divisor by_rep, by_heads;   // by rep, and by the kv-heads
    int target;      // a split has all work / target, in tiles x keys, or more; 0: nothing is split
    int min_len;     // a split's fewest keys
};

// A launch over tiles; part_o [part][dim / 4][row] float4 and part_ml [part][row]
// (reference, as q.k, and sum) hold the splits of split tiles.
struct TileArgs {
    AttendArgs a;
    Cut cut;
    float scale_log2;        // scale log2(e), over 0
    bool q_wide, out_wide;   // q's rows can be read 16 bytes at a time, out's written four values at a time
    int places, parts;       // workgroups; parts that part_o and part_ml have
    float *part_o, *part_ml;
};

constexpr int kChunkRows = 128;   // of a tile of kore_paged_chunk.hip
inline int padded_dim(int hd) { return hd <= 64 ? 64 : hd <= 128 ? 128 : 256; }
hipError_t launch_chunk(const TileArgs &d, hipStream_t s);

namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef half_t half8 __attribute__((ext_vector_type(8)));
typedef bhalf_t bhalf8 __attribute__((ext_vector_type(8)));
typedef short short4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) short4_t lds_short4;

constexpr float kNone = -INFINITY;

// Lane l's and lane l ^ 16's, or l ^ 32's, value.  (The results are copied to
// integers before the bit casts: this hipcc compiles a bit cast of an element of
// the returned vector as its first element for either index.)
__device__ __forceinline__ float max16(float x) {
    const unsigned b = __builtin_bit_cast(unsigned, x);
    const auto r = __builtin_amdgcn_permlane16_swap(b, b, false, false);
    const unsigned r0 = r[0], r1 = r[1];
    return fmaxf(__builtin_bit_cast(float, r0), __builtin_bit_cast(float, r1));
}
__device__ __forceinline__ float max32(float x) {
    const unsigned b = __builtin_bit_cast(unsigned, x);
    const auto r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    const unsigned r0 = r[0], r1 = r[1];
    return fmaxf(__builtin_bit_cast(float, r0), __builtin_bit_cast(float, r1));
}
__device__ __forceinline__ float sum16(float x) {
    const unsigned b = __builtin_bit_cast(unsigned, x);
    const auto r = __builtin_amdgcn_permlane16_swap(b, b, false, false);
    const unsigned r0 = r[0], r1 = r[1];
    return __builtin_bit_cast(float, r0) + __builtin_bit_cast(float, r1);
}
__device__ __forceinline__ float sum32(float x) {
    const unsigned b = __builtin_bit_cast(unsigned, x);
    const auto r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    const unsigned r0 = r[0], r1 = r[1];
    return __builtin_bit_cast(float, r0) + __builtin_bit_cast(float, r1);
}
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// The sum of eight weights, two an instruction, onto s (products with 1: exact; one
// rounding each).
__device__ __forceinline__ float sum_weights(half8 w, float s) {
    typedef half_t half2_t __attribute__((ext_vector_type(2)));
    const half2_t one = {(half_t)1.f, (half_t)1.f};
#pragma unroll
    for (int i = 0; i < 8; i += 2) s = __builtin_amdgcn_fdot2(half2_t{w[i], w[i + 1]}, one, s, false);
    return s;
}
__device__ __forceinline__ float sum_weights(bhalf8 w, float s) {
    typedef bhalf_t bhalf2_t __attribute__((ext_vector_type(2)));
    const bhalf2_t one = {(bhalf_t)1.f, (bhalf_t)1.f};
#pragma unroll
    for (int i = 0; i < 8; i += 2) s = __builtin_amdgcn_fdot2_f32_bf16(bhalf2_t{w[i], w[i + 1]}, one, s, false);
    return s;
}

// A value that is equal in all lanes, in a scalar register.
__device__ __forceinline__ int scalar(int x) { return __builtin_amdgcn_readfirstlane(x); }

// ---- the cut -----------------------------------------------------------------

// A sequence's share of the cut.
struct Share {
    int tiles;      // of its rows, each for every kv-head
    int keys;       // that a tile can span
};

template <int TILE>
__device__ __forceinline__ Share share_of(const Batch &b, int s, int rep, int cap, int window, int &q0, int &n, int &kv) {
    q0 = min(max(b.q_start[s], 0), b.n_tok);
    n = min(max(b.q_start[s + 1], q0), b.n_tok) - q0;
    kv = max(b.kv_len[s], 0);
    Share r;
    r.tiles = (n * rep + TILE - 1) / TILE;
    // the rows of a tile span (TILE - 1) / rep + 2 tokens at most, and its first key is rounded down by up to 63
    const int held = max(0, min(kv, cap)), wide = (TILE - 1) / rep + 65;
    r.keys = window < held - wide ? window + wide : held;
    return r;
}

// A workgroup's place, equal in every lane.
struct Place {
    int seq, tile, split, n_split, head;
    int q0, n, kv;      // of the sequence: first row, rows, positions
    int len;            // keys of a split
    int part;           // number of the split (of the tile's first split, where all are one place) among the parts
};

// Inclusive sums over the wave in six DPP steps (four within rows of 16, then from
// row to row); the last lane's is the whole.
template <class T, int CTRL, int ROWS>
__device__ __forceinline__ T from_lane(T x) {
    return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, ROWS, 0xf, false));
}
template <class T>
__device__ __forceinline__ T prefix_sum(T x) {
    x += from_lane<T, 0x111, 0xf>(x);
    x += from_lane<T, 0x112, 0xf>(x);
    x += from_lane<T, 0x114, 0xf>(x);
    x += from_lane<T, 0x118, 0xf>(x);
    x += from_lane<T, 0x142, 0xa>(x);
    x += from_lane<T, 0x143, 0xc>(x);
    return x;
}
template <class T>
__device__ __forceinline__ T last_lane(T x) {
    return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 63));
}

// The place of number `id`, false where there is none.  Numbers run over the
// sequences, then a sequence's tiles from the last (which has the most keys),
// then its splits, then the kv-heads.  by_tile (the merge): over the split tiles
// alone, one number for all splits.
template <int TILE>
__device__ __forceinline__ bool place_of(const Batch &b, const Cut &c, int id, int nkv, int cap, int window, bool by_tile,
                                         Place &p) {
    const int lane = threadIdx.x & 63;
    int len = INT_MAX, q0 = 0, n = 0, kv = 0;
    const auto share = [&](int s0) {
        return s0 + lane < b.n_seq ? share_of<TILE>(b, s0 + lane, c.rep, cap, window, q0, n, kv) : Share{0, 0};
    };
    Share r = share(0);
    if (c.target) {
        // so that a tile of keys > len has keys / len + 1 < 2 keys / len splits: all splits are at most target and the
        // tiles, those of split tiles at most twice target
        float w = (float)r.tiles * (float)r.keys;
        for (int s0 = 64; s0 < b.n_seq; s0 += 64) {
            const Share t = share(s0);
            w += (float)t.tiles * (float)t.keys;
        }
        const float each = ceilf(last_lane(prefix_sum(w)) * (float)nkv / (float)c.target);
        len = max(c.min_len, ((int)fminf(each, 1e9f) + 63) & ~63);
    }
    int at = 0, part_at = 0;
    for (int s0 = 0; s0 < b.n_seq; s0 += 64) {
        if (b.n_seq > 64) r = share(s0);   // (one round of loads where all sequences have a lane)
        const int n_split = c.target ? max(1, (r.keys + len - 1) / len) : 1;
        const int all = r.tiles * n_split * nkv, part = n_split > 1 ? all : 0;
        const int mine = !by_tile ? all : n_split > 1 ? r.tiles * nkv : 0;
        const int upto = prefix_sum(mine), part_upto = c.target ? prefix_sum(part) : 0;
        const unsigned long long past = __ballot(at + upto > id);
        if (past) {
            const int l = __builtin_ctzll(past);
            const auto of = [&](int x) { return __builtin_amdgcn_readlane(x, l); };
            p.seq = scalar(s0 + l);
            p.n_split = of(n_split);
            p.q0 = of(q0);
            p.n = of(n);
            p.kv = of(kv);
            // the sequence's splits of equal length, in whole steps of 64 keys
            p.len = p.n_split > 1 ? scalar(((of(r.keys) + p.n_split - 1) / p.n_split + 63) & ~63) : INT_MAX;
            int i = id - at - of(upto) + of(mine);
            if (i < 0 || i >= of(mine)) return false;   // (sums past 2^31, of a q_start that is not ascending)
            const int pairs = c.by_heads.of(i);
            p.head = i - pairs * nkv;
            i = pairs;
            p.split = 0;
            if (!by_tile && p.n_split > 1) {
                i = scalar(pairs / p.n_split);
                p.split = pairs - i * p.n_split;
            }
            p.tile = scalar(of(r.tiles) - 1 - i);
            p.part = scalar(part_at + of(part_upto) - of(part) + (i * p.n_split + p.split) * nkv + p.head);
            return true;
        }
        at += last_lane(upto);
        part_at += last_lane(part_upto);
    }
    return false;
}

// The keys of a place: [lo, hi) of its split, of which none before seen_lo is seen; all
// rows of the tile see those in [all_lo, all_hi).
struct Keys {
    int lo, hi, seen_lo, all_lo, all_hi;
};

template <int TILE>
__device__ __forceinline__ Keys keys_of(const Place &p, const Cut &c, int cap, int window) {
    const int t0 = c.by_rep.of(p.tile * TILE), t1 = min(p.n - 1, c.by_rep.of(p.tile * TILE + TILE - 1));
    const int p0 = p.kv - p.n + t0, p1 = p.kv - p.n + t1;   // positions of the first and last row
    Keys k;
    k.seen_lo = window <= p0 ? p0 - window + 1 : 0;
    const int first = k.seen_lo & ~63, end = min(p1 + 1, cap);
    k.lo = first;
    k.hi = end;
    if (p.n_split > 1) {
        const long long a = first + (long long)p.split * p.len, z = a + p.len;
        k.lo = (int)min(a, (long long)INT_MAX - 64);
        k.hi = (int)min(z, (long long)end);
    }
    k.lo = scalar(k.lo);
    k.hi = scalar(k.hi);
    k.seen_lo = scalar(k.seen_lo);
    k.all_lo = scalar(window <= p1 ? p1 - window + 1 : 0);
    k.all_hi = scalar(min(p0 + 1, cap));
    return k;
}

// ---- 16-bit parts ------------------------------------------------------------

// The bits of x cut to 16 (bf16, towards zero).
__device__ __forceinline__ float bf16_cut(float x) {
    return __builtin_bit_cast(float, __builtin_bit_cast(unsigned, x) & 0xffff0000u);
}
__device__ __forceinline__ bool finite(float x) {
    return (__builtin_bit_cast(unsigned, x) & 0x7f800000u) != 0x7f800000u;
}

template <class C> struct Mma;   // the 16-bit matrix instructions of a type

template <> struct Mma<half_t> {
    typedef half8 vec8;
    static __device__ __forceinline__ floatx4 mul16(half8 a, half8 b, floatx4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ floatx16 mul32(half8 a, half8 b, floatx16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
    // Weights reach 2^14 (kLag and kBias below), so that those of 2^-20 of a row's largest are no subnormals.
    static constexpr float kBias = 6.0f;
};
template <> struct Mma<bhalf_t> {
    typedef bhalf8 vec8;
    static __device__ __forceinline__ floatx4 mul16(bhalf8 a, bhalf8 b, floatx4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ floatx16 mul32(bhalf8 a, bhalf8 b, floatx16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
    // Weights reach 1 and no more, so that a V near fp32's largest value overflows no sooner than it must.
    static constexpr float kBias = -8.0f;
};

// Parts that hold an fp32 value: two of fp16 (22 bits of a value near its row's
// largest), three of bf16 (24 bits).
template <class A, class C> struct Parts { static constexpr int q = 1, p = 1; };
template <> struct Parts<float, half_t> { static constexpr int q = 2, p = 2; };
template <> struct Parts<float, bhalf_t> { static constexpr int q = 3, p = 3; };

// The parts of one q value.  All have its sign and none is 0 where q is not, so
// that an infinity of K gives every product the same sign: an infinite score, as
// in exact arithmetic, not NaN.  (A part set to its least value adds 2^-30 of the
// value, or, for fp16, 2^-37 of the row's largest.)
// (An infinite or NaN q makes its row NaN, in parts as in exact arithmetic.)
template <int N>
__device__ __forceinline__ void split_q(float x, bhalf_t (&part)[N]) {
    const float h = bf16_cut(x), least = h * 0x1p-30f, r = x - h, m = bf16_cut(r), l = r - m;
    const auto upper = [](float y) { return __builtin_bit_cast(bhalf_t, (unsigned short)(__builtin_bit_cast(unsigned, y) >> 16)); };
    part[0] = upper(x);
    if constexpr (N == 3) {
        part[1] = upper(m == 0.f ? least : m);
        part[2] = upper(l == 0.f ? least : l);
    }
}
template <int N>
__device__ __forceinline__ void split_q(float x, half_t (&part)[N]) {
    const auto cut = __builtin_amdgcn_cvt_pkrtz(x, x);
    const half_t least = (half_t)__builtin_copysignf(0x1p-24f, x);
    half_t h = (half_t)cut[0];
    const half_t l = (half_t)(x - (float)h);
    if (x != 0.f && (float)h == 0.f) h = least;
    part[0] = h;
    if constexpr (N == 2) part[1] = x != 0.f && (float)l == 0.f ? least : l;
}

// Parts of a weight, each the nearest.
template <int N, class C>
__device__ __forceinline__ void split_p(float x, C (&part)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        part[i] = (C)x;
        if (i + 1 < N) x -= (float)part[i];
    }
}

// A power of two `to` that brings |x| <= big to 2^13 .. 2^14 (2^126 at most: big under
// 2^-112 stays smaller), and the exponent of its inverse.  big >= 0, no NaN.
__device__ __forceinline__ int unit_of(float big, float &to) {
    const unsigned e = __builtin_bit_cast(unsigned, big) >> 23;
    const unsigned up = min(267u - e, 253u);   // 2^(up - 127) 2^(e - 127) = 2^13
    to = __builtin_bit_cast(float, up << 23);
    return 127 - (int)up;
}
__device__ __forceinline__ float power(int e) { return __builtin_bit_cast(float, (unsigned)(127 + e) << 23); }   // -126 .. 127
// scale log2(e) of scores in a unit of q: over 0 and finite (a product with it is used
// with differences of such scores, 0 or 2^-48 at least), so that 0 stays 0.
__device__ __forceinline__ float scale_of(float scale_log2, float unit) {
    return fminf(fmaxf(scale_log2 * unit, 0x1p-126f), 0x1p126f);
}

// ---- the softmax ---------------------------------------------------------------

// A row's weights are 2^((score - ref) s + kBias), score and reference in the units of
// the products, s = scale log2(e) in those.  The difference comes first: it is exact
// for scores near the reference, whatever their size, and what rounding s costs grows
// with the distance from it, as the weights fall.  s is over 0, so that a score of
// -inf (one that is masked) needs no test.  The reference follows the row's largest
// score: it moves when that passes it by kLag, so that the accumulators are rescaled
// rarely.
constexpr float kLag = 8.0f;

// What a state with the reference ref counts beside one with a reference of `to`, the
// largest of all: 0 where there is none, and the smallest float where it is less than that,
// so that an infinite sum stays infinite.
__device__ __forceinline__ float share_at(float ref, float to, float s) {
    return ref == kNone ? 0.f : fmaxf(exp2_((ref - to) * s), 0x1p-149f);
}

// Infinities of V.  A key whose score is over -inf has a weight, however small, and hands an
// infinity or NaN of its V to the row's dim; one whose score is -inf has none and hands on
// nothing, and so does one that the row does not attend.  Products know less: a weight of 0,
// or a part of one that is 0 or of the other sign, times an infinity is NaN.  But they leave
// no sum finite that should not be.  So the keys are gone through as if V were finite, and
// where a sum is not, a second time by a CAREFUL pass, which takes infinities and NaN out of
// the products, notes them, and adds them to the sums by the scores.  (us, finite / a NaN in
// one V row, 28/4/128: 2048 fp16 rows 57 / 190, 512 fp32 rows over 32749 bf16 keys 2.2 times;
// 32 tokens over up to 8192 fp16 keys, a NaN in one sequence's, 59 / 112.)

// Whether a sum is not finite.
template <class V, int N>
__device__ __forceinline__ bool not_finite(const V (&o)[N]) {
    float t = 0;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int x = 0; x < (int)(sizeof(V) / sizeof(float)); ++x) t = fmaf(o[i][x], 0.f, t);
    return t != t;
}
// Which of eight dims are +inf, or -inf (a NaN: both); they become 0.
template <class T, class V>
__device__ __forceinline__ void take_out(V &v, unsigned &up, unsigned &down) {
    up = down = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float x = to_f32((T)v[i]);
        if (!finite(x)) {
            if (!(x < 0.f)) up |= 1u << i;
            if (!(x > 0.f)) down |= 1u << i;
            v[i] = (T)0.f;
        }
    }
}

// The rescale, where a score passes the reference by kLag (or is the first).
template <bool CAREFUL, class V, int N>
__device__ __forceinline__ void follow(float top, float &ref, float &sum, float s, V (&o)[N]) {
    const bool moves = (top - ref) * s > kLag;
    if (__any(moves)) {
        const float next = moves ? top : ref;
        const float f = !moves ? 1.f : CAREFUL ? share_at(ref, next, s) : exp2_((ref - next) * s);
        sum *= f;
#pragma unroll
        for (int i = 0; i < N; ++i) o[i] *= f;
        ref = next;
    }
}

// What a lane knows of its row (column l % 16 of the products).
struct Row {
    int lo, hi;      // sees keys [lo, hi)
    bool real;
    int token, head;
};

__device__ __forceinline__ Row row_of(const Place &p, int r, const Cut &c, int cap, int window) {
    Row x;
    x.real = r < p.n * c.rep;
    x.token = c.by_rep.of(r);
    x.head = p.head * c.rep + (r - x.token * c.rep);
    const int pos = p.kv - p.n + x.token;
    x.lo = window <= pos ? pos - window + 1 : 0;
    x.hi = x.real ? min(pos + 1, cap) : 0;
    return x;
}

// N pieces of a row of q, 8 values each, piece t from dim first + step t: all requested
// before one is used.  What is not there (a row past the last, dims past the head) is
// something else of the row, for zero_q to clear when the rest has arrived.
template <class A>
__device__ __forceinline__ const A *q_row_of(const AttendArgs &a, const Place &p, const Row &row) {
    return (const A *)a.q + (size_t)(row.real ? p.q0 + row.token : p.q0) * a.q_stride + (size_t)(row.real ? row.head : 0) * a.hd;
}
template <class A>
__device__ __forceinline__ void load_piece(const A *src, bool wide, A (&x)[8]) {
    constexpr int kPer = 16 / sizeof(A);
    if (wide) {
        typedef A piece __attribute__((ext_vector_type(kPer)));
#pragma unroll
        for (int i = 0; i < 8; i += kPer) {
            const piece v = *reinterpret_cast<const piece *>(src + i);
#pragma unroll
            for (int j = 0; j < kPer; ++j) x[i + j] = v[j];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = src[i];
    }
}
template <int N, class A>
__device__ __forceinline__ void load_q(const AttendArgs &a, const Place &p, const Row &row, bool wide, int first, int step,
                                       A (&x)[N][8]) {
    const A *const src = q_row_of<A>(a, p, row);
    if (wide) {
#pragma unroll
        for (int t = 0; t < N; ++t) load_piece(src + min(first + step * t, a.hd - 8), true, x[t]);
    } else {
#pragma unroll
        for (int t = 0; t < N; ++t) load_piece(src + min(first + step * t, a.hd - 8), false, x[t]);
    }
}
template <int N, class A>
__device__ __forceinline__ void zero_q(const AttendArgs &a, const Row &row, int first, int step, A (&x)[N][8]) {
#pragma unroll
    for (int t = 0; t < N; ++t)
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (!row.real || first + step * t >= a.hd) x[t][i] = (A)0.f;
}

// The pages of a wave's 16-key groups, 64 at a time in the lanes of a register and
// the next 64 in another, requested long before they are needed.
struct PageRun {
    int now, ahead;
    // group: this lane's
    static __device__ __forceinline__ int load(const AttendArgs &a, const int *table, int group, int hi) {
        const int key = group * 16, at = key >> a.page_shift;
        int p = -1;
        if (key >= 0 && key < hi && at < a.b.pages_stride) p = table[at];   // (a number past the keys may wrap)
        return p < a.n_pages ? p : -1;   // negative: none
    }
    __device__ __forceinline__ int get(int i) const { return __builtin_amdgcn_readlane(now, i); }
};

// 4 elements of a transposed block of LDS: lane i of 16 gives the address of
// elements 4 (i % 4) .. + 3 of row i / 4, and gets element i of the four rows
// (checked on the GPU).
template <class V4>
__device__ __forceinline__ V4 read_transposed(const void *lds) {
    return __builtin_bit_cast(V4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4 *)lds));
}

}  // namespace
}  // namespace kore_paged_gpu

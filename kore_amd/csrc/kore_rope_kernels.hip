// kore_rope_kernels.hip - rotary positions of rows, and the append of rotated
// rows to a paged cache (gfx950).
//
// Both are bound by memory: 12 flops a pair beside 16 bytes (fp32) of traffic,
// and a cosine and sine for each pair of a row, shared by its heads.
#include "kore_paged_device.h"

#include <algorithm>

namespace kore_paged_gpu {
namespace {

constexpr int kThreads = 256;

// m cos(pos f) and m sin(pos f) to within half a float step.  The angle is
// exact (24 + 31 bits) but for one rounding of its 53rd bit; it is reduced by the
// nearest multiple k of pi/2 held as the sum of two doubles, each step one fma,
// so that r is off by some 2^-50 for any int position; then the power series
// about 0 up to where the next term, (pi/4)^15 / 15! = 2e-14 of the sine, is
// nothing beside a float's half step of 3e-8.  fp32 arithmetic would lose the
// angle itself: at position 131072 a float's step is 2^-7.
__device__ __forceinline__ float2 cos_sin(int pos, float freq, double size) {
    constexpr double kHi = 1.57079632679489655800e+00, kLo = 6.12323399573676603587e-17;
    const double a = (double)pos * (double)freq;
    const double k = __builtin_rint(a * 0.63661977236758134308);
    double r = __builtin_fma(-k, kHi, a);
    r = __builtin_fma(-k, kLo, r);
    const double z = r * r;
    double s = 1.0 / 6227020800.0;
    s = __builtin_fma(s, z, -1.0 / 39916800.0);
    s = __builtin_fma(s, z, 1.0 / 362880.0);
    s = __builtin_fma(s, z, -1.0 / 5040.0);
    s = __builtin_fma(s, z, 1.0 / 120.0);
    s = __builtin_fma(s, z, -1.0 / 6.0);
    s = __builtin_fma(s * z, r, r);
    double c = -1.0 / 87178291200.0;
    c = __builtin_fma(c, z, 1.0 / 479001600.0);
    c = __builtin_fma(c, z, -1.0 / 3628800.0);
    c = __builtin_fma(c, z, 1.0 / 40320.0);
    c = __builtin_fma(c, z, -1.0 / 720.0);
    c = __builtin_fma(c, z, 1.0 / 24.0);
    c = __builtin_fma(c, z, -0.5);
    c = __builtin_fma(c, z, 1.0);
    const int q = (int)((long long)k & 3);
    double cc = (q & 1) ? s : c, ss = (q & 1) ? c : s;
    if (q == 1 || q == 2) cc = -cc;
    if (q >= 2) ss = -ss;
    return make_float2((float)(size * cc), (float)(size * ss));
}

// One unit of a head: V pairs, or 2 V dims behind the rotated ones, which are
// copied.  cs: the row's (cos, sin) of every pair.
template <int V, class T, class O>
__device__ __forceinline__ void turn_unit(const T *x, O *y, int unit, int rot, bool interleaved, const float2 *cs,
                                          float sign) {
#pragma clang fp contract(off)
    const int n_turn = rot / (2 * V);
    const bool turned = unit < n_turn, near = !turned || interleaved;
    const int at0 = near ? unit * 2 * V : unit * V, at1 = near ? at0 + V : at0 + rot / 2;
    T a[V], b[V];
    load_n<V>(x + at0, a, true);
    load_n<V>(x + at1, b, true);
    float u[2 * V], w[2 * V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        u[i] = to_f32(a[i]);
        u[V + i] = to_f32(b[i]);
    }
    if (!turned) {
#pragma unroll
        for (int i = 0; i < 2 * V; ++i) w[i] = u[i];
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float2 c = cs[unit * V + i];
            const float sn = sign * c.y;
            const int p0 = interleaved ? 2 * i : i, p1 = interleaved ? 2 * i + 1 : V + i;
            const float e = u[p0] * c.x, f = u[p1] * sn, g = u[p0] * sn, h = u[p1] * c.x;
            w[p0] = e - f;
            w[p1] = g + h;
        }
    }
    O r[V], t[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        r[i] = (O)w[i];
        t[i] = (O)w[V + i];
    }
    store_n<V>(y + at0, r, true);
    store_n<V>(y + at1, t, true);
}

// The (cos, sin) of a block's row, one pair a thread.
__device__ __forceinline__ void stage_turn(const Turn &t, int pos, float2 *cs) {
    for (int i = threadIdx.x; i < t.rot / 2; i += kThreads) cs[i] = cos_sin(pos, t.freq[i], t.size);
    __syncthreads();
}

// A block takes one row; its threads are laid over (head, unit).
template <class T, int V>
__global__ __launch_bounds__(kThreads) void rope_kernel(RopeArgs a) {
    __shared__ float2 cs[kMaxRot / 2];
    const int row = blockIdx.x;
    stage_turn(a.turn, a.pos[row], cs);
    const T *x = (const T *)a.x + (size_t)row * a.x_stride;
    T *y = (T *)a.out + (size_t)row * a.out_stride;
    const int units = a.hd / (2 * V), total = units * a.n_head;
    for (int i = threadIdx.x; i < total; i += kThreads) {
        const int head = i / units, unit = i - head * units;
        turn_unit<V>(x + (size_t)head * a.hd, y + (size_t)head * a.hd, unit, a.turn.rot, a.turn.interleaved, cs,
                     (float)a.sign);
    }
}

// A block takes one row: its k heads into the pool, its v heads into the pool,
// and its q heads (where there are any).
template <class T, class C, int V>
__global__ __launch_bounds__(kThreads) void append_kernel(AppendArgs a) {
    __shared__ float2 cs[kMaxRot / 2];
    const int row = blockIdx.x;
    const int seq = seq_of_row(a.b, row);
    if (seq >= a.b.n_seq || row < a.b.q_start[seq]) return;
    const int pos = a.b.kv_len[seq] - (a.b.q_start[seq + 1] - row);
    const int at = pos >> a.page_shift;
    const int page = pos >= 0 && at < a.b.pages_stride ? a.b.pages[(size_t)seq * a.b.pages_stride + at] : -1;
    const bool stored = page >= 0 && page < a.n_pages;
    stage_turn(a.turn, pos, cs);
    const int units = a.hd / (2 * V), nq = a.q ? a.n_head : 0, total = units * (nq + 2 * a.n_head_kv);
    const int slot = pos & ((1 << a.page_shift) - 1);
    for (int i = threadIdx.x; i < total; i += kThreads) {
        int head = i / units;
        const int unit = i - head * units;
        if (head < nq) {
            turn_unit<V>((const T *)a.q + (size_t)row * a.q_stride + (size_t)head * a.hd,
                         (T *)a.q_out + (size_t)row * a.q_out_stride + (size_t)head * a.hd, unit, a.turn.rot,
                         a.turn.interleaved, cs, 1.0f);
            continue;
        }
        if (!stored) continue;
        head -= nq;
        const bool is_v = head >= a.n_head_kv;
        if (is_v) head -= a.n_head_kv;
        const size_t to = ((((size_t)page * a.n_head_kv + head) << a.page_shift) + slot) * a.hd;
        const T *x = is_v ? (const T *)a.v + (size_t)row * a.v_stride : (const T *)a.k + (size_t)row * a.k_stride;
        turn_unit<V>(x + (size_t)head * a.hd, (C *)(is_v ? a.v_pool : a.k_pool) + to, unit, is_v ? 0 : a.turn.rot,
                     a.turn.interleaved, cs, 1.0f);
    }
}

// Four values at once where rows, heads and the two parts of a head start at
// multiples of four, one otherwise.
bool fours(int rot, int hd) { return rot % 8 == 0 && (hd - rot) % 8 == 0; }
template <class... P>
bool aligned(int bytes, P... p) {
    return ((((uintptr_t)p) % (4 * (size_t)bytes) == 0) && ...);
}

}  // namespace

hipError_t launch_rope(const RopeArgs &a, hipStream_t s) {
    const bool v4 = fours(a.turn.rot, a.hd) && a.x_stride % 4 == 0 && a.out_stride % 4 == 0 &&
                    aligned(type_bytes(a.type), a.x, a.out);
#define KORE_ROPE_CASE(T)                                                             \
    do {                                                                              \
        if (v4) rope_kernel<T, 4><<<a.n_tok, kThreads, 0, s>>>(a);                    \
        else rope_kernel<T, 1><<<a.n_tok, kThreads, 0, s>>>(a);                       \
    } while (0)
    if (a.type == kF32) KORE_ROPE_CASE(float);
    else if (a.type == kF16) KORE_ROPE_CASE(half_t);
    else KORE_ROPE_CASE(bhalf_t);
#undef KORE_ROPE_CASE
    return hipGetLastError();
}

hipError_t launch_append(const AppendArgs &a, hipStream_t s) {
    const int tb = type_bytes(a.type), cb = type_bytes(a.cache_type);
    const bool v4 = fours(a.turn.rot, a.hd) && a.k_stride % 4 == 0 && a.v_stride % 4 == 0 &&
                    (!a.q || (a.q_stride % 4 == 0 && a.q_out_stride % 4 == 0)) &&
                    aligned(tb, a.k, a.v, a.q, a.q_out) && aligned(cb, a.k_pool, a.v_pool);
#define KORE_APPEND_CASE(T, C)                                                        \
    do {                                                                              \
        if (v4) append_kernel<T, C, 4><<<a.b.n_tok, kThreads, 0, s>>>(a);             \
        else append_kernel<T, C, 1><<<a.b.n_tok, kThreads, 0, s>>>(a);                \
    } while (0)
    if (a.type == kF32 && a.cache_type == kF32) KORE_APPEND_CASE(float, float);
    else if (a.type == kF32 && a.cache_type == kF16) KORE_APPEND_CASE(float, half_t);
    else if (a.type == kF32) KORE_APPEND_CASE(float, bhalf_t);
    else if (a.type == kF16) KORE_APPEND_CASE(half_t, half_t);
    else KORE_APPEND_CASE(bhalf_t, bhalf_t);
#undef KORE_APPEND_CASE
    return hipGetLastError();
}

}  // namespace kore_paged_gpu

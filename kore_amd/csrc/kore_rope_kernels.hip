// kore_rope_kernels.hip - rotary positions of rows, and the append of rotated
// rows to a paged cache (gfx950).
//
// Both are bound by memory: 6 flops a pair beside 16 bytes (fp32) of traffic,
// and a cosine and sine for each pair of a row, shared by its heads.  4096 bf16 rows of
// 36 heads of 96: 11.8 us, 4.8 TB/s (a large copy: 5.1); three prompts' 1777 rows of
// 28/4/128 into a bf16 cache: 15.1 us, 5.2 TB/s.  Few rows are a launch and three
// dependent rounds of memory: one row of 32 heads 2.4 us, an append of 16 rows 3.5.
#include "kore_paged_device.h"

#include <algorithm>

namespace kore_paged_gpu {
namespace {

constexpr int kThreads = 256;

// m cos(pos f) and m sin(pos f) to within half a float step.  The angle is
// held as two doubles (24 + 31 bits) and reduced by the nearest multiple k of pi/2,
// itself the sum of two doubles, each step one fma, so that r is off by some 2^-50
// for any int position and frequencies up to 2^20; then the power series
// about 0 up to where the next term, (pi/4)^15 / 15! = 2e-14 of the sine, is
// nothing beside a float's half step of 3e-8.  fp32 arithmetic would lose the
// angle itself: at position 131072 a float's step is 2^-7.
__device__ __forceinline__ float2 cos_sin(int pos, float freq, double size) {
    constexpr double kHi = 1.57079632679489655800e+00, kLo = 6.12323399573676603587e-17;
    const double a = (double)pos * (double)freq;
    const double k = __builtin_rint(a * 0.63661977236758134308);
    double r = __builtin_fma(-k, kHi, a);
    r = __builtin_fma(-k, kLo, r) + __builtin_fma((double)pos, (double)freq, -a);
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

// One unit of a head: V pairs, or 2 V dims behind the rotated ones, which are copied.
// Where its two halves lie, and the turn; cs: the row's (cos, sin) of every pair.
template <int V>
struct Unit {
    int at0, at1;
    bool turned;
    __device__ __forceinline__ Unit(int unit, int rot, bool interleaved) {
        turned = unit < rot / (2 * V);
        const bool near = !turned || interleaved;
        at0 = near ? unit * 2 * V : unit * V;
        at1 = near ? at0 + V : at0 + rot / 2;
    }
};
template <int V, class T, class O>
__device__ __forceinline__ void turn_unit(const Unit<V> &where, const T (&a)[V], const T (&b)[V], O *y, int unit,
                                          bool interleaved, const float2 *cs, float sign) {
#pragma clang fp contract(off)
    float u[2 * V], w[2 * V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        u[i] = to_f32(a[i]);
        u[V + i] = to_f32(b[i]);
    }
    if (!where.turned) {
#pragma unroll
        for (int i = 0; i < 2 * V; ++i) w[i] = u[i];
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float2 c = cs[unit * V + i];
            const float sn = sign * c.y;
            const float u0 = interleaved ? u[2 * i] : u[i], u1 = interleaved ? u[2 * i + 1] : u[V + i];
            const float e = u0 * c.x, f = u1 * sn, g = u0 * sn, h = u1 * c.x;
            w[interleaved ? 2 * i : i] = e - f;
            w[interleaved ? 2 * i + 1 : V + i] = g + h;
        }
    }
    O r[V], t[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        r[i] = (O)w[i];
        t[i] = (O)w[V + i];
    }
    store_n<V>(y + where.at0, r, true);
    store_n<V>(y + where.at1, t, true);
}

// The (cos, sin) of a block's row, one pair a thread.
__device__ __forceinline__ void stage_turn(const Turn &t, int pos, float2 *cs) {
    for (int i = threadIdx.x; i < t.rot / 2; i += kThreads) cs[i] = cos_sin(pos, t.freq[i], t.size);
    __syncthreads();
}

// A block takes one row's units, or a gridDim.y-th of them (of few rows, so that a
// thread has about one); a thread's first kEarly are requested before the turn is
// computed.
constexpr int kEarly = 3;

template <class T, int V, bool INTER>
__global__ __launch_bounds__(kThreads) void rope_kernel(RopeArgs a) {
    __shared__ float2 cs[kMaxRot / 2];
    const int row = blockIdx.x;
    const T *x = (const T *)a.x + (size_t)row * a.x_stride;
    T *y = (T *)a.out + (size_t)row * a.out_stride;
    const int units = a.hd / (2 * V), total = units * a.n_head, step = kThreads * gridDim.y;
    const int first = blockIdx.y * kThreads + threadIdx.x;
    T va[kEarly][V], vb[kEarly][V];
    const auto request = [&](int j, int i) {
        const int head = i / units;
        const Unit<V> u(i - head * units, a.turn.rot, INTER);
        load_n<V>(x + (size_t)head * a.hd + u.at0, va[j]);
        load_n<V>(x + (size_t)head * a.hd + u.at1, vb[j]);
    };
#pragma unroll
    for (int j = 0; j < kEarly; ++j)
        if (first + j * step < total) request(j, first + j * step);
    stage_turn(a.turn, a.pos[row], cs);
    for (int i0 = first; i0 < total; i0 += kEarly * step) {
#pragma unroll
        for (int j = 0; j < kEarly; ++j) {
            const int i = i0 + j * step, head = i / units, unit = i - head * units;
            if (i < total) {
                if (i0 != first) request(j, i);
                turn_unit<V>(Unit<V>(unit, a.turn.rot, INTER), va[j], vb[j], y + (size_t)head * a.hd, unit, INTER, cs, (float)a.sign);
            }
        }
    }
}

// k heads into the pool, v heads into the pool, and q heads (where there are any).
template <class T, class C, int V, bool INTER>
__global__ __launch_bounds__(kThreads) void append_kernel(AppendArgs a) {
    __shared__ float2 cs[kMaxRot / 2];
    const int row = blockIdx.x, lane = threadIdx.x & 63;
    const int units = a.hd / (2 * V), nq = a.q ? a.n_head : 0, total = units * (nq + 2 * a.n_head_kv);
    const int step = kThreads * gridDim.y, first = blockIdx.y * kThreads + threadIdx.x;
    T va[kEarly][V], vb[kEarly][V];
    // head nq + j: k's j, then v's
    const auto request = [&](int j, int i) {
        const int head = i / units, kv = head - nq;
        const bool is_v = kv >= a.n_head_kv;
        const Unit<V> u(i - head * units, is_v ? 0 : a.turn.rot, INTER);
        const T *src = head < nq ? (const T *)a.q + (size_t)row * a.q_stride + (size_t)head * a.hd
                     : is_v ? (const T *)a.v + (size_t)row * a.v_stride + (size_t)(kv - a.n_head_kv) * a.hd
                            : (const T *)a.k + (size_t)row * a.k_stride + (size_t)kv * a.hd;
        load_n<V>(src + u.at0, va[j]);
        load_n<V>(src + u.at1, vb[j]);
    };
#pragma unroll
    for (int j = 0; j < kEarly; ++j)
        if (first + j * step < total) request(j, first + j * step);
    // the row's sequence, each wave for itself, 64 at a time: one round of loads
    int seq = -1, pos = 0;
    for (int s0 = 0; s0 < a.b.n_seq && seq < 0; s0 += 64) {
        const int s = s0 + lane;
        int from = 0, to = 0, len = 0;
        if (s < a.b.n_seq) {
            from = a.b.q_start[s];
            to = a.b.q_start[s + 1];
            len = a.b.kv_len[s];
        }
        const unsigned long long here = __ballot(from <= row && row < to);
        if (here) {
            const int l = __builtin_ctzll(here);
            seq = s0 + l;
            pos = __builtin_amdgcn_readlane(len, l) - (__builtin_amdgcn_readlane(to, l) - row);
        }
    }
    if (seq < 0) return;
    const int at = pos >> a.page_shift;
    const int page = pos >= 0 && at < a.b.pages_stride ? a.b.pages[(size_t)seq * a.b.pages_stride + at] : -1;
    stage_turn(a.turn, pos, cs);
    const bool stored = page >= 0 && page < a.n_pages;
    const int slot = pos & ((1 << a.page_shift) - 1);
    for (int i0 = first; i0 < total; i0 += kEarly * step) {
#pragma unroll
        for (int j = 0; j < kEarly; ++j) {
            const int i = i0 + j * step, head = i / units, unit = i - head * units;
            if (i >= total) continue;
            if (i0 != first) request(j, i);
            if (head < nq) {
                turn_unit<V>(Unit<V>(unit, a.turn.rot, INTER), va[j], vb[j],
                             (T *)a.q_out + (size_t)row * a.q_out_stride + (size_t)head * a.hd, unit, INTER, cs, 1.0f);
            } else if (stored) {
                const bool is_v = head - nq >= a.n_head_kv;
                const int kv = is_v ? head - nq - a.n_head_kv : head - nq;
                const size_t to = ((((size_t)page * a.n_head_kv + kv) << a.page_shift) + slot) * a.hd;
                turn_unit<V>(Unit<V>(unit, is_v ? 0 : a.turn.rot, INTER), va[j], vb[j], (C *)(is_v ? a.v_pool : a.k_pool) + to,
                             unit, INTER, cs, 1.0f);
            }
        }
    }
}

// Workgroups that share a row: as many as give a thread one unit while the launch has
// less than four a CU or so (us, with them / one a row, 32 heads of 128: 1 row 2.39 /
// 2.61, 16 rows 3.07 / 3.50, 333 rows 3.90 / 4.23; an append of 16 rows 3.39 / 4.54).
dim3 row_grid(int n_tok, int total) {
    const int most = (total + kThreads - 1) / kThreads;
    return dim3((unsigned)n_tok, (unsigned)std::clamp(1024 / n_tok, 1, most));
}

// Four values at once where rows, heads and the two parts of a head start at
// multiples of four, one otherwise (4096 rows of 36 heads of 96: 12.0 us, one value at a
// time 16.7).
bool fours(int rot, int hd) { return rot % 8 == 0 && (hd - rot) % 8 == 0; }
template <class... P>
bool aligned(int bytes, P... p) {
    return ((((uintptr_t)p) % (4 * (size_t)bytes) == 0) && ...);
}

}  // namespace

hipError_t launch_rope(const RopeArgs &a, hipStream_t s) {
    const bool v4 = fours(a.turn.rot, a.hd) && a.x_stride % 4 == 0 && a.out_stride % 4 == 0 &&
                    aligned(type_bytes(a.type), a.x, a.out);
    const dim3 grid = row_grid(a.n_tok, a.hd / (v4 ? 8 : 2) * a.n_head);
#define KORE_ROPE_CASE(T)                                                                         \
    do {                                                                                          \
        if (v4 && a.turn.interleaved) return launch(rope_kernel<T, 4, true>, grid, kThreads, 0, s, a);       \
        else if (v4) return launch(rope_kernel<T, 4, false>, grid, kThreads, 0, s, a);                       \
        else if (a.turn.interleaved) return launch(rope_kernel<T, 1, true>, grid, kThreads, 0, s, a);        \
        else return launch(rope_kernel<T, 1, false>, grid, kThreads, 0, s, a);                               \
    } while (0)
    if (a.type == kF32) KORE_ROPE_CASE(float);
    else if (a.type == kF16) KORE_ROPE_CASE(half_t);
    else KORE_ROPE_CASE(bhalf_t);
#undef KORE_ROPE_CASE
}

hipError_t launch_append(const AppendArgs &a, hipStream_t s) {
    const int tb = type_bytes(a.type), cb = type_bytes(a.cache_type);
    const bool v4 = fours(a.turn.rot, a.hd) && a.k_stride % 4 == 0 && a.v_stride % 4 == 0 &&
                    (!a.q || (a.q_stride % 4 == 0 && a.q_out_stride % 4 == 0)) &&
                    aligned(tb, a.k, a.v, a.q, a.q_out) && aligned(cb, a.k_pool, a.v_pool);
    const dim3 grid = row_grid(a.b.n_tok, a.hd / (v4 ? 8 : 2) * ((a.q ? a.n_head : 0) + 2 * a.n_head_kv));
#define KORE_APPEND_CASE(T, C)                                                                    \
    do {                                                                                          \
        if (v4 && a.turn.interleaved) return launch(append_kernel<T, C, 4, true>, grid, kThreads, 0, s, a);  \
        else if (v4) return launch(append_kernel<T, C, 4, false>, grid, kThreads, 0, s, a);                  \
        else if (a.turn.interleaved) return launch(append_kernel<T, C, 1, true>, grid, kThreads, 0, s, a);   \
        else return launch(append_kernel<T, C, 1, false>, grid, kThreads, 0, s, a);                          \
    } while (0)
    if (a.type == kF32 && a.cache_type == kF32) KORE_APPEND_CASE(float, float);
    else if (a.type == kF32 && a.cache_type == kF16) KORE_APPEND_CASE(float, half_t);
    else if (a.type == kF32) KORE_APPEND_CASE(float, bhalf_t);
    else if (a.type == kF16) KORE_APPEND_CASE(half_t, half_t);
    else KORE_APPEND_CASE(bhalf_t, bhalf_t);
#undef KORE_APPEND_CASE
}

}  // namespace kore_paged_gpu

// kore_paged_chunk.hip - paged attention of many rows (chunks of prompts; gfx950).
//
// A tile is 128 rows of a kv-head's (token, q-head) list, 32 for each of four waves,
// and passes over its keys 64 (or 32) at a time through LDS: the flops of a key,
// 512 head_dim for its 4 head_dim bytes, put the kernel between the matrix cores and
// the vector units that make the weights.  Two such teams of waves share a CU as one
// workgroup, each with every other step of the keys, and join their sums through LDS at
// the end: what a step waits for is a wave's own chain of loads, products and weights,
// so a tile takes half as long as with one team, and the long tiles of a causal chunk
// are what the launch waits for (7B, 2048 rows: 56 us with the same waves in two
// workgroups of four).
#include "kore_paged_attend.h"

namespace kore_paged_gpu {
namespace {

constexpr int kWaves = 4, kRows = kChunkRows;   // of a team

// How a (row type, cache type) is computed: fp32 caches in three bf16 parts of
// everything, whose products of parts i and j with i + j < 3 hold 24 bits.
template <class A, class S> struct Form {
    typedef S C;
    static constexpr int qp = Parts<A, S>::q, kp = 1, pp = Parts<A, S>::p;
};
template <> struct Form<float, float> {
    typedef bhalf_t C;
    static constexpr int qp = 3, kp = 3, pp = 3;
};

// What a tile's shape asks of LDS and registers: keys of a step; buffers; teams of a
// workgroup (a CU holds one workgroup).
template <class A, class S, int HDP> struct Shape {
    static constexpr bool parts = Form<A, S>::qp > 1;
    static constexpr int keys = parts ? 32 : 64;
    static constexpr int buffers = HDP <= 128 && Form<A, S>::kp == 1 ? 2 : 1;
    static constexpr int teams = HDP <= 128 ? 2 : 1, threads = 64 * kWaves * teams;
};

// Three bf16 parts of an fp32 value of the cache; an infinity or NaN is all in the first.
__device__ __forceinline__ void split_kv(float x, bhalf_t (&part)[3]) {
    const float h = bf16_cut(x), r = x - h, m = bf16_cut(r), l = r - m;
    const bool f = finite(x);
    part[0] = f ? (bhalf_t)h : (bhalf_t)x;
    part[1] = f ? (bhalf_t)m : (bhalf_t)0.f;
    part[2] = f ? (bhalf_t)l : (bhalf_t)0.f;
}

template <class A, class S, int HDP>
__global__ __launch_bounds__((Shape<A, S, HDP>::threads), 1) void chunk_kernel(TileArgs d) {
    typedef typename Form<A, S>::C C;
    typedef typename Mma<C>::vec8 vec8;
    typedef C vec4 __attribute__((ext_vector_type(4)));
    constexpr int QP = Form<A, S>::qp, KP = Form<A, S>::kp, PP = Form<A, S>::pp;
    constexpr int kKeys = Shape<A, S, HDP>::keys, kBuffers = Shape<A, S, HDP>::buffers, kTeams = Shape<A, S, HDP>::teams;
    constexpr int KS = HDP / 16, DT = HDP / 32, MT = kKeys / 32;         // k-steps, dim tiles, key tiles
    // Rows of LDS: 16 rows' 16-byte pieces of K, and four rows' 64 bytes of V, lie on
    // different banks
    constexpr int kKPitch = HDP + 8, kVPitch = HDP + 32, kPlane = kKeys * (kKPitch + kVPitch);
    constexpr int kPieces = HDP / 8, kWaveRows = 64 / kPieces, kStepRows = kWaves * kWaveRows, kLoads = kKeys / kStepRows;
    typedef S raw8 __attribute__((ext_vector_type(8)));
    __shared__ __attribute__((aligned(16))) C tiles[kTeams][kBuffers][KP * kPlane];
    // of V's pieces in steps that the tile's rows do not all see: which of 8 dims are +inf, or -inf (a NaN: both)
    __shared__ unsigned all_kinds[kTeams][kBuffers][2][kKeys][HDP / 32];
    __shared__ int all_odd[kTeams][kBuffers][kWaves];
    __shared__ float2 team_ml[kWaves][32];   // (reference, sum) of the second team's rows
    static_assert(kTeams == 1 || sizeof tiles >= kWaves * (HDP / 2) * 64 * sizeof(float), "the teams' sums meet in the tiles' place");
    const AttendArgs &a = d.a;
    const int rep = d.cut.rep;
    const int cap = a.b.pages_stride << a.page_shift, lane = threadIdx.x & 63;
    const int wave = scalar(threadIdx.x >> 6) % kWaves, team = scalar(threadIdx.x >> 6) / kWaves;
    auto &tile = tiles[team];
    auto &kinds = all_kinds[team];
    auto &odd_of = all_odd[team];
    Place p;
    if (!place_of<kRows>(a.b, d.cut, blockIdx.x, a.n_head_kv, cap, a.window, false, p)) return;
    const Keys k = keys_of<kRows>(p, rep, cap, a.window);
    const int col = lane & 31, half = lane >> 5;
    const Row row = row_of(p, p.tile * kRows + wave * 32 + col, rep, cap, a.window);
    const int *table = a.b.pages + (size_t)p.seq * a.b.pages_stride;
    const int slot_mask = (1 << a.page_shift) - 1;
    const bool padded = a.hd != HDP;

    // What the wave's rows see: some of them [lo, hi), all of them [all_lo, all_hi)
    int see_lo, see_hi, all_lo, all_hi;
    {
        const int r0 = p.tile * kRows + wave * 32, r1 = min(r0 + 31, p.n * rep - 1);
        const int p0 = p.kv - p.n + scalar(r0 / rep), p1 = p.kv - p.n + scalar(max(r1, 0) / rep);
        see_lo = a.window <= p0 ? p0 - a.window + 1 : 0;
        see_hi = r0 <= r1 ? min(p1 + 1, k.hi) : 0;
        all_lo = a.window <= p1 ? p1 - a.window + 1 : 0;
        all_hi = min(p0 + 1, k.hi);
        see_lo = scalar(see_lo);
        see_hi = scalar(see_hi);
        all_lo = scalar(all_lo);
        all_hi = scalar(all_hi);
    }

    // The team's steps are number team, team + kTeams, ... of the keys; a workgroup runs as many of both
    const int all_steps = k.lo < k.hi ? (k.hi - k.lo + kKeys - 1) / kKeys : 0;
    const int n_run = (all_steps + kTeams - 1) / kTeams, n_step = (all_steps - team + kTeams - 1) / kTeams;
    constexpr int kGroups = kKeys / 16;
    const auto key_of = [&](int step) { return k.lo + (step * kTeams + team) * kKeys; };
    // 16-key group i of the steps' keys is lane i % 64
    const auto pages_from = [&](int step) {
        return PageRun::load(a, table, key_of(step + lane / kGroups) / 16 + lane % kGroups, k.hi);
    };
    PageRun run;
    run.now = pages_from(0);
    run.ahead = pages_from(64 / kGroups);

    // Q: B operand, lane (n, half) has dims 16 t + 8 half .. + 7 of its row
    vec8 q[QP][KS];
    float unit = 1.f;
    {
        const A *src = (const A *)a.q + (size_t)(row.real ? p.q0 + row.token : 0) * a.q_stride + (size_t)(row.real ? row.head : 0) * a.hd;
        const bool vec = ((uintptr_t)src & (8 * sizeof(A) - 1)) == 0;
        A v[KS][8];
        float big = 0;
#pragma unroll
        for (int t = 0; t < KS; ++t) {
            const int dim = 16 * t + 8 * half;
            const bool in = row.real && dim < a.hd;
            if (in) load_n<8>(src + dim, v[t], vec);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (!in) v[t][i] = (A)0.f;
                if (QP == 2) big = fmaxf(big, fabsf(to_f32(v[t][i])));
            }
        }
        float to = 1.f;
        if (QP == 2) unit_of(max32(big), to, unit);
#pragma unroll
        for (int t = 0; t < KS; ++t)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if constexpr (QP == 1) {
                    q[0][t][i] = v[t][i];
                } else {
                    C part[QP];
                    split_q<QP>(to_f32(v[t][i]) * to, part);
#pragma unroll
                    for (int j = 0; j < QP; ++j) q[j][t][i] = part[j];
                }
            }
    }
    const float s_hi = d.sl.hi * unit, s_lo = fmaxf(d.sl.lo * unit, 0x1p-126f);

    // A thread's share of a step: pieces of 8 dims, kWaveRows rows of a wave side by side
    const int my_row = lane / kPieces, my_dim = 8 * (lane % kPieces);
    const bool no_dim = padded && my_dim >= a.hd;
    const unsigned row_bytes = a.hd * sizeof(S), off = my_row * row_bytes + (padded ? min(my_dim, a.hd - 8) : my_dim) * (unsigned)sizeof(S);
    const unsigned first_row = wave * kWaveRows;
    unsigned offs[kLoads];   // from the step's first key
#pragma unroll
    for (int i = 0; i < kLoads; ++i) offs[i] = off + (i * kStepRows + first_row) * row_bytes;
    const unsigned page_bytes = ((unsigned)a.n_head_kv << a.page_shift) * row_bytes;   // (under 2^32: the host's check)
    const size_t head_bytes = ((size_t)p.head << a.page_shift) * row_bytes;
    const char *const k_head = (const char *)a.k_pool + head_bytes, *const v_head = (const char *)a.v_pool + head_bytes;
    raw8 kr[kLoads], vr[kLoads];
    int loaded = 0;                      // step whose K and V are in flight
    unsigned has_next = 0, has_now = 0;  // whether its groups have pages, a bit each
    bool mixed_now = false;              // whether the tile's rows differ in what they see of the step in LDS
    // P groups lie in one page; those without one read page 0.
    const auto load_groups = [&]<int P>(int step) {
        const int group = step * kGroups, key = key_of(step);
        size_t base[kGroups / P];
        has_next = 0;
#pragma unroll
        for (int b = 0; b < kGroups / P; ++b) {
            const int page = run.get((group + b * P) & 63);
            has_next |= page >= 0 ? ((1u << P) - 1) << (b * P) : 0;
            base[b] = (size_t)(unsigned)max(page, 0) * page_bytes + (size_t)(int)((((key + 16 * P * b) & slot_mask) - 16 * P * b) * (int)row_bytes);
        }
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const size_t at = base[kGroups == P ? 0 : (i * kStepRows + first_row) / (16 * P)];
            kr[i] = *reinterpret_cast<const raw8 *>(k_head + at + offs[i]);
            vr[i] = *reinterpret_cast<const raw8 *>(v_head + at + offs[i]);
        }
    };
    const auto load = [&](int step) {
        if (step && (step * kGroups & 63) == 0) {
            run.now = run.ahead;
            run.ahead = pages_from(step + 64 / kGroups);
        }
        if (a.page_shift >= (kKeys == 64 ? 6 : 5)) load_groups.template operator()<kGroups>(step);
        else if (kKeys == 64 && a.page_shift == 5) load_groups.template operator()<kGroups == 4 ? 2 : 1>(step);
        else load_groups.template operator()<1>(step);
        loaded = step;
    };
    // The loaded step into a buffer.  Where the tile's rows differ in what they see, V of
    // positions that none sees is 0, and infinities and NaN are 0 too and noted apart: a
    // product with a weight of 0 would hand them to every row.
    const auto store = [&](int buffer) {
        const int key0 = key_of(loaded);
        C *const ks = tile[buffer], *const vs = ks + kKeys * kKPitch;
        const bool whole = key0 >= k.all_lo && key0 + kKeys <= min(k.all_hi, k.hi) && has_next == (1u << kGroups) - 1;
        bool odd = false;
        if (!whole) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const int first = i * kStepRows + wave * kWaveRows;
                if (!(key0 + first + my_row < k.hi && (has_next >> (first / 16) & 1))) vr[i] = raw8{};
                unsigned up = 0, down = 0;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float v = to_f32(vr[i][e]);
                    if (!finite(v)) {
                        if (!(v < 0.f)) up |= 1u << e;
                        if (!(v > 0.f)) down |= 1u << e;
                        vr[i][e] = (S)0.f;
                    }
                }
                unsigned char *const at = reinterpret_cast<unsigned char *>(kinds[buffer][0][first + my_row]) + my_dim / 8;
                at[0] = (unsigned char)up;
                at[sizeof all_kinds[0][0][0]] = (unsigned char)down;
                odd |= (up | down) != 0;
            }
            odd = __any(odd);
        }
        if (lane == 0) odd_of[buffer][wave] = odd;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int r = i * kStepRows + wave * kWaveRows + my_row;
            if (no_dim) kr[i] = raw8{};
            if constexpr (KP == 1) {
                *reinterpret_cast<raw8 *>(ks + r * kKPitch + my_dim) = kr[i];
                *reinterpret_cast<raw8 *>(vs + r * kVPitch + my_dim) = vr[i];
            } else {
                vec8 x[3], y[3];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    bhalf_t part[3];
                    split_kv(kr[i][e], part);
#pragma unroll
                    for (int j = 0; j < 3; ++j) x[j][e] = part[j];
                    split_kv(vr[i][e], part);
#pragma unroll
                    for (int j = 0; j < 3; ++j) y[j][e] = part[j];
                }
#pragma unroll
                for (int j = 0; j < 3; ++j) {
                    *reinterpret_cast<vec8 *>(ks + j * kPlane + r * kKPitch + my_dim) = x[j];
                    *reinterpret_cast<vec8 *>(vs + j * kPlane + r * kVPitch + my_dim) = y[j];
                }
            }
        }
        has_now = has_next;
        mixed_now = !whole;
    };

    floatx16 o[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i) o[i] = floatx16{};
    float ref = kNone, sum = 0;

    if (n_step) {
        load(0);
        store(0);
        if (n_step > 1) load(1);
    }
    for (int step = 0; step < n_run; ++step) {
        const int buffer = kBuffers == 2 ? step & 1 : 0, key0 = key_of(step);
        __syncthreads();
        const unsigned has = has_now;
        const bool mixed = mixed_now;
        const C *const ks = tile[buffer], *const vs = ks + kKeys * kKPitch;
        const bool any = key0 < see_hi && key0 + kKeys > see_lo && step < n_step;
        const bool whole = key0 >= all_lo && key0 + kKeys <= all_hi && has == (1u << kGroups) - 1;

        // S^T = K Q^T: lane (n, half) gets its row's scores of keys 32 m + 8 (i / 4) + 4 half + i % 4
        floatx16 s[MT];
        if (any) {
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                s[m] = floatx16{};
                const C *const from = ks + (32 * m + col) * kKPitch + 8 * half;
#pragma unroll
                for (int t = 0; t < KS; ++t)
#pragma unroll
                    for (int y = 0; y < KP; ++y) {
                        const vec8 x = *reinterpret_cast<const vec8 *>(from + y * kPlane + 16 * t);
#pragma unroll
                        for (int z = 0; z < QP; ++z)
                            if (KP == 1 || y + z < KP) s[m] = Mma<C>::mul32(x, q[z][t], s[m]);
                    }
            }
            // K's operands are requested kAhead products early
            constexpr int kReads = MT * KS * KP, kAhead = 6, kPer = KP == 3 ? 2 : QP;
            __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
            for (int i = 0; i < kReads - kAhead; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x008, kPer, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            }
            __builtin_amdgcn_sched_group_barrier(0x008, kAhead * kPer, 0);
        }
        if (kBuffers == 2 && step + 1 < n_step) {
            store(buffer ^ 1);
            if (step + 2 < n_step) load(step + 2);
        }
        if (any) {
            if (!whole) {
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int at = 32 * m + 8 * (i / 4) + 4 * half + i % 4, key = key0 + at;
                        if (!(key >= row.lo && key < min(row.hi, k.hi) && (has >> (2 * m + i / 8) & 1))) s[m][i] = kNone;
                    }
            }
            float top = kNone;
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int i = 0; i < 16; ++i) top = fmaxf(top, s[m][i]);
            top = max32(top) * s_hi;
            follow(top, ref, sum, Mma<C>::kBias, o);
            const float base = ref == kNone ? 0.f : ref;
            vec8 w[MT][2][PP];
            float part_sum = 0;
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float e = PP > 1 ? fmaf(s[m][i], s_hi, fmaf(s[m][i], s_lo, -base)) : fmaf(s[m][i], s_hi, -base);
                    const float x = exp2_(e);
                    C part[PP];
                    split_p<PP>(x, part);
                    if (PP > 1) part_sum += x;
#pragma unroll
                    for (int y = 0; y < PP; ++y) w[m][i / 8][y][i % 8] = part[y];
                }
            // one rounded weight is also what is summed: what rounding adds to all of a row's weights divides out
            if constexpr (PP == 1) {
#pragma unroll
                for (int m = 0; m < MT; ++m) part_sum = sum_weights(w[m][1][0], sum_weights(w[m][0][0], part_sum));
            }
            sum += part_sum;
            // O^T += V^T P^T, k order as the scores came: V^T's operand, lane (m, half), has keys 16 t + 4 half + 0..3 and
            // those 8 further of dim 32 i + m
            const C *const from = vs + (4 * half + (lane & 15) / 4) * kVPitch + 16 * (lane >> 4 & 1) + 4 * (lane & 3);
            const auto v_operand = [&](int plane, int t, int i) {
                const C *at = from + plane * kPlane + 16 * t * kVPitch + 32 * i;
                const vec4 x = read_transposed<vec4>(at), y = read_transposed<vec4>(at + 8 * kVPitch);
                return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
            };
#pragma unroll
            for (int t = 0; t < 2 * MT; ++t)
#pragma unroll
                for (int i = 0; i < DT; ++i)
#pragma unroll
                    for (int x = 0; x < KP; ++x) {
                        const vec8 v = v_operand(x, t, i);
#pragma unroll
                        for (int y = 0; y < PP; ++y)
                            if (KP == 1 || x + y < KP) o[i] = Mma<C>::mul32(v, w[t / 2][t & 1][y], o[i]);
                    }
            if (mixed && (odd_of[buffer][0] | odd_of[buffer][1] | odd_of[buffer][2] | odd_of[buffer][3])) {
                for (int e = 0; e < kKeys; ++e) {
                    const bool sees = key0 + e >= row.lo && key0 + e < min(row.hi, k.hi);
#pragma unroll
                    for (int i = 0; i < DT; ++i) {
                        const unsigned up = sees ? kinds[buffer][0][e][i] >> (4 * half) : 0, down = sees ? kinds[buffer][1][e][i] >> (4 * half) : 0;
                        if (!__any((up | down) != 0)) continue;
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            const int bit = 8 * (j / 4) + j % 4;
                            if (up >> bit & 1) o[i][j] += INFINITY;
                            if (down >> bit & 1) o[i][j] -= INFINITY;
                        }
                    }
                }
            }
        }
        if (kBuffers == 1 && step + 1 < n_run) {
            __syncthreads();
            if (step + 1 < n_step) {
                store(0);
                if (step + 2 < n_step) load(step + 2);
            }
        }
    }

    sum = sum32(sum);
    if constexpr (kTeams == 2) {
        float4 *const meet = reinterpret_cast<float4 *>(tiles) + wave * (HDP / 8) * 64 + lane;
        __syncthreads();
        if (team == 1) {
#pragma unroll
            for (int i = 0; i < DT; ++i)
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    meet[(4 * i + x) * 64] = make_float4(o[i][4 * x], o[i][4 * x + 1], o[i][4 * x + 2], o[i][4 * x + 3]);
            if (half == 0) team_ml[wave][col] = make_float2(ref, sum);
        }
        __syncthreads();
        if (team == 1) return;
        const float2 e = team_ml[wave][col];
        const float m = fmaxf(ref, e.x), base = m == kNone ? 0.f : m, f = exp2_(ref - base), g = exp2_(e.x - base);
        ref = m;
        sum = fmaf(e.y, g, sum * f);
#pragma unroll
        for (int i = 0; i < DT; ++i)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const float4 v = meet[(4 * i + x) * 64];
                o[i][4 * x] = fmaf(v.x, g, o[i][4 * x] * f);
                o[i][4 * x + 1] = fmaf(v.y, g, o[i][4 * x + 1] * f);
                o[i][4 * x + 2] = fmaf(v.z, g, o[i][4 * x + 2] * f);
                o[i][4 * x + 3] = fmaf(v.w, g, o[i][4 * x + 3] * f);
            }
    }
    const int r = wave * 32 + col;
    if (p.n_split > 1) {
        const size_t id = blockIdx.x;
#pragma unroll
        for (int i = 0; i < DT; ++i)
#pragma unroll
            for (int x = 0; x < 4; ++x)
                reinterpret_cast<float4 *>(d.part_o)[(id * (HDP / 4) + 8 * i + 2 * x + half) * kRows + r] =
                    make_float4(o[i][4 * x], o[i][4 * x + 1], o[i][4 * x + 2], o[i][4 * x + 3]);
        if (half == 0) reinterpret_cast<float2 *>(d.part_ml)[id * kRows + r] = make_float2(ref, sum);
        return;
    }
    if (!row.real) return;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    A *const out = (A *)a.out + (size_t)(p.q0 + row.token) * a.out_stride + (size_t)row.head * a.hd;
    const bool vec = ((uintptr_t)out & (4 * sizeof(A) - 1)) == 0;
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const int dim = 32 * i + 8 * x + 4 * half;
            const A v[4] = {(A)(o[i][4 * x] * inv), (A)(o[i][4 * x + 1] * inv), (A)(o[i][4 * x + 2] * inv), (A)(o[i][4 * x + 3] * inv)};
            if (dim < a.hd) store_n<4>(out + dim, v, vec);
        }
}

}  // namespace

hipError_t launch_chunk(const TileArgs &d, int places, hipStream_t s) {
    const int hdp = padded_dim(d.a.hd);
    const dim3 grid((unsigned)places);
#define KORE_CHUNK(A, S)                                                        \
    do {                                                                        \
        if (hdp == 64) chunk_kernel<A, S, 64><<<grid, Shape<A, S, 64>::threads, 0, s>>>(d);     \
        else if (hdp == 128) chunk_kernel<A, S, 128><<<grid, Shape<A, S, 128>::threads, 0, s>>>(d); \
        else chunk_kernel<A, S, 256><<<grid, Shape<A, S, 256>::threads, 0, s>>>(d);              \
    } while (0)
    if (d.a.cache_type == kF32) KORE_CHUNK(float, float);
    else if (d.a.type == kF32 && d.a.cache_type == kF16) KORE_CHUNK(float, half_t);
    else if (d.a.type == kF32) KORE_CHUNK(float, bhalf_t);
    else if (d.a.type == kF16) KORE_CHUNK(half_t, half_t);
    else KORE_CHUNK(bhalf_t, bhalf_t);
#undef KORE_CHUNK
    return hipGetLastError();
}

}  // namespace kore_paged_gpu

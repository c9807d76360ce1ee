// kore_paged_chunk.hip - paged attention of many rows (chunks of prompts; gfx950).
//
// A tile is 128 rows of a kv-head's (token, q-head) list, 32 for each of four waves,
// and passes over its keys 64 (or 32) at a time through LDS: the flops of a key,
// 512 head_dim for its 4 head_dim bytes, put the kernel between the matrix cores and
// the vector units that make the weights.  Two such teams of waves share a CU as one
// workgroup, each with every other step of the keys, and join their sums through LDS at
// the end: what a step waits for is a wave's own chain of loads, products and weights,
// so a tile takes half as long as with one team, and the long tiles of a causal chunk
// are what the launch waits for (28/4/128, 2048 fp16 rows: 51 us; the same waves in two
// workgroups of four took 56 where this took 51, an earlier pair of variants).
//
// us, and TFLOP/s of products made (a large bf16 product: 1154 to 1207): 2048 fp16 rows of
// 28/4/128 50 to 60 over several cards, 500 to 600; 512 fp32 rows over 32749 bf16 keys, three
// products each, 589 to 656, 1090 to 1210; 2048 fp32 rows over an fp32 cache, three and
// six, 154 to 180, 750 to 880.  The rest is vector instructions (weights, parts), which
// matrix instructions of another wave hardly overlap, a workgroup's start, and waits at
// the team's two barriers a step.
#include "kore_paged_attend.h"

namespace kore_paged_gpu {
namespace {

constexpr int kWaves = 4, kRows = kChunkRows;   // of a team

// How a (row type, cache type) is computed: the type and parts of q and K, and those
// of the weights and V.  An fp32 cache's K is two fp16 parts, as q, each key in a power
// of two of its own, and its V three bf16 parts, as the weights; the products of parts
// i and j with i + j under the cache's number of parts hold 22 and 24 bits.  (K's units
// leave again with the scores.  V's would have to be the weights': keys of far smaller V
// would lose bits.)
template <class A, class S> struct Form {
    typedef S C;
    typedef S CV;
    static constexpr int qp = Parts<A, S>::q, kp = 1, vp = 1, pp = Parts<A, S>::p;
};
template <> struct Form<float, float> {
    typedef half_t C;
    typedef bhalf_t CV;
    static constexpr int qp = 2, kp = 2, vp = 3, pp = 3;
};

// What a tile's shape asks of LDS and registers: keys of a step; teams of a
// workgroup (a CU holds one workgroup).
template <class A, class S, int HDP> struct Shape {
    static constexpr bool parts = Form<A, S>::qp > 1;
    static constexpr int keys = parts ? 32 : 64;
    static constexpr int teams = HDP <= 128 ? 2 : 1, threads = 64 * kWaves * teams;
    static constexpr bool lag = parts && teams == 2;   // the second team a phase behind
};

// Eight values as one, two or three 16-bit parts.  Three bf16 parts are cut, not
// rounded: 24 bits in all, two values' upper halves an instruction.
__device__ __forceinline__ unsigned upper_halves(float a, float b) {
    return __builtin_amdgcn_perm(__builtin_bit_cast(unsigned, b), __builtin_bit_cast(unsigned, a), 0x07060302);
}
__device__ __forceinline__ void cut3(const float (&x)[8], bhalf8 (&part)[3]) {
    typedef unsigned uint4_t __attribute__((ext_vector_type(4)));
    uint4_t u[3];
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        float r[2], l[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            r[j] = x[i + j] - bf16_cut(x[i + j]);
            l[j] = r[j] - bf16_cut(r[j]);
        }
        u[0][i / 2] = upper_halves(x[i], x[i + 1]);
        u[1][i / 2] = upper_halves(r[0], r[1]);
        u[2][i / 2] = upper_halves(l[0], l[1]);
    }
#pragma unroll
    for (int j = 0; j < 3; ++j) part[j] = __builtin_bit_cast(bhalf8, u[j]);
}
// The largest of PIECES neighbouring lanes' values (8, 16 or 32; none under 0, so that their bits compare as integers).
template <int CTRL>
__device__ __forceinline__ unsigned max_lane(unsigned x) {
    return max(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, true));
}
template <int PIECES>
__device__ __forceinline__ float row_max(float big) {
    if constexpr (PIECES == 32) big = max16(big);
    unsigned x = __builtin_bit_cast(unsigned, big);
    if constexpr (PIECES >= 16) x = max_lane<0x140>(x);    // lane 15 - i of 16
    x = max_lane<0x141>(x);                                 // lane 7 - i of 8
    x = max_lane<0x4e>(max_lane<0xb1>(x));                  // lanes i ^ 1, i ^ 2
    return __builtin_bit_cast(float, x);
}
// Eight weights as N parts of C.
template <int N, class C, class V>
__device__ __forceinline__ void weights(const float (&x)[8], V (&part)[N]) {
    if constexpr (N == 3) {
        cut3(x, part);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            C y[N];
            split_p<N>(x[i], y);
#pragma unroll
            for (int j = 0; j < N; ++j) part[j][i] = y[j];
        }
    }
}

template <class A, class S, int HDP>
__global__ __launch_bounds__((Shape<A, S, HDP>::threads), 1) void chunk_kernel(TileArgs d) {
    typedef typename Form<A, S>::C C;
    typedef typename Form<A, S>::CV CV;
    typedef typename Mma<C>::vec8 vec8;
    typedef typename Mma<CV>::vec8 vvec8;
    typedef CV vec4 __attribute__((ext_vector_type(4)));
    constexpr int QP = Form<A, S>::qp, KP = Form<A, S>::kp, VP = Form<A, S>::vp, PP = Form<A, S>::pp;
    constexpr int kKeys = Shape<A, S, HDP>::keys, kTeams = Shape<A, S, HDP>::teams;
    constexpr bool kLag = Shape<A, S, HDP>::lag;
    constexpr int KS = HDP / 16, DT = HDP / 32, MT = kKeys / 32;         // k-steps, dim tiles, key tiles
    // Rows of LDS: 16 rows' 16-byte pieces of K, and four rows' 64 bytes of V, lie on
    // different banks
    constexpr int kKPitch = HDP + 8, kVPitch = HDP + 32;
    constexpr int kPieces = HDP / 8, kWaveRows = 64 / kPieces, kStepRows = kWaves * kWaveRows, kLoads = kKeys / kStepRows;
    typedef S raw8 __attribute__((ext_vector_type(8)));
    // A team's step of K and of V, in KP and VP planes; at the end half of the second team's sums lie there
    constexpr int kStep = kKeys * (KP * kKPitch + VP * kVPitch), kTileBytes = kTeams * kStep * (int)sizeof(C);
    constexpr int kMeetBytes = kTeams == 2 ? kWaves * HDP / 16 * 64 * 16 : 0;
    // before the first step the tile's rows of q lie there: each is read once, by lanes side by side (in the operands'
    // order a load touches 32 rows, and either team reads all: 28/4/128, 64 fp16 rows over 512 keys 15.4 us instead of 14.7,
    // fp32 22.5 instead of 21.5, a 2048-row fp16 prompt 57.8 instead of 56.1; at HDP = 256 fp32 rows would not fit beside
    // q's third part)
    constexpr bool kStage = kTeams == 2;
    constexpr int kQPitch = HDP + 16 / (int)sizeof(A), kQBytes = kStage ? kRows * kQPitch * (int)sizeof(A) : 0;
    constexpr int kMost = kTileBytes > kMeetBytes ? kTileBytes : kMeetBytes;
    __shared__ __attribute__((aligned(16))) unsigned char tiles[kMost > kQBytes ? kMost : kQBytes];
    // The third part of q, where LDS has room: it would cost the loop its spare registers, and a reload of a spilled
    // one waits for the loads in flight.  (The teams' rows are the same.)
    constexpr bool kThird = QP == 3;
    constexpr int kQReg = kThird ? 2 : QP;
    __shared__ vec8 q_third[kThird ? kWaves : 1][KS][64];
    // a careful pass's notes, of eight dims each (take_out), and whether a wave has any
    __shared__ unsigned all_kinds[kTeams][2][kKeys][HDP / 32];
    __shared__ int all_odd[kTeams][kWaves];
    __shared__ bool all_bad[kTeams * kWaves];   // a wave's sums are not all finite
    __shared__ __attribute__((aligned(16))) int all_back[KP == 2 ? kTeams : 1][kKeys];   // exponents of K's units
    __shared__ float2 team_ml[kWaves][32];   // (reference, sum) of the second team's rows
    const AttendArgs &a = d.a;
    const int rep = d.cut.rep;
    const int cap = a.b.pages_stride << a.page_shift, lane = threadIdx.x & 63;
    const int wave = scalar(threadIdx.x >> 6) % kWaves, team = scalar(threadIdx.x >> 6) / kWaves;
    C *const k_tile = reinterpret_cast<C *>(tiles) + team * kStep;
    CV *const v_tile = reinterpret_cast<CV *>(k_tile + KP * kKeys * kKPitch);
    int *const k_back = all_back[KP == 2 ? team : 0];
    auto &kinds = all_kinds[team];
    auto &odd_of = all_odd[team];
    Place p;
    if (!place_of<kRows>(a.b, d.cut, blockIdx.x, a.n_head_kv, cap, a.window, false, p)) return;
    const Keys k = keys_of<kRows>(p, d.cut, cap, a.window);
    const int col = lane & 31, half = lane >> 5;
    const Row row = row_of(p, p.tile * kRows + wave * 32 + col, d.cut, cap, a.window);
    const int *table = a.b.pages + (size_t)p.seq * a.b.pages_stride;
    const int slot_mask = (1 << a.page_shift) - 1;
    const bool padded = a.hd != HDP;

    // What the wave's rows see: some of them [lo, hi), all of them [all_lo, all_hi)
    int see_lo, see_hi, all_lo, all_hi;
    {
        const int r0 = p.tile * kRows + wave * 32, r1 = min(r0 + 31, p.n * rep - 1);
        const int p0 = p.kv - p.n + d.cut.by_rep.of(r0), p1 = p.kv - p.n + d.cut.by_rep.of(max(r1, 0));
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

    // A thread's share of a step (and of q): pieces of 8 dims, kWaveRows rows of a wave side by side
    const int my_row = lane / kPieces, my_dim = 8 * (lane % kPieces);

    // Q: B operand, lane (n, half) has dims 16 t + 8 half .. + 7 of its row.  Requested here,
    // used when K and V are on their way.
    A q_row[KS][8];
    constexpr int kQPass = kTeams * kStepRows, kQLoads = kRows / kQPass;
    A q_piece[kStage ? kQLoads : 1][8];
    bool q_real[kStage ? kQLoads : 1];
    const int q_first = (team * kWaves + wave) * kWaveRows + my_row;
    if constexpr (kStage) {
        const A *src[kQLoads];
#pragma unroll
        for (int i = 0; i < kQLoads; ++i) {
            const Row r = row_of(p, p.tile * kRows + i * kQPass + q_first, d.cut, cap, a.window);
            q_real[i] = r.real && my_dim < a.hd;
            src[i] = q_row_of<A>(a, p, r) + min(my_dim, a.hd - 8);
        }
        if (d.q_wide) {
#pragma unroll
            for (int i = 0; i < kQLoads; ++i) load_piece(src[i], true, q_piece[i]);
        } else {
#pragma unroll
            for (int i = 0; i < kQLoads; ++i) load_piece(src[i], false, q_piece[i]);
        }
    } else {
        load_q<KS>(a, p, row, d.q_wide, 8 * half, 16, q_row);
    }

    vec8 q[kQReg][KS];
    int q_unit = 0;   // the exponent of q's unit
    const auto make_q = [&] {
        if constexpr (kStage) {
            A *const q_tile = reinterpret_cast<A *>(tiles);
            typedef A piece8 __attribute__((ext_vector_type(8)));
#pragma unroll
            for (int i = 0; i < kQLoads; ++i) {
                piece8 v;
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = q_real[i] ? q_piece[i][e] : (A)0.f;
                *reinterpret_cast<piece8 *>(q_tile + (i * kQPass + q_first) * kQPitch + my_dim) = v;
            }
            __syncthreads();
#pragma unroll
            for (int t = 0; t < KS; ++t) {
                const piece8 v = *reinterpret_cast<const piece8 *>(q_tile + (wave * 32 + col) * kQPitch + 16 * t + 8 * half);
#pragma unroll
                for (int e = 0; e < 8; ++e) q_row[t][e] = v[e];
            }
            __syncthreads();   // K and V take the place
        } else {
            zero_q<KS>(a, row, 8 * half, 16, q_row);
        }
        float to = 1.f;
        if constexpr (QP == 2) {
            float big = 0;
#pragma unroll
            for (int t = 0; t < KS; ++t)
#pragma unroll
                for (int i = 0; i < 8; ++i) big = fmaxf(big, fabsf(q_row[t][i]));
            q_unit = unit_of(max32(big), to);
        }
#pragma unroll
        for (int t = 0; t < KS; ++t) {
            vec8 third = {};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if constexpr (QP == 1) {
                    q[0][t][i] = q_row[t][i];
                } else {
                    C part[QP];
                    split_q<QP>(q_row[t][i] * to, part);
#pragma unroll
                    for (int j = 0; j < kQReg; ++j) q[j][t][i] = part[j];
                    if (kThird) third[i] = part[QP - 1];
                }
            }
            if (kThird && team == 0) q_third[wave][t][lane] = third;
        }
    };
    if constexpr (QP > 1) make_q();   // (behind the loads its registers cost the loop more than the wait)

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
    // Whether a step's groups have pages, a bit each: of the step in LDS, the next and the one after
    unsigned has = 0, has_1 = 0, has_2 = 0;
    constexpr unsigned kAll = (1u << kGroups) - 1;
    // P groups lie in one page; those without one read page 0.
    const auto load_groups = [&]<int P>(int step, const char *pool, raw8 (&x)[kLoads]) {
        const int group = step * kGroups, key = key_of(step);
        size_t base[kGroups / P];
        unsigned bits = 0;
#pragma unroll
        for (int b = 0; b < kGroups / P; ++b) {
            const int page = run.get((group + b * P) & 63);
            bits |= page >= 0 ? ((1u << P) - 1) << (b * P) : 0;
            base[b] = (size_t)(unsigned)max(page, 0) * page_bytes + (size_t)(int)((((key + 16 * P * b) & slot_mask) - 16 * P * b) * (int)row_bytes);
        }
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
            x[i] = *reinterpret_cast<const raw8 *>(pool + base[kGroups == P ? 0 : (i * kStepRows + first_row) / (16 * P)] + offs[i]);
        return bits;
    };
    const auto load = [&](int step, const char *pool, raw8 (&x)[kLoads]) {
        if (a.page_shift >= (kKeys == 64 ? 6 : 5)) return load_groups.template operator()<kGroups>(step, pool, x);
        if (kKeys == 64 && a.page_shift == 5) return load_groups.template operator()<kGroups == 4 ? 2 : 1>(step, pool, x);
        return load_groups.template operator()<1>(step, pool, x);
    };
    const auto load_k = [&](int step) {   // before the same step's V
        if (step && (step * kGroups & 63) == 0) {
            run.now = run.ahead;
            run.ahead = pages_from(step + 64 / kGroups);
        }
        has_2 = load(step, k_head, kr);
    };
    const auto load_v = [&](int step) { load(step, v_head, vr); };
    const auto put_k = [&](raw8 x, int row) {
        C *const at = k_tile + row * kKPitch + my_dim;
        if constexpr (KP == 1) {
            *reinterpret_cast<raw8 *>(at) = x;
        } else {
            // two parts, each the nearest, of the row in its unit
            float big = 0, to;
#pragma unroll
            for (int e = 0; e < 8; ++e) big = fmaxf(big, fabsf(x[e]));
            big = row_max<kPieces>(big);
            const bool odd = __any(big == INFINITY);
            if (odd) {   // the unit of the finite ones
                big = 0;
#pragma unroll
                for (int e = 0; e < 8; ++e) big = fmaxf(big, fabsf(x[e]) < INFINITY ? fabsf(x[e]) : 0.f);
                big = row_max<kPieces>(big);
            }
            const int back = unit_of(big, to);
            vec8 hi, lo;
            typedef C vec2 __attribute__((ext_vector_type(2)));
            typedef float float2_t __attribute__((ext_vector_type(2)));
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const float2_t y = {x[e] * to, x[e + 1] * to};
                const vec2 h = __builtin_convertvector(y, vec2);
                const float2_t r = {__builtin_fmaf((float)h[0], -1.f, y[0]), __builtin_fmaf((float)h[1], -1.f, y[1])};
                const vec2 l = __builtin_convertvector(r, vec2);
                hi[e] = h[0];
                hi[e + 1] = h[1];
                lo[e] = l[0];
                lo[e + 1] = l[1];
            }
            if (odd) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (!(fabsf(x[e]) < INFINITY)) lo[e] = (C)0.f;
            }
            *reinterpret_cast<vec8 *>(at) = hi;
            *reinterpret_cast<vec8 *>(at + kKeys * kKPitch) = lo;
            if (my_dim == 0) k_back[row] = back;
        }
    };
    const auto put_v = [&](raw8 x, int row) {
        CV *const at = v_tile + row * kVPitch + my_dim;
        if constexpr (VP == 1) {
            *reinterpret_cast<raw8 *>(at) = x;
        } else {
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = x[e];
            vvec8 part[3];
            cut3(y, part);   // (of an infinity or NaN some are not finite, and so will the sums be)
#pragma unroll
            for (int j = 0; j < 3; ++j) *reinterpret_cast<vvec8 *>(at + j * kKeys * kVPitch) = part[j];
        }
    };
    const auto store_k = [&] {
        if (padded) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i)
                if (no_dim) kr[i] = raw8{};
        }
#pragma unroll
        for (int i = 0; i < kLoads; ++i) put_k(kr[i], i * kStepRows + wave * kWaveRows + my_row);
    };
    // V into LDS; of positions that no row of the tile sees it is 0: it may hold anything
    const auto store_v = [&]<bool CAREFUL>(int key0, bool mixed) {
        if (mixed) {
            // (a branch: selects cost registers, and 512 fp16 rows over 8192 keys of 16/2/256 170 us instead of 155)
            asm volatile("");
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const int first = i * kStepRows + wave * kWaveRows, key = key0 + first + my_row;
                if (!(key < k.hi && key >= k.seen_lo && (has >> (first / 16) & 1))) vr[i] = raw8{};
            }
        }
        if constexpr (CAREFUL) {
            bool odd = false;
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                unsigned up, down;
                take_out<S>(vr[i], up, down);
                unsigned char *const at = reinterpret_cast<unsigned char *>(kinds[0][i * kStepRows + wave * kWaveRows + my_row]) + my_dim / 8;
                at[0] = (unsigned char)up;
                at[sizeof kinds[0]] = (unsigned char)down;
                odd |= (up | down) != 0;
            }
            odd = __any(odd);
            if (lane == 0) odd_of[wave] = odd;
        }
#pragma unroll
        for (int i = 0; i < kLoads; ++i) put_v(vr[i], i * kStepRows + wave * kWaveRows + my_row);
    };

    floatx16 o[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i) o[i] = floatx16{};
    float ref = kNone, sum = 0;

    // A step is two phases: V into LDS, the scores and their maximum; K of the next step
    // into LDS, the weights and their product with V.  Each reads what the phase before
    // wrote, so K and V need one place each.  With values in parts, whose products are most
    // of a step, the second team runs a phase behind the first: one is at its scores while
    // the other makes weights (512 fp32 rows over 32749 bf16 keys: 686 us against 771 side by
    // side); without, they run side by side (a 2048-row fp16 prompt: 52.7 against 53.9).
    const auto start = [&] {   // run holds the first pages
        load_k(0);
        load_v(0);
        has = has_2;
    };
    if (n_step) start();
    if constexpr (QP == 1) make_q();
    // An fp32 cache's scores leave q's unit with K's, both at once: either alone may pass fp32's range, or their product
    // where the score does not.
    const float unit = KP == 2 ? 1.f : power(q_unit);
    const float s2 = scale_of(d.scale_log2, unit);
    const auto pass = [&]<bool CAREFUL>() __attribute__((always_inline)) {
        if (n_step) {
            store_k();
            if (n_step > 1) load_k(1);
            has_1 = has_2;
        }
        if (kLag && team == 1) __syncthreads();
        for (int step = 0; step < n_run; ++step) {
            const int key0 = key_of(step);
            const bool real = step < n_step;
            const bool mixed = !(key0 >= k.all_lo && key0 + kKeys <= min(k.all_hi, k.hi) && has == kAll);
            const bool any = key0 < see_hi && key0 + kKeys > see_lo && real;
            const bool whole = key0 >= all_lo && key0 + kKeys <= all_hi && has == kAll;
            __syncthreads();
            if (real) {
                store_v.template operator()<CAREFUL>(key0, mixed);
                if (step + 1 < n_step) load_v(step + 1);
            }

            // S^T = K Q^T: lane (n, half) gets its row's scores of keys 32 m + 8 (i / 4) + 4 half + i % 4
            floatx16 s[MT];
            bool far = false;
            unsigned has_weight[MT];   // CAREFUL: of the step's keys, for the lane's row
            if (any) {
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    s[m] = floatx16{};
                    const int from = (32 * m + col) * kKPitch + 8 * half;
#pragma unroll
                    for (int t = 0; t < KS; ++t)
#pragma unroll
                        for (int y = 0; y < KP; ++y) {
                            const vec8 x = *reinterpret_cast<const vec8 *>(&k_tile[y * kKeys * kKPitch + from + 16 * t]);
#pragma unroll
                            for (int z = 0; z < QP; ++z)
                                if (KP == 1 || y + z < KP) s[m] = Mma<C>::mul32(x, z < kQReg ? q[z < kQReg ? z : 0][t] : q_third[wave][t][lane], s[m]);
                        }
                }
                // K's operands are requested kAhead products early
                constexpr int kReads = MT * KS * (KP + kThird), kAhead = 6, kPer = KP == 2 ? 3 : kThird ? 1 : QP;
                __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
                for (int i = 0; i < kReads - kAhead; i += KP) {
                    __builtin_amdgcn_sched_group_barrier(0x008, kPer, 0);
                    __builtin_amdgcn_sched_group_barrier(0x100, KP, 0);
                }
                __builtin_amdgcn_sched_group_barrier(0x008, kAhead / KP * kPer, 0);
                if constexpr (KP == 2) {
#pragma unroll
                    for (int m = 0; m < MT; ++m)
#pragma unroll
                        for (int i = 0; i < 16; i += 4) {
                            const int4 b = *reinterpret_cast<const int4 *>(&k_back[32 * m + 2 * i + 4 * half]);
                            s[m][i] = __builtin_ldexpf(s[m][i], b.x + q_unit);
                            s[m][i + 1] = __builtin_ldexpf(s[m][i + 1], b.y + q_unit);
                            s[m][i + 2] = __builtin_ldexpf(s[m][i + 2], b.z + q_unit);
                            s[m][i + 3] = __builtin_ldexpf(s[m][i + 3], b.w + q_unit);
                        }
                }
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
                follow<CAREFUL>(max32(top), ref, sum, s2, o);
                if constexpr (CAREFUL) {
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        has_weight[m] = 0;
#pragma unroll
                        for (int i = 0; i < 16; ++i) has_weight[m] |= (unsigned)(s[m][i] != kNone) << (8 * (i / 4) + 4 * half + i % 4);
                        has_weight[m] |= __shfl_xor(has_weight[m], 32);
                    }
                }
                // The difference from the reference first, as the softmax's comment says.  16-bit rows: one fma of the score
                // and the scaled reference while that is under 2^11.  Its rounding, at most 2^-14 in the exponent, is the same
                // for the weights of one reference and stays between those of two (a row's teams and splits, and before and
                // after the reference moves): 2^-13.5 of a weight, beside the weights' own half step of 2^-11 (fp16) or 2^-8.
                // (2048 fp16 rows of 28/4/128: 50.2 us with every reference under 2^11, 51.9 with every one over it.)
                if constexpr (PP == 1) {
                    const float base = ref == kNone ? 0.f : ref;
                    far = fabsf(base * s2) >= 0x1p11f;
                    if (__any(far)) {
                        const float off = far ? base : 0.f;   // (a row's bits are not its neighbours' business)
#pragma unroll
                        for (int m = 0; m < MT; ++m)
#pragma unroll
                            for (int i = 0; i < 16; ++i) s[m][i] -= off;
                    }
                }
            }
            __syncthreads();
            if (step + 1 < n_step) {
                store_k();
                if (step + 2 < n_step) load_k(step + 2);
            }
            has = has_1;
            has_1 = has_2;
            if (any) {
                if (CAREFUL && (odd_of[0] | odd_of[1] | odd_of[2] | odd_of[3])) {
                    for (int e = 0; e < kKeys; ++e) {
                        const bool gets = (e < 32 ? has_weight[0] : has_weight[MT - 1]) >> (e & 31) & 1;
#pragma unroll
                        for (int i = 0; i < DT; ++i) {
                            const unsigned up = gets ? kinds[0][e][i] >> (4 * half) : 0, down = gets ? kinds[1][e][i] >> (4 * half) : 0;
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
                const float base = ref == kNone ? 0.f : ref;
                const float minus = PP == 1 && !far ? fmaf(-base, s2, Mma<CV>::kBias) : Mma<CV>::kBias;
                vvec8 w[MT][2][PP];
                float part_sum = 0;
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float x[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float y = s[m][8 * h + i];
                            x[i] = exp2_(fmaf(PP > 1 ? y - base : y, s2, minus));
                            if (PP > 1) part_sum += x[i];
                        }
                        weights<PP, CV>(x, w[m][h]);
                        // one rounded weight is also what is summed: what rounding adds to all of a row's weights divides out
                        if constexpr (PP == 1) part_sum = sum_weights(w[m][h][0], part_sum);
                    }
                sum += part_sum;
                // O^T += V^T P^T, k order as the scores came: V^T's operand, lane (m, half), has keys 16 t + 4 half + 0..3 and
                // those 8 further of dim 32 i + m
                const int from = (4 * half + (lane & 15) / 4) * kVPitch + 16 * (lane >> 4 & 1) + 4 * (lane & 3);
                const auto v_operand = [&](int plane, int t, int i) {
                    const CV *at = &v_tile[plane * kKeys * kVPitch + from + 16 * t * kVPitch + 32 * i];
                    const vec4 x = read_transposed<vec4>(at), y = read_transposed<vec4>(at + 8 * kVPitch);
                    return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
                };
#pragma unroll
                for (int t = 0; t < 2 * MT; ++t)
#pragma unroll
                    for (int i = 0; i < DT; ++i)
#pragma unroll
                        for (int x = 0; x < VP; ++x) {
                            const vvec8 v = v_operand(x, t, i);
#pragma unroll
                            for (int y = 0; y < PP; ++y)
                                if (VP == 1 || x + y < VP) o[i] = Mma<CV>::mul32(v, w[t / 2][t & 1][y], o[i]);
                        }
                // A branch, which ends the block that the compiler schedules: us without / with it, 700 fp32 rows and cache beside
                // eight tokens 106.4 / 100.9, 512 fp32 rows over 8192 keys of 16/2/256 288 / 275 (bf16), 261 / 247 (fp16); over
                // 32749 bf16 keys of 28/4/128 600 / 619, 512 fp16 rows of 16/2/256 156 / 172 (it spills), so not there.
                if constexpr (VP == 3 || (HDP == 256 && QP > 1))
                    if (mixed) asm volatile("s_nop 0");
            }
        }
        if (kLag && team == 0) __syncthreads();
    };
    pass.template operator()<false>();
    const bool bad = __any(not_finite(o));
    if (lane == 0) all_bad[team * kWaves + wave] = bad;
    __syncthreads();   // (and K and V give way)
    bool any_bad = false;
#pragma unroll
    for (int i = 0; i < kTeams * kWaves; ++i) any_bad |= all_bad[i];
    if (__builtin_expect(__any(any_bad), 0)) {
#pragma unroll
        for (int i = 0; i < DT; ++i) o[i] = floatx16{};
        ref = kNone;
        sum = 0;
        run.now = pages_from(0);
        // (as if they were others, so that what this pass makes of them is not kept through the first: 512 fp32 rows over 8192
        // bf16 keys of 16/2/256 287 us without, 283)
#pragma unroll
        for (int i = 0; i < kLoads; ++i) asm volatile("" : "+v"(offs[i]));
        run.ahead = pages_from(64 / kGroups);
        if (n_step) start();
        pass.template operator()<true>();
        __syncthreads();
    }
    sum = sum32(sum);
    if constexpr (kTeams == 2) {
        // the second team's sums through LDS, half of them at a time
        float4 *const meet = reinterpret_cast<float4 *>(tiles) + wave * (HDP / 16) * 64 + lane;
        float f = 1.f, g = 0.f;
#pragma unroll
        for (int part = 0; part < 2; ++part) {
            if (team == 1) {
#pragma unroll
                for (int i = 0; i < DT / 2; ++i)
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const floatx16 &from = o[part * (DT / 2) + i];
                        meet[(4 * i + x) * 64] = make_float4(from[4 * x], from[4 * x + 1], from[4 * x + 2], from[4 * x + 3]);
                    }
                if (part == 0 && half == 0) team_ml[wave][col] = make_float2(ref, sum);
            }
            __syncthreads();
            if (team == 0) {
                if (part == 0) {
                    const float2 e = team_ml[wave][col];
                    const float m = fmaxf(ref, e.x);
                    f = share_at(ref, m, s2);
                    g = share_at(e.x, m, s2);
                    ref = m;
                    sum = fmaf(e.y, g, sum * f);
                }
#pragma unroll
                for (int i = 0; i < DT / 2; ++i)
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const float4 v = meet[(4 * i + x) * 64];
                        floatx16 &to = o[part * (DT / 2) + i];
                        to[4 * x] = fmaf(v.x, g, to[4 * x] * f);
                        to[4 * x + 1] = fmaf(v.y, g, to[4 * x + 1] * f);
                        to[4 * x + 2] = fmaf(v.z, g, to[4 * x + 2] * f);
                        to[4 * x + 3] = fmaf(v.w, g, to[4 * x + 3] * f);
                    }
            }
            if (part == 0) __syncthreads();
        }
        if (team == 1) return;
    }
    const int r = wave * 32 + col;
    if (p.n_split > 1) {
        const size_t id = p.part;
        if (id >= (unsigned)d.parts) return;   // (only where q_start is not ascending)
#pragma unroll
        for (int i = 0; i < DT; ++i)
#pragma unroll
            for (int x = 0; x < 4; ++x)
                reinterpret_cast<float4 *>(d.part_o)[(id * (HDP / 4) + 8 * i + 2 * x + half) * kRows + r] =
                    make_float4(o[i][4 * x], o[i][4 * x + 1], o[i][4 * x + 2], o[i][4 * x + 3]);
        if (half == 0) reinterpret_cast<float2 *>(d.part_ml)[id * kRows + r] = make_float2(ref * unit, sum);
        return;
    }
    if (!row.real) return;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    A *const out = (A *)a.out + (size_t)(p.q0 + row.token) * a.out_stride + (size_t)row.head * a.hd;
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const int dim = 32 * i + 8 * x + 4 * half;
            const A v[4] = {(A)(o[i][4 * x] * inv), (A)(o[i][4 * x + 1] * inv), (A)(o[i][4 * x + 2] * inv), (A)(o[i][4 * x + 3] * inv)};
            if (dim < a.hd) store_n<4>(out + dim, v, d.out_wide);
        }
}

}  // namespace

hipError_t launch_chunk(const TileArgs &d, hipStream_t s) {
    const int hdp = padded_dim(d.a.hd);
    const dim3 grid((unsigned)d.places);
#define KORE_CHUNK(A, S)                                                        \
    do {                                                                        \
        if (hdp == 64) return launch(chunk_kernel<A, S, 64>, grid, Shape<A, S, 64>::threads, 0, s, d);     \
        else if (hdp == 128) return launch(chunk_kernel<A, S, 128>, grid, Shape<A, S, 128>::threads, 0, s, d); \
        else return launch(chunk_kernel<A, S, 256>, grid, Shape<A, S, 256>::threads, 0, s, d);              \
    } while (0)
    if (d.a.cache_type == kF32) KORE_CHUNK(float, float);
    else if (d.a.type == kF32 && d.a.cache_type == kF16) KORE_CHUNK(float, half_t);
    else if (d.a.type == kF32) KORE_CHUNK(float, bhalf_t);
    else if (d.a.type == kF16) KORE_CHUNK(half_t, half_t);
    else KORE_CHUNK(bhalf_t, bhalf_t);
#undef KORE_CHUNK
}

}  // namespace kore_paged_gpu

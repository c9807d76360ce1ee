// kore_paged_decode.hip - paged attention of few rows (a decode step), and the
// merge of split tiles (gfx950).
//
// A tile is 16 rows: the q-heads of one token's kv-head, or of a few tokens.  K and
// V are read once for them, so at 16 flops a cache value the kernel is bound by
// HBM; eight waves a CU, each with its next block in flight, are what carries it.  A
// workgroup is W = 4 waves (8 where little is to be read, launch_attend) that take
// blocks of keys in turn, each with its own softmax state, merged through LDS at the
// end; the next block's K is requested when this one's scores are made, its V when this
// one's is in LDS (or used).
#include "kore_paged_attend.h"

#include <algorithm>

namespace kore_paged_gpu {
namespace {

constexpr int kThreads = 256, kRows = 16;

// The W waves' states (ref, sum, and o as [dim / 4][row] float4) into out, or
// into the split's partial.
template <class A, int HDP, int W>
__device__ __forceinline__ void finish(const TileArgs &d, const Place &p, const float4 (*o)[HDP / 4][kRows],
                                       const float2 (*ml)[kRows]) {
    const AttendArgs &a = d.a;
    __syncthreads();
    const int rep = d.cut.rep;
    for (int i = threadIdx.x; i < HDP / 4 * kRows; i += 64 * W) {
        const int row = i % kRows, d4 = i / kRows;
        float m = kNone, l = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) m = fmaxf(m, ml[w][row].x);
        float4 s = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float2 e = ml[w][row];
            const float f = share_at(e.x, m, d.scale_log2);
            const float4 v = o[w][d4][row];
            l = fmaf(e.y, f, l);
            s.x = fmaf(v.x, f, s.x);
            s.y = fmaf(v.y, f, s.y);
            s.z = fmaf(v.z, f, s.z);
            s.w = fmaf(v.w, f, s.w);
        }
        if (p.n_split > 1) {
            const size_t id = p.part;
            if (id >= (unsigned)d.parts) continue;   // (only where q_start is not ascending)
            reinterpret_cast<float4 *>(d.part_o)[(id * (HDP / 4) + d4) * kRows + row] = s;
            if (d4 == 0) reinterpret_cast<float2 *>(d.part_ml)[id * kRows + row] = make_float2(m, l);
            continue;
        }
        const int r = p.tile * kRows + row;
        if (r >= p.n * rep || 4 * d4 >= a.hd) continue;
        const int token = d.cut.by_rep.of(r), head = p.head * rep + r - token * rep;
        const float inv = l == 0.f ? 0.f : 1.f / l;
        A *out = (A *)a.out + (size_t)(p.q0 + token) * a.out_stride + (size_t)head * a.hd + 4 * d4;
        const A v[4] = {(A)(s.x * inv), (A)(s.y * inv), (A)(s.z * inv), (A)(s.w * inv)};
        store_n<4>(out, v, d.out_wide);
    }
}

// ---- 16-bit caches -----------------------------------------------------------
//
// A block is 32 keys.  S^T = K Q^T on 16x16x32 MFMA: lane (m, g) = (l % 16, l / 16)
// loads 16-byte pieces of K's row m, 64 contiguous bytes for the four g, straight
// into the A operand.  The product leaves a lane the scores of row n = l % 16 and
// keys 4 g + i of either 16, which, rounded, are the B operand of O^T += V^T P^T in a
// k order of its own; V^T's operand in that order comes out of LDS by transposed
// reads (rows padded by 32 bytes: the 8 rows that half a wave reads lie on different
// banks).  No lane ever needs another's score but for the maximum and the sum.
//
// 32 sequences of 1k to 8k keys, 28/4/128, fp32 rows over an fp16 cache: 63 us for 282
// MB, 4.5 TB/s (a large copy: 5.1); one bf16 token over 131072 keys of 16/2/128: 29.6
// us for 134 MB, 4.5 TB/s.
template <class A, class C, int HDP, int W, bool TREE>
__global__ __launch_bounds__(64 * W, HDP <= 128 && W == 4 ? 2 : 1) void decode16_kernel(TileArgs d) {
    // 16-bit rows could have their weights in one part; the second costs nothing beside the loads, and leaves the result
    // no rounding but its own (bf16, one token over 131072 keys: error 1.7e-3 instead of 2.3e-3 of the result)
    constexpr int QP = Parts<A, C>::q, PP = Parts<A, C>::p == 1 ? 2 : Parts<A, C>::p;
    constexpr int KS = HDP / 32, DT = HDP / 16, VR = HDP / 16;   // k-steps, dim tiles, V registers of 16 bytes
    constexpr int kPitch = HDP + 16;                             // of a V row in LDS, elements
    constexpr int kBlock = 32;
    typedef typename Mma<C>::vec8 vec8;
    typedef C vec4 __attribute__((ext_vector_type(4)));
    constexpr size_t kVBytes = sizeof(C) * W * kBlock * kPitch, kOBytes = sizeof(float) * W * HDP * kRows;
    __shared__ __attribute__((aligned(16))) unsigned char shared[kVBytes > kOBytes ? kVBytes : kOBytes];
    __shared__ float2 ml[W][kRows];
    // a careful pass's notes, of eight dims each (take_out)
    __shared__ unsigned kinds[W][2][kBlock][HDP / 32];
    const AttendArgs &a = d.a;
    const int cap = a.b.pages_stride << a.page_shift, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Place p;
    if (!place_of<kRows, TREE>(a.b, d.cut, blockIdx.x, a.n_head_kv, cap, a.window, false, p)) return;
    const Keys k = keys_of<kRows, TREE>(p, d.cut, cap, a.window);
    const int col = lane & 15, g = lane >> 4;
    const Row row = row_of<TREE>(p, p.tile * kRows + col, d, cap);
    const int *table = a.b.pages + (size_t)p.seq * a.b.pages_stride;
    const int slot_mask = (1 << a.page_shift) - 1;
    const bool padded = a.hd != HDP;

    // page groups of this wave: block j's two are lanes 2 (j % 32), + 1
    const int first_block = k.lo / kBlock + wave;
    const auto pages_from = [&](int j) {
        return PageRun::load(a, table, (first_block + W * (j + (lane >> 1))) * 2 + (lane & 1), k.hi);
    };
    const int n_block = k.lo < k.hi ? max(0, ((k.hi + kBlock - 1) / kBlock - first_block + W - 1) / W) : 0;
    PageRun run;
    run.now = pages_from(0);
    run.ahead = -1;

    // Q: B operand, lane (n, g) has dims 32 t + 8 g .. + 7 of its row.  Requested here, used
    // when K and V are on their way.
    A q_row[KS][8];
    load_q<KS>(a, p, row, d.q_wide, 8 * g, 32, q_row);
    // A 16-key group lies in one page: a base that is the wave's, and a lane's offset
    // that does not change.  A group without a page reads page 0.
    const auto base_of = [&](const void *pool, int page, int key) {
        return (const C *)pool + ((((size_t)max(page, 0) * a.n_head_kv + p.head) << a.page_shift) + (key & slot_mask)) * a.hd;
    };
    constexpr int kPerRow = HDP / 8, kRowsPer = 64 / kPerRow;   // 16-byte pieces of a V row; rows a load covers
    const int v_row = lane / kPerRow, v_dim = 8 * (lane % kPerRow);
    unsigned k_off[KS];
#pragma unroll
    for (int t = 0; t < KS; ++t) k_off[t] = col * a.hd + (padded ? min(32 * t + 8 * g, a.hd - 8) : 32 * t + 8 * g);
    const unsigned v_off = v_row * a.hd + (padded ? min(v_dim, a.hd - 8) : v_dim);
    vec8 kr[2][KS], vr[VR];
    int p0 = 0, p1 = 0;   // pages of the block whose K and V are in flight
    const auto load_k = [&](int key0) {
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            const C *src = base_of(a.k_pool, m ? p1 : p0, key0 + 16 * m);
#pragma unroll
            for (int t = 0; t < KS; ++t) kr[m][t] = *reinterpret_cast<const vec8 *>(src + k_off[t]);
        }
    };
    const auto load_v = [&](int key0) {
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            const C *src = base_of(a.v_pool, m ? p1 : p0, key0 + 16 * m);
#pragma unroll
            for (int r = 0; r < VR / 2; ++r) vr[m * (VR / 2) + r] = *reinterpret_cast<const vec8 *>(src + (v_off + kRowsPer * r * a.hd));
        }
    };

    floatx4 o[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i) o[i] = floatx4{0, 0, 0, 0};
    float ref = kNone, sum = 0;
    C *const v_lds = reinterpret_cast<C *>(shared) + wave * kBlock * kPitch;
    // V^T's operand: lane (m, g) needs dim 16 i + m of keys 4 g .. + 3 of either 16
    const C *const v_from = v_lds + (4 * g + (col >> 2)) * kPitch + 4 * (col & 3);
    const auto v_operand = [&](int i) {
        const vec4 x = read_transposed<vec4>(v_from + 16 * i), y = read_transposed<vec4>(v_from + 16 * kPitch + 16 * i);
        return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
    };

    const auto start = [&] {   // run.now holds the first pages
        p0 = run.get(0);
        p1 = run.get(1);
        load_k(first_block * kBlock);
        load_v(first_block * kBlock);
        run.ahead = pages_from(32);
    };
    if (n_block) start();
    vec8 q[QP][KS];
    float unit = 1.f;
    {
        zero_q<KS>(a, row, 8 * g, 32, q_row);
        float to = 1.f;
        if constexpr (QP == 2) {
            float big = 0;
#pragma unroll
            for (int t = 0; t < KS; ++t)
#pragma unroll
                for (int i = 0; i < 8; ++i) big = fmaxf(big, fabsf(q_row[t][i]));
            unit = power(unit_of(max32(max16(big)), to));
        }
#pragma unroll
        for (int t = 0; t < KS; ++t)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if constexpr (QP == 1) {
                    q[0][t][i] = q_row[t][i];
                } else {
                    C part[QP];
                    split_q<QP>(q_row[t][i] * to, part);
#pragma unroll
                    for (int j = 0; j < QP; ++j) q[j][t][i] = part[j];
                }
            }
    }
    const float s2 = scale_of(d.scale_log2, unit);
    const auto pass = [&]<bool CAREFUL>() __attribute__((always_inline)) {
        for (int j = 0; j < n_block; ++j) {
            const int key0 = (first_block + W * j) * kBlock;
            const bool has0 = p0 >= 0, has1 = p1 >= 0;
            const bool whole = key0 >= k.all_lo && key0 + kBlock <= min(k.all_hi, k.hi) && has0 && has1;
            // pages of the next block
            const int next = j + 1, next_key = key0 + W * kBlock;
            if ((next & 31) == 0) {
                run.now = run.ahead;
                run.ahead = pages_from(next + 32);
            }
            p0 = run.get(2 * (next & 31));
            p1 = run.get(2 * (next & 31) + 1);

            if (padded) {
#pragma unroll
                for (int t = 0; t < KS; ++t)
                    if (32 * t + 8 * g >= a.hd) {
                        kr[0][t] = vec8{};
                        kr[1][t] = vec8{};
                    }
            }
            unsigned seen = ~0u;   // keys 16 m + i of the lane's 4 g ..
            if (TREE && !whole) seen = (unsigned)(mask_of(a, p, row, key0) >> (4 * g));
            floatx4 s[2];
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                s[m] = floatx4{0, 0, 0, 0};
#pragma unroll
                for (int t = 0; t < KS; ++t)
#pragma unroll
                    for (int x = 0; x < QP; ++x) s[m] = Mma<C>::mul16(kr[m][t], q[x][t], s[m]);
            }
            if (next < n_block) load_k(next_key);

            // V of positions that no row of the tile sees is 0: it may hold anything
            if (!whole) {
#pragma unroll
                for (int r = 0; r < VR; ++r) {
                    const int key = key0 + kRowsPer * r + v_row;
                    if (!(key < k.hi && key >= k.seen_lo && (kRowsPer * r >= 16 ? has1 : has0))) vr[r] = vec8{};
                }
            }
            bool odd = false;
            if constexpr (CAREFUL) {
#pragma unroll
                for (int r = 0; r < VR; ++r) {
                    unsigned up, down;
                    take_out<C>(vr[r], up, down);
                    unsigned char *const at = reinterpret_cast<unsigned char *>(kinds[wave][0][kRowsPer * r + v_row]) + v_dim / 8;
                    at[0] = (unsigned char)up;
                    at[sizeof kinds[0][0]] = (unsigned char)down;
                    odd |= (up | down) != 0;
                }
                odd = __any(odd);
            }
#pragma unroll
            for (int r = 0; r < VR; ++r) *reinterpret_cast<vec8 *>(v_lds + (kRowsPer * r + v_row) * kPitch + v_dim) = vr[r];
            if (next < n_block) load_v(next_key);

            if (!whole) {
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int key = key0 + 16 * m + 4 * g + i;
                        const bool in = key >= row.lo && key < min(row.hi, k.hi) && (m ? has1 : has0);
                        if (!(in && (!TREE || (seen >> (16 * m + i) & 1)))) s[m][i] = kNone;
                    }
            }
            float top = kNone;
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int i = 0; i < 4; ++i) top = fmaxf(top, s[m][i]);
            top = max32(max16(top));
            follow<CAREFUL>(top, ref, sum, s2, o);
            if (CAREFUL && odd) {
                unsigned has_weight = 0;   // of the block's keys, for the lane's row
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int i = 0; i < 4; ++i) has_weight |= (unsigned)(s[m][i] != kNone) << (16 * m + 4 * g + i);
                has_weight |= __shfl_xor(has_weight, 16);
                has_weight |= __shfl_xor(has_weight, 32);
                for (int e = 0; e < kBlock; ++e) {
                    const bool gets = has_weight >> e & 1;
#pragma unroll
                    for (int i = 0; i < DT; ++i) {
                        const int from = 16 * (i & 1) + 4 * g;
                        const unsigned up = gets ? kinds[wave][0][e][i / 2] >> from : 0, down = gets ? kinds[wave][1][e][i / 2] >> from : 0;
                        if (!__any((up | down) & 15)) continue;
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            if (up >> x & 1) o[i][x] += INFINITY;
                            if (down >> x & 1) o[i][x] -= INFINITY;
                        }
                    }
                }
            }
            const float base = ref == kNone ? 0.f : ref;
            vec8 w[PP];
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float x = exp2_(fmaf(s[m][i] - base, s2, Mma<C>::kBias));
                    C part[PP];
                    split_p<PP>(x, part);
                    sum += x;
#pragma unroll
                    for (int y = 0; y < PP; ++y) w[y][4 * m + i] = part[y];
                }
#pragma unroll
            for (int i = 0; i < DT; ++i) {
                const vec8 v = v_operand(i);
#pragma unroll
                for (int y = 0; y < PP; ++y) o[i] = Mma<C>::mul16(v, w[y], o[i]);
            }
        }
    };
    pass.template operator()<false>();
    if (__builtin_expect(__any(not_finite(o)), 0)) {
#pragma unroll
        for (int i = 0; i < DT; ++i) o[i] = floatx4{0, 0, 0, 0};
        ref = kNone;
        sum = 0;
        run.now = pages_from(0);
        start();
        pass.template operator()<true>();
    }

    sum = sum32(sum16(sum));
    __syncthreads();   // V's rows give way to the states
    float4(*const states)[HDP / 4][kRows] = reinterpret_cast<float4(*)[HDP / 4][kRows]>(shared);
#pragma unroll
    for (int i = 0; i < DT; ++i) states[wave][4 * i + g][col] = make_float4(o[i][0], o[i][1], o[i][2], o[i][3]);
    if (g == 0) ml[wave][col] = make_float2(ref * unit, sum);
    finish<A, HDP, W>(d, p, states, ml);
}

// ---- fp32 caches ---------------------------------------------------------------
//
// A block is 16 keys, both products on 16x16x4 fp32 MFMA (exact products, fp32 sums).
// Lane (m, g) loads K's row m, dims 16 u + 4 g + e: e picks the instruction, g is its
// k.  The scores of keys 4 g + i are its k order of the second product, whose V
// operand, lane (m, g): V[4 g + i][64 j + 4 m + e], comes straight from memory too.
//
// One token over 512 keys of 14/2/64: 6.1 us (a launch's own time is some 2; then three
// rounds of memory); 24 of uneven length, 28/4/128: 100 us for
// 455 MB, 4.5 TB/s.
template <int HDP, int W, bool TREE>
__global__ __launch_bounds__(64 * W, HDP <= 128 && W == 4 ? 2 : 1) void decode32_kernel(TileArgs d) {
    constexpr int KU = HDP / 16, DJ = HDP / 64, kBlock = 16;
    __shared__ float4 states[W][HDP / 4][kRows];
    __shared__ float2 ml[W][kRows];
    const AttendArgs &a = d.a;
    const int cap = a.b.pages_stride << a.page_shift, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Place p;
    if (!place_of<kRows, TREE>(a.b, d.cut, blockIdx.x, a.n_head_kv, cap, a.window, false, p)) return;
    const Keys k = keys_of<kRows, TREE>(p, d.cut, cap, a.window);
    const int col = lane & 15, g = lane >> 4;
    const Row row = row_of<TREE>(p, p.tile * kRows + col, d, cap);
    const int *table = a.b.pages + (size_t)p.seq * a.b.pages_stride;
    const int slot_mask = (1 << a.page_shift) - 1;
    const bool padded = a.hd != HDP;

    // block j's page is lane j % 64
    const int first_block = k.lo / kBlock + wave;
    const auto pages_from = [&](int j) { return PageRun::load(a, table, first_block + W * (j + lane), k.hi); };
    const int n_block = k.lo < k.hi ? max(0, ((k.hi + kBlock - 1) / kBlock - first_block + W - 1) / W) : 0;
    PageRun run;
    run.now = pages_from(0);
    run.ahead = -1;

    floatx4 q[KU];
    {
        const float *const src = (const float *)a.q + (size_t)(row.real ? p.q0 + row.token : p.q0) * a.q_stride +
                                 (size_t)(row.real ? row.head : 0) * a.hd;
#pragma unroll
        for (int u = 0; u < KU; ++u) {
            const float *const at = src + min(16 * u + 4 * g, a.hd - 4);
            if (d.q_wide) q[u] = *reinterpret_cast<const floatx4 *>(at);
            else q[u] = floatx4{at[0], at[1], at[2], at[3]};
        }
    }
    const auto base_of = [&](const void *pool, int page, int key) {
        return (const float *)pool + ((((size_t)max(page, 0) * a.n_head_kv + p.head) << a.page_shift) + (key & slot_mask)) * a.hd;
    };
    unsigned k_off[KU], v_off[DJ];
#pragma unroll
    for (int u = 0; u < KU; ++u) k_off[u] = col * a.hd + (padded ? min(16 * u + 4 * g, a.hd - 4) : 16 * u + 4 * g);
#pragma unroll
    for (int x = 0; x < DJ; ++x) v_off[x] = 4 * g * a.hd + (padded ? min(64 * x + 4 * col, a.hd - 4) : 64 * x + 4 * col);
    floatx4 kr[KU], vr[4][DJ];
    int page = 0;
    const auto load_k = [&](int key0) {
        const float *src = base_of(a.k_pool, page, key0);
#pragma unroll
        for (int u = 0; u < KU; ++u) kr[u] = *reinterpret_cast<const floatx4 *>(src + k_off[u]);
    };
    const auto load_v = [&](int key0) {
        const float *src = base_of(a.v_pool, page, key0);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int x = 0; x < DJ; ++x) vr[i][x] = *reinterpret_cast<const floatx4 *>(src + (v_off[x] + i * a.hd));
    };
    floatx4 o[4 * DJ];
#pragma unroll
    for (int i = 0; i < 4 * DJ; ++i) o[i] = floatx4{0, 0, 0, 0};
    float ref = kNone, sum = 0;

    const auto start = [&] {   // as above
        page = run.get(0);
        load_k(first_block * kBlock);
        load_v(first_block * kBlock);
        run.ahead = pages_from(64);
    };
    if (n_block) start();
#pragma unroll
    for (int u = 0; u < KU; ++u)
        if (!row.real || 16 * u + 4 * g >= a.hd) q[u] = floatx4{0, 0, 0, 0};
    const auto pass = [&]<bool CAREFUL>() __attribute__((always_inline)) {
        for (int j = 0; j < n_block; ++j) {
            const int key0 = (first_block + W * j) * kBlock;
            const bool has = page >= 0, whole = key0 >= k.all_lo && key0 + kBlock <= min(k.all_hi, k.hi) && has;
            const int next = j + 1, next_key = key0 + W * kBlock;
            if ((next & 63) == 0) {
                run.now = run.ahead;
                run.ahead = pages_from(next + 64);
            }
            page = run.get(next & 63);

            if (padded) {
#pragma unroll
                for (int u = 0; u < KU; ++u)
                    if (16 * u + 4 * g >= a.hd) kr[u] = floatx4{0, 0, 0, 0};
            }
            unsigned seen = ~0u;   // keys of the lane's 4 g ..
            if (TREE && !whole) seen = (unsigned)(mask_of(a, p, row, key0) >> (4 * g));
            floatx4 s = floatx4{0, 0, 0, 0}, s2 = floatx4{0, 0, 0, 0};   // two chains
#pragma unroll
            for (int u = 0; u < KU; ++u)
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    s = __builtin_amdgcn_mfma_f32_16x16x4f32(kr[u][e], q[u][e], s, 0, 0, 0);
                    s2 = __builtin_amdgcn_mfma_f32_16x16x4f32(kr[u][e + 1], q[u][e + 1], s2, 0, 0, 0);
                }
            s += s2;
            if (next < n_block) load_k(next_key);

            if (!whole) {   // V as for 16-bit caches
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = key0 + 4 * g + i;
                    const bool in = key < k.hi && key >= k.seen_lo && has;
                    if (!(in && key >= row.lo && key < row.hi && (!TREE || (seen >> i & 1)))) s[i] = kNone;
#pragma unroll
                    for (int x = 0; x < DJ; ++x)
                        if (!in) vr[i][x] = floatx4{0, 0, 0, 0};
                }
            }
            float top = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
            top = max32(max16(top));
            follow<CAREFUL>(top, ref, sum, d.scale_log2, o);
            if constexpr (CAREFUL) {
                unsigned has_weight = 0;   // of the block's keys, for the lane's row
#pragma unroll
                for (int i = 0; i < 4; ++i) has_weight |= (unsigned)(s[i] != kNone) << (4 * g + i);
                has_weight |= __shfl_xor(has_weight, 16);
                has_weight |= __shfl_xor(has_weight, 32);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    bool odd = false;
#pragma unroll
                    for (int x = 0; x < DJ; ++x)
#pragma unroll
                        for (int e = 0; e < 4; ++e) odd |= !finite(vr[i][x][e]);
                    if (!__any(odd)) continue;
                    // key by key, laid over the rows by a product with 1
#pragma unroll 1
                    for (int y = 0; y < 4; ++y) {
                        const bool gets = has_weight >> (4 * y + i) & 1;
#pragma unroll
                        for (int x = 0; x < DJ; ++x)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const floatx4 t = __builtin_amdgcn_mfma_f32_16x16x4f32(g == y && !finite(vr[i][x][e]) ? vr[i][x][e] : 0.f, 1.f,
                                                                                      floatx4{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
                                for (int z = 0; z < 4; ++z)
                                    if (gets) o[4 * x + e][z] += t[z];
                            }
                    }
#pragma unroll
                    for (int x = 0; x < DJ; ++x)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (!finite(vr[i][x][e])) vr[i][x][e] = 0.f;
                }
            }
            const float base = ref == kNone ? 0.f : ref;
            float w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                w[i] = exp2_(fmaf(s[i] - base, d.scale_log2, Mma<bhalf_t>::kBias));
                sum += w[i];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int x = 0; x < DJ; ++x)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        o[4 * x + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(vr[i][x][e], w[i], o[4 * x + e], 0, 0, 0);
            if (next < n_block) load_v(next_key);
        }
    };
    pass.template operator()<false>();
    if (__builtin_expect(__any(not_finite(o)), 0)) {
#pragma unroll
        for (int i = 0; i < 4 * DJ; ++i) o[i] = floatx4{0, 0, 0, 0};
        ref = kNone;
        sum = 0;
        run.now = pages_from(0);
        start();
        pass.template operator()<true>();
    }

    sum = sum32(sum16(sum));
    // o[4 x + e], lane (n, g), element i: dim 64 x + 4 (4 g + i) + e of row n
#pragma unroll
    for (int x = 0; x < DJ; ++x)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            states[wave][16 * x + 4 * g + i][col] = make_float4(o[4 * x][i], o[4 * x + 1][i], o[4 * x + 2][i], o[4 * x + 3][i]);
    if (g == 0) ml[wave][col] = make_float2(ref, sum);
    finish<float, HDP, W>(d, p, states, ml);
}

// ---- the merge of splits ---------------------------------------------------------
//
// TILE rows by 256 / TILE lanes, which are laid over the tile's splits and, what is left
// of them, over the dims, four a lane.  A lane has eight splits' loads in flight and a
// running reference; the lanes' states meet in LDS.  gridDim.y workgroups share a
// tile's dims.  (Few tiles may have hundreds of splits, many tiles two each.)  Bound by
// its launch and two rounds of memory: 4.7 us for two tiles of eight splits, 7.5 for 128
// of three, 12.4 for 112 of 128 rows.
template <class A, int TILE, bool TREE>
__global__ __launch_bounds__(kThreads) void merge_kernel(TileArgs d, int hd4) {
    constexpr int kLanes = kThreads / TILE, kFlight = 8;
    __shared__ float4 so[kLanes][TILE];
    __shared__ float2 sm[kLanes][TILE];
    const AttendArgs &a = d.a;
    const int cap = a.b.pages_stride << a.page_shift;
    Place p;
    if (!place_of<TILE, TREE>(a.b, d.cut, blockIdx.x, a.n_head_kv, cap, a.window, true, p)) return;
    if ((unsigned)p.part + (unsigned)(p.n_split - 1) * (unsigned)a.n_head_kv >= (unsigned)d.parts) return;   // as there
    int parts = 1;
    while (parts < kLanes && parts < p.n_split) parts *= 2;
    const int row = threadIdx.x % TILE, lane = threadIdx.x / TILE, part = lane & (parts - 1), wide = kLanes / parts;
    const size_t step = (size_t)a.n_head_kv * TILE;
    const float2 *const pm = reinterpret_cast<const float2 *>(d.part_ml) + (size_t)p.part * TILE + row;
    const int r = p.tile * TILE + row, token = d.cut.by_rep.of(r), head = p.head * d.cut.rep + r - token * d.cut.rep;
    A *const out = (A *)a.out + (size_t)(p.q0 + token) * a.out_stride + (size_t)head * a.hd;
    for (int d0 = blockIdx.y * wide; 4 * d0 < a.hd; d0 += gridDim.y * wide) {
        const int d4 = d0 + lane / parts;
        const bool real = 4 * d4 < a.hd;
        const float4 *const po = reinterpret_cast<const float4 *>(d.part_o) + ((size_t)p.part * hd4 + d4) * TILE + row;
        float m = kNone, l = 0;
        float4 s = make_float4(0, 0, 0, 0);
        for (int i = part; real && i < p.n_split; i += kFlight * parts) {
            float2 e[kFlight];
            float4 v[kFlight];
#pragma unroll
            for (int x = 0; x < kFlight; ++x) {
                const int n = i + x * parts;
                e[x] = make_float2(kNone, 0.f);
                v[x] = make_float4(0, 0, 0, 0);
                if (n < p.n_split) {
                    e[x] = pm[n * step];
                    v[x] = po[n * step * hd4];
                }
            }
            float next = m;
#pragma unroll
            for (int x = 0; x < kFlight; ++x) next = fmaxf(next, e[x].x);
            const float f = share_at(m, next, d.scale_log2);
            l *= f;
            s = make_float4(s.x * f, s.y * f, s.z * f, s.w * f);
#pragma unroll
            for (int x = 0; x < kFlight; ++x) {
                const float g = share_at(e[x].x, next, d.scale_log2);
                l = fmaf(e[x].y, g, l);
                s = make_float4(fmaf(v[x].x, g, s.x), fmaf(v[x].y, g, s.y), fmaf(v[x].z, g, s.z), fmaf(v[x].w, g, s.w));
            }
            m = next;
        }
        so[lane][row] = s;
        sm[lane][row] = make_float2(m, l);
        __syncthreads();
        if (real && part == 0 && r < p.n * d.cut.rep) {
            for (int i = 1; i < parts; ++i) m = fmaxf(m, sm[lane + i][row].x);
            l = 0;
            s = make_float4(0, 0, 0, 0);
            for (int i = 0; i < parts; ++i) {
                const float2 e = sm[lane + i][row];
                const float4 v = so[lane + i][row];
                const float g = share_at(e.x, m, d.scale_log2);
                l = fmaf(e.y, g, l);
                s = make_float4(fmaf(v.x, g, s.x), fmaf(v.y, g, s.y), fmaf(v.z, g, s.z), fmaf(v.w, g, s.w));
            }
            const float inv = l == 0.f ? 0.f : 1.f / l;
            const A w[4] = {(A)(s.x * inv), (A)(s.y * inv), (A)(s.z * inv), (A)(s.w * inv)};
            store_n<4>(out + 4 * d4, w, d.out_wide);
        }
        __syncthreads();
    }
}

template <int W, bool TREE>
hipError_t launch_decode(const TileArgs &d, hipStream_t s) {
    const int hdp = padded_dim(d.a.hd);
    const dim3 grid((unsigned)d.places);
#define KORE_DECODE(KERNEL, ...)                                                                \
    do {                                                                                        \
        if (hdp == 64) return launch(KERNEL<__VA_ARGS__ 64, W, TREE>, grid, 64 * W, 0, s, d);                    \
        else if (hdp == 128) return launch(KERNEL<__VA_ARGS__ 128, W, TREE>, grid, 64 * W, 0, s, d);             \
        else if constexpr (W == 4) return launch(KERNEL<__VA_ARGS__ 256, W, TREE>, grid, 64 * W, 0, s, d);       \
    } while (0)
#define KORE_COMMA ,
    if (d.a.cache_type == kF32) KORE_DECODE(decode32_kernel);
    else if (d.a.type == kF32 && d.a.cache_type == kF16) KORE_DECODE(decode16_kernel, float KORE_COMMA half_t KORE_COMMA);
    else if (d.a.type == kF32) KORE_DECODE(decode16_kernel, float KORE_COMMA bhalf_t KORE_COMMA);
    else if (d.a.type == kF16) KORE_DECODE(decode16_kernel, half_t KORE_COMMA half_t KORE_COMMA);
    else KORE_DECODE(decode16_kernel, bhalf_t KORE_COMMA bhalf_t KORE_COMMA);
#undef KORE_COMMA
#undef KORE_DECODE
    return hipErrorInvalidValue;   // (a head of more than 128 in eight waves: launch_attend makes no such call)
}

constexpr int kPerCu = 2;                              // workgroups of a CU, of the 16-row kernels
constexpr int kShort = 1280;                           // keys that a tile among many is not split for

template <bool TREE>
hipError_t launch_attend(const AttendArgs &a, hipStream_t s) {
    TileArgs d{};
    d.a = a;
    d.cut.rep = a.n_head / a.n_head_kv;
    d.cut.by_rep = divisor(d.cut.rep);
    d.cut.by_heads = divisor(a.n_head_kv);
    const int size = type_bytes(a.type);   // (a head is a multiple of 8 values)
    d.q_wide = (uintptr_t)a.q % 16 == 0 && a.q_stride * size % 16 == 0;
    d.out_wide = (uintptr_t)a.out % (4 * size) == 0 && a.out_stride % 4 == 0;
    const int max_q = a.max_q ? a.max_q : (a.b.n_tok + a.b.n_seq - 1) / a.b.n_seq;
    // Tiles of 16 rows read a sequence's keys once each, most of it from L2: up to three of them beat one of 128.  us, 16 /
    // 128 rows a tile, 28/4/128 at 32768 keys, new rows 2, 6, 9, 18: fp16 20.7 / 26.6, 27.5 / 26.7, 42.3 / 26.7, 53.3 /
    // 28.8; fp32 rows and cache 32 / 55, 56 / 57, 80 / 56, 124 / 61; 16 sequences of 2048, fp16: 23.4 / 27.8, 30.9 / 27.9,
    // 30.0 / 28.3, 47.5 / 36.5.
    bool chunk = (long long)max_q * d.cut.rep > 3 * kRows;
    // Trees have up to some hundred rows a kv-head, and every tile reads all keys of its sequence: which tiles take less time
    // goes by both.  A launch of either takes a start, the merge in it (more of it for wide heads in tiles of 16, and for many
    // tiles of 128), and so much for each key of each tile: us, heads of 128, fitted to 1 to 16 trees of 8 to 32 tokens over
    // 500 to 8000 keys, run with both.  The keys are those that the table's width and the window allow, since the host knows no
    // lengths: over 171 such cases and other heads, with tables as wide as the longest sequence, it takes 1.02 times the better
    // tiles' time (1.42 at most); behind wide tables it may take 128 rows where 16 would do (us, tight / 4096 / 32768 positions:
    // 1 tree of 8 over 500 fp16 keys 10.7 / 11.4 / 14.7, of 32 10.7 / 18.0 / 14.5, fp32 rows 12.2 / 20.2 / 18.3, fp32 cache 20.2 /
    // 23.2 / 23.2; 16 trees of 32 over 1000 29.5 / 31.4 / 31.2, 43.8 / 41.6 / 41.6, 96.9 / 70.9 / 70.9).  us, 16 / 128 rows a tile, 28/4/128, 1 tree of 8 over 500, of 32 over 8000, 16 of 32 over 2000: fp16 10.5 /
    // 14.3, 32.4 / 20.8, 82 / 44; fp32 rows over fp16 12.2 / 18.3, 34.0 / 28.4, 86 / 62; fp32 cache 12.4 / 23.1, 58 / 42, 199 / 118.
    if (TREE) {
        const bool f32 = a.cache_type == kF32, parts = a.type == kF32;
        const auto us = [&](int tile, double start, double each, double full) {
            const long long of_all = (long long)a.b.n_tok * d.cut.rep / tile + a.b.n_seq;
            const long long of_each = ((long long)max_q * d.cut.rep + tile - 1) / tile * a.b.n_seq;
            const double tiles = (double)std::min(of_all, of_each) * a.n_head_kv;
            const double keys = (double)std::min((long long)a.b.pages_stride << a.page_shift, (long long)a.window + max_q);
            return start + full * std::min(tiles / 64, 1.0) + each * tiles * keys * padded_dim(a.hd) / 128;
        };
        chunk = us(kChunkRows, f32 ? 24 : parts ? 18 : 16, f32 ? 33e-5 : parts ? 15e-5 : 9e-5, 4) <
                us(kRows, a.hd > 128 ? 22 : f32 ? 12 : 10, f32 ? 10.5e-5 : 4e-5, 0);
    }
    const int rows = chunk ? kChunkRows : kRows;
    // the most (tile, kv-head)s that n_tok rows of n_seq sequences can be
    const long long tiles = ((long long)a.b.n_tok * d.cut.rep / rows + std::min(a.b.n_seq, a.b.n_tok)) * a.n_head_kv;
    // Few tiles: splits make up the workgroups that the card holds at once.  From half of those on it is the longest tiles
    // alone that are split, those of some twice the mean (chunks) or over it (16 rows), and none where a tile cannot have
    // many keys or all are one sequence's: the merge's launch and the partials cost every call.  us, split / not, 28/4/128:
    //   rows of one sequence over 4096 keys, tiles 34 %, 50 %, 59 % of the CUs: fp16 55 / 80, 60 / 79, 80 / 77; fp32 160 /
    //   271, 172 / 278, 276 / 272;
    //   four prompts of 512 beside a token over 1024, 2048, 65536: fp16 44.7 / 41.0, 49.1 / 56.7, 77 / 1041; fp32 122 / 119,
    //   128 / 179, 208 / 4025;
    //   100 tokens over 300 keys, one over 1024, 2048, 65536: 23.0 / 20.6, 24.8 / 29.5, 60 / 645;
    //   300 tokens over 1000 keys, one over 65536: 186 / 776; 300 over 1100: 137 / 124 (the price of being ready for it).
    const int at_once = chunk ? a.num_cu : kPerCu * a.num_cu;
    const long long most = std::min((long long)a.b.pages_stride << a.page_shift,
                                    (long long)a.window + (TREE ? a.b.n_tok : (rows - 1) / d.cut.rep) + 65);
    // A split's fewest keys, of 64, 128 and 256: 64 fp32 rows over 512 keys 22.6, 25.1, 32.4 us; 64 fp16 rows 15.5, 15.3,
    // 16.8; one token over 512 keys 9.6, 10.1, 11.2.
    d.cut.min_len = chunk && size == 2 ? 128 : 64;
    // Few tiles of 16 rows whose K and V cannot be much stay whole, with twice the waves, and need no merge: up to some 240
    // KB, and more where there are more tiles to split.  us, split / whole: a token over 256 keys of 14/2/64 fp32 (128 KB)
    // 9.6 / 7.3, over 512 9.9 / 10.1; of 28/4/128 fp16 over 256 (128 KB) 11.8 / 9.6, 512 12.1 / 10.9, 1024 12.5 / 15.3; 32
    // tokens of those over 512 15.5 / 12.3, 1024 23.0 / 16.9.  (16 waves for heads of 64: 8.5 and 11.1 in the first case.)
    const bool few = 2 * tiles <= at_once;
    const bool wide = !chunk && few && a.hd <= 128 && most > d.cut.min_len &&
                      2 * most * a.hd * type_bytes(a.cache_type) <= (240 + 2 * tiles) << 10;
    if (wide) d.cut.target = 0;
    else if (few) d.cut.target = most > d.cut.min_len ? (int)(at_once - tiles) : 0;
    else if (a.b.n_seq == 1 || most <= kShort) d.cut.target = 0;
    else d.cut.target = (int)(chunk ? std::min<long long>(tiles / 2, at_once) : std::min<long long>(tiles, at_once / 2));
    // Trees that are split at all fill the card once, where a lane has each sequence (fitting_len).  us, by target / so,
    // 28/4/128: 16 of up to 32 over up to 8000 fp16 keys, fp32 rows 200 / 91; 8 of 32 over 4000, fp16 41 / 37; 32 of up to 16
    // over up to 2000 fp32 keys 132 / 89; one of 63 over 131000 bf16 keys of 16/2/128 97 / 91.
    if (TREE && d.cut.target && a.b.n_seq <= 64) d.cut.at_once = at_once;
    d.scale_log2 = (float)((double)a.scale * 1.4426950408889634074);
    const int hdp = padded_dim(a.hd);
    d.places = std::max((int)tiles + d.cut.target, d.cut.at_once);
    d.part_o = a.part;
    d.parts = std::max(d.cut.target + (int)std::min<long long>(d.cut.target, tiles), d.cut.at_once);
    d.part_ml = a.part + (size_t)d.parts * rows * hdp;
    const hipError_t e = chunk ? launch_chunk(d, s) : wide ? launch_decode<8, TREE>(d, s) : launch_decode<4, TREE>(d, s);
    if (e != hipSuccess || !d.cut.target) return e;
    // some eight workgroups a CU, where there are dims enough (32 sequences, fp16 cache: 57.8 us from cache, with one a CU
    // 78.3, with 32 59.9)
    const int joined = (int)std::min<long long>(std::max(d.cut.target, d.cut.at_once / 2), tiles);   // the most tiles that can be split
    const dim3 merge((unsigned)joined, (unsigned)std::clamp(8 * a.num_cu / joined, 1, a.hd / 4));
#define KORE_MERGE(A)                                                                    \
    do {                                                                                 \
        if (chunk) return launch(merge_kernel<A, kChunkRows, TREE>, merge, kThreads, 0, s, d, hdp / 4);   \
        else return launch(merge_kernel<A, kRows, TREE>, merge, kThreads, 0, s, d, hdp / 4);              \
    } while (0)
    if (a.type == kF32) KORE_MERGE(float);
    else if (a.type == kF16) KORE_MERGE(half_t);
    else KORE_MERGE(bhalf_t);
#undef KORE_MERGE
}

}  // namespace

size_t attend_workspace_bytes(int hd, int num_cu) {
    return 2 * (size_t)num_cu * kChunkRows * ((size_t)padded_dim(hd) + 2) * sizeof(float);
}

hipError_t launch_attend(const AttendArgs &a, hipStream_t s) {
    return a.tree.mask ? launch_attend<true>(a, s) : launch_attend<false>(a, s);
}

}  // namespace kore_paged_gpu

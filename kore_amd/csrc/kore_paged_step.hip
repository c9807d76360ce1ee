// kore_paged_step.hip - the tables of a step of drafted tokens, and what is kept of
// it (gfx950).
//
// Whole numbers and copies, a few bytes a row: both are launches and rounds of
// dependent loads, not bandwidth, but for the rows that keep moves.
#include "kore_paged_device.h"

#include <algorithm>

namespace kore_paged_gpu {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;

// ---- sums over a workgroup ------------------------------------------------------

// Inclusive sums over the wave of 64-bit numbers: in DPP steps as in kore_paged_attend.h.
template <int CTRL, int ROWS>
__device__ __forceinline__ long long from_lane(long long x) {
    const int lo = __builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false);
    const int hi = __builtin_amdgcn_update_dpp(0, (int)(x >> 32), CTRL, ROWS, 0xf, false);
    return (long long)(unsigned)lo | (long long)hi << 32;
}
__device__ __forceinline__ long long wave_prefix(long long x) {
    x += from_lane<0x111, 0xf>(x);
    x += from_lane<0x112, 0xf>(x);
    x += from_lane<0x114, 0xf>(x);
    x += from_lane<0x118, 0xf>(x);
    x += from_lane<0x142, 0xa>(x);
    x += from_lane<0x143, 0xc>(x);
    return x;
}

// Two numbers a thread: what the threads before it have, and all of them.  (One barrier:
// `waves` is not used again before another.)
struct Sums {
    long long before[2], all[2];
};
__device__ __forceinline__ long long of_lane(long long x, int lane) {
    return (long long)(unsigned)__builtin_amdgcn_readlane((int)x, lane) | (long long)__builtin_amdgcn_readlane((int)(x >> 32), lane) << 32;
}
__device__ __forceinline__ Sums block_sums(long long x, long long y, long long (*waves)[2]) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = blockDim.x >> 6;
    const long long px = wave_prefix(x), py = wave_prefix(y);
    Sums s{{px - x, py - y}, {of_lane(px, 63), of_lane(py, 63)}};
    if (n == 1) return s;
    if (lane == 63) {
        waves[wave][0] = px;
        waves[wave][1] = py;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {   // the waves' sums, one a lane
        const long long of = wave_prefix(lane < n ? waves[lane][i] : 0);
        if (wave) s.before[i] += of_lane(of, wave - 1);
        s.all[i] = of_lane(of, 63);
    }
    return s;
}

// ---- the plan ---------------------------------------------------------------------

// A request: its rows, what it holds, the pages it has and those it needs.  One that no
// table holds asks for more rows than any step has.
constexpr long long kBad = 1LL << 40;
struct Request {
    int held, n, had, need;
    bool bad;
    __device__ __forceinline__ long long rows() const { return bad ? kBad : n; }
};
__device__ __forceinline__ Request request(const PlanArgs &a, int s) {
    Request r{0, 0, 0, 0, false};
    if (s >= a.n_seq) return r;
    const int n = a.n_new[s], mask = (1 << a.page_shift) - 1;
    r.held = a.kv_held[s];
    r.bad = n < 0 || r.held < 0 || (long long)n + r.held > (long long)a.pages_stride << a.page_shift || (a.words && n > 64 * a.words);
    if (r.bad) return r;
    r.n = n;
    r.had = (int)(((long long)r.held + mask) >> a.page_shift);
    r.need = (int)(((long long)r.held + n + mask) >> a.page_shift) - r.had;
    return r;
}

// What comes of the sums of all: 0, or why there is no step.
__device__ __forceinline__ int status_of(const PlanArgs &a, const Sums &all, int n_free) {
    if (n_free < 0 || n_free > a.n_pages || all.all[0] > a.n_tok) return -1;
    return (int)min(max(all.all[1] - n_free, 0LL), (long long)INT_MAX);
}

// A row's depth in its tree and its mask: a walk from parent to parent, each before the
// row, so that it ends.  parent: of the sequence's rows.  A row holds one bit for itself
// and each row before it, or the last `window` of them, which are the highest.
__device__ __forceinline__ int ancestors(const PlanArgs &a, int i, const int *parent, unsigned long long *mask) {
    int at = i, depth = -1;
    for (int w = a.words - 1; w >= 0; --w) {
        unsigned long long bits = 0;
        while (at >= 64 * w) {
            bits |= 1ULL << (at & 63);
            const int up = parent[at];
            at = (unsigned)up < (unsigned)at ? up : -1;   // (a negative one is a large one)
        }
        mask[w] = bits;
        depth += __popcll(bits);
    }
    // (taken off afterwards, by the rows that are so deep alone: the walk itself is what a plan of deep trees takes)
    for (int w = 0, off = depth + 1 - a.window; off > 0; ++w) {
        unsigned long long bits = mask[w];
        const int n = __popcll(bits);
        if (n <= off) {
            bits = 0;
            off -= n;
        } else {
            for (; off > 0; --off) bits &= bits - 1;
        }
        mask[w] = bits;
    }
    return depth;
}

// A row's entries: the i-th new one of a sequence that held `held`, its slot on `page`.
__device__ __forceinline__ void put_row(const PlanArgs &a, int row, bool real, int i, int held, int page, const int *parent) {
    unsigned long long *const mask = a.mask + (size_t)row * a.words;
    const int at = held + i;
    int pos = -1;
    long long slot = -1;
    if (real) {
        pos = a.words ? held + ancestors(a, i, parent, mask) : at;
        if (page >= 0 && page < a.n_pages) slot = ((long long)page << a.page_shift) + (at & ((1 << a.page_shift) - 1));
    } else {
        for (int w = 0; w < a.words; ++w) mask[w] = 0;
    }
    a.pos[row] = pos;
    a.slot[row] = slot;
}

// The last of n numbers, ascending from one that is x or less, that is x or less.
template <class F>
__device__ __forceinline__ int last_upto(const F &number, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int m = (lo + hi) >> 1;
        if (number(m) <= x) lo = m;
        else hi = m;
    }
    return lo;
}

// A step whose sequences have a thread each: every workgroup sums them all and takes
// some of the rows; the first one also writes what is the sequences'.  Two rounds
// of memory: the requests, the parents of the workgroup's rows and the number of free
// pages; then the pages that rows go into, a sequence's last and those at the end of the
// free ones.  The rest is in LDS: a row's sequence by halves, its ancestors one after the
// other.  (Workgroups but the first need inputs that the first does not overwrite.)
//
// A token of one sequence 3.1 us (up to 3.9 where the host issues more slowly), 64 trees of
// up to 32 4.3, 24 thousand rows of 1000 sequences 5.4: a launch of some 2 and the rounds.
// Deep trees walk an LDS latency a row above: 8 of up to 320 rows, half as deep, 12 us.
__global__ __launch_bounds__(kThreads) void plan_kernel(PlanArgs a) {
    __shared__ long long waves[kWaves][2];
    __shared__ int starts[kThreads], firsts[kThreads], helds[kThreads], lasts[kThreads], tops[kThreads];
    __shared__ int parents[kThreads + 64 * kMaxWords];   // of the rows before the workgroup's that their trees may have, and of its own
    const int tid = threadIdx.x, T = blockDim.x, page_mask = (1 << a.page_shift) - 1;
    int base = blockIdx.x * T;
    const int before = 64 * a.words, n_free = a.n_free[0];
    const auto stage_parents = [&] {
        for (int x = tid; x < before + T; x += T) {
            const int row = base - before + x;
            parents[x] = row >= 0 && row < a.n_tok ? a.parent[row] : -1;
        }
    };
    if (a.words) stage_parents();
    const Request r = request(a, tid);
    if (a.n_seq && tid < n_free && n_free <= a.n_pages) tops[tid] = a.free_pages[n_free - 1 - tid];
    // of the pages that a sequence holds only the last has room
    lasts[tid] = !r.bad && r.held & page_mask ? a.pages[(size_t)tid * a.pages_stride + (r.held >> a.page_shift)] : -1;
    helds[tid] = r.held;
    const Sums sum = block_sums(r.rows(), r.need, waves);
    const int status = status_of(a, sum, n_free), n_rows = status ? 0 : (int)sum.all[0], start = status ? 0 : (int)sum.before[0];
    starts[tid] = start;
    firsts[tid] = status ? 0 : (int)sum.before[1] - r.had;   // page j of the sequence is new page firsts + j of all
    if (blockIdx.x == 0) {
        if (tid == 0) {
            a.status[0] = status;
            a.n_free_out[0] = status ? n_free : n_free - (int)sum.all[1];
            a.q_start[0] = 0;
        }
        if (tid < a.n_seq) {
            a.q_start[tid + 1] = status ? 0 : start + r.n;
            a.kv_len[tid] = status ? r.held : r.held + r.n;
        }
    }
    __syncthreads();
    for (bool again = false; base < a.n_tok; base += gridDim.x * T, again = true) {
        if (a.words && again) {
            __syncthreads();
            stage_parents();
            __syncthreads();
        }
        const int row = base + tid;
        if (row >= a.n_tok) continue;
        const bool real = row < n_rows;
        int first = 0, i = 0, held = 0, page = -1;
        if (real) {
            const int l = last_upto([&](int m) { return starts[m]; }, a.n_seq, row);
            first = starts[l];
            i = row - first;
            held = helds[l];
            const int j = (held + i) >> a.page_shift;
            if (j << a.page_shift >= held) {
                const int number = firsts[l] + j;
                page = number < T ? tops[number] : a.free_pages[n_free - 1 - number];
                if (((held + i) & page_mask) == 0) a.pages[(size_t)l * a.pages_stride + j] = page;
            } else {
                page = lasts[l];
            }
        }
        put_row(a, row, real, i, held, page, parents + (first - base + before));
    }
}

// Steps of more sequences, or of many rows whose outputs take the place of the inputs: one
// workgroup for what is the sequences', kThreads of them at a time, then the rows.  2500
// sequences of four rows 14 us.
__global__ __launch_bounds__(kThreads) void plan_sequences_kernel(PlanArgs a) {
    __shared__ long long waves[kWaves][2];
    __shared__ int firsts[kThreads], hads[kThreads];   // of a round's sequences
    const int tid = threadIdx.x, n_free = a.n_free[0];
    long long rows = 0, need = 0;
    for (int s = tid; s < a.n_seq; s += kThreads) {
        const Request r = request(a, s);
        rows += r.rows();
        need += r.need;
    }
    const Sums all = block_sums(rows, need, waves);
    const int status = status_of(a, all, n_free);
    if (tid == 0) {
        a.status[0] = status;
        a.n_free_out[0] = status ? n_free : n_free - (int)all.all[1];
        a.q_start[0] = 0;
    }
    long long row_at = 0, need_at = 0;
    for (int s0 = 0; s0 < a.n_seq; s0 += kThreads) {
        const int s = s0 + tid;
        Request r = request(a, s);
        if (status) r.n = r.need = 0;
        __syncthreads();
        const Sums sum = block_sums(r.n, r.need, waves);
        if (s < a.n_seq) {
            a.q_start[s + 1] = (int)(row_at + sum.before[0]) + r.n;
            a.kv_len[s] = r.held + r.n;
        }
        firsts[tid] = (int)(need_at + sum.before[1]);
        hads[tid] = r.had;
        __syncthreads();
        for (int x = tid; x < (int)sum.all[1]; x += kThreads) {   // the round's new pages
            const int number = (int)need_at + x;
            const int l = last_upto([&](int m) { return firsts[m]; }, min(kThreads, a.n_seq - s0), number);
            a.pages[(size_t)(s0 + l) * a.pages_stride + hads[l] + number - firsts[l]] = a.free_pages[n_free - 1 - number];
        }
        row_at += sum.all[0];
        need_at += sum.all[1];
    }
}
__global__ __launch_bounds__(256) void plan_rows_kernel(PlanArgs a) {
    const int row = blockIdx.x * 256 + threadIdx.x;
    if (row >= a.n_tok) return;
    const bool real = row < a.q_start[a.n_seq];
    int first = 0, i = 0, held = 0, page = -1;
    if (real) {
        const int s = last_upto([&](int m) { return a.q_start[m]; }, a.n_seq, row);
        first = a.q_start[s];
        i = row - first;
        held = a.kv_len[s] - (a.q_start[s + 1] - first);
        page = a.pages[(size_t)s * a.pages_stride + ((held + i) >> a.page_shift)];
    }
    put_row(a, row, real, i, held, page, a.parent + first);
}

// ---- what is kept -------------------------------------------------------------------

// A sequence's end: positions before and after.
struct End {
    int start, n, keep, kv, after;
};
__device__ __forceinline__ End end_of(const KeepArgs &a, int s) {
    End e;
    e.start = min(max(a.q_start[s], 0), a.n_tok);
    e.n = min(max(a.q_start[s + 1], e.start), a.n_tok) - e.start;
    e.kv = max(a.kv_len[s], 0);
    const int keep = a.n_keep[s];
    e.keep = min(keep, e.n);
    e.after = keep < 0 ? 0 : max(0, e.kv - e.n + e.keep);
    return e;
}

// The moves of a sequence, by workgroup `part` of `share`.  A thread has 16 bytes of a
// position's K or V, of one kv-head of a layer, and moves them from row to row, eight rows
// in flight: what it overwrites lies before all that it has still to read, since the rows
// ascend.
constexpr int kMoveThreads = 256, kFlight = 8;   // (at most)

__device__ __forceinline__ void move_rows(const KeepArgs &a, int seq, int part, int share) {
    __shared__ long long from[kMoveThreads], to[kMoveThreads];   // 16-byte pieces, from the head's first; from -1: nothing moves
    __shared__ int near[kMoveThreads];               // the first pages of the new rows
    const int T = blockDim.x;
    const End e = end_of(a, seq);
    if (e.keep <= 0) return;
    const int row_pieces = a.hd * type_bytes(a.cache_type) / 16, held = e.kv - e.n;
    const long long head_pieces = (long long)row_pieces << a.page_shift, page_pieces = head_pieces * a.n_head_kv;
    const int per_pool = a.n_head_kv * row_pieces;   // pieces of a position's K or V
    const long long pieces = 2LL * per_pool * a.n_layer;
    const int *const table = a.pages + (size_t)seq * a.pages_stride;
    const int first_page = max(held, 0) >> a.page_shift;
    const int at_page = first_page + (int)threadIdx.x;
    const int my_page = at_page < a.pages_stride && at_page <= (e.kv - 1) >> a.page_shift ? table[at_page] : -1;
    int next_row = (int)threadIdx.x < e.keep ? a.rows[e.start + threadIdx.x] : -1;
    near[threadIdx.x] = my_page;
    const auto piece_of = [&](int pos) -> long long {
        const int at = pos >> a.page_shift;
        if (pos < 0 || at >= a.pages_stride) return -1;
        const int page = at - first_page < T ? near[at - first_page] : table[at];
        if (page < 0 || page >= a.n_pages) return -1;
        return page * page_pieces + (long long)(pos & ((1 << a.page_shift) - 1)) * row_pieces;
    };
    for (int i0 = 0; i0 < e.keep; i0 += T) {
        const int n = min(T, e.keep - i0), i = i0 + threadIdx.x;
        const int row = next_row;
        next_row = i + T < e.keep ? a.rows[e.start + i + T] : -1;
        __syncthreads();
        if ((int)threadIdx.x < n) {
            long long f = -1, t = -1;
            if (row >= 0 && row < e.n && row != i) {
                f = piece_of(held + row);
                t = piece_of(held + i);
            }
            from[threadIdx.x] = t < 0 ? -1 : f;
            to[threadIdx.x] = t;
        }
        __syncthreads();
        for (long long id = (long long)part * T + threadIdx.x; id < pieces; id += share * T) {
            // K and V of a layer side by side (a division of 32 bits where it does)
            const int pool = id >> 32 ? (int)(id / per_pool) : (int)((unsigned)id / (unsigned)per_pool);
            const unsigned in_pos = (unsigned)(id - (long long)pool * per_pool), head = in_pos / (unsigned)row_pieces;
            const unsigned piece = in_pos - head * row_pieces;
            uint4 *const base = (uint4 *)(pool & 1 ? a.v_pool : a.k_pool) + (long long)(pool >> 1) * a.n_pages * page_pieces +
                                head * head_pieces + piece;
            for (int i = 0; i < n; i += kFlight) {
                uint4 x[kFlight];
#pragma unroll
                for (int j = 0; j < kFlight; ++j)
                    if (i + j < n && from[i + j] >= 0) x[j] = base[from[i + j]];
#pragma unroll
                for (int j = 0; j < kFlight; ++j)
                    if (i + j < n && from[i + j] >= 0) base[to[i + j]] = x[j];
            }
        }
    }
}

// The lengths, and the pages that no position needs any more, by one workgroup.  A wave
// has a run of the sequences, 64 at a time in its lanes; a lane takes a few pages of its
// sequence, the wave together a sequence's many.  The pages are counted, the waves add
// up, and each writes its own.
constexpr int kFew = 4;
struct Given {
    int lo, hi, count;      // of the lane's sequence: entries of the table, those that are pages
    int page[kFew];         // where they are few
    __device__ __forceinline__ bool many() const { return hi - lo > kFew; }
};
__device__ __forceinline__ void give_back(const KeepArgs &a) {
    __shared__ long long waves[kWaves][2];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n_wave = blockDim.x >> 6;
    const int each = (a.n_seq + n_wave - 1) / n_wave, s_first = wave * each, s_end = min(a.n_seq, s_first + each);
    const int mask = (1 << a.page_shift) - 1;
    const int n_free = a.n_free ? min(max(a.n_free[0], 0), a.n_pages) : 0;
    const auto is_page = [&](int page) { return page >= 0 && page < a.n_pages; };
    const auto pages_of = [&](int kv) { return (int)min(((long long)kv + mask) >> a.page_shift, (long long)a.pages_stride); };
    // the pages of lane l's sequence, which has many: visit(a page, or not, in each lane)
    const auto each_page = [&](const Given &g, int s0, int l, const auto &visit) {
        const int from = __builtin_amdgcn_readlane(g.lo, l), to = __builtin_amdgcn_readlane(g.hi, l);
        const int *const table = a.pages + (size_t)(s0 + l) * a.pages_stride;
        for (int j0 = from; j0 < to; j0 += 64 * kFlight) {
            int page[kFlight];
#pragma unroll
            for (int x = 0; x < kFlight; ++x) {
                const int j = j0 + 64 * x + lane;
                page[x] = j < to ? table[j] : -1;
            }
#pragma unroll
            for (int x = 0; x < kFlight; ++x)
                if (j0 + 64 * x < to) visit(is_page(page[x]), page[x]);
        }
    };
    const auto find = [&](int s0) {
        Given g{0, 0, 0, {}};
        if (s0 + lane < s_end) {
            const End e = end_of(a, s0 + lane);
            g.lo = pages_of(e.after);
            g.hi = pages_of(e.kv);
        }
        const int *const table = a.pages + (size_t)min(s0 + lane, a.n_seq - 1) * a.pages_stride;
#pragma unroll
        for (int j = 0; j < kFew; ++j) {
            g.page[j] = !g.many() && g.lo + j < g.hi ? table[g.lo + j] : -1;
            g.count += is_page(g.page[j]);
        }
        for (unsigned long long left = __ballot(g.many()); left; left &= left - 1) {
            const int l = __builtin_ctzll(left);
            int count = 0;
            each_page(g, s0, l, [&](bool real, int) { count += __popcll(__ballot(real)); });
            if (lane == l) g.count = count;
        }
        return g;
    };
    // the first page of the batch becomes free page number `at`; the number behind its last
    const auto put = [&](const Given &g, int s0, long long at) {
        const long long upto = wave_prefix(g.count);
        long long to = at + upto - g.count;
#pragma unroll
        for (int j = 0; j < kFew; ++j)
            if (is_page(g.page[j])) {
                if (to < a.n_pages) a.free_pages[to] = g.page[j];
                ++to;
            }
        for (unsigned long long left = __ballot(g.many()); left; left &= left - 1) {
            const int l = __builtin_ctzll(left);
            long long next = at + __shfl(upto - g.count, l);
            each_page(g, s0, l, [&](bool real, int page) {
                const unsigned long long here = __ballot(real);
                const long long mine = next + __popcll(here & ((1ULL << lane) - 1));
                if (real && mine < a.n_pages) a.free_pages[mine] = page;
                next += __popcll(here);
            });
        }
        return at + __shfl(upto, 63);
    };
    if (a.n_free) {
        Given g = find(s_first);
        long long count = g.count;
        for (int s0 = s_first + 64; s0 < s_end; s0 += 64) count += find(s0).count;
        const Sums sum = block_sums(count, 0, waves);
        long long at = put(g, s_first, n_free + __shfl(sum.before[0], 0));
        for (int s0 = s_first + 64; s0 < s_end; s0 += 64) at = put(find(s0), s0, at);
        if (threadIdx.x == 0) a.n_free_out[0] = (int)min(n_free + sum.all[0], (long long)a.n_pages);
    }
    __syncthreads();
    for (int s = threadIdx.x; s < a.n_seq; s += blockDim.x) a.kv_out[s] = end_of(a, s).after;
}

// One launch for both, where the lengths that the moves read are not those that are written.
// 16 drafted tokens of which four stay, 24 layers: 3.7 to 4.5 us, a launch and three rounds (ends and
// rows, pages, the rows themselves); 32 sequences' seven rows, 28 layers of 4 kv-heads of 128:
// 7.0, since rows of a head are 256 bytes each, and lie apart.
__global__ __launch_bounds__(kMoveThreads) void keep_kernel(KeepArgs a, int share) {
    if (blockIdx.x == 0) return give_back(a);
    const int id = blockIdx.x - 1, seq = id / share;
    move_rows(a, seq, id - seq * share, share);
}
__global__ __launch_bounds__(kMoveThreads) void move_kernel(KeepArgs a, int share) {
    const int seq = blockIdx.x / share;
    move_rows(a, seq, blockIdx.x - seq * share, share);
}
__global__ __launch_bounds__(kThreads) void ends_kernel(KeepArgs a) { give_back(a); }

// Rows that one workgroup takes where others must not be.
constexpr int kOneRows = 4096;
// Sequences whose pages four waves give back beside the moves.
constexpr int kOneSeqs = 1024;

}  // namespace

hipError_t launch_plan(const PlanArgs &a, hipStream_t s) {
    const bool in_place = a.kv_len == a.kv_held || a.n_free_out == a.n_free;
    if (a.n_seq <= kThreads && (!in_place || a.n_tok <= kOneRows)) {
        // No more threads than sequences, where other workgroups take the rest of the rows (us, 64 / 256 / 1024 threads: 64 trees
        // 4.6 / 5.0 / 5.4; 8000 rows of 4 prompts 3.4 / 3.8 / 4.3).
        const int threads = (std::clamp(in_place ? std::max(a.n_seq, a.n_tok) : a.n_seq, 1, kThreads) + 63) & ~63;
        const int blocks = in_place ? 1 : std::max(1, (a.n_tok + threads - 1) / threads);
        return launch(plan_kernel, dim3((unsigned)blocks), threads, 0, s, a);
    }
    const hipError_t e = launch(plan_sequences_kernel, dim3(1), kThreads, 0, s, a);
    if (e != hipSuccess || a.n_tok == 0) return e;
    return launch(plan_rows_kernel, dim3((unsigned)((a.n_tok + 255) / 256)), 256, 0, s, a);
}

hipError_t launch_keep(const KeepArgs &a, hipStream_t s) {
    if (a.n_seq == 0 && !a.n_free) return hipSuccess;
    if (a.rows && a.n_seq && a.n_tok) {
        // (a launch has fewer than 2^32 threads)
        const long long pieces = 2LL * a.n_layer * a.n_head_kv * a.hd * type_bytes(a.cache_type) / 16;
        // One wave a workgroup waits for no other; it also has a lane for each of 64 sequences' pages, and more take four (us, of
        // 64 / 128 / 256 threads: 2 sequences' 20 rows of 28 layers 8.6 / 9.4 / 10.8; 32 sequences' 7 rows 6.9 / 7.3 / 8.3; 300
        // sequences in 2 layers 9.4 / 7.3 / 5.1).
        const int threads = a.n_seq <= 64 ? 64 : kMoveThreads;
        const int share = (int)std::min<long long>((pieces + threads - 1) / threads, (1 << 23) / a.n_seq);
        if (a.n_seq <= kOneSeqs && a.kv_out != a.kv_len)
            return launch(keep_kernel, dim3((unsigned)(1 + share * a.n_seq)), threads, 0, s, a, share);
        const hipError_t e = launch(move_kernel, dim3((unsigned)(share * a.n_seq)), threads, 0, s, a, share);
        if (e != hipSuccess) return e;
    }
    return launch(ends_kernel, dim3(1), kThreads, 0, s, a);
}

}  // namespace kore_paged_gpu

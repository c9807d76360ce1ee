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

// Two numbers a thread: what the threads before it have, and all of them.
struct Sums {
    long long before[2], all[2];
};
__device__ __forceinline__ Sums block_sums(long long x, long long y, long long (*waves)[2]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long px = wave_prefix(x), py = wave_prefix(y);
    if (lane == 63) {
        waves[wave][0] = px;
        waves[wave][1] = py;
    }
    __syncthreads();
    Sums s{{px - x, py - y}, {0, 0}};
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (w < wave) s.before[i] += waves[w][i];
            s.all[i] += waves[w][i];
        }
    __syncthreads();
    return s;
}

// ---- the plan ---------------------------------------------------------------------

// A request: its rows, what it holds, the pages it has and those it needs.  One that no
// table holds is bad and asks for nothing.
struct Request {
    long long held;
    int n, had, need;
    bool bad;
};
__device__ __forceinline__ Request request(const PlanArgs &a, int s) {
    Request r{0, 0, 0, 0, false};
    if (s >= a.n_seq) return r;
    const int n = a.n_new[s], held = a.kv_held[s];
    const int mask = (1 << a.page_shift) - 1;
    r.bad = n < 0 || held < 0 || (long long)n + held > (long long)a.pages_stride << a.page_shift || n > a.n_tok ||
            (a.words && n > 64 * a.words);
    r.held = held;
    if (r.bad) return r;
    r.n = n;
    r.had = (int)(((long long)held + mask) >> a.page_shift);
    r.need = (int)(((long long)held + n + mask) >> a.page_shift) - r.had;
    return r;
}

// A row's depth in its tree and its mask: a walk from parent to parent, each before the
// row, so that it ends.
__device__ __forceinline__ int ancestors(const PlanArgs &a, int first, int i, unsigned long long *mask) {
    const int *const parent = a.parent + first;
    int at = i, depth = 0;
    for (int w = a.words - 1; w >= 0; --w) {
        unsigned long long bits = 0;
        while (at >= 64 * w) {
            bits |= 1ULL << (at & 63);
            const int up = parent[at];
            const bool root = up < 0 || up >= at;
            at = root ? -1 : up;
            if (!root) ++depth;
        }
        mask[w] = bits;
    }
    return depth;
}

// What a row gets: sequence s, its i-th new row (s < 0: no row).  page: of the row's slot.
__device__ __forceinline__ void put_row(const PlanArgs &a, int row, bool real, int first, int i, int held, int page) {
    const int at = held + i;
    int pos = -1;
    long long slot = -1;
    if (real) {
        pos = a.words ? held + ancestors(a, first, i, a.mask + (size_t)row * a.words) : at;
        if (page >= 0 && page < a.n_pages) slot = ((long long)page << a.page_shift) + (at & ((1 << a.page_shift) - 1));
    } else {
        for (int w = 0; w < a.words; ++w) a.mask[(size_t)row * a.words + w] = 0;
    }
    a.pos[row] = pos;
    a.slot[row] = slot;
}

// One workgroup: the requests' sums, what comes of them, and the tables of the sequences;
// ROWS: also those of the rows (at most kThreads sequences).
template <bool ROWS>
__global__ __launch_bounds__(kThreads) void plan_kernel(PlanArgs a) {
    __shared__ long long waves[kWaves][2];
    __shared__ int any_bad;
    __shared__ int starts[kThreads + 1], firsts[kThreads + 1], helds[kThreads];   // of a round's sequences
    const int tid = threadIdx.x, n_free = a.n_free[0];
    if (tid == 0) any_bad = n_free < 0 || n_free > a.n_pages;
    __syncthreads();
    // the sums of all
    long long rows = 0, need = 0;
    bool bad = false;
    Request r = request(a, tid);
    for (int s = tid; s < a.n_seq; s += kThreads) {
        if (s != tid) r = request(a, s);
        rows += r.n;
        need += r.need;
        bad |= r.bad;
    }
    if (bad) any_bad = 1;
    const Sums all = block_sums(rows, need, waves);
    const long long missing = all.all[1] - n_free;
    const int status = any_bad || all.all[0] > a.n_tok ? -1 : missing > 0 ? (int)min(missing, (long long)INT_MAX) : 0;
    if (tid == 0) {
        a.status[0] = status;
        a.n_free_out[0] = status ? n_free : n_free - (int)all.all[1];
        a.q_start[0] = 0;
    }
    // the sequences, a round of them at a time
    long long row_at = 0, need_at = 0;
    for (int s0 = 0; s0 < a.n_seq; s0 += kThreads) {
        const int s = s0 + tid;
        if (a.n_seq > kThreads) r = request(a, s);
        if (status) r.n = r.need = 0;
        const Sums sum = block_sums(r.n, r.need, waves);
        if (s < a.n_seq) {
            a.q_start[s + 1] = (int)(row_at + sum.before[0]) + r.n;
            a.kv_len[s] = (int)r.held + r.n;
        }
        starts[tid + 1] = (int)(row_at + sum.before[0]) + r.n;   // (behind the last sequence: all rows)
        firsts[tid] = (int)(need_at + sum.before[1]) - r.had;    // the j-th page of the sequence is number firsts + j
        helds[tid] = (int)r.held;
        if (tid == 0) starts[0] = (int)row_at;
        __syncthreads();
        // whose the number x is: the last sequence of the round that begins no later
        const auto owner = [&](const auto &begins, int x) {
            int lo = 0, hi = min(kThreads, a.n_seq - s0);   // begins(lo) <= x < begins(hi)
            while (hi - lo > 1) {
                const int m = (lo + hi) >> 1;
                if (begins(m) <= x) lo = m;
                else hi = m;
            }
            return lo;
        };
        if constexpr (ROWS) {
            const int n_rows = (int)all.all[0];
            for (int row = tid; row < a.n_tok; row += kThreads) {
                const bool real = !status && row < n_rows;
                int first = 0, i = 0, held = 0, page = -1;
                if (real) {
                    const int l = owner([&](int m) { return starts[m]; }, row);
                    first = starts[l];
                    i = row - first;
                    held = helds[l];
                    const int j = (held + i) >> a.page_shift;
                    int *const entry = a.pages + (size_t)l * a.pages_stride + j;
                    if (j << a.page_shift >= held) {   // a page that is new
                        page = a.free_pages[n_free - 1 - (firsts[l] + j)];
                        if (((held + i) & ((1 << a.page_shift) - 1)) == 0) *entry = page;
                    } else {
                        page = *entry;
                    }
                }
                put_row(a, row, real, first, i, held, page);
            }
        } else {
            // the round's new pages
            const int n_need = (int)sum.all[1];
            const int had = r.had;
            __syncthreads();
            firsts[tid] += had;
            starts[tid] = had;   // (not needed any more)
            __syncthreads();
            for (int x = tid; x < n_need; x += kThreads) {
                const int number = (int)need_at + x;
                const int l = owner([&](int m) { return firsts[m]; }, number);
                a.pages[(size_t)(s0 + l) * a.pages_stride + starts[l] + number - firsts[l]] = a.free_pages[n_free - 1 - number];
            }
        }
        row_at += sum.all[0];
        need_at += sum.all[1];
        __syncthreads();
    }
    if (ROWS && a.n_seq == 0)
        for (int row = tid; row < a.n_tok; row += kThreads) put_row(a, row, false, 0, 0, 0, -1);
}

// The rows of a plan whose sequences are done, a thread each.
__global__ __launch_bounds__(256) void plan_rows_kernel(PlanArgs a) {
    const int row = blockIdx.x * 256 + threadIdx.x;
    if (row >= a.n_tok) return;
    const bool real = row < a.q_start[a.n_seq];
    int first = 0, i = 0, held = 0, page = -1;
    if (real) {
        int lo = 0, hi = a.n_seq;   // q_start[lo] <= row < q_start[hi]
        while (hi - lo > 1) {
            const int m = (lo + hi) >> 1;
            if (a.q_start[m] <= row) lo = m;
            else hi = m;
        }
        first = a.q_start[lo];
        i = row - first;
        held = a.kv_len[lo] - (a.q_start[lo + 1] - first);
        page = a.pages[(size_t)lo * a.pages_stride + ((held + i) >> a.page_shift)];
    }
    put_row(a, row, real, first, i, held, page);
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

// A thread has 16 bytes of a position's K or V, of one kv-head of a layer, and moves them
// from row to row, eight rows in flight: what it overwrites lies before all that it has
// still to read, since the rows ascend.
constexpr int kMoves = 256, kFlight = 8;

// Workgroups seq * share .. of a sequence share its pieces.
__global__ __launch_bounds__(256) void move_kernel(KeepArgs a, int share) {
    __shared__ long long from[kMoves], to[kMoves];   // 16-byte pieces, from the head's first; from -1: nothing moves
    const int seq = blockIdx.x / share, part = blockIdx.x - seq * share;
    const End e = end_of(a, seq);
    if (e.keep <= 0) return;
    const int row_pieces = a.hd * type_bytes(a.cache_type) / 16;
    const long long head_pieces = (long long)row_pieces << a.page_shift, page_pieces = head_pieces * a.n_head_kv;
    const int per_pool = a.n_head_kv * row_pieces;   // pieces of a position's K or V
    const long long pieces = 2LL * per_pool * a.n_layer;
    const int *const table = a.pages + (size_t)seq * a.pages_stride;
    const auto piece_of = [&](int pos) -> long long {
        const int at = pos >> a.page_shift;
        if (pos < 0 || at >= a.pages_stride) return -1;
        const int page = table[at];
        if (page < 0 || page >= a.n_pages) return -1;
        return page * page_pieces + (long long)(pos & ((1 << a.page_shift) - 1)) * row_pieces;
    };
    for (int i0 = 0; i0 < e.keep; i0 += kMoves) {
        const int n = min(kMoves, e.keep - i0);
        __syncthreads();
        if ((int)threadIdx.x < n) {
            const int i = i0 + threadIdx.x, row = a.rows[e.start + i];
            long long f = -1, t = -1;
            if (row >= 0 && row < e.n && row != i) {
                f = piece_of(e.kv - e.n + row);
                t = piece_of(e.kv - e.n + i);
            }
            from[threadIdx.x] = t < 0 ? -1 : f;
            to[threadIdx.x] = t;
        }
        __syncthreads();
        for (long long id = (long long)part * 256 + threadIdx.x; id < pieces; id += share * 256) {
            const int pool = (int)(id / per_pool), in_pos = (int)(id - (long long)pool * per_pool);   // K and V of a layer side by side
            const int head = in_pos / row_pieces, piece = in_pos - head * row_pieces;
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

// The lengths, and the pages that no position needs any more, by one workgroup: a wave
// has a run of the sequences, 64 at a time in its lanes; it counts their pages, the waves
// add up, and it goes through them again and writes.
__global__ __launch_bounds__(kThreads) void ends_kernel(KeepArgs a) {
    __shared__ long long waves[kWaves][2];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int each = (a.n_seq + kWaves - 1) / kWaves, s_first = wave * each, s_end = min(a.n_seq, s_first + each);
    const int mask = (1 << a.page_shift) - 1;
    const int n_free = a.n_free ? min(max(a.n_free[0], 0), a.n_pages) : 0;
    const auto pages_of = [&](int kv) { return (int)min(((long long)kv + mask) >> a.page_shift, (long long)a.pages_stride); };
    // every page of the run's sequences: visit(valid in this lane, page, lanes before it)
    const auto each_page = [&](const auto &visit) {
        for (int s0 = s_first; s0 < s_end; s0 += 64) {
            int lo = 0, hi = 0;
            if (s0 + lane < s_end) {
                const End e = end_of(a, s0 + lane);
                lo = pages_of(e.after);
                hi = pages_of(e.kv);
            }
            for (unsigned long long left = __ballot(hi > lo); left; left &= left - 1) {
                const int l = __builtin_ctzll(left), from = __builtin_amdgcn_readlane(lo, l), to = __builtin_amdgcn_readlane(hi, l);
                const int *const table = a.pages + (size_t)(s0 + l) * a.pages_stride;
                for (int j = from; j < to; j += 64) {
                    const int page = j + lane < to ? table[j + lane] : -1;
                    visit(page >= 0 && page < a.n_pages, page);
                }
            }
        }
    };
    long long count = 0;
    if (a.free_pages) each_page([&](bool valid, int) { count += __popcll(__ballot(valid)); });
    const Sums sum = block_sums(lane == 0 ? count : 0, 0, waves);
    long long at = n_free + __shfl(sum.before[0], 0);
    if (a.free_pages)
        each_page([&](bool valid, int page) {
            const unsigned long long here = __ballot(valid);
            const long long to = at + __popcll(here & ((1ULL << lane) - 1));
            if (valid && to < a.n_pages) a.free_pages[to] = page;
            at += __popcll(here);
        });
    if (a.n_free && threadIdx.x == 0) a.n_free_out[0] = (int)min(n_free + sum.all[0], (long long)a.n_pages);
    __syncthreads();
    for (int s = threadIdx.x; s < a.n_seq; s += kThreads) a.kv_out[s] = end_of(a, s).after;
}

// Steps of up to so many rows and sequences are one workgroup's, rows and all.
constexpr int kOneRows = 4096;

}  // namespace

hipError_t launch_plan(const PlanArgs &a, hipStream_t s) {
    if (a.n_tok <= kOneRows && a.n_seq <= kThreads) return launch(plan_kernel<true>, dim3(1), kThreads, 0, s, a);
    const hipError_t e = launch(plan_kernel<false>, dim3(1), kThreads, 0, s, a);
    if (e != hipSuccess || a.n_tok == 0) return e;
    return launch(plan_rows_kernel, dim3((unsigned)((a.n_tok + 255) / 256)), 256, 0, s, a);
}

hipError_t launch_keep(const KeepArgs &a, hipStream_t s) {
    if (a.n_seq == 0 && !a.n_free) return hipSuccess;
    if (a.rows && a.n_seq && a.n_tok) {
        // (a launch has fewer than 2^32 threads)
        const long long pieces = 2LL * a.n_layer * a.n_head_kv * a.hd * type_bytes(a.cache_type) / 16;
        const int share = (int)std::min<long long>((pieces + 255) / 256, (1 << 23) / a.n_seq);
        const hipError_t e = launch(move_kernel, dim3((unsigned)(share * a.n_seq)), 256, 0, s, a, share);
        if (e != hipSuccess) return e;
    }
    return launch(ends_kernel, dim3(1), kThreads, 0, s, a);
}

}  // namespace kore_paged_gpu

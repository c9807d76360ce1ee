// kore_paged_kernels.h - launch interface between kore_paged_api.cpp and the
// rotary, append and paged-attention kernels.  Internal to libkore_paged.so.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

namespace kore_paged_gpu {

constexpr int kMaxHeadDim = 256;        // of the paged cache
constexpr int kMaxRopeHeadDim = 1024;   // of the rotary call
constexpr int kMaxRot = 512;
constexpr int kMaxKeys = 1 << 30;       // positions of a sequence's row of the page table
// A launch has fewer than 2^32 threads: rows of a call (256 threads each); rows x heads and sequences x kv-heads
// of a batch, which make at most 2^23 + 2^22 tiles of 256 threads, or 2^20 + 2^22 of 512.
constexpr int kMaxRows = 1 << 23, kMaxRowHeads = 1 << 27, kMaxSeqHeads = 1 << 22;
// Every row of an append and every tile of an attention scans the sequences, 64 a round: at 2^16 of them a call takes
// seconds at its largest, at 2^22 it would hold the device for many minutes.
constexpr int kMaxSeq = 1 << 16;

constexpr int kMaxWords = 16;           // of 64 bits, of a tree's mask

enum Type { kF32 = 0, kF16 = 1, kBF16 = 2 };
constexpr int type_bytes(int t) { return t == kF32 ? 4 : 2; }

// Frequencies of rot / 2 pairs (device) and what turns with them.
struct Turn {
    const float *freq;
    double size;       // m: c and s are multiplied by it
    int rot;           // 0: nothing is rotated
    int interleaved;
};

struct RopeArgs {
    Turn turn;
    const void *x;
    void *out;
    const int *pos;
    int64_t x_stride, out_stride;
    int n_tok, n_head, hd;
    int sign;          // -1: transpose
    int type;
};

// Heads that are normalised (where a set has weights) and turned, of up to two sets of rows, into rows of their
// own or, with a slot for each row, q's rows and a pool's slots.
struct HeadSet {
    const void *x;
    void *out;               // rows; of a pool's k: the layer's pool
    int64_t x_stride, out_stride;
    int n_head;
    const float *norm;       // or NULL
};
struct HeadsArgs {
    Turn turn;
    HeadSet set[2];          // q, k; sets without rows have no heads
    const int *pos;          // negative: the row is left
    float eps;
    double per_dim;          // 1 / hd
    int n_tok, hd, type;
    // the store: v's rows, and where k's and v's go
    const int64_t *slot;     // NULL: no store
    const void *v;
    int64_t v_stride;
    void *v_pool;
    int n_pages, page_shift, cache_type;
};

// The batch as the kernels see it.
struct Batch {
    const int *q_start, *kv_len, *pages;
    int n_seq, n_tok, pages_stride;
};

struct AppendArgs {
    Turn turn;
    Batch b;
    const void *k, *v, *q;
    void *q_out;
    int64_t k_stride, v_stride, q_stride, q_out_stride;
    void *k_pool, *v_pool;   // of the layer
    int n_pages, page_shift, n_head, n_head_kv, hd;
    int type, cache_type;
};

// Which new rows a row attends: mask NULL, those up to itself.
struct Tree {
    const unsigned long long *mask;
    const int *pos;
    int words;
};

struct AttendArgs {
    Batch b;
    const void *q;
    void *out;
    int64_t q_stride, out_stride;
    const void *k_pool, *v_pool;   // of the layer
    int n_pages, page_shift, n_head, n_head_kv, hd;
    int window;                    // INT_MAX: none
    float scale;
    int type, cache_type;
    int max_q, num_cu;
    float *part;                   // workspace
    Tree tree;
};

struct PlanArgs {
    int n_seq, n_tok, n_pages, page_shift, pages_stride, words;   // words 0: no trees
    int window;              // of the masks; INT_MAX: none
    const int *n_new, *kv_held, *free_pages, *n_free, *parent;
    int *kv_len, *pages, *n_free_out, *q_start, *pos, *status;
    int64_t *slot;
    unsigned long long *mask;
};

struct KeepArgs {
    int n_seq, n_tok, n_layer, n_pages, page_shift, pages_stride, n_head_kv, hd, cache_type;
    const int *q_start, *n_keep, *rows, *kv_len, *pages, *n_free;
    int *kv_out, *free_pages, *n_free_out;
    void *k_pool, *v_pool;
};

hipError_t launch_rope(const RopeArgs &a, hipStream_t s);
hipError_t launch_heads(const HeadsArgs &a, hipStream_t s);
hipError_t launch_append(const AppendArgs &a, hipStream_t s);
hipError_t launch_plan(const PlanArgs &a, hipStream_t s);
hipError_t launch_keep(const KeepArgs &a, hipStream_t s);
hipError_t launch_attend(const AttendArgs &a, hipStream_t s);
size_t attend_workspace_bytes(int hd, int num_cu);

}  // namespace kore_paged_gpu

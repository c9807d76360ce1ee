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

enum Type { kF32 = 0, kF16 = 1, kBF16 = 2 };
inline int type_bytes(int t) { return t == kF32 ? 4 : 2; }

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
};

hipError_t launch_rope(const RopeArgs &a, hipStream_t s);
hipError_t launch_append(const AppendArgs &a, hipStream_t s);
hipError_t launch_attend(const AttendArgs &a, hipStream_t s);
size_t attend_workspace_bytes(int hd, int num_cu);

}  // namespace kore_paged_gpu

// kore_paged_device.h - device helpers shared by the rotary, append and
// paged-attention kernels.  Internal to libkore_paged.so.
#pragma once

#include "kore_launch.h"
#include "kore_paged_kernels.h"

#include <climits>

namespace kore_paged_gpu {
namespace {

using kore_gpu::launch;

typedef _Float16 half_t;
typedef __bf16 bhalf_t;

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(half_t x) { return (float)x; }
__device__ __forceinline__ float to_f32(bhalf_t x) { return (float)x; }

// N elements from an address that is aligned to N elements, and to one such (vec) or to an element.
template <int N, class T>
__device__ __forceinline__ void load_n(const T *p, T (&x)[N]) {
    typedef T vec_t __attribute__((ext_vector_type(N)));
    const vec_t v = *reinterpret_cast<const vec_t *>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = v[i];
}
template <int N, class T>
__device__ __forceinline__ void store_n(T *p, const T (&x)[N], bool vec) {
    typedef T vec_t __attribute__((ext_vector_type(N)));
    if (vec) {
        vec_t v;
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = x[i];
        *reinterpret_cast<vec_t *>(p) = v;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) p[i] = x[i];
    }
}

}  // namespace
}  // namespace kore_paged_gpu

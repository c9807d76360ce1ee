// kore_paged_attend.hip - attention of new rows over a paged KV cache (gfx950).
#include "kore_paged_device.h"

namespace kore_paged_gpu {
namespace {

// One wave per (row, q-head), a key at a time: lanes over the head's dims.
template <class T, class C>
__global__ __launch_bounds__(64) void attend_kernel(AttendArgs a) {
    const int row = blockIdx.x, head = blockIdx.y, lane = threadIdx.x;
    const int seq = seq_of_row(a.b, row);
    if (seq >= a.b.n_seq || row < a.b.q_start[seq]) return;
    const int pos = a.b.kv_len[seq] - (a.b.q_start[seq + 1] - row);
    const int kv_head = head / (a.n_head / a.n_head_kv);
    const int ps = 1 << a.page_shift;
    const int end = min(pos + 1, a.b.pages_stride << a.page_shift);
    const int begin = a.window <= pos ? pos - a.window + 1 : 0;
    const T *q = (const T *)a.q + (size_t)row * a.q_stride + (size_t)head * a.hd;
    float qv[4], o[4] = {0, 0, 0, 0}, m = -INFINITY, l = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) qv[i] = lane + 64 * i < a.hd ? to_f32(q[lane + 64 * i]) : 0.f;
    for (int j = begin; j < end; ++j) {
        const int page = a.b.pages[(size_t)seq * a.b.pages_stride + (j >> a.page_shift)];
        if (page < 0 || page >= a.n_pages) continue;
        const size_t at = ((((size_t)page * a.n_head_kv + kv_head) << a.page_shift) + (j & (ps - 1))) * a.hd;
        const C *k = (const C *)a.k_pool + at, *v = (const C *)a.v_pool + at;
        float dot = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (lane + 64 * i < a.hd) dot = fmaf(qv[i], to_f32(k[lane + 64 * i]), dot);
#pragma unroll
        for (int d = 32; d; d >>= 1) dot += __shfl_xor(dot, d);
        const float s = dot * a.scale, mn = fmaxf(m, s);
        const float base = mn == -INFINITY ? 0.f : mn;
        const float f = __expf(m - base), p = __expf(s - base);
        l = l * f + p;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (lane + 64 * i < a.hd) o[i] = fmaf(p, to_f32(v[lane + 64 * i]), o[i] * f);
        m = mn;
    }
    T *out = (T *)a.out + (size_t)row * a.out_stride + (size_t)head * a.hd;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (lane + 64 * i < a.hd) out[lane + 64 * i] = (T)(l == 0.f ? 0.f : o[i] / l);
}

}  // namespace

size_t attend_workspace_bytes(int n_head, int n_head_kv, int hd, int num_cu) { return 16; }

hipError_t launch_attend(const AttendArgs &a, hipStream_t s) {
    const dim3 grid(a.b.n_tok, a.n_head);
    if (a.type == kF32 && a.cache_type == kF32) attend_kernel<float, float><<<grid, 64, 0, s>>>(a);
    else if (a.type == kF32 && a.cache_type == kF16) attend_kernel<float, half_t><<<grid, 64, 0, s>>>(a);
    else if (a.type == kF32) attend_kernel<float, bhalf_t><<<grid, 64, 0, s>>>(a);
    else if (a.type == kF16) attend_kernel<half_t, half_t><<<grid, 64, 0, s>>>(a);
    else attend_kernel<bhalf_t, bhalf_t><<<grid, 64, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace kore_paged_gpu

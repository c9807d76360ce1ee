// kore_launch.h - kernel launches that report their own result.  Internal to the
// libraries.
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

namespace kore_gpu {

// Launches kernel(args...) and returns what that launch says: hipGetLastError() would
// also report an error that another call of the thread has left, and take it away.
template <class... P>
inline hipError_t launch(void (*kernel)(P...), dim3 grid, dim3 block, size_t lds, hipStream_t s, std::type_identity_t<P>... args) {
    void *at[] = {static_cast<void *>(&args)...};
    return hipLaunchKernel(reinterpret_cast<const void *>(kernel), grid, block, at, lds, s);
}

}  // namespace kore_gpu

// launch.h -- what the short calls need at every launch, asked of the runtime
// once for each device.
#pragma once
#include <cuda_runtime.h>

#include <atomic>

#include "internal.h"

namespace nrn {

constexpr int kMaxDevices = 64;

inline int device_index() {
    int d = 0;
    cudaGetDevice(&d);
    return d;
}

// sm_count_current, kept.
inline int sm_count() {
    static std::atomic<int> known[kMaxDevices];
    const int d = device_index();
    if (d < 0 || d >= kMaxDevices) return sm_count_current();
    int n = known[d].load(std::memory_order_relaxed);
    if (n == 0) known[d].store(n = sm_count_current(), std::memory_order_relaxed);
    return n;
}

// Lets a kernel use `bytes` of dynamic shared memory.
template <auto Kernel>
cudaError_t allow_shared(int bytes) {
    static std::atomic<int> most[kMaxDevices];
    const int d = device_index();
    if (d >= 0 && d < kMaxDevices && most[d].load(std::memory_order_relaxed) >= bytes) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && d >= 0 && d < kMaxDevices) most[d].store(bytes, std::memory_order_relaxed);
    return e;
}

}  // namespace nrn

// launch.h -- what the short calls need at every launch, asked of the runtime
// once for each device.
#pragma once
#include <cuda_runtime.h>

#include <atomic>
#include <mutex>

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

// Lets a kernel use `bytes` of dynamic shared memory.  The limit is only ever
// raised, and one thread at a time sets it: another thread's launch may need
// the larger one.
template <auto Kernel>
cudaError_t allow_shared(int bytes) {
    static std::atomic<int> most[kMaxDevices];
    static std::mutex turn;
    const int d = device_index();
    if (d < 0 || d >= kMaxDevices) return cudaErrorInvalidDevice;
    if (most[d].load(std::memory_order_acquire) >= bytes) return cudaSuccess;
    std::lock_guard<std::mutex> lock(turn);
    if (most[d].load(std::memory_order_relaxed) >= bytes) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) most[d].store(bytes, std::memory_order_release);
    return e;
}

// Kernels that follow one another in one call: with `after`, the blocks of
// this one take their places as those of the one before leave, and wait
// (previous_done) before they touch what it wrote, or write what it reads.
// Each kernel of such a chain lets the next one in (let_next) and waits on
// every path, so that the end of one is the end of all before it; a kernel that
// does neither may stand in the chain, launched as usual.  A kernel that
// allocates TMEM does so before it lets the next one in: the allocation waits
// for as long as another block of its SM holds the columns.
template <typename... P, typename... A>
cudaError_t launch_chained(void (*kernel)(P...), dim3 grid, dim3 block, int shared, cudaStream_t s, bool after, const A&... args) {
    cudaLaunchConfig_t c{};
    c.gridDim = grid, c.blockDim = block, c.dynamicSmemBytes = static_cast<size_t>(shared), c.stream = s;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    c.attrs = &at, c.numAttrs = after ? 1 : 0;
    return cudaLaunchKernelEx(&c, kernel, args...);
}
__device__ __forceinline__ void let_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void previous_done() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

}  // namespace nrn

// waits.cu -- the device word in which the operators' kernels note that one
// of their bounded waits gave up: one for each device, made once, never freed.
#include <cuda_runtime.h>

#include <mutex>

#include "common.cuh"
#include "launch.h"

namespace nrn {
namespace {

std::mutex g_turn;
int32_t* g_flag[kMaxDevices];

// A word of zeros on the current device, made beside whatever is being
// captured: the thread's capture mode is relaxed meanwhile, and the zeros are
// written on a stream of their own and waited for.
cudaError_t make_flag(int32_t** flag) {
    int32_t* p = nullptr;
    cudaStream_t s = nullptr;
    cudaError_t e = cudaMalloc(&p, sizeof(int32_t));
    if (e == cudaSuccess) e = cudaStreamCreateWithFlags(&s, cudaStreamNonBlocking);
    if (e == cudaSuccess) e = cudaMemsetAsync(p, 0, sizeof(int32_t), s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    if (s) cudaStreamDestroy(s);
    if (e == cudaSuccess) *flag = p;
    else if (p) cudaFree(p);
    return e;
}

}  // namespace
}  // namespace nrn

using namespace nrn;

extern "C" nrn_status_t nrn_cuda_wait_flag(int32_t device, int32_t** flag) {
    NRN_CHECK_ARG(flag != nullptr, "nrn_cuda_wait_flag: null result");
    NRN_CHECK_ARG(device >= 0 && device < kMaxDevices, "nrn_cuda_wait_flag: no such device");
    std::lock_guard<std::mutex> turn(g_turn);
    if (g_flag[device] == nullptr) {
        int before = 0;
        NRN_CUDA_TRY(cudaGetDevice(&before));
        NRN_CUDA_TRY(cudaSetDevice(device));
        cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
        cudaError_t e = cudaThreadExchangeStreamCaptureMode(&mode);
        if (e == cudaSuccess) {
            e = make_flag(&g_flag[device]);
            const cudaError_t back = cudaThreadExchangeStreamCaptureMode(&mode);
            if (e == cudaSuccess) e = back;
        }
        const cudaError_t back = cudaSetDevice(before);
        if (e == cudaSuccess) e = back;
        NRN_CUDA_TRY(e);
    }
    *flag = g_flag[device];
    return NRN_OK;
}

// scaled.cuh -- e4m3 values with a scale for each block of 128.
#pragma once
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace nrn {

// A block's scale from its largest magnitude, given as the largest bit
// pattern of |x|: a NaN or infinity there wins and makes the scale one.  The
// floor keeps 1 / scale finite; a block below it is noise.
__device__ __forceinline__ float block_scale(uint32_t amax_bits) {
    const float a = __uint_as_float(amax_bits);
    return (a < 0x1p-64f ? 0x1p-64f : a) * (1.0f / 448.0f);
}

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// Four values as e4m3, the first in the low byte.
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
}

}  // namespace nrn

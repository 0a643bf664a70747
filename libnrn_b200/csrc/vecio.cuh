// vecio.cuh -- eight consecutive elements of a row as fp32, for bf16, fp16
// and fp32 rows: one or two 16-byte accesses where the row allows it, single
// elements where it is not aligned or ends.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace nrn {

template <typename T>
__device__ __forceinline__ float to_f32(T x);
template <>
__device__ __forceinline__ float to_f32(float x) { return x; }
template <>
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32(float x) { return __float2bfloat16_rn(x); }

// Raw storage of eight elements (16 or 32 bytes).
template <typename T>
struct alignas(16) Raw8 {
    T e[8];
};

// Elements [0, n) of p; the rest is 0.  `vec`: p is 16-byte aligned.
template <typename T>
__device__ __forceinline__ Raw8<T> load8(const T* p, int n, bool vec) {
    Raw8<T> r;
    if (vec && n >= 8) {
        const uint4* s = reinterpret_cast<const uint4*>(p);
        uint4* d = reinterpret_cast<uint4*>(&r);
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(r) / 16); ++i) d[i] = s[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) r.e[i] = i < n ? p[i] : from_f32<T>(0.0f);
    }
    return r;
}

// Two results as one word (16-bit types), the first in the low half.
__device__ __forceinline__ uint32_t pack2_f32(__nv_bfloat16, float a, float b) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
__device__ __forceinline__ uint32_t pack2_f32(__half, float a, float b) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float* x, int n, bool vec) {
    if (vec && n >= 8) {
        uint4* d = reinterpret_cast<uint4*>(p);
        if constexpr (sizeof(T) == 2) {
            const T k{};
            d[0] = make_uint4(pack2_f32(k, x[0], x[1]), pack2_f32(k, x[2], x[3]), pack2_f32(k, x[4], x[5]), pack2_f32(k, x[6], x[7]));
        } else {
            d[0] = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
            d[1] = make_uint4(__float_as_uint(x[4]), __float_as_uint(x[5]), __float_as_uint(x[6]), __float_as_uint(x[7]));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = from_f32<T>(x[i]);
    }
}

}  // namespace nrn

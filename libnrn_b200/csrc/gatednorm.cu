// gatednorm.cu -- the norms before and after a block, with the block's gate
// and residual scale, in one pass, and their gradients.
//
//     y = r + alpha * act(gate) * norm(h) * w_post       norm(x) = x / sqrt(mean(x^2) + eps)
//     z = norm(y) * w_pre                                 (the next block's input)
//
// Everything is fp32 between the loads and the stores; z takes y before y is
// rounded.  z may go out as e4m3 with a scale for each row and 128 columns,
// ready for the 8-bit product.
//
// Bound by HBM: three rows in, two out (five and three backward), if the
// operations an element stay near 30: the sigmoid is two special-function
// operations for 16-bit types, alpha and w_post are one factor, and a block keeps
// its columns' factors in registers over all the rows it takes in turn.  A row
// is held in registers, eight elements a thread and vector (16 bytes of bf16):
// 32 threads a row where the row is short, else a block a row.  The reductions
// over a row are barriers that a block waits at, so its next rows must be on
// their way meanwhile: rows on 16-byte boundaries come by bulk copies into a
// ring of two to four in shared memory.  Measured, bf16 rows of 4096: forward
// with z as e4m3 606 MB in 129 us (71% of the measured copy); backward, rows
// of 2560, 336 MB in 99 us (52%): there the operations an element, about 60,
// and two reductions a row count as much as the bytes.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "internal.h"
#include "launch.h"
#include "scaled.cuh"
#include "tc.cuh"
#include "vecio.cuh"

namespace nrn {
namespace {

constexpr int kMaxD = 16384;

struct RowArrays {                     // kernel arguments: read where they are used, not kept in registers
    const void* from[5];
    int64_t stride[5];
    int64_t rows;
    int32_t d, stages;
    int32_t vec, pad;
    int32_t* err;
};

struct NormArgs {
    nrn_gatednorm_t f;
    RowArrays in;                      // residual, h, gate
    uint8_t* zv;
    float* zs;
    int64_t zv_stride, zs_row, zs_col;
};

struct GradArgs {
    nrn_gatednorm_t f;
    nrn_gatednorm_grad_t g;
    RowArrays in;                      // residual, h, gate, dy, dz
    float* part;                       // [parts][2][d]: sums over rows
};

RowArrays row_arrays(const nrn_gatednorm_t& f, bool vec) {
    RowArrays r{};
    r.from[0] = f.residual, r.from[1] = f.h, r.from[2] = f.gate;
    r.stride[0] = f.residual_stride, r.stride[1] = f.h_stride, r.stride[2] = f.gate_stride;
    r.rows = f.rows, r.d = f.d, r.vec = vec, r.err = f.err;
    return r;
}

// The sigmoid's error, relative: for 16-bit types ex2.approx (2^-22), its
// argument's rounding (|x| 2^-23: 2^-18 at 30) and rcp.approx (2^-23), far
// below the results' 2^-9 and 2^-12; fp32 takes expf (2^-22 in all).  Below
// -87 a 16-bit type's is 0.
template <typename T>
__device__ __forceinline__ float exp_of(float x) {
    if constexpr (sizeof(T) == 4) return expf(x);
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x * 1.4426950408889634f));
    return e;
}
__device__ __forceinline__ float inverse(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
template <typename T>
__device__ __forceinline__ float sigmoid(float x) { return inverse(1.0f + exp_of<T>(-x)); }
// sigmoid(x) and its derivative sigmoid(x) sigmoid(-x).  1 - sigmoid(x) in
// place of sigmoid(-x) would have none of its bits left at 17.
template <typename T>
__device__ __forceinline__ float2 sigmoid_grad(float x) {
    const float t = exp_of<T>(-fabsf(x)), r = inverse(1.0f + t), u = t * r;
    return make_float2(x < 0.0f ? u : r, u * r);
}

__device__ __forceinline__ float max_or_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// N sums over the threads of a row; every thread gets them.  A row of one
// warp needs no barrier; else `red` is [2][N][32] floats used in turn.
template <int N, bool WARP>
__device__ __forceinline__ void row_sum(float (&x)[N], float* red, int& turn) {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) x[i] += __shfl_xor_sync(0xffffffffu, x[i], d);
    if constexpr (!WARP) {
        float* at = red + (turn & 1) * 64;
        ++turn;
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        if (lane == 0)
#pragma unroll
            for (int i = 0; i < N; ++i) at[i * 32 + warp] = x[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float s = lane < static_cast<int>(blockDim.x >> 5) ? at[i * 32 + lane] : 0.0f;
#pragma unroll
            for (int d = 8; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);   // at most 16 warps
            x[i] = __shfl_sync(0xffffffffu, s, 0);
        }
    }
}

__device__ __forceinline__ void load_param(const float* p, int c, int n, float* out) {
    if (p == nullptr) {
#pragma unroll
        for (int e = 0; e < 8; ++e) out[e] = 1.0f;
    } else if (n >= 8 && (reinterpret_cast<uintptr_t>(p + c) & 15) == 0) {
        const float4 a = *reinterpret_cast<const float4*>(p + c), b = *reinterpret_cast<const float4*>(p + c + 4);
        out[0] = a.x, out[1] = a.y, out[2] = a.z, out[3] = a.w;
        out[4] = b.x, out[5] = b.y, out[6] = b.z, out[7] = b.w;
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) out[e] = e < n ? p[c + e] : 0.0f;
    }
}

// Threads of a block, at most: 128 with a row for each warp, else 512 (128
// registers a thread; 64 where it has eight elements).
template <bool WARP>
constexpr int most_threads() {
    return WARP ? 128 : 512;
}

// The rows a block reads, as a ring in shared memory filled by one thread's
// bulk copies (RING), or straight from global memory.
constexpr int kMostStages = 4;
constexpr int kRingHead = 128;
enum { ERR_NORM_TIMEOUT = 5 };

template <typename T, int N, bool RING>
struct Rows {
    const RowArrays& a;
    int64_t step;
    int32_t stage;
    uint32_t phase;
    uint64_t* bars;
    unsigned char* ring;

    __device__ __forceinline__ Rows(const RowArrays& arrays, int64_t step_) : a(arrays), step(step_) {}

    __device__ __forceinline__ void start(unsigned char* smem, int64_t row) {
        if constexpr (RING) {
            bars = reinterpret_cast<uint64_t*>(smem);
            ring = smem + kRingHead;
            stage = 0;
            phase = 0;
            if (threadIdx.x == 0) {
                for (int i = 0; i < a.stages; ++i) tc::mbar_init(&bars[i], 1);
                asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
                for (int i = 0; i < a.stages; ++i) fill(row + i * step, i);
            }
            __syncthreads();
        }
    }
    __device__ __forceinline__ void fill(int64_t row, int st) {
        if (row >= a.rows) return;
        const uint32_t bytes = static_cast<uint32_t>(a.d * sizeof(T));
        uint32_t all = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) all += a.from[i] ? bytes : 0u;
        tc::mbar_expect_tx(&bars[st], all);
        const uint64_t once = tc::policy_evict_first();
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (a.from[i]) tc::bulk_load(ring + (st * N + i) * static_cast<size_t>(bytes), static_cast<const T*>(a.from[i]) + row * a.stride[i], bytes, &bars[st], once);
    }
    // this row is in shared memory
    __device__ __forceinline__ void wait() {
        if constexpr (RING) {
            if (!tc::mbar_wait(&bars[stage], phase, nullptr) && a.err) atomicCAS(a.err, 0, ERR_NORM_TIMEOUT);
        }
    }
    __device__ __forceinline__ Raw8<T> get(int i, int64_t row, int c) const {
        if constexpr (RING) {
            const uint4* s = reinterpret_cast<const uint4*>(ring + (stage * N + i) * (a.d * sizeof(T)) + (c < a.d ? c : 0) * sizeof(T));
            Raw8<T> r;
            uint4* t = reinterpret_cast<uint4*>(&r);
#pragma unroll
            for (int k = 0; k < static_cast<int>(sizeof(r) / 16); ++k) t[k] = c < a.d ? s[k] : make_uint4(0, 0, 0, 0);
            return r;
        } else {
            const int n = a.d - c;
            return load8(static_cast<const T*>(a.from[i]) + row * a.stride[i] + (n > 0 ? c : 0), n, a.vec != 0);
        }
    }
    // every thread of the block has what it needs of this row
    __device__ __forceinline__ void done(int64_t row) {
        if constexpr (RING) {
            if (threadIdx.x == 0) fill(row + a.stages * step, stage);
            if (++stage == a.stages) {
                stage = 0;
                phase ^= 1u;
            }
        }
    }
};

// A warp or a block a row, VPT vectors of eight a thread.  Elements past the row's
// end are loaded as 0 and stay 0: they add nothing to the sums.
template <typename T, bool WARP, int VPT, bool RING>
__global__ void __launch_bounds__(most_threads<WARP>(), WARP ? 8 / VPT : 1)
    norm_kernel(const __grid_constant__ NormArgs a) {
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ float red[128];
    const nrn_gatednorm_t& f = a.f;
    const int tpr = WARP ? 32 : blockDim.x, tid = WARP ? (threadIdx.x & 31) : threadIdx.x;
    const int64_t step = static_cast<int64_t>(gridDim.x) * (WARP ? 4 : 1);
    int64_t row = WARP ? static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5) : blockIdx.x;
    if (row >= f.rows) return;
    const bool vec = a.in.vec != 0, gated = f.gate != nullptr, silu = f.act == NRN_ACT_SILU;
    Rows<T, 3, RING> in(a.in, step);
    in.start(smem, row);
    const float inv_d = 1.0f / static_cast<float>(f.d);
    int turn = 0;
    float aw[VPT][8], wp[VPT][8];
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
        const int c = (tid + v * tpr) * 8, n = f.d - c;
        float al[8];
        load_param(f.w_post, n > 0 ? c : 0, n, aw[v]);
        load_param(f.alpha, n > 0 ? c : 0, n, al);
        load_param(f.w_pre, n > 0 ? c : 0, n, wp[v]);
#pragma unroll
        for (int e = 0; e < 8; ++e) aw[v][e] *= al[e];
    }
    const bool want_z = f.z != nullptr || a.zv != nullptr;
    for (; row < f.rows; row += step) {
        float y[VPT][8];
        in.wait();
        if (f.h) {
            Raw8<T> r[VPT], gate[VPT];
            float s[1] = {0.0f};
#pragma unroll
            for (int v = 0; v < VPT; ++v) {
                const int c = (tid + v * tpr) * 8;
                const Raw8<T> h = in.get(1, row, c);
                r[v] = in.get(0, row, c);
                if (gated) gate[v] = in.get(2, row, c);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    y[v][e] = to_f32(h.e[e]);
                    s[0] = fmaf(y[v][e], y[v][e], s[0]);
                }
            }
            row_sum<1, WARP>(s, red, turn);
            in.done(row);
            const float inv = rsqrtf(fmaf(s[0], inv_d, f.eps));
#pragma unroll
            for (int v = 0; v < VPT; ++v)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float u = inv * aw[v][e];
                    if (gated) {
                        const float g = to_f32(gate[v].e[e]), sg = sigmoid<T>(g);
                        u *= silu ? g * sg : sg;
                    }
                    y[v][e] = fmaf(y[v][e], u, to_f32(r[v].e[e]));
                }
            if (f.y) {
#pragma unroll
                for (int v = 0; v < VPT; ++v) {
                    const int c = (tid + v * tpr) * 8, n = f.d - c;
                    if (n > 0) store8(static_cast<T*>(f.y) + row * f.y_stride + c, y[v], n, vec);
                }
            }
            if (!want_z) continue;
        } else {
#pragma unroll
            for (int v = 0; v < VPT; ++v) {
                const Raw8<T> r = in.get(0, row, (tid + v * tpr) * 8);
#pragma unroll
                for (int e = 0; e < 8; ++e) y[v][e] = to_f32(r.e[e]);
            }
        }
        float s[1] = {0.0f};
#pragma unroll
        for (int v = 0; v < VPT; ++v)
#pragma unroll
            for (int e = 0; e < 8; ++e) s[0] = fmaf(y[v][e], y[v][e], s[0]);
        row_sum<1, WARP>(s, red, turn);
        if (!f.h) in.done(row);
        const float inv = rsqrtf(fmaf(s[0], inv_d, f.eps));
#pragma unroll
        for (int v = 0; v < VPT; ++v) {
            const int c = (tid + v * tpr) * 8, n = f.d - c;
#pragma unroll
            for (int e = 0; e < 8; ++e) y[v][e] *= inv * wp[v][e];
            if (a.zv == nullptr) {
                if (n > 0) store8(static_cast<T*>(f.z) + row * f.z_stride + c, y[v], n, vec);
                continue;
            }
            // an infinity in y gives a NaN among zeros, which has to win
            float m = fabsf(y[v][0]);
#pragma unroll
            for (int e = 1; e < 8; ++e) m = max_or_nan(m, fabsf(y[v][e]));
#pragma unroll
            for (int d = 1; d < 16; d <<= 1) m = max_or_nan(m, __shfl_xor_sync(0xffffffffu, m, d));   // 16 lanes: 128 columns
            if (n <= 0) continue;
            const float sc = block_scale(__float_as_uint(m)), q = __frcp_rn(sc);
            if ((tid & 15) == 0) a.zs[row * a.zs_row + (c / 128) * a.zs_col] = sc;
            *reinterpret_cast<uint2*>(a.zv + row * a.zv_stride + c) =
                make_uint2(e4m3x4(y[v][0] * q, y[v][1] * q, y[v][2] * q, y[v][3] * q),
                           e4m3x4(y[v][4] * q, y[v][5] * q, y[v][6] * q, y[v][7] * q));
        }
    }
}

// Backward.  With hh = norm(h), a = act(gate), f = alpha w_post, yh = norm(y):
//     d  = dy + inv_y (dz w_pre - yh mean(dz w_pre yh))            = dresidual
//     dgate = d f hh act'(gate);   t = d f a;   dh = inv_h (t - hh mean(t hh))
//     s1 = sum over rows of d a hh: dalpha = s1 w_post, dw_post = s1 alpha
//     s2 = sum over rows of dz yh = dw_pre
// y is computed again from h, gate and r: reading it would cost a fifth of
// the reads and its rounding.  Blocks take rows in turn and keep their part of
// the two sums in registers; a second kernel adds the parts.  What a row
// gives is read again from the ring by each of the four passes over it, and
// the gate's sigmoid computed twice: kept in registers they would leave room
// for half the threads, and spilled they cost more than the rest (d 1024:
// 191 us with 48 bytes spilled a thread, 85 us without).
template <typename T, bool WARP, int VPT, bool RING>
__global__ void __launch_bounds__(most_threads<WARP>(), WARP ? 8 / VPT : 1)
    norm_grad_kernel(const __grid_constant__ GradArgs a) {
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ float red[128];
    const nrn_gatednorm_t& f = a.f;
    const nrn_gatednorm_grad_t& g = a.g;
    const int tpr = WARP ? 32 : blockDim.x, tid = WARP ? (threadIdx.x & 31) : threadIdx.x;
    const int slot = WARP ? blockIdx.x * 4 + (threadIdx.x >> 5) : blockIdx.x;
    const int64_t step = static_cast<int64_t>(gridDim.x) * (WARP ? 4 : 1);
    const bool vec = a.in.vec != 0, block = f.h != nullptr, gated = f.gate != nullptr, silu = f.act == NRN_ACT_SILU;
    const float inv_d = 1.0f / static_cast<float>(f.d);
    int turn = 0;
    float s1[VPT][8], s2[VPT][8];
#pragma unroll
    for (int v = 0; v < VPT; ++v)
#pragma unroll
        for (int e = 0; e < 8; ++e) s1[v][e] = s2[v][e] = 0.0f;
    // a column's factors: in registers while there is room for them
    constexpr bool kKeep = VPT <= 2;
    float kaw[kKeep ? VPT : 1][8], kwp[kKeep ? VPT : 1][8];
    auto factors = [&](int v, float* aw, float* wp) {
        const int c = (tid + v * tpr) * 8, n = f.d - c;
        float al[8];
        load_param(f.w_post, n > 0 ? c : 0, n, aw);
        load_param(f.alpha, n > 0 ? c : 0, n, al);
        load_param(f.w_pre, n > 0 ? c : 0, n, wp);
#pragma unroll
        for (int e = 0; e < 8; ++e) aw[e] *= al[e];
    };
    if constexpr (kKeep)
#pragma unroll
        for (int v = 0; v < VPT; ++v) factors(v, kaw[v], kwp[v]);
    Rows<T, 5, RING> in(a.in, step);
    in.start(smem, slot);
    for (int64_t row = slot; row < f.rows; row += step) {
        in.wait();
        float y[VPT][8], inv_h = 0.0f;
        if (block) {
            float s[1] = {0.0f};
#pragma unroll
            for (int v = 0; v < VPT; ++v) {
                const Raw8<T> h = in.get(1, row, (tid + v * tpr) * 8);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float x = to_f32(h.e[e]);
                    s[0] = fmaf(x, x, s[0]);
                }
            }
            row_sum<1, WARP>(s, red, turn);
            inv_h = rsqrtf(fmaf(s[0], inv_d, f.eps));
        }
        float sy[2] = {0.0f, 0.0f};
#pragma unroll
        for (int v = 0; v < VPT; ++v) {
            const int c = (tid + v * tpr) * 8;
            float taw[8], twp[8];
            if constexpr (!kKeep) factors(v, taw, twp);
            const float *aw = kKeep ? kaw[kKeep ? v : 0] : taw, *wp = kKeep ? kwp[kKeep ? v : 0] : twp;
            const Raw8<T> r = in.get(0, row, c);
#pragma unroll
            for (int e = 0; e < 8; ++e) y[v][e] = to_f32(r.e[e]);
            if (block) {
                const Raw8<T> h = in.get(1, row, c);
                if (gated) {
                    const Raw8<T> gate = in.get(2, row, c);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float t = to_f32(gate.e[e]), sg = sigmoid<T>(t);
                        y[v][e] = fmaf(to_f32(h.e[e]) * inv_h * aw[e], silu ? t * sg : sg, y[v][e]);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) y[v][e] = fmaf(to_f32(h.e[e]) * inv_h, aw[e], y[v][e]);
                }
            }
            if (g.dz) {
                const Raw8<T> dz = in.get(4, row, c);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    sy[0] = fmaf(y[v][e], y[v][e], sy[0]);
                    sy[1] = fmaf(to_f32(dz.e[e]) * wp[e], y[v][e], sy[1]);
                }
            }
        }
        float inv_y = 0.0f, my = 0.0f;
        if (g.dz) {
            row_sum<2, WARP>(sy, red, turn);
            inv_y = rsqrtf(fmaf(sy[0], inv_d, f.eps));
            my = inv_y * inv_y * sy[1] * inv_d;      // mean(dz w_pre yh) inv_y
        }
        float st[1] = {0.0f};
#pragma unroll
        for (int v = 0; v < VPT; ++v) {
            const int c = (tid + v * tpr) * 8, n = f.d - c;
            float taw[8], twp[8], d[8];
            if constexpr (!kKeep) factors(v, taw, twp);
            const float *aw = kKeep ? kaw[kKeep ? v : 0] : taw, *wp = kKeep ? kwp[kKeep ? v : 0] : twp;
#pragma unroll
            for (int e = 0; e < 8; ++e) d[e] = 0.0f;
            if (g.dy) {
                const Raw8<T> dy = in.get(3, row, c);
#pragma unroll
                for (int e = 0; e < 8; ++e) d[e] = to_f32(dy.e[e]);
            }
            if (g.dz) {
                const Raw8<T> dz = in.get(4, row, c);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float z = to_f32(dz.e[e]);
                    s2[v][e] = fmaf(z, y[v][e] * inv_y, s2[v][e]);
                    d[e] = fmaf(inv_y, z * wp[e] - y[v][e] * my, d[e]);
                }
            }
            if (n > 0 && g.dresidual) store8(static_cast<T*>(g.dresidual) + row * g.dresidual_stride + c, d, n, vec);
            if (!block) continue;
            const Raw8<T> h = in.get(1, row, c);
            if (gated) {
                const Raw8<T> gate = in.get(2, row, c);
                float dg[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float hh = to_f32(h.e[e]) * inv_h, t = to_f32(gate.e[e]), da = d[e] * aw[e];
                    const float2 sg = sigmoid_grad<T>(t);
                    const float act = silu ? t * sg.x : sg.x, dact = silu ? fmaf(t, sg.y, sg.x) : sg.y;
                    s1[v][e] = fmaf(d[e] * act, hh, s1[v][e]);
                    dg[e] = da * hh * dact;
                    y[v][e] = da * act;
                    st[0] = fmaf(y[v][e], hh, st[0]);
                }
                if (n > 0 && g.dgate) store8(static_cast<T*>(g.dgate) + row * g.dgate_stride + c, dg, n, vec);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float hh = to_f32(h.e[e]) * inv_h;
                    s1[v][e] = fmaf(d[e], hh, s1[v][e]);
                    y[v][e] = d[e] * aw[e];
                    st[0] = fmaf(y[v][e], hh, st[0]);
                }
            }
        }
        if (block) {
            row_sum<1, WARP>(st, red, turn);
            const float mh = st[0] * inv_d * inv_h;
#pragma unroll
            for (int v = 0; v < VPT; ++v) {
                const int c = (tid + v * tpr) * 8, n = f.d - c;
                const Raw8<T> h = in.get(1, row, c);
#pragma unroll
                for (int e = 0; e < 8; ++e) y[v][e] = inv_h * (y[v][e] - to_f32(h.e[e]) * mh);
                if (n > 0 && g.dh) store8(static_cast<T*>(g.dh) + row * g.dh_stride + c, y[v], n, vec);
            }
        }
        if constexpr (RING) __syncthreads();             // the row is read: its place may be filled again
        in.done(row);
    }
    if (a.part == nullptr) return;
    float* at = a.part + static_cast<int64_t>(slot) * 2 * f.d;
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
        const int c = (tid + v * tpr) * 8, n = f.d - c;
        if (n <= 0) continue;
        store8(at + c, s1[v], n, f.d % 4 == 0);
        store8(at + f.d + c, s2[v], n, f.d % 4 == 0);
    }
}

// Adds the blocks' parts of one of the two sums, in their order: 32 columns a
// block, 32 runs of parts at once.
__global__ void __launch_bounds__(1024) norm_parts_kernel(const float* part, int parts, int d, const float* alpha, const float* w_post,
                                                          float* dalpha, float* dw_post, float* dw_pre) {
    __shared__ float sum[32][33];
    const int c = blockIdx.x * 32 + (threadIdx.x & 31), run = threadIdx.x >> 5;
    float s = 0.0f;
    if (c < d)
#pragma unroll 4
        for (int p = run; p < parts; p += 32) s += part[(static_cast<int64_t>(p) * 2 + blockIdx.y) * d + c];
    sum[run][threadIdx.x & 31] = s;
    __syncthreads();
    if (run != 0 || c >= d) return;
#pragma unroll
    for (int r = 1; r < 32; ++r) s += sum[r][threadIdx.x];
    if (blockIdx.y == 1) {
        if (dw_pre) dw_pre[c] = s;
    } else {
        if (dalpha) dalpha[c] = w_post ? s * w_post[c] : s;
        if (dw_post) dw_post[c] = alpha ? s * alpha[c] : s;
    }
}

// A row of up to 512 elements has a warp, a longer one a block whose threads
// have 16 elements each (measured at d 4096: 8 elements a thread 131 us, 16
// 111 us: the reductions cost each thread the same), past 8,192 elements 32.
struct Shape {
    bool warp;
    int vpt, threads;
};
Shape shape_of(int d) {
    const int vecs = (d + 7) / 8;
    if (vecs <= 64) return {true, vecs <= 32 ? 1 : 2, 128};
    const int vpt = vecs <= 1024 ? 2 : 4;
    return {false, vpt, ((vecs + vpt - 1) / vpt + 31) / 32 * 32};
}

// Blocks that take the rows in turn: as many as are on the GPU at once.
int blocks_per_sm(const Shape& sh) { return (sh.vpt == 1 ? 1024 : 512) / sh.threads; }
unsigned blocks_for(const Shape& sh, int64_t rows) {
    const int rows_per = sh.warp ? 4 : 1;
    return static_cast<unsigned>(std::min<int64_t>((rows + rows_per - 1) / rows_per, static_cast<int64_t>(blocks_per_sm(sh)) * sm_count()));
}
// Parts of the sums over rows that the backward kernel leaves: one for each block, or warp where a warp has a row.
int grad_parts(int64_t rows, int d) {
    const Shape sh = shape_of(d);
    return static_cast<int>(blocks_for(sh, rows)) * (sh.warp ? 4 : 1);
}

// Rows that a block's share of the SM's shared memory holds; below two there is no ring.
int ring_stages(const Shape& sh, int arrays, int d, int size, bool vec) {
    if (sh.warp || !vec || d % 8 != 0) return 0;
    const int room = (227 * 1024 / blocks_per_sm(sh) - 2048 - kRingHead) / (arrays * d * size);
    return room < 2 ? 0 : std::min(room, kMostStages);
}

template <auto Kernel, typename A>
cudaError_t launch(const Shape& sh, const A& a, int bytes, cudaStream_t s) {
    const cudaError_t e = bytes ? allow_shared<Kernel>(bytes) : cudaSuccess;
    if (e != cudaSuccess) return e;
    Kernel<<<blocks_for(sh, a.f.rows), sh.threads, bytes, s>>>(a);
    return cudaGetLastError();
}

template <typename T>
cudaError_t forward_any(NormArgs a, cudaStream_t s) {
    const Shape sh = shape_of(a.f.d);
    const int size = static_cast<int>(sizeof(T));
    a.in.stages = ring_stages(sh, 3, a.f.d, size, a.in.vec != 0);
    const int bytes = a.in.stages ? kRingHead + a.in.stages * 3 * a.f.d * size : 0;
    if (sh.warp) return sh.vpt == 1 ? launch<norm_kernel<T, true, 1, false>>(sh, a, 0, s) : launch<norm_kernel<T, true, 2, false>>(sh, a, 0, s);
    if (sh.vpt == 2) return bytes ? launch<norm_kernel<T, false, 2, true>>(sh, a, bytes, s) : launch<norm_kernel<T, false, 2, false>>(sh, a, 0, s);
    return bytes ? launch<norm_kernel<T, false, 4, true>>(sh, a, bytes, s) : launch<norm_kernel<T, false, 4, false>>(sh, a, 0, s);
}

template <typename T>
cudaError_t backward_any(GradArgs a, cudaStream_t s) {
    const Shape sh = shape_of(a.f.d);
    const int size = static_cast<int>(sizeof(T));
    a.in.stages = ring_stages(sh, 5, a.f.d, size, a.in.vec != 0);
    const int bytes = a.in.stages ? kRingHead + a.in.stages * 5 * a.f.d * size : 0;
    if (sh.warp) return sh.vpt == 1 ? launch<norm_grad_kernel<T, true, 1, false>>(sh, a, 0, s) : launch<norm_grad_kernel<T, true, 2, false>>(sh, a, 0, s);
    if (sh.vpt == 2)
        return bytes ? launch<norm_grad_kernel<T, false, 2, true>>(sh, a, bytes, s) : launch<norm_grad_kernel<T, false, 2, false>>(sh, a, 0, s);
    return bytes ? launch<norm_grad_kernel<T, false, 4, true>>(sh, a, bytes, s) : launch<norm_grad_kernel<T, false, 4, false>>(sh, a, 0, s);
}

bool row_ok(const void* p, int64_t stride, int size) {
    return p == nullptr || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * size % 16 == 0);
}

nrn_status_t check_norm(const nrn_gatednorm_t* a, const std::string& who) {
    NRN_CHECK_ARG(a != nullptr, who + ": null arguments");
    NRN_CHECK_ARG(a->dtype == NRN_BF16 || a->dtype == NRN_FP16 || a->dtype == NRN_FP32, who + ": unknown type");
    NRN_CHECK_ARG(a->act == NRN_ACT_SILU || a->act == NRN_ACT_SIGMOID, who + ": unknown activation");
    NRN_CHECK_ARG(a->rows >= 0 && a->rows < (int64_t(1) << 31), who + ": rows out of range");
    NRN_CHECK_ARG(a->d >= 1 && a->d <= kMaxD, who + ": rows have 1 to 16,384 elements");
    NRN_CHECK_ARG(std::isfinite(a->eps) && a->eps >= 0.0f, who + ": eps must be finite and not negative");
    NRN_CHECK_ARG(a->rows == 0 || a->residual, who + ": null residual");
    NRN_CHECK_ARG(a->rows == 0 || a->h || (!a->gate && !a->y), who + ": a gate and y belong to a block's output h");
    return NRN_OK;
}

}  // namespace
}  // namespace nrn

using namespace nrn;

extern "C" nrn_status_t nrn_cuda_gatednorm_forward(const nrn_gatednorm_t* in, nrn_stream_t stream) {
    const std::string who = "nrn_cuda_gatednorm_forward";
    NRN_TRY(check_norm(in, who));
    NRN_CHECK_ARG(!(in->z && in->z_scaled), who + ": z goes out in one form");
    NormArgs a{};
    a.f = *in;
    const int size = in->dtype == NRN_FP32 ? 4 : 2;
    if (const nrn_scaled_t* q = in->z_scaled) {
        NRN_CHECK_ARG(q->row_block == 1 && q->rows == in->rows && q->cols == in->d, who + ": z_scaled has another shape");
        NRN_CHECK_ARG(in->rows == 0 || (q->values && q->scales), who + ": null array");
        NRN_CHECK_ARG(reinterpret_cast<uintptr_t>(q->values) % 16 == 0 && q->value_stride % 16 == 0 && q->value_stride >= q->cols,
                      who + ": values must be 16-byte aligned with rows a multiple of 16 bytes apart");
        a.zv = q->values;
        a.zs = q->scales;
        a.zv_stride = q->value_stride;
        a.zs_row = q->scale_stride[0], a.zs_col = q->scale_stride[1];
    }
    if (in->rows == 0 || (!in->y && !in->z && !a.zv)) return NRN_OK;
    a.in = row_arrays(*in, row_ok(in->residual, in->residual_stride, size) && row_ok(in->h, in->h_stride, size) &&
                               row_ok(in->gate, in->gate_stride, size) && row_ok(in->y, in->y_stride, size) && row_ok(in->z, in->z_stride, size));
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (in->dtype == NRN_BF16) NRN_CUDA_TRY(forward_any<__nv_bfloat16>(a, s));
    else if (in->dtype == NRN_FP16) NRN_CUDA_TRY(forward_any<__half>(a, s));
    else NRN_CUDA_TRY(forward_any<float>(a, s));
    return NRN_OK;
}

extern "C" nrn_status_t nrn_cuda_gatednorm_workspace(const nrn_gatednorm_t* a, int64_t* bytes) {
    NRN_CHECK_ARG(a && bytes, "nrn_cuda_gatednorm_workspace: null argument");
    NRN_CHECK_ARG(a->rows >= 0 && a->d >= 1 && a->d <= kMaxD, "nrn_cuda_gatednorm_workspace: sizes out of range");
    *bytes = static_cast<int64_t>(grad_parts(a->rows, a->d)) * 2 * a->d * 4;
    return NRN_OK;
}

extern "C" nrn_status_t nrn_cuda_gatednorm_backward(const nrn_gatednorm_t* in, const nrn_gatednorm_grad_t* g, nrn_stream_t stream) {
    const std::string who = "nrn_cuda_gatednorm_backward";
    NRN_TRY(check_norm(in, who));
    NRN_CHECK_ARG(g != nullptr, who + ": null gradients");
    NRN_CHECK_ARG(in->rows == 0 || in->h || !(g->dh || g->dgate || g->dalpha || g->dw_post), who + ": no block output, no gradients of it");
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const bool sums = g->dalpha || g->dw_post || g->dw_pre;
    if (in->rows == 0) {
        for (float* p : {g->dalpha, g->dw_post, g->dw_pre})
            if (p) NRN_CUDA_TRY(cudaMemsetAsync(p, 0, static_cast<size_t>(in->d) * 4, s));
        return NRN_OK;
    }
    GradArgs a{};
    a.f = *in;
    a.g = *g;
    const int size = in->dtype == NRN_FP32 ? 4 : 2;
    const int parts = grad_parts(in->rows, in->d);
    if (sums) {
        NRN_CHECK_ARG(g->workspace && g->workspace_bytes >= static_cast<int64_t>(parts) * 2 * in->d * 4, who + ": workspace too small");
        a.part = static_cast<float*>(g->workspace);
    }
    a.in = row_arrays(*in, row_ok(in->residual, in->residual_stride, size) && row_ok(in->h, in->h_stride, size) &&
                               row_ok(in->gate, in->gate_stride, size) && row_ok(g->dy, g->dy_stride, size) && row_ok(g->dz, g->dz_stride, size) &&
                               row_ok(g->dresidual, g->dresidual_stride, size) && row_ok(g->dh, g->dh_stride, size) && row_ok(g->dgate, g->dgate_stride, size));
    a.in.from[3] = g->dy, a.in.from[4] = g->dz;
    a.in.stride[3] = g->dy_stride, a.in.stride[4] = g->dz_stride;
    if (in->dtype == NRN_BF16) NRN_CUDA_TRY(backward_any<__nv_bfloat16>(a, s));
    else if (in->dtype == NRN_FP16) NRN_CUDA_TRY(backward_any<__half>(a, s));
    else NRN_CUDA_TRY(backward_any<float>(a, s));
    if (sums) {
        norm_parts_kernel<<<dim3(static_cast<unsigned>((in->d + 31) / 32), 2), 1024, 0, s>>>(a.part, parts, in->d, in->alpha, in->w_post, g->dalpha, g->dw_post,
                                                                                          g->dw_pre);
        NRN_CUDA_TRY(cudaGetLastError());
    }
    return NRN_OK;
}

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
// Bound by HBM: three rows in, two out (six and three backward), a few dozen
// operations an element.  A row is held in registers, eight elements a thread
// and vector (16 bytes of bf16): 32 threads a row where the row is short, else
// a block a row.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "internal.h"
#include "scaled.cuh"
#include "vecio.cuh"

namespace nrn {
namespace {

constexpr int kMaxD = 16384;

struct NormArgs {
    nrn_gatednorm_t f;
    uint8_t* zv;
    float* zs;
    int64_t zv_stride, zs_row, zs_col;
    int32_t vec;                       // every row starts on a 16-byte boundary
};

struct GradArgs {
    nrn_gatednorm_t f;
    nrn_gatednorm_grad_t g;
    float* part;                       // [blocks][3][d]: dalpha, dw_post, dw_pre
    int32_t vec;
};

__device__ __forceinline__ float sigmoid(float x) { return 1.0f / (1.0f + expf(-x)); }

// N sums over the threads of a row; every thread gets them.  Rows of one
// warp need no barrier; else `red` is [2][N][32] floats used in turn.
template <int N, int TPR>
__device__ __forceinline__ void row_sum(float (&x)[N], float* red, int& turn) {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) x[i] += __shfl_xor_sync(0xffffffffu, x[i], d);
    if constexpr (TPR > 32) {
        float* at = red + (turn & 1) * 64;
        ++turn;
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        if (lane == 0)
#pragma unroll
            for (int i = 0; i < N; ++i) at[i * 32 + warp] = x[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float s = lane < TPR / 32 ? at[i * 32 + lane] : 0.0f;
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
            x[i] = s;
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

// TPR threads a row, VPT vectors of eight a thread; ROWS rows a block.
template <typename T, int TPR, int VPT>
__global__ void __launch_bounds__(TPR == 32 ? 128 : TPR) norm_kernel(const __grid_constant__ NormArgs a) {
    __shared__ float red[128];
    const nrn_gatednorm_t& f = a.f;
    const int tid = TPR == 32 ? (threadIdx.x & 31) : threadIdx.x;
    const int rows_per = TPR == 32 ? 4 : 1;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * rows_per + (TPR == 32 ? threadIdx.x >> 5 : 0);
    if (row >= f.rows) return;
    const bool vec = a.vec != 0;
    const float inv_d = 1.0f / static_cast<float>(f.d);
    int turn = 0;
    Raw8<T> rr[VPT], rh[VPT], rg[VPT];
    auto left = [&](int v) { return f.d - (tid + v * TPR) * 8; };
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
        const int n = left(v);
        const int64_t c = n > 0 ? (tid + v * TPR) * 8 : 0;
        rr[v] = load8(static_cast<const T*>(f.residual) + row * f.residual_stride + c, n, vec);
        if (f.h) rh[v] = load8(static_cast<const T*>(f.h) + row * f.h_stride + c, n, vec);
        if (f.gate) rg[v] = load8(static_cast<const T*>(f.gate) + row * f.gate_stride + c, n, vec);
    }
    float y[VPT][8];
    if (f.h) {
        float s[1] = {0.0f};
#pragma unroll
        for (int v = 0; v < VPT; ++v)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float x = to_f32(rh[v].e[e]);
                s[0] = fmaf(x, x, s[0]);
            }
        row_sum<1, TPR>(s, red, turn);
        const float inv = rsqrtf(s[0] * inv_d + f.eps);
#pragma unroll
        for (int v = 0; v < VPT; ++v) {
            const int n = left(v), c = (tid + v * TPR) * 8;
            float w[8], al[8];
            load_param(f.w_post, n > 0 ? c : 0, n, w);
            load_param(f.alpha, n > 0 ? c : 0, n, al);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float u = to_f32(rh[v].e[e]) * inv * w[e] * al[e];
                if (f.gate) {
                    const float g = to_f32(rg[v].e[e]), sg = sigmoid(g);
                    u *= f.act == NRN_ACT_SILU ? g * sg : sg;
                }
                y[v][e] = to_f32(rr[v].e[e]) + u;
            }
            if (f.y && n > 0) store8(static_cast<T*>(f.y) + row * f.y_stride + c, y[v], n, vec);
        }
    } else {
#pragma unroll
        for (int v = 0; v < VPT; ++v)
#pragma unroll
            for (int e = 0; e < 8; ++e) y[v][e] = to_f32(rr[v].e[e]);
    }
    if (f.z == nullptr && a.zv == nullptr) return;
    float s[1] = {0.0f};
#pragma unroll
    for (int v = 0; v < VPT; ++v)
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < left(v)) s[0] = fmaf(y[v][e], y[v][e], s[0]);
    row_sum<1, TPR>(s, red, turn);
    const float inv = rsqrtf(s[0] * inv_d + f.eps);
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
        const int n = left(v), c = (tid + v * TPR) * 8;
        float w[8];
        load_param(f.w_pre, n > 0 ? c : 0, n, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) y[v][e] = e < n ? y[v][e] * inv * w[e] : 0.0f;
        if (a.zv == nullptr) {
            if (n > 0) store8(static_cast<T*>(f.z) + row * f.z_stride + c, y[v], n, vec);
            continue;
        }
        uint32_t m = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) m = max(m, abs_bits(y[v][e]));
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));   // 16 lanes: 128 columns
        if (n <= 0) continue;
        const float sc = block_scale(m), q = 1.0f / sc;
        if ((tid & 15) == 0) a.zs[row * a.zs_row + (c / 128) * a.zs_col] = sc;
        *reinterpret_cast<uint2*>(a.zv + row * a.zv_stride + c) =
            make_uint2(e4m3x4(y[v][0] * q, y[v][1] * q, y[v][2] * q, y[v][3] * q),
                       e4m3x4(y[v][4] * q, y[v][5] * q, y[v][6] * q, y[v][7] * q));
    }
}

// Backward.  With hh = norm(h), u = hh w_post, a = act(gate), yh = norm(y):
//     dzw = dz w_pre;   dy' = dy + inv_y (dzw - yh mean(dzw yh))      = dresidual
//     dgate = dy' alpha u act'(gate);  dalpha += dy' a u
//     dhh = dy' alpha a w_post;  dh = inv_h (dhh - hh mean(dhh hh))
//     dw_post += dy' alpha a hh;  dw_pre += dz yh
// y is computed again from h, gate and r: reading it would cost a fourth of
// the reads and its rounding.  Blocks take rows in turn and keep their part of
// the three sums over rows in registers; a second kernel adds the parts.
template <typename T, int TPR, int VPT>
__global__ void __launch_bounds__(TPR == 32 ? 128 : TPR) norm_grad_kernel(const __grid_constant__ GradArgs a) {
    __shared__ float red[256];
    const nrn_gatednorm_t& f = a.f;
    const nrn_gatednorm_grad_t& g = a.g;
    const int tid = TPR == 32 ? (threadIdx.x & 31) : threadIdx.x;
    const int rows_per = TPR == 32 ? 4 : 1;
    const int slot = blockIdx.x * rows_per + (TPR == 32 ? threadIdx.x >> 5 : 0);
    const int64_t step = static_cast<int64_t>(gridDim.x) * rows_per;
    const bool vec = a.vec != 0;
    const float inv_d = 1.0f / static_cast<float>(f.d);
    int turn = 0;
    float sal[VPT][8], spo[VPT][8], spr[VPT][8];
#pragma unroll
    for (int v = 0; v < VPT; ++v)
#pragma unroll
        for (int e = 0; e < 8; ++e) sal[v][e] = spo[v][e] = spr[v][e] = 0.0f;
    auto left = [&](int v) { return f.d - (tid + v * TPR) * 8; };

    for (int64_t row = slot; row < f.rows; row += step) {
        Raw8<T> rr[VPT], rh[VPT], rg[VPT], ry[VPT], rz[VPT];
#pragma unroll
        for (int v = 0; v < VPT; ++v) {
            const int n = left(v);
            const int64_t c = n > 0 ? (tid + v * TPR) * 8 : 0;
            rr[v] = load8(static_cast<const T*>(f.residual) + row * f.residual_stride + c, n, vec);
            if (f.h) rh[v] = load8(static_cast<const T*>(f.h) + row * f.h_stride + c, n, vec);
            if (f.gate) rg[v] = load8(static_cast<const T*>(f.gate) + row * f.gate_stride + c, n, vec);
            if (g.dy) ry[v] = load8(static_cast<const T*>(g.dy) + row * g.dy_stride + c, n, vec);
            if (g.dz) rz[v] = load8(static_cast<const T*>(g.dz) + row * g.dz_stride + c, n, vec);
        }
        float inv_h = 0.0f;
        if (f.h) {
            float s[1] = {0.0f};
#pragma unroll
            for (int v = 0; v < VPT; ++v)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float x = to_f32(rh[v].e[e]);
                    s[0] = fmaf(x, x, s[0]);
                }
            row_sum<1, TPR>(s, red, turn);
            inv_h = rsqrtf(s[0] * inv_d + f.eps);
        }
        // y, and the two sums its norm's gradient needs
        float y[VPT][8];
        float s2[2] = {0.0f, 0.0f};
#pragma unroll
        for (int v = 0; v < VPT; ++v) {
            const int n = left(v), c = n > 0 ? (tid + v * TPR) * 8 : 0;
            float w[8], al[8], wp[8];
            load_param(f.w_post, c, n, w);
            load_param(f.alpha, c, n, al);
            load_param(f.w_pre, c, n, wp);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                y[v][e] = to_f32(rr[v].e[e]);
                if (f.h) {
                    float u = to_f32(rh[v].e[e]) * inv_h * w[e] * al[e];
                    if (f.gate) {
                        const float x = to_f32(rg[v].e[e]), sg = sigmoid(x);
                        u *= f.act == NRN_ACT_SILU ? x * sg : sg;
                    }
                    y[v][e] += u;
                }
                if (e < n) {
                    s2[0] = fmaf(y[v][e], y[v][e], s2[0]);
                    if (g.dz) s2[1] = fmaf(to_f32(rz[v].e[e]) * wp[e], y[v][e], s2[1]);
                }
            }
        }
        float inv_y = 0.0f, my = 0.0f;
        if (g.dz) {
            row_sum<2, TPR>(s2, red, turn);
            inv_y = rsqrtf(s2[0] * inv_d + f.eps);
            my = inv_y * inv_y * s2[1] * inv_d;      // mean(dzw yh) inv_y
        }
        // dy' into y; dgate out; mean(dhh hh)
        float s3[1] = {0.0f};
#pragma unroll
        for (int v = 0; v < VPT; ++v) {
            const int n = left(v), c = n > 0 ? (tid + v * TPR) * 8 : 0;
            float w[8], al[8], wp[8], dg[8];
            load_param(f.w_post, c, n, w);
            load_param(f.alpha, c, n, al);
            load_param(f.w_pre, c, n, wp);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float d = g.dy ? to_f32(ry[v].e[e]) : 0.0f;
                if (g.dz) {
                    const float z = to_f32(rz[v].e[e]);
                    spr[v][e] = fmaf(z, y[v][e] * inv_y, spr[v][e]);
                    d += inv_y * (z * wp[e] - y[v][e] * my);
                }
                y[v][e] = d;
                if (f.h) {
                    const float hh = to_f32(rh[v].e[e]) * inv_h;
                    float act = 1.0f, dact = 0.0f;
                    if (f.gate) {
                        const float x = to_f32(rg[v].e[e]), sg = sigmoid(x);
                        act = f.act == NRN_ACT_SILU ? x * sg : sg;
                        dact = f.act == NRN_ACT_SILU ? sg * fmaf(x, 1.0f - sg, 1.0f) : sg * (1.0f - sg);
                    }
                    const float u = hh * w[e];
                    sal[v][e] = fmaf(d * act, u, sal[v][e]);
                    const float da = d * al[e];
                    dg[e] = da * u * dact;
                    spo[v][e] = fmaf(da * act, hh, spo[v][e]);
                    s3[0] = fmaf(da * act * w[e], hh, s3[0]);
                }
            }
            if (n > 0) {
                if (g.dresidual) store8(static_cast<T*>(g.dresidual) + row * g.dresidual_stride + c, y[v], n, vec);
                if (g.dgate && f.h && f.gate) store8(static_cast<T*>(g.dgate) + row * g.dgate_stride + c, dg, n, vec);
            }
        }
        if (f.h && g.dh) {
            row_sum<1, TPR>(s3, red, turn);
            const float mh = s3[0] * inv_d;
#pragma unroll
            for (int v = 0; v < VPT; ++v) {
                const int n = left(v), c = n > 0 ? (tid + v * TPR) * 8 : 0;
                float w[8], al[8], dh[8];
                load_param(f.w_post, c, n, w);
                load_param(f.alpha, c, n, al);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float act = 1.0f;
                    if (f.gate) {
                        const float x = to_f32(rg[v].e[e]), sg = sigmoid(x);
                        act = f.act == NRN_ACT_SILU ? x * sg : sg;
                    }
                    dh[e] = inv_h * (y[v][e] * al[e] * act * w[e] - to_f32(rh[v].e[e]) * inv_h * mh);
                }
                if (n > 0) store8(static_cast<T*>(g.dh) + row * g.dh_stride + c, dh, n, vec);
            }
        }
    }
    if (a.part == nullptr) return;
    float* at = a.part + static_cast<int64_t>(slot) * 3 * f.d;
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
        const int n = left(v), c = (tid + v * TPR) * 8;
        if (n <= 0) continue;
        store8(at + c, sal[v], n, false);
        store8(at + f.d + c, spo[v], n, false);
        store8(at + 2 * f.d + c, spr[v], n, false);
    }
}

// Adds the parts of one of the three sums, in their order: 32 columns a
// block, eight runs of parts at once.
__global__ void __launch_bounds__(256) norm_parts_kernel(const float* part, int parts, int d, float* dalpha, float* dw_post,
                                                         float* dw_pre) {
    __shared__ float sum[8][32];
    float* out = blockIdx.y == 0 ? dalpha : (blockIdx.y == 1 ? dw_post : dw_pre);
    if (out == nullptr) return;
    const int c = blockIdx.x * 32 + (threadIdx.x & 31), run = threadIdx.x >> 5;
    float s = 0.0f;
    if (c < d)
        for (int p = run; p < parts; p += 8) s += part[(static_cast<int64_t>(p) * 3 + blockIdx.y) * d + c];
    sum[run][threadIdx.x & 31] = s;
    __syncthreads();
    if (run == 0 && c < d) {
#pragma unroll
        for (int r = 1; r < 8; ++r) s += sum[r][threadIdx.x];
        out[c] = s;
    }
}

// Threads of a row and vectors of a thread.
struct Shape {
    int tpr, vpt;
};
Shape shape_of(int d) {
    const int vecs = (d + 7) / 8;
    if (vecs <= 32) return {32, 1};
    if (vecs <= 64) return {32, 2};
    if (vecs <= 128) return {128, 1};
    if (vecs <= 256) return {256, 1};
    if (vecs <= 320) return {320, 1};
    if (vecs <= 512) return {512, 1};
    if (vecs <= 1024) return {1024, 1};
    return {1024, 2};
}

template <typename T, int TPR, int VPT>
void run_forward(const NormArgs& a, cudaStream_t s) {
    const int rows_per = TPR == 32 ? 4 : 1;
    norm_kernel<T, TPR, VPT><<<static_cast<unsigned>((a.f.rows + rows_per - 1) / rows_per), TPR == 32 ? 128 : TPR, 0, s>>>(a);
}

// Blocks of the backward kernel: enough threads for every SM, but a part of
// the sums for each, which the second kernel reads.
int grad_blocks(int64_t rows, int tpr) {
    const int threads = tpr == 32 ? 128 : tpr, per = std::max(1, 1024 / threads), rows_per = tpr == 32 ? 4 : 1;
    return static_cast<int>(std::min<int64_t>((rows + rows_per - 1) / rows_per, static_cast<int64_t>(per) * sm_count_current()));
}
int grad_parts(int64_t rows, int tpr) { return grad_blocks(rows, tpr) * (tpr == 32 ? 4 : 1); }

template <typename T, int TPR, int VPT>
void run_backward(const GradArgs& a, cudaStream_t s) {
    norm_grad_kernel<T, TPR, VPT><<<grad_blocks(a.f.rows, TPR), TPR == 32 ? 128 : TPR, 0, s>>>(a);
}

#define NRN_NORM_SHAPES(T, CALL)                                \
    do {                                                        \
        const Shape sh = shape_of(a.f.d);                       \
        if (sh.tpr == 32 && sh.vpt == 1) CALL<T, 32, 1>(a, s);  \
        else if (sh.tpr == 32) CALL<T, 32, 2>(a, s);            \
        else if (sh.tpr == 128) CALL<T, 128, 1>(a, s);          \
        else if (sh.tpr == 256) CALL<T, 256, 1>(a, s);          \
        else if (sh.tpr == 320) CALL<T, 320, 1>(a, s);          \
        else if (sh.tpr == 512) CALL<T, 512, 1>(a, s);          \
        else if (sh.vpt == 1) CALL<T, 1024, 1>(a, s);           \
        else CALL<T, 1024, 2>(a, s);                            \
    } while (0)

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
    a.vec = row_ok(in->residual, in->residual_stride, size) && row_ok(in->h, in->h_stride, size) &&
            row_ok(in->gate, in->gate_stride, size) && row_ok(in->y, in->y_stride, size) && row_ok(in->z, in->z_stride, size);
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (in->dtype == NRN_BF16) NRN_NORM_SHAPES(__nv_bfloat16, run_forward);
    else if (in->dtype == NRN_FP16) NRN_NORM_SHAPES(__half, run_forward);
    else NRN_NORM_SHAPES(float, run_forward);
    NRN_CUDA_TRY(cudaGetLastError());
    return NRN_OK;
}

extern "C" nrn_status_t nrn_cuda_gatednorm_workspace(const nrn_gatednorm_t* a, int64_t* bytes) {
    NRN_CHECK_ARG(a && bytes, "nrn_cuda_gatednorm_workspace: null argument");
    NRN_CHECK_ARG(a->rows >= 0 && a->d >= 1 && a->d <= kMaxD, "nrn_cuda_gatednorm_workspace: sizes out of range");
    *bytes = static_cast<int64_t>(grad_parts(a->rows, shape_of(a->d).tpr)) * 3 * a->d * 4;
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
    const int size = in->dtype == NRN_FP32 ? 4 : 2, tpr = shape_of(in->d).tpr;
    const int parts = grad_parts(in->rows, tpr);
    if (sums) {
        NRN_CHECK_ARG(g->workspace && g->workspace_bytes >= static_cast<int64_t>(parts) * 3 * in->d * 4, who + ": workspace too small");
        a.part = static_cast<float*>(g->workspace);
    }
    a.vec = row_ok(in->residual, in->residual_stride, size) && row_ok(in->h, in->h_stride, size) &&
            row_ok(in->gate, in->gate_stride, size) && row_ok(g->dy, g->dy_stride, size) && row_ok(g->dz, g->dz_stride, size) &&
            row_ok(g->dresidual, g->dresidual_stride, size) && row_ok(g->dh, g->dh_stride, size) && row_ok(g->dgate, g->dgate_stride, size);
    if (in->dtype == NRN_BF16) NRN_NORM_SHAPES(__nv_bfloat16, run_backward);
    else if (in->dtype == NRN_FP16) NRN_NORM_SHAPES(__half, run_backward);
    else NRN_NORM_SHAPES(float, run_backward);
    NRN_CUDA_TRY(cudaGetLastError());
    if (sums) {
        norm_parts_kernel<<<dim3(static_cast<unsigned>((in->d + 31) / 32), 3), 256, 0, s>>>(a.part, parts, in->d, g->dalpha, g->dw_post, g->dw_pre);
        NRN_CUDA_TRY(cudaGetLastError());
    }
    return NRN_OK;
}

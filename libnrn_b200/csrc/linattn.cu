// linattn.cu -- linear attention with a decay for each head: a fast Hebbian
// projection with forgetting, read by queries.
//
// For each sequence and head, with lam = exp(log_decay[head]):
//     S_t = lam S_{t-1} + k_t v_t^T            (S: dk x dv, fp32)
//     o_t = scale S_t^T q_t
// The rate form of the exponentially decaying traces of the pair STDP rule
// (src/plasticity/stdp.cpp:89-141): presynaptic key times postsynaptic value,
// summed with forgetting.
//
// One scan serves the forward pass and, with the roles of its operands
// exchanged, all gradients.  In general form, over tokens p = 0, 1, ..
//     o_p = out_mul (lam^(p+off) X0^T a_p + sum_{j<=p} lam^(p-j) (a_p . b_j) c_j)
//   forward:  a, b, c = q, k, v            off = 1, X0 = S_0
//   dq:       a, b, c = do, v, k           off = 1, X0 = S_0^T
//   dk:       a, b, c = v, do, q reversed  off = 0, X0 = dS^T / scale
//   dv:       a, b, c = k, q, do reversed  off = 0, X0 = dS / scale
// (dS: gradient of the final state; the state the reversed scan ends with,
// times scale, is the gradient of S_0).  `off` says whether the state that
// enters a token decays before it is read.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "internal.h"
#include "launch.h"
#include "tc.cuh"
#include "tensor_map.h"
#include "vecio.cuh"

namespace nrn {
namespace {

constexpr int kMaxDim = 256;       // largest key or value dimension
constexpr int kChunk = 64;         // tokens of a chunk

struct Strided {
    const void* p;
    int64_t seq, tok, head;        // strides in elements
    int32_t share;                 // heads of the scan that read one head here
    int32_t d;                     // innermost extent (stride 1)
};

struct ScanArgs {
    Strided a, b, c;
    void* o;
    int64_t o_seq, o_tok, o_head;
    int32_t o_f32;                 // o is fp32 whatever the inputs' type (partial sums of shared heads)
    int32_t vec;                   // rows of a, b, c start on 16-byte boundaries
    int32_t o_vec;                 // rows of o do
    int32_t heads;
    int32_t seqs;
    int64_t tokens;                // per sequence, or of all packed sequences
    const int32_t* cu;             // [seqs + 1] starts of packed sequences, or null
    const float* log_decay;
    float out_mul, in_mul, end_mul;
    int32_t off, reverse;
    const float* s_in;             // [seqs][heads] states, element (i of b, j of c) at i*s_i + j*s_j; or null
    float* s_out;                  // the same layout, or null
    int64_t s_i, s_j;
    float* seg;                    // [units][heads]: states of segments, element (i of b, j of c) at i*g_i + j*g_j; or null
    int64_t g_i, g_j;
    int32_t seg_made;              // the states that enter the segments are there already
    int64_t seg_len;               // tokens of a segment (a multiple of the chunk)
    int32_t units;
    int32_t* err;                  // set when a device-side wait gives up, or null
};

// ------------------------------------------------------------------ units
//
// A unit is one segment of one sequence.  Units of sequence s start at
// first(s) = floor(start of s / seg_len) + s: a place that needs no sum over
// the sequences before it and leaves room for ceil(length / seg_len)
// segments; a unit past its sequence's last segment is empty.
struct Unit {
    int64_t row0;                  // first token of the sequence in packed arrays (0 otherwise)
    int64_t len;                   // tokens of the sequence
    int64_t begin, end;            // this segment's tokens
    int32_t seq;
    bool last;                     // it ends the sequence
    bool any;
};

__device__ __forceinline__ int64_t clamp_start(const ScanArgs& p, int s) {
    const int64_t x = p.cu[s];
    return x < 0 ? 0 : (x > p.tokens ? p.tokens : x);
}

__device__ __forceinline__ Unit unit_of(const ScanArgs& p, int u) {
    Unit r;
    int64_t seg;
    if (p.cu == nullptr) {
        const int64_t per = p.tokens > 0 ? (p.tokens + p.seg_len - 1) / p.seg_len : 1;
        r.seq = static_cast<int32_t>(u / per);
        seg = u - r.seq * per;
        r.row0 = 0;
        r.len = p.tokens;
    } else {
        int lo = 0, hi = p.seqs - 1;          // the last sequence whose first unit is <= u
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (clamp_start(p, mid) / p.seg_len + mid <= u) lo = mid;
            else hi = mid - 1;
        }
        r.seq = lo;
        r.row0 = clamp_start(p, lo);
        const int64_t next = clamp_start(p, lo + 1);
        r.len = next > r.row0 ? next - r.row0 : 0;
        seg = u - (r.row0 / p.seg_len + lo);
    }
    r.begin = seg * p.seg_len;
    r.end = r.begin + p.seg_len < r.len ? r.begin + p.seg_len : r.len;
    r.any = seg >= 0 && (r.begin < r.len || (r.len == 0 && seg == 0));
    r.last = r.end == r.len;
    return r;
}

// lam^n: n = 0 is 1 whatever the decay (log_decay may be -inf: the state is
// dropped at every token).  In double, so that a power is off by its rounding
// to fp32 alone: it is applied once for every chunk of a long memory.
__device__ __forceinline__ float decay_power(float log_decay, int64_t n) {
    return n == 0 ? 1.0f : static_cast<float>(exp(static_cast<double>(log_decay) * static_cast<double>(n)));
}

template <typename T>
__device__ __forceinline__ const T* row_ptr(const Strided& m, const Unit& u, int64_t t, int head) {
    return static_cast<const T*>(m.p) + (u.row0 + t) * m.tok + static_cast<int64_t>(u.seq) * m.seq +
           static_cast<int64_t>(head / m.share) * m.head;
}

// ------------------------------------------------------- token by token
//
// The recurrence itself, for every type and dimension.  A block has 32
// columns (c) of one state: 8 lanes share a column, each with every eighth
// group of four rows in registers, so a token costs each thread
// 3 * b.d / 8 operations and three shuffles; 16 tokens at a time are staged
// in shared memory as fp32.  It does 3 b.d c.d operations a token and head on
// the fp32 pipe, at about a sixth of the pipe's rate (256 x 64 fp32 tokens of
// 16 heads of 128 x 128: 2.1 ms, 13 times their bytes; bf16 of 200 x 200 5.8
// ms): every token is a chain of shared-memory loads, products and shuffles
// that the next one waits for.  It serves fp16, fp32 and b.d > 128; bf16 with
// b.d <= 128 has the kernels below.
//
// lam in fp32 is off by up to 3e-8, which over a memory of thousands of
// tokens would show; the error of its powers is taken out of the state after
// every 16 tokens.
constexpr int kSerialThreads = 256;
constexpr int kSerialCols = 32;
constexpr int kSerialTokens = 16;

template <typename T, int G>   // G groups of 4 rows a thread: b.d <= 32 G
__global__ void __launch_bounds__(kSerialThreads) scan_serial_kernel(const __grid_constant__ ScanArgs p, int state_only) {
    __shared__ __align__(16) float sa[kSerialTokens][32 * G];
    __shared__ __align__(16) float sb[kSerialTokens][32 * G];
    __shared__ float sc[kSerialTokens][kSerialCols];
    const int db = p.b.d, dc = p.c.d;
    const int tiles = (dc + kSerialCols - 1) / kSerialCols;
    const int tile = blockIdx.x % tiles;
    const int head = (blockIdx.x / tiles) % p.heads;
    const int unit = blockIdx.x / tiles / p.heads;
    const Unit u = unit_of(p, unit);
    if (!u.any) return;
    const int part = threadIdx.x & 7, col_l = threadIdx.x >> 3, col = tile * kSerialCols + col_l;
    const float lam = decay_power(p.log_decay[head], 1);
    // lam^16 / (fp32 lam)^16 - 1; where lam^16 vanishes there is nothing to mend
    double l2 = static_cast<double>(lam) * lam, l4 = l2 * l2, l16 = l4 * l4 * (l4 * l4);
    const float mend = l16 > 1e-30 ? static_cast<float>(exp(16.0 * static_cast<double>(p.log_decay[head])) / l16 - 1.0) : 0.0f;

    float s[4 * G];
#pragma unroll
    for (int g = 0; g < 4 * G; ++g) s[g] = 0.0f;
    const int64_t sh = (static_cast<int64_t>(u.seq) * p.heads + head) * db * dc;
    const int64_t gh = (static_cast<int64_t>(unit) * p.heads + head) * db * dc;
    if (!state_only && col < dc && (p.seg != nullptr || p.s_in != nullptr)) {
#pragma unroll
        for (int g = 0; g < 4 * G; ++g) {
            const int i = ((g >> 2) * 8 + part) * 4 + (g & 3);
            if (i < db)
                s[g] = p.seg ? p.seg[gh + i * p.g_i + col * p.g_j] : p.s_in[sh + i * p.s_i + col * p.s_j] * p.in_mul;
        }
    }
    for (int64_t t0 = u.begin; t0 < u.end; t0 += kSerialTokens) {
        const int n = static_cast<int>(u.end - t0 < kSerialTokens ? u.end - t0 : kSerialTokens);
        __syncthreads();
        for (int e = threadIdx.x; e < kSerialTokens * 32 * G; e += kSerialThreads) {
            const int t = e / (32 * G), i = e - t * 32 * G;
            float x = 0.0f, y = 0.0f;
            if (t < n && i < db) {
                const int64_t tok = p.reverse ? u.len - 1 - (t0 + t) : t0 + t;
                y = to_f32(row_ptr<T>(p.b, u, tok, head)[i]);
                if (!state_only) x = to_f32(row_ptr<T>(p.a, u, tok, head)[i]);
            }
            sa[t][i] = x;
            sb[t][i] = y;
        }
        for (int e = threadIdx.x; e < kSerialTokens * kSerialCols; e += kSerialThreads) {
            const int t = e / kSerialCols, j = tile * kSerialCols + e % kSerialCols;
            float x = 0.0f;
            if (t < n && j < dc) {
                const int64_t tok = p.reverse ? u.len - 1 - (t0 + t) : t0 + t;
                x = to_f32(row_ptr<T>(p.c, u, tok, head)[j]);
            }
            sc[t][e % kSerialCols] = x;
        }
        __syncthreads();
        for (int t = 0; t < n; ++t) {
            const float c = sc[t][col_l];
            float o = 0.0f;
            // off = 1: decay, add, read.  off = 0: add, read, decay.
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const float4 b = *reinterpret_cast<const float4*>(&sb[t][(g * 8 + part) * 4]);
                const float4 a = *reinterpret_cast<const float4*>(&sa[t][(g * 8 + part) * 4]);
                if (p.off) {
                    s[4 * g + 0] = fmaf(b.x, c, lam * s[4 * g + 0]);
                    s[4 * g + 1] = fmaf(b.y, c, lam * s[4 * g + 1]);
                    s[4 * g + 2] = fmaf(b.z, c, lam * s[4 * g + 2]);
                    s[4 * g + 3] = fmaf(b.w, c, lam * s[4 * g + 3]);
                } else {
                    s[4 * g + 0] = fmaf(b.x, c, s[4 * g + 0]);
                    s[4 * g + 1] = fmaf(b.y, c, s[4 * g + 1]);
                    s[4 * g + 2] = fmaf(b.z, c, s[4 * g + 2]);
                    s[4 * g + 3] = fmaf(b.w, c, s[4 * g + 3]);
                }
                o = fmaf(a.x, s[4 * g + 0], o);
                o = fmaf(a.y, s[4 * g + 1], o);
                o = fmaf(a.z, s[4 * g + 2], o);
                o = fmaf(a.w, s[4 * g + 3], o);
                if (!p.off) {
                    s[4 * g + 0] *= lam;
                    s[4 * g + 1] *= lam;
                    s[4 * g + 2] *= lam;
                    s[4 * g + 3] *= lam;
                }
            }
            if (state_only) continue;
            o += __shfl_xor_sync(0xffffffffu, o, 1);
            o += __shfl_xor_sync(0xffffffffu, o, 2);
            o += __shfl_xor_sync(0xffffffffu, o, 4);
            if (part == 0 && col < dc) {
                const int64_t tok = p.reverse ? u.len - 1 - (t0 + t) : t0 + t;
                const int64_t at = (u.row0 + tok) * p.o_tok + static_cast<int64_t>(u.seq) * p.o_seq + head * p.o_head + col;
                if (p.o_f32) static_cast<float*>(p.o)[at] = o * p.out_mul;
                else static_cast<T*>(p.o)[at] = from_f32<T>(o * p.out_mul);
            }
        }
        if (n == kSerialTokens) {
#pragma unroll
            for (int g = 0; g < 4 * G; ++g) {
                const float x = fmaf(s[g], mend, s[g]);
                s[g] = x == x ? x : s[g];            // an infinity times the error would leave no number
            }
        }
    }
    if (col >= dc) return;
    if (state_only) {
#pragma unroll
        for (int g = 0; g < 4 * G; ++g) {
            const int i = ((g >> 2) * 8 + part) * 4 + (g & 3);
            if (i < db) p.seg[gh + i * p.g_i + col * p.g_j] = s[g];
        }
    } else if (u.last && p.s_out != nullptr && p.seg == nullptr) {
#pragma unroll
        for (int g = 0; g < 4 * G; ++g) {
            const int i = ((g >> 2) * 8 + part) * 4 + (g & 3);
            if (i < db) p.s_out[sh + i * p.s_i + col * p.s_j] = s[g] * p.end_mul;
        }
    }
}

// ------------------------------------------------------- chunks of 32 tokens
//
// bf16 inputs with rows off 16-byte boundaries, b.d <= 128.  For a chunk of
// tokens p with entering state X:
//     o_p = lam^(p+off) X^T a_p + sum_{j<=p} lam^(p-j) (a_p . b_j) c_j
//     X'  = lam^n X + sum_j lam^(n-off-j) b_j c_j^T
// A block holds 64 columns (c) of one state, a warp 16 of them: X^T as
// 16 x b.d fp32 accumulators in registers for the whole scan, which are, cast
// to bf16, the left operand of X^T a^T as they lie.  All products are 16x8x16
// tensor-core instructions:
//     P    = decayed a b^T, lower triangle only, once for the block (shared)
//     o^T  = c^T P^T + (X^T a^T) lam^(p+off), written through shared memory
//     X'^T = lam^n X^T + (w c)^T b
// Roundings: P and the copy of X that is read are bf16, as the result is
// (each at most 2^-9, sums fp32).  The state itself keeps fp32: the decayed
// values w c are split into bf16 terms (TERMS = 3: all 24 bits; 2 where the
// state that comes out is made elsewhere: 16 bits, below the results' 8).
//
// A token that is no number must not reach earlier tokens of its chunk
// through the zeros of P (0 * inf): where the product with P has an element
// that is not finite, the warp sums it again over j <= p alone.
constexpr int kMmaThreads = 128;
constexpr int kMmaCols = 64;
constexpr int kMmaChunk = 32;

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], const void* p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(p))));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], const void* p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(p))));
}
__device__ __forceinline__ void stsm4t(void* p, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(
                     static_cast<uint32_t>(__cvta_generic_to_shared(p))),
                 "r"(a), "r"(b), "r"(c), "r"(d)
                 : "memory");
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Two fp32 as bf16, the first in the low half.
__device__ __forceinline__ uint32_t bf16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float low_f32(uint32_t x) { return __uint_as_float(x << 16); }
__device__ __forceinline__ float high_f32(uint32_t x) { return __uint_as_float(x & 0xffff0000u); }

// One operand's rows of CH tokens as CH x COLS bf16 in shared memory, zeros
// past the tokens and past the operand's columns.  A thread has one place in
// every kRows-th row; its address moves on by additions alone.
template <int CH, int COLS>
struct RowLoader {
    static constexpr int kPitch = COLS + 8, kRows = kMmaThreads / (COLS / 8), kLoads = CH / kRows;
    const __nv_bfloat16* src;
    int64_t step;                  // kRows tokens on
    int t, left;                   // first row; columns of the operand from this place on
    uint32_t place;                // bytes from the start of the rows

    __device__ __forceinline__ RowLoader(const Strided& m, const ScanArgs& p, const Unit& u, int head, int col0) {
        t = threadIdx.x / (COLS / 8);
        const int c = (threadIdx.x % (COLS / 8)) * 8;
        left = m.d - col0 - c;
        const int64_t first = p.reverse ? u.len - 1 - (u.begin + t) : u.begin + t;
        src = row_ptr<__nv_bfloat16>(m, u, 0, head) + first * m.tok + col0 + c;
        step = (p.reverse ? -m.tok : m.tok) * kRows;
        place = static_cast<uint32_t>((t * kPitch + c) * 2);
    }
    // the next CH tokens, n of which there are, element by element: rows on
    // 16-byte boundaries go to the kernel below
    __device__ __forceinline__ void load(void* dst, int n) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i, src += step) {
            const bool in = t + i * kRows < n && left > 0;
            const Raw8<__nv_bfloat16> r = load8(src, in ? left : 0, false);
            *reinterpret_cast<uint4*>(static_cast<char*>(dst) + place + i * kRows * kPitch * 2) = *reinterpret_cast<const uint4*>(&r);
        }
    }
};

template <int DK, int CH>
struct MmaSmem {
    __nv_bfloat16 a[2][CH][DK + 8];
    __nv_bfloat16 b[2][CH][DK + 8];
    __nv_bfloat16 c[2][CH][kMmaCols + 8];
    __nv_bfloat16 prob[CH][CH + 8];
    __nv_bfloat16 out[4][32][24];
    float pw[CH + 4];                  // lam^0 .. lam^CH
};

template <int DK, int CH, int TERMS, bool STATE_ONLY>
__global__ void __launch_bounds__(kMmaThreads, DK == 64 ? 4 : 3) scan_mma_kernel(const __grid_constant__ ScanArgs p) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    MmaSmem<DK, CH>& M = *reinterpret_cast<MmaSmem<DK, CH>*>(smem_raw);
    const int dc = p.c.d, db = p.b.d;
    const int tiles = (dc + kMmaCols - 1) / kMmaCols;
    const int tile = blockIdx.x % tiles;
    const int head = (blockIdx.x / tiles) % p.heads;
    const int unit = blockIdx.x / tiles / p.heads;
    const Unit u = unit_of(p, unit);
    if (!u.any) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, q = lane & 3;                  // row and column group of a fragment
    constexpr int kTiles = (CH / 16) * (CH / 16 + 1) / 2;
    const int l7 = lane & 7, l8 = (lane >> 3) & 1, l16 = lane >> 4;
    const int col0 = tile * kMmaCols, wcol = col0 + warp * 16;
    for (int i = threadIdx.x; i <= CH; i += kMmaThreads) M.pw[i] = decay_power(p.log_decay[head], i);

    // X^T: element (wcol + g + 8 (e >> 1), 8 nt + 2 q + (e & 1)) in s[nt][e]
    float s[DK / 8][4];
    const int64_t sh = (static_cast<int64_t>(u.seq) * p.heads + head) * db * dc;
    const int64_t gh = (static_cast<int64_t>(unit) * p.heads + head) * db * dc;
    const bool given = !STATE_ONLY && (p.seg != nullptr || p.s_in != nullptr);
#pragma unroll
    for (int nt = 0; nt < DK / 8; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = nt * 8 + 2 * q + (e & 1), j = wcol + g + 8 * (e >> 1);
            s[nt][e] = 0.0f;
            if (given && i < db && j < dc)
                s[nt][e] = p.seg ? p.seg[gh + i * p.g_i + j * p.g_j] : p.s_in[sh + i * p.s_i + j * p.s_j] * p.in_mul;
        }

    RowLoader<CH, DK> la(p.a, p, u, head, 0), lb(p.b, p, u, head, 0);
    RowLoader<CH, kMmaCols> lc(p.c, p, u, head, col0);
    // the results' place of this lane: token begin + lane / 2, eight of the warp's columns
    const int oj = wcol + 8 * (lane & 1);
    const int64_t ofirst = u.begin + (lane >> 1), ostep = p.reverse ? -p.o_tok : p.o_tok;
    int64_t oat = (u.row0 + (p.reverse ? u.len - 1 - ofirst : ofirst)) * p.o_tok + static_cast<int64_t>(u.seq) * p.o_seq + head * p.o_head + oj;
    auto fetch = [&](int64_t t0, int stage) {
        const int n = static_cast<int>(u.end - t0 < CH ? u.end - t0 : CH);
        lb.load(&M.b[stage][0][0], n);
        lc.load(&M.c[stage][0][0], n);
        if (!STATE_ONLY) la.load(&M.a[stage][0][0], n);
    };
    if (u.begin < u.end) fetch(u.begin, 0);

    int stage = 0;
    for (int64_t t0 = u.begin; t0 < u.end; t0 += CH, stage ^= 1) {
        const int n = static_cast<int>(u.end - t0 < CH ? u.end - t0 : CH);
        __syncthreads();                 // this chunk is here, and everybody is done with the last one
        if (t0 + CH < u.end) fetch(t0 + CH, stage ^ 1);
        const auto& A = M.a[stage];
        const auto& B = M.b[stage];
        const auto& C = M.c[stage];

        if constexpr (!STATE_ONLY) {
            // P: the 16 x 16 tiles of the lower triangle, in turn over the warps
#pragma unroll
            for (int t = 0; t < (kTiles + 3) / 4; ++t) {
                const int id = warp + 4 * t;
                if (id >= kTiles) break;
                const int r = id < 1 ? 0 : (id < 3 ? 1 : (id < 6 ? 2 : 3)), c = id - r * (r + 1) / 2;
                float acc[2][2][4] = {};
#pragma unroll
                for (int kk = 0; kk < DK / 16; ++kk) {
                    uint32_t fa[4], fb[4];
                    ldsm4(fa, &A[r * 16 + l7 + 8 * l8][kk * 16 + 8 * l16]);
                    ldsm4(fb, &B[c * 16 + l7 + 8 * l16][kk * 16 + 8 * l8]);
                    mma16816(acc[kk & 1][0], fa, fb[0], fb[1]);
                    mma16816(acc[kk & 1][1], fa, fb[2], fb[3]);
                }
#pragma unroll
                for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int i = r * 16 + g + 8 * h, j = c * 16 + nt * 8 + 2 * q;
                        const float x = acc[0][nt][2 * h] + acc[1][nt][2 * h], y = acc[0][nt][2 * h + 1] + acc[1][nt][2 * h + 1];
                        *reinterpret_cast<uint32_t*>(&M.prob[i][j]) =
                            bf16x2(j <= i ? x * M.pw[i - j] : 0.0f, j + 1 <= i ? y * M.pw[i - j - 1] : 0.0f);
                    }
            }
            __syncthreads();

            // o^T: element (wcol + g + 8 (e >> 1), token 8 nt + 2 q + (e & 1))
            float o[CH / 8][4] = {};
#pragma unroll
            for (int kk = 0; kk < CH / 16; ++kk) {
                uint32_t fc[4];
                ldsm4t(fc, &C[kk * 16 + l7 + 8 * l16][warp * 16 + 8 * l8]);
#pragma unroll
                for (int np = kk; np < CH / 16; ++np) {
                    uint32_t fp[4];
                    ldsm4(fp, &M.prob[np * 16 + l7 + 8 * l16][kk * 16 + 8 * l8]);
                    mma16816(o[2 * np], fc, fp[0], fp[1]);
                    mma16816(o[2 * np + 1], fc, fp[2], fp[3]);
                }
            }
            bool bad = false;
#pragma unroll
            for (int nt = 0; nt < CH / 8; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) bad |= !(fabsf(o[nt][e]) <= 3.4028234e38f);
            if (__any_sync(0xffffffffu, bad)) {
#pragma unroll
                for (int nt = 0; nt < CH / 8; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int i = nt * 8 + 2 * q + (e & 1);
                        float x = 0.0f;
                        for (int j = 0; j <= i; ++j)
                            x = fmaf(to_f32(M.prob[i][j]), to_f32(C[j][warp * 16 + g + 8 * (e >> 1)]), x);
                        o[nt][e] = x;
                    }
            }
            {
                float x[CH / 8][4] = {};
#pragma unroll
                for (int kk = 0; kk < DK / 16; ++kk) {
                    const uint32_t fs[4] = {bf16x2(s[2 * kk][0], s[2 * kk][1]), bf16x2(s[2 * kk][2], s[2 * kk][3]),
                                            bf16x2(s[2 * kk + 1][0], s[2 * kk + 1][1]), bf16x2(s[2 * kk + 1][2], s[2 * kk + 1][3])};
#pragma unroll
                    for (int np = 0; np < CH / 16; ++np) {
                        uint32_t fa[4];
                        ldsm4(fa, &A[np * 16 + l7 + 8 * l16][kk * 16 + 8 * l8]);
                        mma16816(x[2 * np], fs, fa[0], fa[1]);
                        mma16816(x[2 * np + 1], fs, fa[2], fa[3]);
                    }
                }
#pragma unroll
                for (int nt = 0; nt < CH / 8; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        o[nt][e] = p.out_mul * fmaf(M.pw[nt * 8 + 2 * q + (e & 1) + p.off], x[nt][e], o[nt][e]);
            }
            if (p.o_f32) {
#pragma unroll
                for (int nt = 0; nt < CH / 8; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int t = nt * 8 + 2 * q + (e & 1), j = wcol + g + 8 * (e >> 1);
                        const int64_t tok = p.reverse ? u.len - 1 - (t0 + t) : t0 + t;
                        if (t < n && j < dc)
                            static_cast<float*>(p.o)[(u.row0 + tok) * p.o_tok + static_cast<int64_t>(u.seq) * p.o_seq + head * p.o_head + j] = o[nt][e];
                    }
            } else {
                // 32 tokens at a time through the warp's own 32 x 16 elements: 32 bytes a token
#pragma unroll
                for (int half = 0; half < CH / 32; ++half) {
                    __syncwarp();
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const int nt = half * 4 + 2 * k;
                        stsm4t(&M.out[warp][k * 16 + l7 + 8 * l16][8 * l8], bf16x2(o[nt][0], o[nt][1]), bf16x2(o[nt][2], o[nt][3]),
                               bf16x2(o[nt + 1][0], o[nt + 1][1]), bf16x2(o[nt + 1][2], o[nt + 1][3]));
                    }
                    __syncwarp();
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const int r = k * 16 + (lane >> 1), t = half * 32 + r;
                        __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(p.o) + oat;
                        oat += 16 * ostep;
                        if (t >= n || oj >= dc) continue;
                        const __nv_bfloat16* src = &M.out[warp][r][8 * (lane & 1)];
                        if (p.o_vec) {
                            *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(src);
                        } else {
                            for (int e = 0; e < 8 && oj + e < dc; ++e) dst[e] = src[e];
                        }
                    }
                }
            }
        }

        // the state
        const float whole = M.pw[n];
#pragma unroll
        for (int nt = 0; nt < DK / 8; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[nt][e] *= whole;
#pragma unroll
        for (int kk = 0; kk < CH / 16; ++kk) {
            if (kk * 16 >= n) break;
            uint32_t fc[4], term[3][4];
            ldsm4t(fc, &C[kk * 16 + l7 + 8 * l16][warp * 16 + 8 * l8]);
#pragma unroll
            for (int h = 0; h < 2; ++h) {           // tokens 2 q and 2 q + 1 of the first and second eight
                const int j = kk * 16 + 8 * h + 2 * q;
                const float w0 = j < n ? M.pw[n - p.off - j] : 0.0f, w1 = j + 1 < n ? M.pw[n - p.off - j - 1] : 0.0f;
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    float x = low_f32(fc[2 * h + r]) * w0, y = high_f32(fc[2 * h + r]) * w1;
#pragma unroll
                    for (int k = 0; k < TERMS; ++k) {
                        const uint32_t z = bf16x2(x, y);
                        term[k][2 * h + r] = z;
                        x -= low_f32(z);
                        y -= high_f32(z);
                    }
                }
            }
#pragma unroll
            for (int n4 = 0; n4 < DK / 16; n4 += 4) {   // eight accumulators between the terms of one
                uint32_t fb[4][4];
#pragma unroll
                for (int i = 0; i < 4; ++i) ldsm4t(fb[i], &B[kk * 16 + l7 + 8 * l8][(n4 + i) * 16 + 8 * l16]);
#pragma unroll
                for (int k = 0; k < TERMS; ++k)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        mma16816(s[2 * (n4 + i)], term[k], fb[i][0], fb[i][1]);
                        mma16816(s[2 * (n4 + i) + 1], term[k], fb[i][2], fb[i][3]);
                    }
            }
        }
    }

    float* to = STATE_ONLY ? p.seg : (u.last && p.seg == nullptr ? p.s_out : nullptr);
    if (to == nullptr) return;
#pragma unroll
    for (int nt = 0; nt < DK / 8; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = nt * 8 + 2 * q + (e & 1), j = wcol + g + 8 * (e >> 1);
            if (i >= db || j >= dc) continue;
            if (STATE_ONLY) to[gh + i * p.g_i + j * p.g_j] = s[nt][e];
            else to[sh + i * p.s_i + j * p.s_j] = s[nt][e] * p.end_mul;
        }
}

// -------------------------------------------------- the same on tcgen05
//
// bf16 rows on 16-byte boundaries, b.d <= 128: chunks of 64 tokens, 128
// columns (c) of one state a block, products on tcgen05 with fp32
// accumulators in TMEM, in the transposed form (TMEM lane = column of c):
//     P     [64 x 64]   = a b^T                 lanes: tokens i
//     inter [128 x 64]  = X16^T a^T             X16: the entering state in bf16
//     U     [128 x b.d] = sum over terms of (w c)^T b
//     intra [128 x 64]  = c^T P^T
// The left operands of the last three (X16, the terms, c^T) are written to
// TMEM from registers; a, b, b^T and P lie in shared memory.  20 warps, one
// block an SM:
//   warp 0      copies: a, b and c of a chunk by TMA into one of three stages;
//   warp 1      issues the MMAs (one thread); warps 2 and 3 only give up
//               their registers;
//   warps 4-11  (1) c's decayed terms and b^T, while P and inter run; (2) P
//               out of TMEM, decay and mask, bf16, and c^T, while U runs;
//   warps 12-19 (3) the fp32 state, kept in registers (64 a thread):
//               lam^n X + U, and its bf16 copy; (4) the results.
// The two groups work on neighbouring chunks at once: with all sixteen warps
// on one phase after the other a chunk took 6,600 cycles, of which 2,700 were
// issue slots; it takes 3,500 so.  The pass that makes segments' states has
// only U to compute and two buffers of terms and b^T: 0.9 us a chunk.
//
// What bounds it: neither HBM (9 x 4096 tokens of 16 heads of 128: 604 MB in
// 142 us, 65% of the measured copy) nor the MMAs, but the chain P -> mask ->
// intra -> results and U -> state -> inter, each through TMEM and registers.
// The third stage of copies brought 5%.  64 tokens a chunk:
// 128 would halve the chain but double P's work and does not fit shared
// memory; 128 columns a block: with 64 a and b are read and P is made twice.
// With mma.sync (the kernel above) operands pass through every warp's
// registers, about 270 warp instructions a token and head.
//
// A value of c that is no number must not reach earlier tokens of its chunk
// through the zeros of P (0 * inf): it goes into the tiles as 0, and from its
// token on the column's results are NaN.
constexpr int kTcThreads = 640;
constexpr int kTcGroup = 8;             // warps of each of the two groups
constexpr int kTcCols = 128;
constexpr int kTcStages = 3;            // chunks of a, b and c in shared memory
enum { ERR_LINATTN_TIMEOUT = 5 };

using namespace tc;

template <int DK, int TERMS, bool STATE_ONLY>
struct TcSmem {
    static constexpr int kTile = kChunk * 128;                        // 64 rows of 64 bf16: 8 KB
    static constexpr int kTilesA = STATE_ONLY ? 0 : DK / 64, kTilesB = DK / 64, kTilesC = 2;
    static constexpr int kStage = (kTilesA + kTilesB + kTilesC) * kTile;
    static constexpr int kHead = 3072;
    static constexpr int kBt = kHead + kTcStages * kStage;                    // b^T [DK][64]
    static constexpr int kBuffers = STATE_ONLY ? 2 : 1;   // of the left operand's terms and b^T: the state's pass has room
    static constexpr int kProb = kBt + kBuffers * DK * 128;           // [64][64]
    static constexpr int kOut = kProb + (STATE_ONLY ? 0 : kTile);          // 4 KB for each warp of results
    static constexpr int kBytes = kOut + (STATE_ONLY ? 0 : kTcGroup * 4096);
};
static_assert(TcSmem<128, 3, false>::kBytes <= 227 * 1024, "shared memory of one block");

struct TcHead {
    uint64_t full[kTcStages], empty[kTcStages], oready[2], uready[2], vk[2], pready, psm, x16, iready, odone, drain;
    uint32_t tmem;
    int abort;
    alignas(16) float lag[128];    // factor of P at token i - token j, from -63 on
    alignas(16) float w[kChunk];   // decay of each token to the chunk's end
    alignas(16) float out[2][kChunk];   // and of the entering state to each token, times out_mul; [1]: of a shorter last chunk
    float whole[2];                // lam^(tokens of the chunk), likewise
    uint8_t bad[2][kTcGroup];      // 16 columns of c hold a value that is no number, and each column's first, in scan order
    uint8_t first_bad[2][kTcCols];
};
static_assert(sizeof(TcHead) <= 3072, "barriers and factors");

// No swizzle: rows of 16 bytes, eight rows to a core matrix, core matrices of
// one row group 128 bytes apart, row groups `group` bytes apart.
__device__ __forceinline__ uint64_t desc_plain(uint32_t addr, uint32_t group) {
    return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(128 >> 4) << 16) |
           (static_cast<uint64_t>(group >> 4) << 32) | (1ull << 46);
}
// 128-byte swizzle as TMA writes it.
__device__ __forceinline__ uint64_t desc_swizzled(uint32_t addr) {
    return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | (1ull << 16) | (static_cast<uint64_t>(1024 >> 4) << 32) |
           (1ull << 46) | (2ull << 61);
}
// The same with A in TMEM: lane = row, two elements of K a column.
template <int NN>
__device__ __forceinline__ void mma_bf16_ta(uint32_t d, uint32_t a, uint64_t b, bool accumulate) {
    constexpr uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(NN >> 3) << 17) | (128u >> 4 << 24);
    const uint32_t zero = 0;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1u : 0u), "r"(zero)
        : "memory");
}
// One thread of a converged warp, chosen so that the compiler keeps what the warp computed alike in uniform registers.
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}
// 16 lanes by 32 columns from eight pairs of fragment registers (row g and g + 8 of four columns each).
__device__ __forceinline__ void tc_st_frag(uint32_t taddr, const uint32_t (&v)[4][4]) {
    asm volatile(
        "tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
        "r"(v[0][0]), "r"(v[0][1]), "r"(v[0][2]), "r"(v[0][3]), "r"(v[1][0]), "r"(v[1][1]), "r"(v[1][2]), "r"(v[1][3]), "r"(v[2][0]),
        "r"(v[2][1]), "r"(v[2][2]), "r"(v[2][3]), "r"(v[3][0]), "r"(v[3][1]), "r"(v[3][2]), "r"(v[3][3])
        : "memory");
}
__device__ __forceinline__ void tc_st16(uint32_t taddr, const uint32_t* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]),
        "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
template <int MM, int NN>
__device__ __forceinline__ void mma_bf16(uint32_t d, uint64_t a, uint64_t b, bool accumulate) {
    constexpr uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(NN >> 3) << 17) | (static_cast<uint32_t>(MM >> 4) << 24);
    const uint32_t zero = 0;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1u : 0u), "r"(zero)
        : "memory");
}
__device__ __forceinline__ void stsm4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void ldsm4t_at(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const void* map, int x, int y, int z, int w, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
        : "memory");
}
// 16 lanes x 32 columns as the fragments of four 16x8 accumulators.
__device__ __forceinline__ void tc_ld_frag(uint32_t taddr, uint32_t* v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
          "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr));
}
constexpr uint64_t kMinusOnes = 0xbf800000bf800000ull;
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// F32: the results are fp32 parts (shared heads); both kinds in one kernel cost it registers (4%)
template <int DK, int TERMS, bool STATE_ONLY, bool F32>
__global__ void __launch_bounds__(kTcThreads, 1)
    scan_tc_kernel(const __grid_constant__ CUtensorMap amap, const __grid_constant__ CUtensorMap bmap,
                   const __grid_constant__ CUtensorMap cmap, const __grid_constant__ ScanArgs p) {
    using L = TcSmem<DK, TERMS, STATE_ONLY>;
    extern __shared__ __align__(1024) unsigned char smem[];
    TcHead& M = *reinterpret_cast<TcHead*>(smem);
    const uint32_t base = smem_u32(smem);
    volatile int* abort = &M.abort;
    const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const int db = p.b.d, dc = p.c.d;
    const int tiles = (dc + kTcCols - 1) / kTcCols;
    const int tile = blockIdx.x % tiles;
    const int head = (blockIdx.x / tiles) % p.heads;
    const int unit = blockIdx.x / tiles / p.heads;
    const Unit u = unit_of(p, unit);
    if (!u.any) {
        let_next();
        previous_done();
        return;
    }
    const int chunks = static_cast<int>((u.end - u.begin + kChunk - 1) / kChunk);
    // TMEM columns: accumulators, then the left operands X16, c^T's terms and c^T
    constexpr uint32_t kP = 0, kU = 64, kIntra = kU + DK, kInter = kIntra + 64, kX16 = kInter + 64, kCt = kX16 + DK / 2,
                       kTerms = STATE_ONLY ? kIntra : kCt + 32;
    static_assert(kTerms + L::kBuffers * 96 <= 512, "columns of TMEM");

    if (threadIdx.x == 0) {
        for (int i = 0; i < kTcStages; ++i) {
            mbar_init(&M.full[i], 1);
            mbar_init(&M.empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            // two of each: the next chunk's may come before this one's is looked at
            mbar_init(&M.uready[i], 1);
            mbar_init(&M.oready[i], 1);
            mbar_init(&M.vk[i], kTcGroup);
        }
        mbar_init(&M.pready, 1);
        mbar_init(&M.iready, 1);
        mbar_init(&M.drain, 1);
        mbar_init(&M.psm, kTcGroup);
        mbar_init(&M.x16, kTcGroup);
        mbar_init(&M.odone, kTcGroup);
        M.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&M.tmem)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = M.tmem;
    let_next();              // not before this block has its TMEM: a block of the next kernel could take it and wait for this one
    previous_done();
    auto fail = [&]() {
        *abort = 1;
        if (p.err) atomicCAS(p.err, 0, ERR_LINATTN_TIMEOUT);
    };
    // tokens of chunk c, and the first of them in memory order
    auto tokens = [&](int c) { return static_cast<int>(u.end - u.begin - static_cast<int64_t>(c) * kChunk < kChunk ? u.end - u.begin - static_cast<int64_t>(c) * kChunk : kChunk); };
    auto first = [&](int c) {
        const int64_t t = u.begin + static_cast<int64_t>(c) * kChunk;
        return p.reverse ? u.len - t - tokens(c) : t;
    };

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        if (warp == 0 && lane == 0) {
            int c = 0, st = 0;
            uint32_t phase = 0;
            for (; c < chunks; ++c) {
                if (!mbar_wait(&M.empty[st], phase ^ 1u, abort)) {
                    fail();
                    break;
                }
                const uint32_t dst = base + L::kHead + st * L::kStage;
                const int tok = static_cast<int>(u.row0 + first(c)), seq = p.cu ? 0 : u.seq;
                mbar_expect_tx(&M.full[st], L::kStage);
                for (int i = 0; i < L::kTilesA; ++i)
                    tma_load_4d(dst + i * L::kTile, &amap, 64 * i, head / p.a.share, tok, seq, &M.full[st]);
                for (int i = 0; i < L::kTilesB; ++i)
                    tma_load_4d(dst + (L::kTilesA + i) * L::kTile, &bmap, 64 * i, head / p.b.share, tok, seq, &M.full[st]);
                for (int i = 0; i < L::kTilesC; ++i)
                    tma_load_4d(dst + (L::kTilesA + L::kTilesB + i) * L::kTile, &cmap, tile * kTcCols + 64 * i, head / p.c.share, tok, seq, &M.full[st]);
                if (++st == kTcStages) {
                    st = 0;
                    phase ^= 1u;
                }
            }
            // the copies still in flight land before the block ends
            for (int q = c - 1; q >= 0 && q >= c - kTcStages; --q) mbar_wait(&M.full[q % kTcStages], (q / kTcStages) & 1, nullptr);
        } else if (warp == 1) {
            // the whole warp walks the chunks, one thread issues
            const bool leader = elect_one();
            bool ok = true;
            int stage = 0;
            uint32_t phase = 0;
            for (int c = 0; c < chunks; ++c) {
                const uint32_t ph = c & 1;
                const uint32_t sa = base + L::kHead + stage * L::kStage, sb = sa + L::kTilesA * L::kTile;
                ok = __all_sync(0xffffffffu, mbar_wait(&M.full[stage], phase, abort));
                if (!ok) break;
                tc_fence_after();
                if constexpr (!STATE_ONLY) {
                    // P: the last chunk's was read before psm of that chunk, on which intra waited
                    if (leader) {
#pragma unroll
                        for (int kk = 0; kk < DK / 16; ++kk)
                            mma_bf16<64, 64>(tmem + kP, desc_swizzled(sa + (kk >> 2) * L::kTile + (kk & 3) * 32),
                                             desc_swizzled(sb + (kk >> 2) * L::kTile + (kk & 3) * 32), kk > 0);
                        tc_commit(&M.pready);
                    }
                    __syncwarp();
                }
                // X16 is there, U of the last chunk read, and c's terms are there: U first, the state waits for it
                ok = __all_sync(0xffffffffu, mbar_wait(&M.x16, ph, abort) && mbar_wait(&M.vk[ph], (c >> 1) & 1, abort));
                if (!ok) break;
                tc_fence_after();
                if (leader) {
#pragma unroll
                    for (int t = 0; t < TERMS; ++t)
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk)
                            mma_bf16_ta<DK>(tmem + kU, tmem + kTerms + (L::kBuffers == 2 ? ph * 96 : 0) + t * 32 + kk * 8,
                                            desc_plain(base + L::kBt + (L::kBuffers == 2 ? ph * DK * 128 : 0) + kk * 256, 1024), t + kk > 0);
                    tc_commit(&M.uready[ph]);
                }
                __syncwarp();
                if constexpr (!STATE_ONLY) {
                    // the last chunk's results have been read
                    if (c > 0) ok = __all_sync(0xffffffffu, mbar_wait(&M.odone, ph ^ 1u, abort));
                    if (!ok) break;
                    tc_fence_after();
                    if (leader) {
#pragma unroll
                        for (int kk = 0; kk < DK / 16; ++kk)
                            mma_bf16_ta<64>(tmem + kInter, tmem + kX16 + kk * 8, desc_swizzled(sa + (kk >> 2) * L::kTile + (kk & 3) * 32), kk > 0);
                        tc_commit(&M.iready);
                    }
                    __syncwarp();
                }
                if constexpr (!STATE_ONLY) {
                    ok = __all_sync(0xffffffffu, mbar_wait(&M.psm, ph, abort));
                    if (!ok) break;
                    tc_fence_after();
                    if (leader) {
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk)
                            mma_bf16_ta<64>(tmem + kIntra, tmem + kCt + kk * 8, desc_plain(base + L::kProb + kk * 256, 1024), kk > 0);
                        tc_commit(&M.oready[ph]);
                    }
                    __syncwarp();
                }
                if (leader) tc_commit(&M.empty[stage]);
                __syncwarp();
                if (++stage == kTcStages) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
            if (!ok && leader) fail();
            // every MMA issued has completed before the accumulators are freed
            if (leader) {
                tc_commit(&M.drain);
                mbar_wait(&M.drain, 0, nullptr);
            }
        }
    } else if (warp < 4 + kTcGroup) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
        const int ew = warp - 4, sub = warp & 3, half = ew >> 2;      // rows 16 sub and columns 32 half of P; 16 columns of c and b
        const int ccol = 2 * sub + half;                              // these 16 of c: this warp's lanes of TMEM
        const int et = threadIdx.x - 128;
        const int l7 = lane & 7, l8 = (lane >> 3) & 1, l16 = lane >> 4, q = lane & 3, g8 = lane >> 2;
        const float g = p.log_decay[head];
        // the factors of a chunk of n tokens, one thread each; the results' group reads its own after the MMAs that follow these
        auto factors = [&](int n, int last) {
            int64_t power = -1;
            if (et < 127) power = last ? -1 : (p.reverse ? 63 - et : et - 63);
            else if (et == 127) power = n;
            else if (et < 192) power = et - 128 < n ? n - p.off - (p.reverse ? n - 1 - (et - 128) : et - 128) : -1;
            else power = et - 192 < n ? (p.reverse ? n - 1 - (et - 192) : et - 192) + p.off : -1;
            const float f = power < 0 ? 0.0f : decay_power(g, power);
            if (et < 127 && !last) M.lag[et] = p.out_mul * f;
            if (et == 127) M.whole[last] = f;
            if (et >= 128 && et < 192) M.w[et - 128] = f;
            if (et >= 192) M.out[last][et - 192] = p.out_mul * f;
        };
        bool ok = true;
        int stage = kTcStages - 1;
        uint32_t phase = 1;
        for (int c = 0; c < chunks; ++c) {
            if (++stage == kTcStages) {
                stage = 0;
                phase ^= 1u;
            }
            const int st = c & 1, n = tokens(c);
            const uint32_t ph = c & 1;
            const uint32_t sb = base + L::kHead + stage * L::kStage + L::kTilesA * L::kTile, sc = sb + L::kTilesB * L::kTile;
            // U has read the terms that were in this place
            if (c >= L::kBuffers) ok = ok && __all_sync(0xffffffffu, mbar_wait(&M.uready[(c - L::kBuffers) & 1], ((c - L::kBuffers) >> 1) & 1, abort));
            if (c == 0 || n < kChunk) {
                asm volatile("bar.sync 1, 256;" ::: "memory");
                factors(n, c > 0);
                asm volatile("bar.sync 1, 256;" ::: "memory");
            }
            ok = ok && __all_sync(0xffffffffu, mbar_wait(&M.full[stage], phase, abort));
            uint32_t f[4][4];                            // two tokens of two columns each
            uint64_t numbers = 0;                        // stays 0 while all values are
            if (ok) {
                tc_fence_after();
                // (1) 16 columns of c
                const uint32_t lrow = (l7 + 8 * l16) * 128;
                const uint32_t cfrom = sc + (ccol >> 2) * L::kTile + lrow + (((2 * (ccol & 3) + l8) ^ l7) << 4);
                const uint32_t lanes = tmem + (static_cast<uint32_t>(16 * ccol) << 16);
#pragma unroll
                for (int kk = 0; kk < 4; ++kk) ldsm4t_at(f[kk], cfrom + kk * 2048);
                if (n < kChunk) {
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk)
#pragma unroll
                        for (int h = 0; h < 4; ++h) {
                            const int j = kk * 16 + (h >> 1) * 8 + 2 * q;
                            f[kk][h] &= j + 1 < n ? 0xffffffffu : (j < n ? 0xffffu : 0u);
                        }
                }
                {
                    uint64_t y[4][4];                    // two tokens' values
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk)
#pragma unroll
                        for (int h = 0; h < 4; ++h) {
                            const uint64_t w = *reinterpret_cast<const uint64_t*>(&M.w[kk * 16 + 8 * (h >> 1) + 2 * q]);
                            y[kk][h] = pack2(f[kk][h] << 16, f[kk][h] & 0xffff0000u);
                            if (!STATE_ONLY) numbers = fma2(y[kk][h], 0ull, numbers);
                            y[kk][h] = mul2(y[kk][h], w);
                        }
                    uint32_t term[4][4];
#pragma unroll
                    for (int k = 0; k < TERMS; ++k) {
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk)
#pragma unroll
                            for (int h = 0; h < 4; ++h) {
                                const float2 v = unpack2(y[kk][h]);
                                term[kk][h] = bf16x2(v.x, v.y);
                                if (k + 1 < TERMS)       // what the term leaves
                                    y[kk][h] = fma2(pack2(term[kk][h] << 16, term[kk][h] & 0xffff0000u), kMinusOnes, y[kk][h]);
                            }
                        tc_st_frag(lanes + kTerms + (L::kBuffers == 2 ? ph * 96 : 0) + 32 * k, term);
                    }
                }
                // and 16 of b
                const uint32_t to = (L::kBuffers == 2 ? ph * DK * 128 : 0) + (2 * ew + l8) * 1024 + l16 * 128 + l7 * 16;
                const uint32_t from = (ew >> 2) * L::kTile + lrow + (((2 * (ew & 3) + l8) ^ l7) << 4);
                if (ew < DK / 16) {
                    uint32_t t[4][4];
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk) ldsm4t_at(t[kk], sb + from + kk * 2048);
                    if (n < kChunk) {
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk)
#pragma unroll
                            for (int h = 0; h < 4; ++h) {
                                const int j = kk * 16 + (h >> 1) * 8 + 2 * q;
                                t[kk][h] &= j + 1 < n ? 0xffffffffu : (j < n ? 0xffffu : 0u);
                            }
                    }
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk) stsm4(base + L::kBt + to + kk * 256, t[kk][0], t[kk][1], t[kk][2], t[kk][3]);
                }
                tc_wait_st();
                tc_fence_before();
                proxy_fence();
                __syncwarp();
                if (lane == 0) mbar_arrive(&M.vk[ph]);
            }
            if constexpr (!STATE_ONLY) {
                // c^T itself goes out with P: intra of the last chunk has read its own, and the results' group what is said of it
                if (c > 0) ok = ok && __all_sync(0xffffffffu, mbar_wait(&M.oready[st ^ 1], ((c - 1) >> 1) & 1, abort));
                if (ok) {
                    tc_fence_after();
                    const float2 finite = unpack2(numbers);
                    const bool bad = __any_sync(0xffffffffu, finite.x != 0.0f || finite.y != 0.0f);
                    if (bad) {
                        int first[2] = {255, 255};
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk)
#pragma unroll
                            for (int h = 0; h < 4; ++h)
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    const uint32_t part = e ? f[kk][h] >> 16 : f[kk][h] & 0xffffu;
                                    if ((part & 0x7f80u) != 0x7f80u) continue;
                                    f[kk][h] &= e ? 0xffffu : 0xffff0000u;
                                    const int j = kk * 16 + (h >> 1) * 8 + 2 * q + e;
                                    first[h & 1] = min(first[h & 1], p.reverse ? n - 1 - j : j);
                                }
#pragma unroll
                        for (int r = 0; r < 2; ++r) {
                            first[r] = min(first[r], __shfl_xor_sync(0xffffffffu, first[r], 1));
                            first[r] = min(first[r], __shfl_xor_sync(0xffffffffu, first[r], 2));
                            if (q == 0) M.first_bad[st][16 * ccol + 8 * r + g8] = static_cast<uint8_t>(first[r]);
                        }
                    }
                    if (lane == 0) M.bad[st][ccol] = bad;
                    tc_st_frag(tmem + (static_cast<uint32_t>(16 * ccol) << 16) + kCt, f);
                }
                // (2) rows i = 16 sub + g and + 8, columns j = 32 half + 8 nt + 2 q and + 1: v[4 nt ..]
                ok = ok && __all_sync(0xffffffffu, mbar_wait(&M.pready, ph, abort));
                if (ok) {
                    tc_fence_after();
                    uint32_t v[16];
                    tc_ld_frag(tmem + (static_cast<uint32_t>(32 * sub) << 16) + kP + 32 * half, v);
                    tc_wait_ld16(v);
                    const int i = 16 * sub + g8, j0 = 32 * half + 2 * q;
                    const float* lag = &M.lag[63 + i - j0];
                    // token j of column e from here counts for token i if before < e <= upto
                    const int d = i - j0, before = p.reverse ? d - 1 : -1000, upto = p.reverse ? n - 1 - j0 : d;
                    uint32_t r[8];
#pragma unroll
                    for (int nt = 0; nt < 4; ++nt)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int e = 8 * nt - 8 * h;                // against row i + 8 h
                            // in reverse the tokens past the sequence's end come before: they are masked by upto
                            const bool s0 = e > before && (p.reverse ? 8 * nt : e) <= upto;
                            const bool s1 = e + 1 > before && (p.reverse ? 8 * nt + 1 : e + 1) <= upto;
                            r[2 * nt + h] = bf16x2(s0 ? __uint_as_float(v[4 * nt + 2 * h]) * lag[-e] : 0.0f,
                                                   s1 ? __uint_as_float(v[4 * nt + 2 * h + 1]) * lag[-e - 1] : 0.0f);
                        }
                    // matrices (rows 0-7, 8-15) x (columns 8 nt, 8 nt + 8)
                    const uint32_t at = base + L::kProb + (2 * sub + l8) * 1024 + (4 * half + l16) * 128 + l7 * 16;
                    stsm4(at, r[0], r[1], r[2], r[3]);
                    stsm4(at + 256, r[4], r[5], r[6], r[7]);
                    tc_wait_st();
                    tc_fence_before();
                    proxy_fence();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&M.psm);
                }
            }
        }
        if (!ok && lane == 0) fail();
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 120;");
        const int ew = warp - 4 - kTcGroup, sub = warp & 3, half = ew >> 2;   // TMEM lanes 32 sub ..; half of their columns
        const uint32_t lanes = tmem + (static_cast<uint32_t>(32 * sub) << 16);
        const int row = tile * kTcCols + 32 * sub + lane;             // column of c
        const int64_t sh = (static_cast<int64_t>(u.seq) * p.heads + head) * db * dc;
        const int64_t gh = (static_cast<int64_t>(unit) * p.heads + head) * db * dc;
        constexpr int kX = DK / 2;
        const int x0 = half * kX;                                     // first row of b's dimension of this thread
        uint64_t x[kX / 2];                                           // pairs
        {
            // the state that enters: sixteen elements' loads at a time (one after the other they took 18,000 cycles)
            const float* from = STATE_ONLY ? nullptr : (p.seg ? p.seg + gh + x0 * p.g_i + row * p.g_j : (p.s_in ? p.s_in + sh + x0 * p.s_i + row * p.s_j : nullptr));
            const int64_t si = p.seg ? p.g_i : p.s_i;
            const float mul = p.seg ? 1.0f : p.in_mul;
            const int rows = from != nullptr && row < dc ? db - x0 : 0;       // elements there are
#pragma unroll
            for (int i0 = 0; i0 < kX; i0 += 16) {
                float v[16];
                if (si == 1 && rows >= i0 + 16 && (reinterpret_cast<uintptr_t>(from) & 15) == 0) {
#pragma unroll
                    for (int i = 0; i < 16; i += 4) *reinterpret_cast<float4*>(v + i) = *reinterpret_cast<const float4*>(from + i0 + i);
                } else if (rows >= i0 + 16) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) v[i] = from[(i0 + i) * si];
                } else {
#pragma unroll
                    for (int i = 0; i < 16; ++i) v[i] = i0 + i < rows ? from[(i0 + i) * si] : 0.0f;
                }
#pragma unroll
                for (int i = 0; i < 16; i += 2) x[(i0 + i) / 2] = pack2(__float_as_uint(v[i] * mul), __float_as_uint(v[i + 1] * mul));
            }
        }
        // the bf16 copy of this thread's part of the state; U has been read
        auto copy_state = [&]() {
            if constexpr (!STATE_ONLY) {
#pragma unroll
                for (int i = 0; i < kX; i += 32) {
                    uint32_t v[16];
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        const float2 y = unpack2(x[i / 2 + k]);
                        v[k] = bf16x2(y.x, y.y);
                    }
                    tc_st16(lanes + kX16 + (x0 + i) / 2, v);
                }
                tc_wait_st();
                tc_fence_before();
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&M.x16);
        };
        if (chunks > 0) copy_state();
        bool ok = true;
        for (int c = 0; c < chunks; ++c) {
            const int st = c & 1, n = tokens(c);
            const uint32_t ph = c & 1;
            // (3) the state
            ok = ok && __all_sync(0xffffffffu, mbar_wait(&M.uready[ph], (c >> 1) & 1, abort));
            const int last = c > 0 && n < kChunk;
            if (ok) {
                tc_fence_after();
                const uint32_t whole = __float_as_uint(M.whole[last]);
                const uint64_t whole2 = pack2(whole, whole);
#pragma unroll
                for (int i0 = 0; i0 < kX; i0 += 16) {
                    uint32_t v[16];
                    tc_ld16(lanes + kU + x0 + i0, v);
                    tc_wait_ld16(v);
#pragma unroll
                    for (int i = 0; i < 16; i += 2) x[(i0 + i) / 2] = fma2(whole2, x[(i0 + i) / 2], pack2(v[i], v[i + 1]));
                }
                tc_fence_before();
                if (c + 1 < chunks) {
                    if (!STATE_ONLY) ok = __all_sync(0xffffffffu, mbar_wait(&M.iready, ph, abort));   // inter has read the last copy
                    tc_fence_after();
                    if (ok) copy_state();
                }
            }
            if constexpr (!STATE_ONLY) {
                // (4) the results: 32 tokens of this lane's column
                ok = ok && __all_sync(0xffffffffu, mbar_wait(&M.oready[st], (c >> 1) & 1, abort));
                if (ok) {
                    tc_fence_after();
                    const bool bad = (M.bad[st][2 * sub] | M.bad[st][2 * sub + 1]) != 0;
                    const int64_t at = (u.row0 + first(c) + 32 * half) * p.o_tok + static_cast<int64_t>(u.seq) * p.o_seq + head * p.o_head;
                    const int m = n - 32 * half;             // tokens of this half
                    // results pass through shared memory of this warp's own, bf16 ones two tokens a word
                    unsigned char* own = smem + L::kOut + ew * 4096;
#pragma unroll
                    for (int t0 = 0; t0 < 32; t0 += 16) {
                        uint32_t a[16], b[16];
                        tc_ld16(lanes + kIntra + 32 * half + t0, a);
                        tc_ld16(lanes + kInter + 32 * half + t0, b);
                        tc_wait_ld16(a);
                        tc_wait_ld16(b);
#pragma unroll
                        for (int t = 0; t < 16; t += 4) {
                            const ulonglong2 w = *reinterpret_cast<const ulonglong2*>(&M.out[last][32 * half + t0 + t]);
                            const float2 lo = unpack2(fma2(w.x, pack2(b[t], b[t + 1]), pack2(a[t], a[t + 1])));
                            const float2 hi = unpack2(fma2(w.y, pack2(b[t + 2], b[t + 3]), pack2(a[t + 2], a[t + 3])));
                            a[t] = __float_as_uint(lo.x), a[t + 1] = __float_as_uint(lo.y);
                            a[t + 2] = __float_as_uint(hi.x), a[t + 3] = __float_as_uint(hi.y);
                        }
                        if (bad && M.bad[st][2 * sub + (lane >> 4)]) {
                            const int from = M.first_bad[st][32 * sub + lane];
#pragma unroll
                            for (int t = 0; t < 16; ++t) {
                                const int i = 32 * half + t0 + t;
                                if ((p.reverse ? n - 1 - i : i) >= from) a[t] = 0x7fffffffu;
                            }
                        }
                        if constexpr (F32) {
#pragma unroll
                            for (int t = 0; t < 16; ++t) *reinterpret_cast<uint32_t*>(own + (t0 + t) * 128 + lane * 4) = a[t];
                        } else {
#pragma unroll
                            for (int t = 0; t < 16; t += 2)
                                *reinterpret_cast<uint32_t*>(own + (t0 + t) * 64 + lane * 4) = bf16x2(__uint_as_float(a[t]), __uint_as_float(a[t + 1]));
                        }
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&M.odone);    // read: the next chunk's may come
                    const int j4 = tile * kTcCols + 32 * sub + 4 * (lane & 7);
                    if constexpr (F32) {
                        // four tokens at a time, 128 bytes each (a store a token straight from the registers: a scan of 106 us takes 78 so)
                        float* to = static_cast<float*>(p.o) + at + (lane >> 3) * p.o_tok + j4;
#pragma unroll
                        for (int t = lane >> 3; t < 32; t += 4, to += 4 * p.o_tok) {
                            const float4 r = *reinterpret_cast<const float4*>(own + t * 128 + (lane & 7) * 16);
                            if (t >= m || j4 >= dc) continue;
                            if (p.o_vec) {
                                *reinterpret_cast<float4*>(to) = r;
                            } else {
                                to[0] = r.x;
                                if (j4 + 1 < dc) to[1] = r.y;
                                if (j4 + 2 < dc) to[2] = r.z;
                                if (j4 + 3 < dc) to[3] = r.w;
                            }
                        }
                        __syncwarp();
                    } else {
                        // out of there as four columns of two tokens a lane: 64 bytes a token
                        const int t8 = 2 * (lane >> 3);
                        __nv_bfloat16* to = static_cast<__nv_bfloat16*>(p.o) + at + t8 * p.o_tok + j4;
#pragma unroll
                        for (int k = 0; k < 4; ++k, to += 8 * p.o_tok) {
                            const uint4 r = *reinterpret_cast<const uint4*>(own + (4 * k + (lane >> 3)) * 128 + (lane & 7) * 16);
                            const uint2 even = make_uint2(__byte_perm(r.x, r.y, 0x5410), __byte_perm(r.z, r.w, 0x5410));
                            const uint2 odd = make_uint2(__byte_perm(r.x, r.y, 0x7632), __byte_perm(r.z, r.w, 0x7632));
                            const int left = m - 8 * k - t8;
                            if (j4 >= dc) continue;
                            if (p.o_vec) {
                                if (left > 0) *reinterpret_cast<uint2*>(to) = even;
                                if (left > 1) *reinterpret_cast<uint2*>(to + p.o_tok) = odd;
                            } else {
                                const __nv_bfloat16 *e0 = reinterpret_cast<const __nv_bfloat16*>(&even), *e1 = reinterpret_cast<const __nv_bfloat16*>(&odd);
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    if (j4 + e >= dc) continue;
                                    if (left > 0) to[e] = e0[e];
                                    if (left > 1) to[p.o_tok + e] = e1[e];
                                }
                            }
                        }
                        __syncwarp();
                    }
                }
            }
        }
        float* to = STATE_ONLY ? p.seg : (u.last && p.seg == nullptr ? p.s_out : nullptr);
        if (to != nullptr && row < dc && ok) {
            const int64_t si = STATE_ONLY ? p.g_i : p.s_i;
            const float mul = STATE_ONLY ? 1.0f : p.end_mul;
            to += STATE_ONLY ? gh + x0 * p.g_i + row * p.g_j : sh + x0 * p.s_i + row * p.s_j;
#pragma unroll
            for (int i = 0; i < kX; i += 2, to += 2 * si) {
                const float2 y = unpack2(x[i / 2]);
                if (x0 + i < db) to[0] = y.x * mul;
                if (x0 + i + 1 < db) to[si] = y.y * mul;
            }
        }
        if (!ok && lane == 0) fail();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

// ---------------------------------------------------------- segment states
//
// The segments' own end states (from zero) become the states that enter
// them: X_{g+1} = lam^len(g) X_g + E_g with X_0 the given state; the state
// after the last segment is the final one.  One thread an element (two at
// once where they lie in pairs), the loads of four segments in flight; a
// segment's state is read and written once.
template <int V>
__global__ void __launch_bounds__(128) scan_join_kernel(const __grid_constant__ ScanArgs p) {
    __shared__ float power[2];
    const int64_t n = static_cast<int64_t>(p.b.d) * p.c.d;
    const int head = blockIdx.y % p.heads, seq = blockIdx.y / p.heads;
    int64_t len = p.tokens, first;
    if (p.cu == nullptr) {
        first = static_cast<int64_t>(seq) * (p.tokens > 0 ? (p.tokens + p.seg_len - 1) / p.seg_len : 1);
    } else {
        const int64_t a = clamp_start(p, seq), b = clamp_start(p, seq + 1);
        len = b > a ? b - a : 0;
        first = a / p.seg_len + seq;
    }
    const int64_t segs = (len + p.seg_len - 1) / p.seg_len;
    if (threadIdx.x == 0) power[0] = decay_power(p.log_decay[head], p.seg_len);
    if (threadIdx.x == 32) power[1] = decay_power(p.log_decay[head], len - (segs - 1) * p.seg_len);
    __syncthreads();
    let_next();
    previous_done();
    const int64_t e = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) * V;
    if (e >= n) return;
    const int64_t sh = (static_cast<int64_t>(seq) * p.heads + head) * n;
    float x[V];
    int64_t at_state[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int64_t i = (e + v) / p.c.d, j = e + v - i * p.c.d;
        at_state[v] = sh + i * p.s_i + j * p.s_j;
        x[v] = p.s_in ? p.s_in[at_state[v]] * p.in_mul : 0.0f;
    }
    const int64_t step = static_cast<int64_t>(p.heads) * n;
    float* at = p.seg + (first * p.heads + head) * n + e;
    for (int64_t g = 0; g < segs; g += 4) {
        float own[4][V];
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int v = 0; v < V; ++v) own[k][v] = 0.0f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (g + k >= segs) break;
            if constexpr (V == 2) *reinterpret_cast<float2*>(own[k]) = *reinterpret_cast<const float2*>(at + k * step);
            else own[k][0] = at[k * step];
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (g + k >= segs) break;
            if constexpr (V == 2) *reinterpret_cast<float2*>(at + k * step) = make_float2(x[0], x[1]);
            else at[k * step] = x[0];
            const float w = power[g + k == segs - 1];
#pragma unroll
            for (int v = 0; v < V; ++v) x[v] = fmaf(w, x[v], own[k][v]);
        }
        at += 4 * step;
    }
    if (p.s_out)
#pragma unroll
        for (int v = 0; v < V; ++v) p.s_out[at_state[v]] = x[v] * p.end_mul;
}

// Sums the partial gradients of `share` heads that read one key or value
// head, in the heads' order: out[token][kv][d] = sum_h part[token][kv*share + h][d].
// V elements a thread, bound by HBM: 4 share bytes in and one result out an
// element.
template <typename T, int V>
__global__ void __launch_bounds__(256) sum_heads_kernel(const float* part, uint32_t tokens, uint32_t kv, uint32_t share, uint32_t d, T* out,
                                                        int64_t o_seq, int64_t o_tok, int64_t o_head, uint32_t per_seq) {
    const uint32_t vecs = d / V, row = kv * vecs;
    const uint32_t t = blockIdx.x * blockDim.y + threadIdx.y;
    let_next();
    previous_done();
    if (t >= tokens) return;
    const float* from = part + static_cast<int64_t>(t) * kv * share * d;
    const uint32_t s = t / per_seq;
    T* to = out + s * o_seq + (t - s * per_seq) * o_tok;
    for (uint32_t e = threadIdx.x; e < row; e += blockDim.x) {
        const uint32_t h = e / vecs, i = (e - h * vecs) * V;
        const float* at = from + static_cast<int64_t>(h) * share * d + i;
        float x[V];
#pragma unroll
        for (int k = 0; k < V; ++k) x[k] = 0.0f;
        for (uint32_t g = 0; g < share; ++g, at += d) {
            if constexpr (V == 8) {
                const float4 a = *reinterpret_cast<const float4*>(at), b = *reinterpret_cast<const float4*>(at + 4);
                x[0] += a.x, x[1] += a.y, x[2] += a.z, x[3] += a.w;
                x[4] += b.x, x[5] += b.y, x[6] += b.z, x[7] += b.w;
            } else {
                x[0] += at[0];
            }
        }
        if constexpr (V == 8) store8(to + h * o_head + i, x, 8, true);
        else to[h * o_head + i] = from_f32<T>(x[0]);
    }
}

// Always after the scan that made the parts.
template <typename T>
cudaError_t sum_heads(const float* part, int64_t tokens, int kv, int share, int d, void* out, const int64_t* st, int64_t per_seq, cudaStream_t s) {
    const int64_t n = 16 / static_cast<int64_t>(sizeof(T));
    const bool vec = d % 8 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0 && st[0] % n == 0 && st[1] % n == 0 && st[2] % n == 0;
    const unsigned row = static_cast<unsigned>(kv * d / (vec ? 8 : 1));
    const dim3 block(row >= 256 ? 256 : (row > 128 ? 256 : (row > 64 ? 128 : (row > 32 ? 64 : 32))), 1);
    const dim3 threads(block.x, 256 / block.x);
    const unsigned blocks = static_cast<unsigned>((tokens + threads.y - 1) / threads.y);
    if (vec)
        return launch_chained(sum_heads_kernel<T, 8>, blocks, threads, 0, s, true, part, static_cast<uint32_t>(tokens), kv, share, d, static_cast<T*>(out),
                              st[0], st[1], st[2], static_cast<uint32_t>(per_seq));
    return launch_chained(sum_heads_kernel<T, 1>, blocks, threads, 0, s, true, part, static_cast<uint32_t>(tokens), kv, share, d, static_cast<T*>(out), st[0],
                          st[1], st[2], static_cast<uint32_t>(per_seq));
}

// -------------------------------------------------------------- one token
//
// One token for each sequence: the state is read, updated and written once,
// 8 bytes an element, which is all that counts.  A block has 32 columns of
// one state (8 lanes of float4 a row, 32 rows at a time): every load of a
// thread is in flight at once and small batches still spread over the GPU.
// Bound by HBM: 192 sequences of 16 heads of 128 x 128 (405 MB) in 78 us, 79%
// of the measured copy; with lam after the loads, where it would seem hidden,
// 91.  One sequence is a launch's latency.
constexpr int kStepThreads = 256;

struct StepArgs {
    const void *q, *k, *v;
    void* o;
    int64_t q_seq, q_head, k_seq, k_head, v_seq, v_head, o_seq, o_head;
    float* state;
    int64_t s_slot;                // elements from slot to slot
    const int32_t* slots;          // [seqs] or null
    int32_t n_slots;
    int32_t heads, share, dk, dv;
    const float* log_decay;
    float scale;
};

template <typename T, int V>
__global__ void __launch_bounds__(kStepThreads) step_kernel(const __grid_constant__ StepArgs p) {
    __shared__ float part[8][8 * V];
    const int tiles = (p.dv + 8 * V - 1) / (8 * V);
    const int tile = blockIdx.x % tiles;
    const int head = (blockIdx.x / tiles) % p.heads;
    const int seq = blockIdx.x / tiles / p.heads;
    const int slot = p.slots ? p.slots[seq] : seq;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int cl = (threadIdx.x & 7) * V, col = tile * 8 * V + cl, r0 = threadIdx.x >> 3;
    T* o = static_cast<T*>(p.o) + seq * p.o_seq + head * p.o_head;
    if (slot < 0 || slot >= p.n_slots) {
        // a negative slot is padding; one past the cache is a caller's error that must not go unseen
        if (threadIdx.x < 8 * V && tile * 8 * V + static_cast<int>(threadIdx.x) < p.dv)
            o[tile * 8 * V + threadIdx.x] = from_f32<T>(slot < 0 ? 0.0f : __int_as_float(0x7fc00000));
        return;
    }
    const T* q = static_cast<const T*>(p.q) + seq * p.q_seq + head * p.q_head;
    const T* k = static_cast<const T*>(p.k) + seq * p.k_seq + (head / p.share) * p.k_head;
    const T* v = static_cast<const T*>(p.v) + seq * p.v_seq + (head / p.share) * p.v_head;
    float* s = p.state + slot * p.s_slot + static_cast<int64_t>(head) * p.dk * p.dv;
    // lam to 48 bits: a long run of steps applies it thousands of times
    const double whole = exp(static_cast<double>(p.log_decay[head]));
    const float lam = static_cast<float>(whole), lam_lo = static_cast<float>(whole - lam);
    const bool in = col < p.dv;
    float vv[V], acc[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        vv[e] = in ? to_f32(v[col + e]) : 0.0f;
        acc[e] = 0.0f;
    }
#pragma unroll
    for (int g = 0; g < kMaxDim / 32; g += 4) {
        if (32 * g >= p.dk) break;
        float x[4][V];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = r0 + 32 * (g + i);
            if (in && r < p.dk) {
                if constexpr (V == 4) {
                    const float4 y = *reinterpret_cast<const float4*>(s + static_cast<int64_t>(r) * p.dv + col);
                    x[i][0] = y.x, x[i][1] = y.y, x[i][2] = y.z, x[i][3] = y.w;
                } else {
                    x[i][0] = s[static_cast<int64_t>(r) * p.dv + col];
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = r0 + 32 * (g + i);
            if (in && r < p.dk) {
                const float kk = to_f32(k[r]), qq = to_f32(q[r]);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    x[i][e] = fmaf(lam, x[i][e], fmaf(lam_lo, x[i][e], kk * vv[e]));
                    acc[e] = fmaf(qq, x[i][e], acc[e]);
                }
                if constexpr (V == 4)
                    *reinterpret_cast<float4*>(s + static_cast<int64_t>(r) * p.dv + col) =
                        make_float4(x[i][0], x[i][1], x[i][2], x[i][3]);
                else
                    s[static_cast<int64_t>(r) * p.dv + col] = x[i][0];
            }
        }
    }
#pragma unroll
    for (int e = 0; e < V; ++e) {
        acc[e] += __shfl_xor_sync(0xffffffffu, acc[e], 8);
        acc[e] += __shfl_xor_sync(0xffffffffu, acc[e], 16);
        if (lane < 8) part[warp][cl + e] = acc[e];
    }
    __syncthreads();
    if (threadIdx.x < 8 * V) {
        const int j = tile * 8 * V + threadIdx.x;
        float x = 0.0f;
#pragma unroll
        for (int w = 0; w < 8; ++w) x += part[w][threadIdx.x];
        if (j < p.dv) o[j] = from_f32<T>(x * p.scale);
    }
}

// ---------------------------------------------------------------- launches

template <typename T>
cudaError_t launch_serial(const ScanArgs& p, bool state_only, cudaStream_t s) {
    const int64_t blocks = static_cast<int64_t>(p.units) * p.heads * ((p.c.d + kSerialCols - 1) / kSerialCols);
    const unsigned g = static_cast<unsigned>(blocks);
    if (p.b.d <= 64) scan_serial_kernel<T, 2><<<g, kSerialThreads, 0, s>>>(p, state_only);
    else if (p.b.d <= 128) scan_serial_kernel<T, 4><<<g, kSerialThreads, 0, s>>>(p, state_only);
    else scan_serial_kernel<T, 8><<<g, kSerialThreads, 0, s>>>(p, state_only);
    return cudaGetLastError();
}

template <int DK, int CH, int TERMS, bool STATE_ONLY>
cudaError_t launch_mma(const ScanArgs& p, cudaStream_t s) {
    const int64_t blocks = static_cast<int64_t>(p.units) * p.heads * ((p.c.d + kMmaCols - 1) / kMmaCols);
    constexpr int bytes = sizeof(MmaSmem<DK, CH>);
    const cudaError_t e = allow_shared<scan_mma_kernel<DK, CH, TERMS, STATE_ONLY>>(bytes);
    if (e != cudaSuccess) return e;
    scan_mma_kernel<DK, CH, TERMS, STATE_ONLY><<<static_cast<unsigned>(blocks), kMmaThreads, bytes, s>>>(p);
    return cudaGetLastError();
}

template <int DK>
cudaError_t launch_mma_any(const ScanArgs& p, bool state_only, cudaStream_t s) {
    if (state_only) return launch_mma<DK, kMmaChunk, 3, true>(p, s);
    // the final state comes out of this scan only where sequences are whole
    return p.seg == nullptr && p.s_out != nullptr ? launch_mma<DK, kMmaChunk, 3, false>(p, s) : launch_mma<DK, kMmaChunk, 2, false>(p, s);
}

// Tensor map of one operand: d, head, token, sequence; boxes of 64 elements of 64 tokens.
bool make_scan_map(const Strided& m, const ScanArgs& p, CUtensorMap* map) {
    const TensorMapEncode fn = tensor_map_encode();
    if (!fn) return false;
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(m.d), static_cast<cuuint64_t>(p.heads / m.share), static_cast<cuuint64_t>(p.tokens),
                                static_cast<cuuint64_t>(p.cu ? 1 : p.seqs)};
    // the stride of a dimension of one says nothing, and may be anything
    const cuuint64_t strides[3] = {dims[1] > 1 ? static_cast<cuuint64_t>(m.head) * 2 : 16, dims[2] > 1 ? static_cast<cuuint64_t>(m.tok) * 2 : 16,
                                   dims[3] > 1 ? static_cast<cuuint64_t>(m.seq) * 2 : 16};
    const cuuint32_t box[4] = {64, 1, kChunk, 1}, one[4] = {1, 1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(m.p), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DK, int TERMS, bool STATE_ONLY, bool F32>
cudaError_t launch_tc(const ScanArgs& p, const CUtensorMap* maps, bool after, cudaStream_t s) {
    const int64_t blocks = static_cast<int64_t>(p.units) * p.heads * ((p.c.d + kTcCols - 1) / kTcCols);
    constexpr int bytes = TcSmem<DK, TERMS, STATE_ONLY>::kBytes;
    const cudaError_t e = allow_shared<scan_tc_kernel<DK, TERMS, STATE_ONLY, F32>>(bytes);
    if (e != cudaSuccess) return e;
    return launch_chained(scan_tc_kernel<DK, TERMS, STATE_ONLY, F32>, dim3(static_cast<unsigned>(blocks)), dim3(kTcThreads), bytes, s, after, maps[0], maps[1],
                          maps[2], p);
}

template <int DK>
cudaError_t launch_tc_any(const ScanArgs& p, const CUtensorMap* maps, bool state_only, bool after, cudaStream_t s) {
    if (state_only) return launch_tc<DK, 3, true, false>(p, maps, after, s);
    const bool whole = p.seg == nullptr && p.s_out != nullptr;
    if (p.o_f32) return whole ? launch_tc<DK, 3, false, true>(p, maps, after, s) : launch_tc<DK, 2, false, true>(p, maps, after, s);
    return whole ? launch_tc<DK, 3, false, false>(p, maps, after, s) : launch_tc<DK, 2, false, false>(p, maps, after, s);
}

// Which kernel a scan runs on.
enum class Scan { kTensor, kMma, kSerial };
Scan scan_of(int dtype, int bd, bool vec, int64_t tokens) {
    if (dtype != NRN_BF16 || bd > 128) return Scan::kSerial;
    return vec && tokens > 0 && tokens < (int64_t(1) << 31) - kChunk ? Scan::kTensor : Scan::kMma;
}

// after: a kernel of the same call comes before it
cudaError_t launch_scan(const ScanArgs& p, int dtype, bool state_only, bool after, cudaStream_t s) {
    const Scan scan = scan_of(dtype, p.b.d, p.vec != 0, p.tokens);
    if (scan == Scan::kTensor) {
        CUtensorMap maps[3];
        if (make_scan_map(p.a, p, &maps[0]) && make_scan_map(p.b, p, &maps[1]) && make_scan_map(p.c, p, &maps[2]))
            return p.b.d <= 64 ? launch_tc_any<64>(p, maps, state_only, after, s) : launch_tc_any<128>(p, maps, state_only, after, s);
    }
    if (scan != Scan::kSerial) return p.b.d <= 64 ? launch_mma_any<64>(p, state_only, s) : launch_mma_any<128>(p, state_only, s);
    if (dtype == NRN_BF16) return launch_serial<__nv_bfloat16>(p, state_only, s);
    if (dtype == NRN_FP16) return launch_serial<__half>(p, state_only, s);
    return launch_serial<float>(p, state_only, s);
}

int elem_size(int dtype) { return dtype == NRN_FP32 ? 4 : 2; }

// Tokens of a segment.  A scan is serial in time, so its parallelism is
// sequences x heads x tiles of columns; where that leaves SMs idle, or a last
// round of blocks nearly empty, the sequences are split.  Splitting costs a
// pass over b and c for the segments' states and the join, so the least time
// is looked for, by a model of microseconds measured for each kernel.  Packed
// sequences' lengths are not known here: their segments are counted as if half
// of them were cut short, and whole ones as if the longest were twice the mean.
//
// scan_tc_kernel, one block an SM (d 128): 2.0 a chunk of 64 tokens and 5 a
// block, 0.9 and 4 for the states, 4 for the join and its bytes.
int64_t tensor_segment(const nrn_linattn_t* a, int dc) {
    const int64_t rows = static_cast<int64_t>(a->heads) * ((dc + kTcCols - 1) / kTcCols), sms = sm_count();
    const bool packed = a->cu_seqlens != nullptr;
    const int64_t chunks = (a->tokens + kChunk - 1) / kChunk;              // of each sequence, or of all packed ones
    if (chunks <= 1) return kChunk;
    const auto rounds = [&](double blocks) {
        const double r = blocks / static_cast<double>(sms);
        return packed ? std::max(1.0, r + 0.5) : std::ceil(r);
    };
    int64_t best = 0;
    double cost = 1e300;
    for (int64_t k = 1; k <= std::min<int64_t>(chunks, 4 * sms); ++k) {     // segments of a sequence, or of all
        const int64_t s = (chunks + k - 1) / k;
        const double units = packed ? static_cast<double>(chunks) / s + 0.5 * a->seqs
                                    : static_cast<double>(a->seqs) * ((chunks + s - 1) / s);
        const double r = rounds(units * rows);
        double t = r * (2.0 * s + 5.0);
        // packed sequences that are whole: the longest is about twice the mean
        if (packed && k == 1) t = std::max(rounds(static_cast<double>(a->seqs) * rows) * (2.0 * chunks / std::max(1, a->seqs) + 5.0),
                                           2.0 * std::min<double>(chunks, 2.0 * chunks / std::max(1, a->seqs)) + 5.0);
        else if (k > 1) t += r * (0.9 * s + 4.0) + 4.0 + units * rows * a->dk * static_cast<double>(std::min(dc, kTcCols)) * 8.0 / 3e6;
        if (t < cost) {
            cost = t;
            best = s;
        }
        if (units * rows > 4.0 * sms) break;
    }
    return best * kChunk;
}

// The others have several blocks on an SM: the first costs `main` a chunk of
// 64 tokens, each further one `more`, and likewise for the states (one head's
// 16,384 tokens, and 64 sequences of 1,024 tokens of 16 heads; fp32 and fp16
// alike).  Whole and split: 4 x 2,048 fp32 tokens of 16 heads of 128 take 1.65
// ms whole, 1.96 to 2.94 split; 65,536 fp16 tokens of 8 heads of 64 take 32 ms
// whole, 3.4 in 18 segments, 2.2 in 64.
struct ScanCost {
    int cols;
    double main, more, state, state_more;
};
ScanCost cost_of(Scan scan, int bd) {
    if (scan == Scan::kMma) return bd <= 64 ? ScanCost{kMmaCols, 3.7, 2.8, 1.6, 1.4} : ScanCost{kMmaCols, 5.5, 3.9, 2.7, 2.7};
    if (bd <= 64) return {kSerialCols, 24.0, 12.0, 14.0, 7.0};
    return bd <= 128 ? ScanCost{kSerialCols, 33.0, 19.0, 22.0, 13.5} : ScanCost{kSerialCols, 56.0, 30.0, 41.0, 24.0};
}

// passes: of states to scans (in a backward pass two of three, the values' and
// the keys' scan have one).
int64_t segment_length(const nrn_linattn_t* a, int bd, int dc, Scan scan, double passes) {
    if (scan == Scan::kTensor) return tensor_segment(a, dc);
    const ScanCost c = cost_of(scan, bd);
    const double rows = static_cast<double>(a->heads) * ((dc + c.cols - 1) / c.cols), sms = std::max(1, sm_count());
    const bool packed = a->cu_seqlens != nullptr;
    const int64_t chunks = (a->tokens + kChunk - 1) / kChunk;
    if (chunks <= 1) return kChunk;
    int64_t best = chunks;
    double cost = 1e300;
    for (int64_t k = 1; k <= chunks; k += k < 8 ? 1 : k / 4) {
        const int64_t s = (chunks + k - 1) / k;
        const double mean = packed && k == 1 ? static_cast<double>(chunks) / std::max(1, a->seqs) : static_cast<double>(s);
        const double units = !packed ? static_cast<double>(a->seqs) * ((chunks + s - 1) / s)
                                     : (k == 1 ? static_cast<double>(a->seqs) : static_cast<double>(chunks) / s + 0.5 * a->seqs);
        const double further = std::max(0.0, units * rows / sms - 1.0);          // blocks an SM past the first
        double t = mean * (c.main + c.more * further) + 5.0;
        if (packed && k == 1) t = std::max(t, std::min<double>(static_cast<double>(chunks), 2.0 * mean) * c.main + 5.0);
        if (k > 1) t += passes * (mean * (c.state + c.state_more * further) + 8.0 + units * a->heads * a->dk * a->dv * 8.0 / 3e6);
        if (t < cost) {
            cost = t;
            best = s;
        }
        if (units * rows > 16.0 * sms) break;
    }
    return best * kChunk;
}

int64_t unit_count(const nrn_linattn_t* a, int64_t seg_len) {
    if (a->cu_seqlens) return a->tokens / seg_len + a->seqs;
    return a->seqs * std::max<int64_t>(1, (a->tokens + seg_len - 1) / seg_len);
}

bool is_split(const nrn_linattn_t* a, int64_t seg_len) {
    return a->cu_seqlens ? a->tokens > seg_len : a->tokens > seg_len;
}

int64_t align256(int64_t x) { return (x + 255) / 256 * 256; }

int64_t all_tokens(const nrn_linattn_t* a) { return a->cu_seqlens ? a->tokens : a->tokens * a->seqs; }

// Segments of the scans whose b has the keys' dimension (the forward one and
// the values') and of those whose b has the values' (the queries' and keys').
struct Segments {
    int64_t by_k = 0, by_v = 0;        // tokens

    Segments(const nrn_linattn_t* a, bool vec, bool backward) {
        const Scan k = scan_of(a->dtype, a->dk, vec, a->tokens), v = scan_of(a->dtype, a->dv, vec, a->tokens);
        const double passes = backward ? 2.0 / 3.0 : 1.0;
        by_k = segment_length(a, a->dk, a->dv, k, passes);
        by_v = !backward || (k == v && a->dk == a->dv) ? by_k : segment_length(a, a->dv, a->dk, v, passes);
    }
    // of the segments' states
    int64_t bytes(const nrn_linattn_t* a) const {
        int64_t most = 0;
        for (int64_t l : {by_k, by_v})
            if (is_split(a, l)) most = std::max(most, unit_count(a, l));
        return align256(most * a->heads * a->dk * a->dv * 4);
    }
};

// of the fp32 parts of shared heads
int64_t part_bytes(const nrn_linattn_t* a) {
    return a->kv_heads == a->heads ? 0 : align256(all_tokens(a) * a->heads * std::max(a->dk, a->dv) * 4);
}

nrn_status_t run_scan(ScanArgs p, const nrn_linattn_t* a, bool after, cudaStream_t s) {
    const int per16 = 16 / elem_size(a->dtype);
    p.o_vec = reinterpret_cast<uintptr_t>(p.o) % 16 == 0 && p.o_seq % per16 == 0 && p.o_tok % per16 == 0 && p.o_head % per16 == 0 && p.c.d % per16 == 0;
    if (p.cu) p.a.seq = p.b.seq = p.c.seq = p.o_seq = 0;      // packed: a token's row counts from the arrays' start
    const int64_t units = unit_count(a, p.seg_len);
    NRN_CHECK_ARG(units * p.heads * ((p.c.d + 31) / 32) < (int64_t(1) << 31), "nrn_cuda_linattn: too many sequences, heads and segments for one launch");
    NRN_CHECK_ARG(static_cast<int64_t>(p.seqs) * p.heads < 65536 || !is_split(a, p.seg_len),
                  "nrn_cuda_linattn: at most 65,535 sequences times heads when sequences are split");
    p.units = static_cast<int32_t>(units);
    p.seg = is_split(a, p.seg_len) ? static_cast<float*>(a->workspace) : nullptr;
    if (!p.seg_made) p.g_i = p.c.d, p.g_j = 1;
    if (p.seg != nullptr && !p.seg_made) {
        NRN_CUDA_TRY(launch_scan(p, a->dtype, true, after, s));
        const int64_t n = static_cast<int64_t>(p.b.d) * p.c.d;
        const int v = n % 2 == 0 ? 2 : 1;      // every state starts on an even element then
        const dim3 grid(static_cast<unsigned>((n / v + 127) / 128), static_cast<unsigned>(p.seqs * p.heads));
        NRN_CUDA_TRY(launch_chained(v == 2 ? scan_join_kernel<2> : scan_join_kernel<1>, grid, dim3(128), 0, s, true, p));
        after = true;
    }
    NRN_CUDA_TRY(launch_scan(p, a->dtype, false, after, s));
    return NRN_OK;
}

Strided strided(const void* p, const int64_t* st, int share, int d) {
    Strided r;
    r.p = p;
    r.seq = st[0], r.tok = st[1], r.head = st[2];
    r.share = share;
    r.d = d;
    return r;
}

bool rows_aligned(const Strided& m, int dtype) {
    const int64_t n = 16 / elem_size(dtype);
    return reinterpret_cast<uintptr_t>(m.p) % 16 == 0 && m.seq % n == 0 && m.tok % n == 0 && m.head % n == 0 && m.d % n == 0;
}

nrn_status_t check_common(const nrn_linattn_t* a, const char* who) {
    const std::string w(who);
    NRN_CHECK_ARG(a != nullptr, w + ": null arguments");
    NRN_CHECK_ARG(a->dtype == NRN_BF16 || a->dtype == NRN_FP16 || a->dtype == NRN_FP32, w + ": unknown type");
    NRN_CHECK_ARG(a->seqs >= 0 && a->tokens >= 0, w + ": negative sizes");
    NRN_CHECK_ARG(a->tokens < (int64_t(1) << 31) && (a->cu_seqlens || a->tokens * a->seqs < (int64_t(1) << 31)), w + ": at most 2^31 - 1 tokens");
    NRN_CHECK_ARG(a->heads >= 1 && a->kv_heads >= 1 && a->heads % a->kv_heads == 0,
                  w + ": heads must be a multiple of kv_heads");
    NRN_CHECK_ARG(a->dk >= 1 && a->dk <= kMaxDim && a->dv >= 1 && a->dv <= kMaxDim, w + ": key and value dimensions are 1 to 256");
    NRN_CHECK_ARG(std::isfinite(a->scale) && a->scale != 0.0f, w + ": scale must be finite and not 0");
    NRN_CHECK_ARG(a->log_decay != nullptr, w + ": null log_decay");
    return NRN_OK;
}

ScanArgs scan_args(const nrn_linattn_t* a) {
    ScanArgs p{};
    p.heads = a->heads;
    p.seqs = a->seqs;
    p.tokens = a->tokens;
    p.cu = a->cu_seqlens;
    p.log_decay = a->log_decay;
    p.err = a->err;
    p.out_mul = a->scale;
    p.in_mul = p.end_mul = 1.0f;
    p.off = 1;
    return p;
}

template <typename T>
void launch_step(const StepArgs& p, int seqs, bool vec, cudaStream_t s) {
    if (vec) {
        const int64_t n = static_cast<int64_t>(seqs) * p.heads * ((p.dv + 31) / 32);
        step_kernel<T, 4><<<static_cast<unsigned>(n), kStepThreads, 0, s>>>(p);
    } else {
        const int64_t n = static_cast<int64_t>(seqs) * p.heads * ((p.dv + 7) / 8);
        step_kernel<T, 1><<<static_cast<unsigned>(n), kStepThreads, 0, s>>>(p);
    }
}

}  // namespace
}  // namespace nrn

using namespace nrn;

extern "C" nrn_status_t nrn_cuda_linattn_workspace(const nrn_linattn_t* a, int32_t backward, int64_t* bytes) {
    NRN_TRY(check_common(a, "nrn_cuda_linattn_workspace"));
    NRN_CHECK_ARG(bytes != nullptr, "nrn_cuda_linattn_workspace: null result");
    // whatever the arrays' alignment turns out to be
    *bytes = std::max(Segments(a, false, backward != 0).bytes(a), Segments(a, true, backward != 0).bytes(a)) + (backward ? part_bytes(a) : 0);
    return NRN_OK;
}

extern "C" nrn_status_t nrn_cuda_linattn_forward(const nrn_linattn_t* a, nrn_stream_t stream) {
    NRN_TRY(check_common(a, "nrn_cuda_linattn_forward"));
    if (a->seqs == 0) return NRN_OK;
    NRN_CHECK_ARG(all_tokens(a) == 0 || (a->q && a->k && a->v && a->o), "nrn_cuda_linattn_forward: null array");
    ScanArgs p = scan_args(a);
    const int share = a->heads / a->kv_heads;
    p.a = strided(a->q, a->q_stride, 1, a->dk);
    p.b = strided(a->k, a->k_stride, share, a->dk);
    p.c = strided(a->v, a->v_stride, share, a->dv);
    p.vec = rows_aligned(p.a, a->dtype) && rows_aligned(p.b, a->dtype) && rows_aligned(p.c, a->dtype);
    const Segments segs(a, p.vec != 0, false);
    const int64_t need = segs.bytes(a);
    NRN_CHECK_ARG(need == 0 || (a->workspace && a->workspace_bytes >= need), "nrn_cuda_linattn_forward: workspace too small");
    p.seg_len = segs.by_k;
    p.o = a->o;
    p.o_seq = a->o_stride[0], p.o_tok = a->o_stride[1], p.o_head = a->o_stride[2];
    p.s_in = a->state_in, p.s_out = a->state_out;
    p.s_i = a->dv, p.s_j = 1;
    return run_scan(p, a, false, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" nrn_status_t nrn_cuda_linattn_backward(const nrn_linattn_t* a, const nrn_linattn_grad_t* g, nrn_stream_t stream) {
    NRN_TRY(check_common(a, "nrn_cuda_linattn_backward"));
    NRN_CHECK_ARG(g != nullptr, "nrn_cuda_linattn_backward: null gradients");
    NRN_CHECK_ARG(std::isfinite(1.0f / a->scale), "nrn_cuda_linattn_backward: 1 / scale must be finite");   // the final states' gradient goes through it
    if (a->seqs == 0) return NRN_OK;
    NRN_CHECK_ARG(all_tokens(a) == 0 || (a->q && a->k && a->v && g->d_o && g->dq && g->dk && g->dv),
                  "nrn_cuda_linattn_backward: null array");
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const int share = a->heads / a->kv_heads;
    const Strided q = strided(a->q, a->q_stride, 1, a->dk), k = strided(a->k, a->k_stride, share, a->dk);
    const Strided v = strided(a->v, a->v_stride, share, a->dv), d = strided(g->d_o, g->d_o_stride, 1, a->dv);
    const int vec = rows_aligned(q, a->dtype) && rows_aligned(k, a->dtype) && rows_aligned(v, a->dtype) && rows_aligned(d, a->dtype);

    const Segments segs(a, vec != 0, true);
    const int64_t states = segs.bytes(a), need = states + part_bytes(a);
    NRN_CHECK_ARG(need == 0 || (a->workspace && a->workspace_bytes >= need), "nrn_cuda_linattn_backward: workspace too small");
    ScanArgs p = scan_args(a);
    p.vec = vec;
    p.seg_len = segs.by_v;
    p.a = d, p.b = v, p.c = k;
    p.o = g->dq;
    p.o_seq = g->dq_stride[0], p.o_tok = g->dq_stride[1], p.o_head = g->dq_stride[2];
    p.s_in = a->state_in;
    p.s_i = 1, p.s_j = a->dv;
    NRN_TRY(run_scan(p, a, false, s));

    // the gradients of keys and values run backwards in time; heads that
    // share one key or value head leave fp32 parts, summed in a fixed order
    p.reverse = 1;
    p.off = 0;
    p.in_mul = 1.0f / a->scale;
    p.end_mul = a->scale;
    p.s_in = g->dstate_out;
    float* part = reinterpret_cast<float*>(static_cast<char*>(a->workspace) + states);
    // both carry the state of q and do, one transposed: where their segments
    // are alike, the values' scan leaves the keys' its entering states
    const bool alike = segs.by_k == segs.by_v;
    for (int which : {1, 0}) {
        p.seg_len = which ? segs.by_k : segs.by_v;
        p.a = which ? k : v, p.b = which ? q : d, p.c = which ? d : q;
        p.seg_made = !which && alike;
        p.g_i = 1, p.g_j = a->dv;
        const int dd = which ? a->dv : a->dk;
        const int64_t* st = which ? g->dv_stride : g->dk_stride;
        void* out = which ? g->dv : g->dk;
        p.s_i = which ? a->dv : 1, p.s_j = which ? 1 : a->dv;
        p.s_out = which ? g->dstate_in : nullptr;
        if (share == 1) {
            p.o = out;
            p.o_seq = st[0], p.o_tok = st[1], p.o_head = st[2];
        } else {
            p.o = part;
            p.o_f32 = 1;
            p.o_head = dd;
            p.o_tok = static_cast<int64_t>(a->heads) * dd;
            p.o_seq = a->cu_seqlens ? 0 : p.o_tok * a->tokens;
        }
        NRN_TRY(run_scan(p, a, true, s));
        const int64_t n = all_tokens(a);
        if (share == 1 || n == 0) continue;
        const int64_t per = a->cu_seqlens ? n : a->tokens;
        if (a->dtype == NRN_BF16) NRN_CUDA_TRY(sum_heads<__nv_bfloat16>(part, n, a->kv_heads, share, dd, out, st, per, s));
        else if (a->dtype == NRN_FP16) NRN_CUDA_TRY(sum_heads<__half>(part, n, a->kv_heads, share, dd, out, st, per, s));
        else NRN_CUDA_TRY(sum_heads<float>(part, n, a->kv_heads, share, dd, out, st, per, s));
    }
    return NRN_OK;
}

extern "C" nrn_status_t nrn_cuda_linattn_step(const nrn_linattn_t* a, float* state, int64_t slot_stride, int32_t n_slots,
                                              const int32_t* slots, nrn_stream_t stream) {
    NRN_TRY(check_common(a, "nrn_cuda_linattn_step"));
    NRN_CHECK_ARG(a->tokens == 1 && a->cu_seqlens == nullptr, "nrn_cuda_linattn_step: one token for each sequence");
    NRN_CHECK_ARG(n_slots >= 0 && (slots || n_slots >= a->seqs), "nrn_cuda_linattn_step: fewer states than sequences");
    NRN_CHECK_ARG(n_slots <= 1 || slot_stride >= static_cast<int64_t>(a->heads) * a->dk * a->dv, "nrn_cuda_linattn_step: states lie on one another");
    if (a->seqs == 0) return NRN_OK;
    NRN_CHECK_ARG(a->q && a->k && a->v && a->o && state, "nrn_cuda_linattn_step: null array");
    NRN_CHECK_ARG(static_cast<int64_t>(a->seqs) * a->heads * ((a->dv + 7) / 8) < (int64_t(1) << 31),
                  "nrn_cuda_linattn_step: too many sequences and heads for one launch");
    StepArgs p{};
    p.q = a->q, p.k = a->k, p.v = a->v, p.o = a->o;
    p.q_seq = a->q_stride[0], p.q_head = a->q_stride[2];
    p.k_seq = a->k_stride[0], p.k_head = a->k_stride[2];
    p.v_seq = a->v_stride[0], p.v_head = a->v_stride[2];
    p.o_seq = a->o_stride[0], p.o_head = a->o_stride[2];
    p.state = state;
    p.s_slot = slot_stride;
    p.slots = slots;
    p.n_slots = n_slots;
    p.heads = a->heads;
    p.share = a->heads / a->kv_heads;
    p.dk = a->dk, p.dv = a->dv;
    p.log_decay = a->log_decay;
    p.scale = a->scale;
    const bool vec = a->dv % 4 == 0 && slot_stride % 4 == 0 && reinterpret_cast<uintptr_t>(state) % 16 == 0;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (a->dtype == NRN_BF16) launch_step<__nv_bfloat16>(p, a->seqs, vec, s);
    else if (a->dtype == NRN_FP16) launch_step<__half>(p, a->seqs, vec, s);
    else launch_step<float>(p, a->seqs, vec, s);
    NRN_CUDA_TRY(cudaGetLastError());
    return NRN_OK;
}

// scaled.cu -- matrix products in 8-bit floating point (e4m3) with a scale
// for each block of 128 columns, and the quantisers that make their operands.
//
//     out[m][n] = sum over blocks kb of sa[m][kb] sb[n][kb] (sum over k in kb of a[m][k] b[n][k])
//
// A scale belongs to one row (activations, gradients) or to 128 rows
// (weights).  The inner sums run on the tensor cores (tcgen05, fp32 in
// TMEM); because the scales change with every block, each block's sums leave
// TMEM and are scaled and added in fp32 registers.
//
// Kernel (persistent, one CTA per SM, 12 warps), for a tile of 128 rows of
// one operand ("rows", the MMA's M) by NT rows of the other ("cols", its N):
//   warp 0    producer: per block one TMA box of each operand (128-byte
//             swizzle, zeros outside the matrix) into a ring of stages;
//   warp 1    issuer (one thread): per block four tcgen05.mma (K = 32) into
//             one of the TMEM accumulators; the commit frees the stage and
//             hands the accumulator on;
//   warps 4-11 two warpgroups, each half of the columns: tcgen05.ld, scale,
//             add, and at the end write the tile.  With NT = 256 a thread
//             holds 128 sums: the first warpgroup gives its registers up
//             (12 x 168 at launch: 4 x 56 + 8 x 224).
// With NT = 256 an accumulator is 128 x 256: per block 512 cycles of MMA at
// the dense e4m3 rate against 256 cycles of TMEM reads and 256 (128 as
// packed pairs) of FMA issue, so the promotion hides behind the MMA of the
// next block; NT = 128 would read as much shared memory per cycle as there is
// (128 bytes).
// Measured, 8192 x 8192 by 4096 columns: 305 us, 1,800 TFLOP/s: more than the
// measured bf16 rate, 55% of twice it.  Run for a second it takes 350: at 1000
// W the clock falls to 1.70 GHz.  With a scale for each row on both sides 466.
// A block takes 1,200 cycles on a full GPU: two accumulators fill TMEM, so an
// MMA starts only when the sums of the block before last are out.  Pairs of
// CTAs sharing the cols operand (305 us) and sixteen promoting warps (351 us,
// for their registers) brought nothing.
//
// Few rows (decode): the weights take the MMA's rows and the few activations
// its columns, NT = 16 up.  Too few tiles for the GPU: the columns k are
// split; the last CTA of a tile to finish adds the parts in their order
// (nobody waits), so results repeat bit for bit.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <mutex>
#include <type_traits>

#include "common.cuh"
#include "internal.h"
#include "launch.h"
#include "scaled.cuh"
#include "tc.cuh"
#include "tensor_map.h"
#include "vecio.cuh"

namespace nrn {
namespace {

using namespace tc;

constexpr int kBlock = 128;            // columns (and weight rows) of a scale block
constexpr int kRowTile = 128;
constexpr int kEpiThreads = 256;
constexpr int kThreads = 128 + kEpiThreads;
constexpr int kMaxStages = 8;
enum { ERR_SCALED_TIMEOUT = 5 };

struct ProductArgs {
    const float* rs;                   // scales of the rows operand
    const float* cs;                   // scales of the cols operand
    int64_t rs_row, rs_col, cs_row, cs_col;
    int32_t r_shift, c_shift;          // log2 of the row block (0 or 7)
    int32_t n_rows, n_cols, blocks;    // blocks of 128 along k
    int32_t row_tiles, col_tiles, splits, stages;
    void* out;
    int64_t out_row, out_col;          // strides of the output along rows and cols (one of them 1)
    int32_t dtype, vec;
    float* part;                       // [tile][split][128 * NT] partial sums
    int32_t* count;                    // [tile] parts finished
    int32_t* err;
};

struct Smem {
    uint64_t full[kMaxStages];
    uint64_t empty[kMaxStages];
    uint64_t tfull[4];
    uint64_t tempty[4];
    uint64_t drain;
    uint32_t tmem;
    int abort;
    int last;
    int stop;
    alignas(16) float cscale[2][256];
};
constexpr int kSmemHead = 4096;        // Smem, padded so that the tiles start 1 KB aligned
static_assert(sizeof(Smem) <= kSmemHead, "barrier block too large");

// K-major, 128-byte swizzle: 8-row groups of 1 KB; descriptor version 1.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr) {
    return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | (1ull << 16) | (static_cast<uint64_t>(1024 >> 4) << 32) |
           (1ull << 46) | (2ull << 61);
}

// kind::f8f6f4: D f32, A and B e4m3, both K-major, M = 128.
template <int NT>
__device__ __forceinline__ void mma_e4m3(uint32_t d, uint64_t a, uint64_t b, uint32_t accumulate) {
    constexpr uint32_t idesc = (1u << 4) | (static_cast<uint32_t>(NT >> 3) << 17) | ((128u >> 4) << 24);
    const uint32_t zero = 0;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(zero)
        : "memory");
}

__device__ __forceinline__ void epi_barrier() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

template <int NT>
struct Shape {
    static constexpr int kCols = NT / 2;                       // columns of a thread
    static constexpr int kChunk = kCols < 16 ? kCols : 16;     // columns of one TMEM load
    static constexpr int kBufs = NT == 256 ? 2 : 4;
    static constexpr uint32_t kTmem = NT * kBufs < 32 ? 32 : NT * kBufs;
    static constexpr int kStageBytes = (kRowTile + NT) * kBlock;
};
// Results whose rows do not start on 16 bytes, or that end inside a tile, pass
// through 32 x 16 floats of a warp's own, so that a store covers two rows: one
// element of 32 rows a store made 6992 x 4411 results (213 columns) 336 us
// that take 53.  A kernel of its own (ODD): in one with the rest the backward
// pass took 175 us where it takes 166.
constexpr int kOutPitch = 17;          // floats: no bank conflicts either way
constexpr int kOutBytes = kEpiThreads / 32 * 32 * kOutPitch * 4;

template <typename T>
__device__ __forceinline__ void put(void* out, int64_t at, float x) {
    static_cast<T*>(out)[at] = from_f32<T>(x);
}
__device__ __forceinline__ void put_any(void* out, int dtype, int64_t at, float x) {
    if (dtype == NRN_BF16) put<__nv_bfloat16>(out, at, x);
    else if (dtype == NRN_FP16) put<__half>(out, at, x);
    else put<float>(out, at, x);
}

// CBLOCK: the cols operand has one scale for 128 rows (uniform over a
// warpgroup's columns); otherwise one for each, staged in shared memory.
template <int NT, bool CBLOCK, bool ODD>
__global__ void __launch_bounds__(kThreads, 1)
    product_kernel(const __grid_constant__ CUtensorMap rmap, const __grid_constant__ CUtensorMap cmap,
                   const __grid_constant__ ProductArgs a) {
    using S = Shape<NT>;
    extern __shared__ __align__(1024) unsigned char smem[];
    Smem& M = *reinterpret_cast<Smem*>(smem);
    unsigned char* tiles = smem + kSmemHead;
    volatile int* abort = &M.abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int stages = a.stages;

    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) {
            mbar_init(&M.full[s], 1);
            mbar_init(&M.empty[s], 1);
        }
        for (int i = 0; i < S::kBufs; ++i) {
            mbar_init(&M.tfull[i], 1);
            mbar_init(&M.tempty[i], kEpiThreads / 32);
        }
        mbar_init(&M.drain, 1);
        M.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&M.tmem)),
                     "r"(S::kTmem)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = M.tmem;
    let_next();
    previous_done();
    const int items = a.row_tiles * a.col_tiles * a.splits;

    auto fail = [&]() {
        *abort = 1;
        if (a.err) atomicCAS(a.err, 0, ERR_SCALED_TIMEOUT);
    };
    // item -> tile and its blocks [k0, k1); the row tile runs fastest
    auto work = [&](int item, int& rt, int& ct, int& k0, int& k1) {
        const int tile = item / a.splits, sp = item - tile * a.splits;
        ct = tile / a.row_tiles;
        rt = tile - ct * a.row_tiles;
        k0 = static_cast<int>(static_cast<int64_t>(a.blocks) * sp / a.splits);
        k1 = static_cast<int>(static_cast<int64_t>(a.blocks) * (sp + 1) / a.splits);
    };

    if (warp < 4) {
        if constexpr (NT == 256) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == 0 && lane == 0) {
            long long it = 0;
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int i = blockIdx.x; i < items && ok; i += gridDim.x) {
                int rt, ct, k0, k1;
                work(i, rt, ct, k0, k1);
                for (int kb = k0; kb < k1; ++kb, ++it) {
                    if (!mbar_wait(&M.empty[stage], phase ^ 1u, abort)) {
                        fail();
                        ok = false;
                        break;
                    }
                    unsigned char* dst = tiles + stage * S::kStageBytes;
                    mbar_expect_tx(&M.full[stage], S::kStageBytes);
                    tma_load_2d(dst, &rmap, kb * kBlock, rt * kRowTile, &M.full[stage]);
                    tma_load_2d(dst + kRowTile * kBlock, &cmap, kb * kBlock, ct * NT, &M.full[stage]);
                    if (++stage == stages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
            // the copies still in flight land before the CTA exits
            for (long long q = it - 1; q >= 0 && q >= it - stages; --q)
                mbar_wait(&M.full[q % stages], static_cast<uint32_t>((q / stages) & 1), nullptr);
        } else if (warp == 1 && lane == 0) {
            int stage = 0, buf = 0;
            uint32_t phase = 0, bphase = 0;
            bool ok = true;
            for (int i = blockIdx.x; i < items && ok; i += gridDim.x) {
                int rt, ct, k0, k1;
                work(i, rt, ct, k0, k1);
                for (int kb = k0; kb < k1; ++kb) {
                    if (!mbar_wait(&M.tempty[buf], bphase ^ 1u, abort) || !mbar_wait(&M.full[stage], phase, abort)) {
                        fail();
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t pa = smem_u32(tiles + stage * S::kStageBytes), pb = pa + kRowTile * kBlock;
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk)
                        mma_e4m3<NT>(tmem + static_cast<uint32_t>(buf * NT), smem_desc(pa + kk * 32), smem_desc(pb + kk * 32),
                                     kk > 0 ? 1u : 0u);
                    tc_commit(&M.empty[stage]);
                    tc_commit(&M.tfull[buf]);
                    if (++stage == stages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                    if (++buf == S::kBufs) {
                        buf = 0;
                        bphase ^= 1u;
                    }
                }
            }
            // every MMA issued has completed before the accumulators are freed
            tc_commit(&M.drain);
            mbar_wait(&M.drain, 0, nullptr);
        }
    } else {
        if constexpr (NT == 256) asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        const int et = threadIdx.x - 128;            // 0 .. 255
        const int half = et >> 7;                    // this warpgroup's half of the columns
        const int sub = warp & 3;                    // TMEM lanes 32 sub ..
        const int row_l = sub * 32 + lane;
        int buf = 0;
        uint32_t bphase = 0;
        for (int i = blockIdx.x; i < items; i += gridDim.x) {
            int rt, ct, k0, k1;
            work(i, rt, ct, k0, k1);
            const int row = rt * kRowTile + row_l, col0 = ct * NT + half * S::kCols;
            const float* rs = row < a.n_rows ? a.rs + (row >> a.r_shift) * a.rs_row : nullptr;
            // CBLOCK: this warpgroup's scale; else: the scale of column `et` of the tile, for everybody
            const int ccol = CBLOCK ? col0 : ct * NT + et;
            const float* cs = ccol < a.n_cols && (CBLOCK || et < NT) ? a.cs + (ccol >> a.c_shift) * a.cs_row : nullptr;
            uint64_t acc[S::kCols / 2];
#pragma unroll
            for (int j = 0; j < S::kCols / 2; ++j) acc[j] = 0;
            float rnext = rs && k0 < k1 ? rs[k0 * a.rs_col] : 0.0f;
            float cnext = cs && k0 < k1 ? cs[k0 * a.cs_col] : 0.0f;
            bool ok = true;
            for (int kb = k0; kb < k1; ++kb) {
                const float rsc = rnext, csc = cnext;
                if (kb + 1 < k1) {
                    if (rs) rnext = rs[(kb + 1) * a.rs_col];
                    if (cs) cnext = cs[(kb + 1) * a.cs_col];
                }
                if (!CBLOCK) {
                    if (et < NT) M.cscale[kb & 1][et] = csc;
                    epi_barrier();
                }
                const bool got = mbar_wait(&M.tfull[buf], bphase, abort);
                if (!__all_sync(0xffffffffu, got)) {
                    if (lane == 0) fail();
                    ok = false;
                }
                if (ok) {
                    tc_fence_after();
                    const uint32_t at = tmem + (static_cast<uint32_t>(32 * sub) << 16) +
                                        static_cast<uint32_t>(buf * NT + half * S::kCols);
                    const float u = CBLOCK ? rsc * csc : rsc;
                    const uint64_t uu = pack2(__float_as_uint(u), __float_as_uint(u));
                    const float* sc = &M.cscale[kb & 1][half * S::kCols];
                    auto add = [&](const uint32_t* v, int c0) {
#pragma unroll
                        for (int j = 0; j < S::kChunk; j += 4) {
                            uint64_t f = uu, h = uu;
                            if (!CBLOCK) {
                                const ulonglong2 s4 = *reinterpret_cast<const ulonglong2*>(sc + c0 + j);
                                f = mul2(uu, s4.x);
                                h = mul2(uu, s4.y);
                            }
                            acc[(c0 + j) / 2] = fma2(pack2(v[j], v[j + 1]), f, acc[(c0 + j) / 2]);
                            acc[(c0 + j) / 2 + 1] = fma2(pack2(v[j + 2], v[j + 3]), h, acc[(c0 + j) / 2 + 1]);
                        }
                    };
                    if constexpr (S::kCols == 8) {
                        uint32_t v[8];
                        tc_ld8(at, v);
                        tc_wait_ld8(v);
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&M.tempty[buf]);
                        add(v, 0);
                    } else {
                        uint32_t v[2][16];
                        tc_ld16(at, v[0]);
#pragma unroll
                        for (int c = 0; c < S::kCols / 16; ++c) {
                            tc_wait_ld16(v[c & 1]);
                            if (c + 1 < S::kCols / 16) {
                                tc_ld16(at + 16 * (c + 1), v[(c + 1) & 1]);
                            } else {
                                tc_fence_before();
                                __syncwarp();
                                if (lane == 0) mbar_arrive(&M.tempty[buf]);
                            }
                            add(v[c & 1], 16 * c);
                        }
                    }
                } else if (CBLOCK) {
                    break;                 // without CBLOCK the barrier above counts every warp to the end
                }
                if (++buf == S::kBufs) {
                    buf = 0;
                    bphase ^= 1u;
                }
            }
            if (a.splits > 1 || !CBLOCK) {
                // barriers follow: one thread decides for all whether to go on
                epi_barrier();
                if (et == 0) M.stop = *abort;
                epi_barrier();
                if (M.stop) break;
            } else if (!ok) {
                break;
            }
            if (a.splits > 1) {
                const int tile = i / a.splits;
                float* mine = a.part + static_cast<int64_t>(i) * kRowTile * NT;
#pragma unroll
                for (int j = 0; j < S::kCols / 2; ++j) {
                    const float2 x = unpack2(acc[j]);
                    mine[(2 * j) * kEpiThreads + et] = x.x;
                    mine[(2 * j + 1) * kEpiThreads + et] = x.y;
                }
                __threadfence();
                epi_barrier();
                if (et == 0) M.last = atomicAdd(&a.count[tile], 1) == a.splits - 1;
                epi_barrier();
                if (!M.last) continue;
                __threadfence();
                const float* all = a.part + static_cast<int64_t>(tile) * a.splits * kRowTile * NT;
#pragma unroll
                for (int j = 0; j < S::kCols / 2; ++j) {
                    float2 x = make_float2(0.0f, 0.0f);
                    for (int s = 0; s < a.splits; ++s) {
                        x.x += __ldcg(all + static_cast<int64_t>(s) * kRowTile * NT + (2 * j) * kEpiThreads + et);
                        x.y += __ldcg(all + static_cast<int64_t>(s) * kRowTile * NT + (2 * j + 1) * kEpiThreads + et);
                    }
                    acc[j] = pack2(__float_as_uint(x.x), __float_as_uint(x.y));
                }
                if (et == 0) a.count[tile] = 0;
            }
            const bool whole = a.vec && col0 + S::kCols <= a.n_cols;      // this warpgroup's columns
            if (ODD && !whole) {
                float* st = reinterpret_cast<float*>(tiles + stages * S::kStageBytes) + (et >> 5) * 32 * kOutPitch;
                const int e = lane % S::kChunk, first = rt * kRowTile + sub * 32;
#pragma unroll
                for (int j = 0; j < S::kCols; j += S::kChunk) {
                    if (col0 + j >= a.n_cols) continue;
#pragma unroll
                    for (int c = 0; c < S::kChunk; c += 2) {
                        const float2 y = unpack2(acc[(j + c) / 2]);
                        st[lane * kOutPitch + c] = y.x, st[lane * kOutPitch + c + 1] = y.y;
                    }
                    __syncwarp();
                    if (col0 + j + e < a.n_cols) {
                        const int64_t at = first * a.out_row + col0 + j + e;
                        const int rows = min(a.n_rows - first, 32);
                        if (a.dtype == NRN_FP32) {
                            for (int r = lane / S::kChunk; r < rows; r += 32 / S::kChunk) static_cast<float*>(a.out)[at + r * a.out_row] = st[r * kOutPitch + e];
                        } else if (a.dtype == NRN_BF16) {
                            for (int r = lane / S::kChunk; r < rows; r += 32 / S::kChunk) put<__nv_bfloat16>(a.out, at + r * a.out_row, st[r * kOutPitch + e]);
                        } else {
                            for (int r = lane / S::kChunk; r < rows; r += 32 / S::kChunk) put<__half>(a.out, at + r * a.out_row, st[r * kOutPitch + e]);
                        }
                    }
                    __syncwarp();
                }
            } else if (row < a.n_rows) {
                if (whole) {
                    // 8 columns at a time: 16 bytes (32 in fp32)
#pragma unroll
                    for (int j = 0; j < S::kCols; j += 8) {
                        float x[8];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float2 y = unpack2(acc[j / 2 + e]);
                            x[2 * e] = y.x, x[2 * e + 1] = y.y;
                        }
                        const int64_t at = row * a.out_row + col0 + j;
                        if (a.dtype == NRN_BF16) store8(static_cast<__nv_bfloat16*>(a.out) + at, x, 8, true);
                        else if (a.dtype == NRN_FP16) store8(static_cast<__half*>(a.out) + at, x, 8, true);
                        else store8(static_cast<float*>(a.out) + at, x, 8, true);
                    }
                } else if constexpr (!ODD) {
                    // swapped: neighbouring lanes' rows are neighbours in the result
#pragma unroll
                    for (int j = 0; j < S::kCols; ++j) {
                        const float2 y = unpack2(acc[j / 2]);
                        if (col0 + j < a.n_cols)
                            put_any(a.out, a.dtype, row * a.out_row + static_cast<int64_t>(col0 + j) * a.out_col, j & 1 ? y.y : y.x);
                    }
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::kTmem)
                                : "memory");
}

// ------------------------------------------------------------- quantisers

constexpr int kQuantThreads = 256;

// A scale for each row and 128 columns: 16 lanes of eight elements a block,
// two blocks of the result at a time so that enough loads are in flight.  One
// read and a write of half or a quarter of it: 32,768 x 4096 bf16 (403 MB) in
// 108 us, 57% of the measured copy (8192 x 4096, partly from L2, in 26): it
// issues in 71% of its cycles, most of them an element's arithmetic.
template <typename T>
__global__ void __launch_bounds__(kQuantThreads)
    quant_rows_kernel(const T* x, uint32_t rows, uint32_t cols, int64_t x_stride, int vec, uint8_t* values, int64_t v_stride,
                      float* scales, int64_t s_row, int64_t s_col, uint32_t blocks) {
    const uint32_t total = rows * blocks, part = threadIdx.x & 15;
    const uint32_t step = gridDim.x * (kQuantThreads / 16);
    constexpr int kAtOnce = 2;
    // every lane of a warp takes part in the shuffles: the loop is uniform
    for (uint32_t w0 = blockIdx.x * (kQuantThreads / 16) + (threadIdx.x >> 5) * 2; w0 < total; w0 += kAtOnce * step) {
        Raw8<T> raw[kAtOnce];
        uint32_t r[kAtOnce], b[kAtOnce];
        int n[kAtOnce];
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
            const uint32_t w = w0 + k * step + ((threadIdx.x >> 4) & 1);
            r[k] = w / blocks;
            b[k] = w - r[k] * blocks;
            const int left = static_cast<int>(cols - b[k] * kBlock) - static_cast<int>(part) * 8;
            n[k] = w < total && left > 0 ? min(left, 8) : (w < total ? 0 : -1);
            raw[k] = load8(x + (n[k] > 0 ? r[k] * x_stride + b[k] * kBlock + part * 8 : 0), n[k], vec != 0);
        }
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
            float f[8];
            uint32_t m = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                f[e] = to_f32(raw[k].e[e]);
                m = max(m, abs_bits(f[e]));
            }
#pragma unroll
            for (int d = 1; d < 16; d <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
            const float s = block_scale(m), inv = __frcp_rn(s);
            if (n[k] >= 0 && part == 0) scales[r[k] * s_row + b[k] * s_col] = s;
            if (n[k] > 0)          // rows are padded to 16 bytes: a whole store fits
                *reinterpret_cast<uint2*>(values + r[k] * v_stride + b[k] * kBlock + part * 8) =
                    make_uint2(e4m3x4(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv), e4m3x4(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv));
        }
    }
}

struct QuantOut {
    uint8_t* values;
    int64_t v_stride;
    float* scales;
    int64_t s_row, s_col;
};

// x^T with a scale for each of its rows (columns of x) and 128 rows of x, and
// with ROWS also x itself with a scale for each row and 128 columns, from one
// read: a gradient is wanted both ways.  A block has a 128 x 128 tile, a
// thread eight rows by eight columns of it in registers; the transposed bytes
// pass through shared memory, eight at a time, their places exclusive-ored
// with the column's so that neither way has bank conflicts.
//
// In a backward pass the kernels that make operands follow one another but do
// not need one another: each waits for the one before only at its end, so
// that the product after the last one has all of them.
//
// Three blocks an SM where a thread's 80 registers do for it (4096 columns of
// 4097 rows: 20.3 us against 24.7 with two); with ROWS they do not (22.7
// against 19 with two).
template <typename T, bool ROWS>
__global__ void __launch_bounds__(kQuantThreads, ROWS || sizeof(T) == 4 ? 2 : 3)
    quant_cols_kernel(const T* x, int64_t rows, int64_t cols, int64_t x_stride, int vec, const QuantOut by_cols, const QuantOut by_rows) {
    __shared__ alignas(16) uint8_t bytes[kBlock][kBlock];
    __shared__ uint32_t amax[kQuantThreads / 16][kBlock];
    __shared__ float inv_s[kBlock];
    const int64_t r0 = static_cast<int64_t>(blockIdx.y) * kBlock, c0 = static_cast<int64_t>(blockIdx.x) * kBlock;
    const int part = threadIdx.x & 15, rg = threadIdx.x >> 4;        // columns 8 part ..; rows 8 rg ..
    let_next();
    const int64_t left = cols - c0 - part * 8;
    const int n = static_cast<int>(left < 0 ? 0 : (left < 8 ? left : 8));
    Raw8<T> raw[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t r = r0 + rg * 8 + i;
        raw[i] = load8(x + (r < rows && n > 0 ? r * x_stride + c0 + part * 8 : 0), r < rows ? n : 0, vec != 0);
    }
    uint32_t m[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) m[e] = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        uint32_t mr = 0;
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            f[e] = to_f32(raw[i].e[e]);
            const uint32_t a = abs_bits(f[e]);
            m[e] = max(m[e], a);
            if (ROWS) mr = max(mr, a);
        }
        if constexpr (ROWS) {
#pragma unroll
            for (int d = 1; d < 16; d <<= 1) mr = max(mr, __shfl_xor_sync(0xffffffffu, mr, d));
            const float s = block_scale(mr), inv = __frcp_rn(s);
            const int64_t r = r0 + rg * 8 + i;
            if (r < rows) {
                if (part == 0) by_rows.scales[r * by_rows.s_row + blockIdx.x * by_rows.s_col] = s;
                if (n > 0)
                    *reinterpret_cast<uint2*>(by_rows.values + r * by_rows.v_stride + c0 + part * 8) =
                        make_uint2(e4m3x4(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv), e4m3x4(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv));
            }
        }
    }
#pragma unroll
    for (int e = 0; e < 8; e += 4) *reinterpret_cast<uint4*>(&amax[rg][part * 8 + e]) = make_uint4(m[e], m[e + 1], m[e + 2], m[e + 3]);
    __syncthreads();
    if (threadIdx.x < kBlock) {
        uint32_t a = 0;
#pragma unroll
        for (int g = 0; g < kQuantThreads / 16; ++g) a = max(a, amax[g][threadIdx.x]);
        const float s = block_scale(a);
        inv_s[threadIdx.x] = __frcp_rn(s);
        if (c0 + threadIdx.x < cols) by_cols.scales[(c0 + threadIdx.x) * by_cols.s_row + blockIdx.y * by_cols.s_col] = s;
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int c = part * 8 + e;
        const float inv = inv_s[c];
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = to_f32(raw[i].e[e]) * inv;
        *reinterpret_cast<uint2*>(&bytes[c][(rg ^ part) * 8]) = make_uint2(e4m3x4(f[0], f[1], f[2], f[3]), e4m3x4(f[4], f[5], f[6], f[7]));
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int c = k * 32 + (threadIdx.x >> 3), q = threadIdx.x & 7, pc = c >> 3;      // rows 16 q .. of column c
        if (c0 + c >= cols || r0 + q * 16 >= rows) continue;
        uint4 v = *reinterpret_cast<const uint4*>(&bytes[c][(q ^ (pc >> 1)) * 16]);
        if (pc & 1) v = make_uint4(v.z, v.w, v.x, v.y);
        *reinterpret_cast<uint4*>(by_cols.values + (c0 + c) * by_cols.v_stride + r0 + q * 16) = v;   // rows are padded to 16 bytes
    }
    previous_done();
}

// A scale for each 128 x 128 block: weights, once.  32,768 x 4096 bf16 (403
// MB) in 184 us, a third of the measured copy.
template <typename T>
__global__ void __launch_bounds__(kQuantThreads)
    quant_blocks_kernel(const T* x, int64_t rows, int64_t cols, int64_t x_stride, int vec, uint8_t* values, int64_t v_stride,
                        float* scales, int64_t s_row, int64_t s_col) {
    __shared__ uint32_t amax[kQuantThreads / 32];
    const int64_t r0 = static_cast<int64_t>(blockIdx.y) * kBlock, c0 = static_cast<int64_t>(blockIdx.x) * kBlock;
    const int part = threadIdx.x & 15;
    const int64_t c = c0 + part * 8, left = cols - c;
    const int n = static_cast<int>(left < 0 ? 0 : (left < 8 ? left : 8));
    Raw8<T> raw[8];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t r = r0 + (threadIdx.x >> 4) + 16 * i;
        raw[i] = load8(x + (r < rows && n > 0 ? r * x_stride + c : 0), r < rows ? n : 0, vec != 0);
#pragma unroll
        for (int e = 0; e < 8; ++e) m = max(m, abs_bits(to_f32(raw[i].e[e])));
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if ((threadIdx.x & 31) == 0) amax[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kQuantThreads / 32; ++w) m = max(m, amax[w]);
    const float s = block_scale(m), inv = 1.0f / s;
    if (threadIdx.x == 0) scales[blockIdx.y * s_row + blockIdx.x * s_col] = s;
    if (n <= 0) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t r = r0 + (threadIdx.x >> 4) + 16 * i;
        if (r >= rows) break;
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = to_f32(raw[i].e[e]) * inv;
        *reinterpret_cast<uint2*>(values + r * v_stride + c) =
            make_uint2(e4m3x4(f[0], f[1], f[2], f[3]), e4m3x4(f[4], f[5], f[6], f[7]));
    }
}

// Values of a matrix transposed, 128 x 128 bytes at a time: four rows by
// four columns a step, through shared memory on both sides.
__global__ void __launch_bounds__(kQuantThreads)
    transpose_kernel(const uint8_t* in, int64_t rows, int64_t cols, int64_t in_stride, uint8_t* out, int64_t out_stride) {
    __shared__ alignas(8) uint32_t from[kBlock][34], to[kBlock][34];   // 34: four rows on are 8 banks on
    let_next();
    const int64_t r0 = static_cast<int64_t>(blockIdx.y) * kBlock, c0 = static_cast<int64_t>(blockIdx.x) * kBlock;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int r = k * 32 + (threadIdx.x >> 3), q = threadIdx.x & 7;
        // rows are padded to 16 bytes: 16 that start inside a row end inside its storage
        const uint4 v = r0 + r < rows && c0 + q * 16 < cols ? *reinterpret_cast<const uint4*>(in + (r0 + r) * in_stride + c0 + q * 16) : make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint2*>(&from[r][q * 4]) = make_uint2(v.x, v.y);
        *reinterpret_cast<uint2*>(&from[r][q * 4 + 2]) = make_uint2(v.z, v.w);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        // columns 4 cw .., rows 4 rw ..: a warp has eight by four of them
        const int e = k * (kQuantThreads / 32) + (threadIdx.x >> 5), cw = (e & 3) * 8 + (threadIdx.x & 7), rw = (e >> 2) * 4 + ((threadIdx.x >> 3) & 3);
        const uint32_t a = from[4 * rw][cw], b = from[4 * rw + 1][cw], c = from[4 * rw + 2][cw], d = from[4 * rw + 3][cw];
        const uint32_t ab = __byte_perm(a, b, 0x5140), cd = __byte_perm(c, d, 0x5140), ab2 = __byte_perm(a, b, 0x7362), cd2 = __byte_perm(c, d, 0x7362);
        to[4 * cw][rw] = __byte_perm(ab, cd, 0x5410);
        to[4 * cw + 1][rw] = __byte_perm(ab, cd, 0x7632);
        to[4 * cw + 2][rw] = __byte_perm(ab2, cd2, 0x5410);
        to[4 * cw + 3][rw] = __byte_perm(ab2, cd2, 0x7632);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int c = k * 32 + (threadIdx.x >> 3), q = threadIdx.x & 7;
        if (c0 + c < cols && r0 + q * 16 < rows) {
            const uint2 lo = *reinterpret_cast<const uint2*>(&to[c][q * 4]), hi = *reinterpret_cast<const uint2*>(&to[c][q * 4 + 2]);
            *reinterpret_cast<uint4*>(out + (c0 + c) * out_stride + r0 + q * 16) = make_uint4(lo.x, lo.y, hi.x, hi.y);
        }
    }
    previous_done();
}

// --------------------------------------------------------------- launches

nrn_status_t make_map(const nrn_scaled_t* m, int box_rows, CUtensorMap* map) {
    const TensorMapEncode fn = tensor_map_encode();
    if (!fn) return fail(NRN_ERR_UNSUPPORTED, "nrn_cuda_scaled_product: the driver has no cuTensorMapEncodeTiled");
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(m->cols), static_cast<cuuint64_t>(m->rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(m->value_stride)};
    const cuuint32_t box[2] = {kBlock, static_cast<cuuint32_t>(box_rows)}, one[2] = {1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, m->values, dims, strides, box, one,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(NRN_ERR_INVALID, "nrn_cuda_scaled_product: cuTensorMapEncodeTiled refused the operand");
    return NRN_OK;
}

// The counters have a place of their own at the workspace's start, whatever
// the sizes: one call's parts never lie where another's counters are.
constexpr int64_t kMaxSplitTiles = 1024;
constexpr int64_t kCountBytes = kMaxSplitTiles * 4;

struct Plan {
    bool swap;
    int nt, splits;
    int64_t row_tiles, col_tiles, blocks;
};

// The tile width and the split of k: the fewest cycles by a model of what
// bounds the kernel.  Rounds of tiles over the SMs; per block of 128 columns
// both operands' way from L2, which all SMs together get at about 36 bytes a
// cycle each and one alone at 64 (measured: 128 x 256 tiles 1,300 cycles a
// block on a full GPU, 128 x 128 tiles 1,000, against 512 and 256 of MMA); per
// tile a fixed cost and the result's way out; where k is split, the parts' way
// out and, in the last block of a tile, all parts' way back.
Plan plan_of(int64_t m, int64_t n, int64_t k) {
    Plan best{};
    best.swap = m <= 128;
    const int64_t rows = best.swap ? n : m, cols = best.swap ? m : n;
    best.row_tiles = (rows + kRowTile - 1) / kRowTile;
    best.blocks = (k + kBlock - 1) / kBlock;
    const int64_t sms = std::max(1, sm_count());
    double cost = 1e300;
    for (int nt : {256, 128, 64, 32, 16}) {
        if (nt > 16 && nt / 2 >= cols) continue;                 // a narrower tile holds them all
        const int64_t ct = (cols + nt - 1) / nt;
        for (int splits : {1, 2, 3, 4, 6, 8, 12, 16}) {
            if (splits > 1 && (best.blocks / splits < 2 || best.row_tiles * ct > kMaxSplitTiles)) break;
            const int64_t items = best.row_tiles * ct * splits;
            const double rounds = static_cast<double>((items + sms - 1) / sms);
            const double busy = static_cast<double>(std::min(items, sms)) / static_cast<double>(sms);
            const double per = static_cast<double>(kRowTile + nt) * std::max(2.0, 3.6 * busy);
            const double c = rounds * (static_cast<double>((best.blocks + splits - 1) / splits) * per + 1000 + 7.0 * nt +
                                       (splits > 1 ? 1500 + 14.0 * nt * (1 + splits) : 0.0));
            if (c < cost) {
                cost = c;
                best.nt = nt;
                best.splits = splits;
                best.col_tiles = ct;
            }
        }
    }
    return best;
}

int64_t plan_workspace(const Plan& p) {
    if (p.splits == 1) return 0;
    return kCountBytes + p.row_tiles * p.col_tiles * p.splits * kRowTile * p.nt * 4;
}

nrn_status_t check_scaled(const nrn_scaled_t* m, const std::string& who) {
    NRN_CHECK_ARG(m != nullptr, who + ": null matrix");
    NRN_CHECK_ARG(m->rows >= 0 && m->cols >= 0 && m->rows < (int64_t(1) << 31) - 256 && m->cols < (int64_t(1) << 31) - 256,
                  who + ": sizes out of range");
    NRN_CHECK_ARG(m->row_block == 1 || m->row_block == kBlock, who + ": row_block is 1 or 128");
    NRN_CHECK_ARG(m->rows == 0 || m->cols == 0 || (m->values && m->scales), who + ": null array");
    NRN_CHECK_ARG(reinterpret_cast<uintptr_t>(m->values) % 16 == 0 && m->value_stride % 16 == 0 && m->value_stride >= m->cols,
                  who + ": values must be 16-byte aligned with rows a multiple of 16 bytes apart");
    NRN_CHECK_ARG(m->value_stride < (int64_t(1) << 40), who + ": row stride out of range");
    return NRN_OK;
}

template <int NT, bool CB, bool ODD>
nrn_status_t launch_product(const CUtensorMap& rm, const CUtensorMap& cm, ProductArgs a, bool after, cudaStream_t s) {
    constexpr int stage = Shape<NT>::kStageBytes;
    a.stages = std::min(kMaxStages, (227 * 1024 - kSmemHead - (ODD ? kOutBytes : 0)) / stage);
    const int bytes = kSmemHead + a.stages * stage + (ODD ? kOutBytes : 0);
    NRN_CUDA_TRY((allow_shared<product_kernel<NT, CB, ODD>>(bytes)));
    const int grid = std::min(a.row_tiles * a.col_tiles * a.splits, sm_count());
    NRN_CUDA_TRY(launch_chained(product_kernel<NT, CB, ODD>, dim3(static_cast<unsigned>(grid)), dim3(kThreads), bytes, s, after, rm, cm, a));
    return NRN_OK;
}

template <bool CB>
nrn_status_t launch_nt(int nt, const CUtensorMap& rm, const CUtensorMap& cm, const ProductArgs& a, bool after, cudaStream_t s) {
    // rows of results that end inside a warpgroup's columns, or start anywhere
    const bool odd = a.out_col == 1 && !(a.vec && a.n_cols % (nt / 2) == 0);
    const auto run = [&](auto width) {
        return odd ? launch_product<width(), CB, true>(rm, cm, a, after, s) : launch_product<width(), CB, false>(rm, cm, a, after, s);
    };
    switch (nt) {
        case 256: return run(std::integral_constant<int, 256>());
        case 128: return run(std::integral_constant<int, 128>());
        case 64: return run(std::integral_constant<int, 64>());
        case 32: return run(std::integral_constant<int, 32>());
        default: return run(std::integral_constant<int, 16>());
    }
}

QuantOut quant_out(const nrn_scaled_t* o) {
    return QuantOut{o->values, o->value_stride, o->scales, o->scale_stride[0], o->scale_stride[1]};
}

// x both ways, for a gradient.
template <typename T>
nrn_status_t quantize_both(const void* x, int64_t rows, int64_t cols, int64_t stride, const nrn_scaled_t* by_cols, const nrn_scaled_t* by_rows,
                           cudaStream_t s) {
    const int vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && stride * sizeof(T) % 16 == 0;
    const dim3 grid(static_cast<unsigned>((cols + kBlock - 1) / kBlock), static_cast<unsigned>((rows + kBlock - 1) / kBlock));
    quant_cols_kernel<T, true><<<grid, kQuantThreads, 0, s>>>(static_cast<const T*>(x), rows, cols, stride, vec, quant_out(by_cols), quant_out(by_rows));
    NRN_CUDA_TRY(cudaGetLastError());
    return NRN_OK;
}

template <typename T>
nrn_status_t quantize(const void* x, int64_t rows, int64_t cols, int64_t stride, bool transpose, const nrn_scaled_t* o,
                      bool after, cudaStream_t s) {
    const T* p = static_cast<const T*>(x);
    const int vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && stride * sizeof(T) % 16 == 0;
    const int64_t rb = (rows + kBlock - 1) / kBlock;
    if (!transpose && o->row_block == 1) {
        const int64_t per_row = (cols + kBlock - 1) / kBlock, work = rows * per_row;
        NRN_CHECK_ARG(work < (int64_t(1) << 30), "nrn_cuda_scaled_quantize: too many blocks for one launch");
        const int64_t blocks = std::min<int64_t>((work + kQuantThreads / 16 - 1) / (kQuantThreads / 16), 16LL * sm_count());
        quant_rows_kernel<T><<<static_cast<unsigned>(blocks), kQuantThreads, 0, s>>>(
            p, static_cast<uint32_t>(rows), static_cast<uint32_t>(cols), stride, vec, o->values, o->value_stride, o->scales, o->scale_stride[0],
            o->scale_stride[1], static_cast<uint32_t>(per_row));
    } else {
        NRN_CHECK_ARG(rb < 65536, "nrn_cuda_scaled_quantize: at most 8,388,480 rows");
        const dim3 grid(static_cast<unsigned>((cols + kBlock - 1) / kBlock), static_cast<unsigned>(rb));
        if (transpose)
            NRN_CUDA_TRY(launch_chained(quant_cols_kernel<T, false>, grid, dim3(kQuantThreads), 0, s, after, p, rows, cols, stride, vec, quant_out(o), QuantOut{}));
        else
            quant_blocks_kernel<T><<<grid, kQuantThreads, 0, s>>>(
                p, rows, cols, stride, vec, o->values, o->value_stride, o->scales, o->scale_stride[0], o->scale_stride[1]);
    }
    NRN_CUDA_TRY(cudaGetLastError());
    return NRN_OK;
}

}  // namespace

TensorMapEncode tensor_map_encode() {
    static std::once_flag once;
    static TensorMapEncode fn = nullptr;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<TensorMapEncode>(p);
    });
    return fn;
}

}  // namespace nrn

using namespace nrn;

extern "C" nrn_status_t nrn_cuda_scaled_quantize(const void* x, int32_t dtype, int64_t rows, int64_t cols, int64_t row_stride,
                                                 int32_t transpose, const nrn_scaled_t* out, nrn_stream_t stream) {
    const std::string who = "nrn_cuda_scaled_quantize";
    NRN_TRY(check_scaled(out, who));
    NRN_CHECK_ARG(dtype == NRN_BF16 || dtype == NRN_FP16 || dtype == NRN_FP32, who + ": unknown type");
    NRN_CHECK_ARG(rows >= 0 && cols >= 0 && row_stride >= 0, who + ": negative sizes");
    NRN_CHECK_ARG(out->rows == (transpose ? cols : rows) && out->cols == (transpose ? rows : cols), who + ": the result has another shape");
    NRN_CHECK_ARG(!transpose || out->row_block == 1, who + ": a transposed result has a scale for each row");
    if (rows == 0 || cols == 0) return NRN_OK;
    NRN_CHECK_ARG(x != nullptr, who + ": null array");
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (dtype == NRN_BF16) return quantize<__nv_bfloat16>(x, rows, cols, row_stride, transpose != 0, out, false, s);
    if (dtype == NRN_FP16) return quantize<__half>(x, rows, cols, row_stride, transpose != 0, out, false, s);
    return quantize<float>(x, rows, cols, row_stride, transpose != 0, out, false, s);
}

extern "C" nrn_status_t nrn_cuda_scaled_workspace(const nrn_scaled_t* a, const nrn_scaled_t* b, int64_t* bytes) {
    const std::string who = "nrn_cuda_scaled_workspace";
    NRN_CHECK_ARG(a && b && bytes, who + ": null argument");
    NRN_CHECK_ARG(a->rows >= 0 && b->rows >= 0 && a->cols >= 0, who + ": negative sizes");
    *bytes = a->rows == 0 || b->rows == 0 || a->cols == 0 ? 0 : plan_workspace(plan_of(a->rows, b->rows, a->cols));
    return NRN_OK;
}

namespace nrn {
namespace {

// after: a kernel of the same call comes before it
nrn_status_t run_transpose(const nrn_scaled_t* in, const nrn_scaled_t* out, bool after, cudaStream_t s) {
    const std::string who = "nrn_cuda_scaled_transpose";
    NRN_TRY(check_scaled(in, who));
    NRN_TRY(check_scaled(out, who));
    NRN_CHECK_ARG(in->row_block == kBlock && out->row_block == kBlock, who + ": both have a row_block of 128");
    NRN_CHECK_ARG(in->rows == out->cols && in->cols == out->rows, who + ": the result has another shape");
    if (in->rows == 0 || in->cols == 0) return NRN_OK;
    const int64_t rb = (in->rows + kBlock - 1) / kBlock, cb = (in->cols + kBlock - 1) / kBlock;
    NRN_CHECK_ARG(rb < 65536, who + ": at most 8,388,480 rows");
    NRN_CUDA_TRY(launch_chained(transpose_kernel, dim3(static_cast<unsigned>(cb), static_cast<unsigned>(rb)), dim3(kQuantThreads), 0, s, after, in->values,
                                in->rows, in->cols, in->value_stride, out->values, out->value_stride));
    return NRN_OK;
}

nrn_status_t run_product(const nrn_scaled_t* a, const nrn_scaled_t* b, void* out, int32_t dtype, int64_t out_stride, void* workspace,
                         int64_t workspace_bytes, int32_t* err, bool after, cudaStream_t s) {
    const std::string who = "nrn_cuda_scaled_product";
    NRN_TRY(check_scaled(a, who));
    NRN_TRY(check_scaled(b, who));
    NRN_CHECK_ARG(dtype == NRN_BF16 || dtype == NRN_FP16 || dtype == NRN_FP32, who + ": unknown type");
    NRN_CHECK_ARG(a->cols == b->cols, who + ": the operands have different numbers of columns");
    NRN_CHECK_ARG(out_stride >= b->rows, who + ": rows of the result overlap");
    if (a->rows == 0 || b->rows == 0) return NRN_OK;
    NRN_CHECK_ARG(out != nullptr, who + ": null array");
    const int size = dtype == NRN_FP32 ? 4 : 2;
    if (a->cols == 0) {
        NRN_CUDA_TRY(cudaMemset2DAsync(out, out_stride * size, 0, b->rows * size, a->rows, s));
        return NRN_OK;
    }
    const Plan p = plan_of(a->rows, b->rows, a->cols);
    NRN_CHECK_ARG(p.row_tiles * p.col_tiles * p.splits < (int64_t(1) << 31), who + ": the result is too large for one launch");
    const int64_t need = plan_workspace(p);
    NRN_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need), who + ": workspace too small");
    const nrn_scaled_t *r = p.swap ? b : a, *c = p.swap ? a : b;
    CUtensorMap rm, cm;
    NRN_TRY(make_map(r, kRowTile, &rm));
    NRN_TRY(make_map(c, p.nt, &cm));
    ProductArgs g{};
    g.rs = r->scales, g.cs = c->scales;
    g.rs_row = r->scale_stride[0], g.rs_col = r->scale_stride[1];
    g.cs_row = c->scale_stride[0], g.cs_col = c->scale_stride[1];
    g.r_shift = r->row_block == 1 ? 0 : 7;
    g.c_shift = c->row_block == 1 ? 0 : 7;
    g.n_rows = static_cast<int32_t>(r->rows), g.n_cols = static_cast<int32_t>(c->rows);
    g.blocks = static_cast<int32_t>(p.blocks);
    g.row_tiles = static_cast<int32_t>(p.row_tiles), g.col_tiles = static_cast<int32_t>(p.col_tiles);
    g.splits = p.splits;
    g.out = out;
    g.out_row = p.swap ? 1 : out_stride;
    g.out_col = p.swap ? out_stride : 1;
    g.dtype = dtype;
    g.vec = !p.swap && reinterpret_cast<uintptr_t>(out) % 16 == 0 && out_stride * size % 16 == 0;
    g.count = static_cast<int32_t*>(workspace);
    g.part = need ? reinterpret_cast<float*>(static_cast<char*>(workspace) + kCountBytes) : nullptr;
    g.err = err;
    return c->row_block == 1 ? launch_nt<false>(p.nt, rm, cm, g, after, s) : launch_nt<true>(p.nt, rm, cm, g, after, s);
}

// The 8-bit operands of a backward pass, one after the other in the workspace.
struct BackwardPlan {
    nrn_scaled_t dy, dyt, xt, wt;
    int64_t product_bytes, bytes;
};

BackwardPlan backward_plan(int64_t rows, const nrn_scaled_t* w, uint8_t* base) {
    BackwardPlan p{};
    // the products' own workspace first, its counters at least: they stay zero from call to call
    const auto need = [](int64_t m, int64_t n, int64_t k) { return m == 0 || n == 0 || k == 0 ? 0 : plan_workspace(plan_of(m, n, k)); };
    p.product_bytes = std::max({kCountBytes, need(rows, w->cols, w->rows), need(w->rows, w->cols, rows)});
    int64_t at = (p.product_bytes + 255) / 256 * 256;
    const auto make = [&](int64_t r, int64_t c, bool scales) {
        nrn_scaled_t m{};
        m.rows = r, m.cols = c, m.row_block = 1;
        m.value_stride = (std::max<int64_t>(c, 1) + 15) / 16 * 16;
        m.values = base + at;
        at += (r * m.value_stride + 255) / 256 * 256;
        if (scales) {
            const int64_t kb = (c + kBlock - 1) / kBlock;
            m.scales = reinterpret_cast<float*>(base + at);
            m.scale_stride[0] = 1, m.scale_stride[1] = std::max<int64_t>(r, 1);
            at += (r * kb * 4 + 255) / 256 * 256;
        }
        return m;
    };
    p.dy = make(rows, w->rows, true);
    p.dyt = make(w->rows, rows, true);
    p.xt = make(w->cols, rows, true);
    p.wt = make(w->cols, w->rows, false);
    p.wt.row_block = kBlock;
    p.wt.scales = w->scales;
    p.wt.scale_stride[0] = w->scale_stride[1], p.wt.scale_stride[1] = w->scale_stride[0];
    p.bytes = at;
    return p;
}

}  // namespace
}  // namespace nrn

extern "C" nrn_status_t nrn_cuda_scaled_transpose(const nrn_scaled_t* in, const nrn_scaled_t* out, nrn_stream_t stream) {
    return run_transpose(in, out, false, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" nrn_status_t nrn_cuda_scaled_product(const nrn_scaled_t* a, const nrn_scaled_t* b, void* out, int32_t dtype,
                                                int64_t out_stride, void* workspace, int64_t workspace_bytes, int32_t* err,
                                                nrn_stream_t stream) {
    return run_product(a, b, out, dtype, out_stride, workspace, workspace_bytes, err, false, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" nrn_status_t nrn_cuda_scaled_backward_workspace(int64_t rows, const nrn_scaled_t* w, int64_t* bytes, int64_t* zeroed) {
    const std::string who = "nrn_cuda_scaled_backward_workspace";
    NRN_CHECK_ARG(w && bytes && zeroed, who + ": null argument");
    NRN_CHECK_ARG(rows >= 0 && w->rows >= 0 && w->cols >= 0, who + ": negative sizes");
    const BackwardPlan p = backward_plan(rows, w, nullptr);
    *bytes = p.bytes;
    *zeroed = kCountBytes;
    return NRN_OK;
}

extern "C" nrn_status_t nrn_cuda_scaled_backward(const void* dy, const void* x, int32_t dtype, int64_t rows, int64_t dy_stride, int64_t x_stride,
                                                 const nrn_scaled_t* w, void* dx, int32_t dx_dtype, void* dw, int32_t dw_dtype, void* workspace,
                                                 int64_t workspace_bytes, int32_t* err, nrn_stream_t stream) {
    const std::string who = "nrn_cuda_scaled_backward";
    NRN_TRY(check_scaled(w, who));
    NRN_CHECK_ARG(w->row_block == kBlock, who + ": weights have a row_block of 128");
    NRN_CHECK_ARG(dtype == NRN_BF16 || dtype == NRN_FP16 || dtype == NRN_FP32, who + ": unknown type");
    NRN_CHECK_ARG(rows >= 0 && rows < (int64_t(1) << 23) - 128 && w->rows < (int64_t(1) << 23) - 128, who + ": at most 8,388,480 rows");
    NRN_CHECK_ARG(dy_stride >= 0 && x_stride >= 0, who + ": negative strides");
    NRN_CHECK_ARG(dx_dtype == NRN_BF16 || dx_dtype == NRN_FP16 || dx_dtype == NRN_FP32, who + ": unknown type of dx");
    NRN_CHECK_ARG(dw_dtype == NRN_BF16 || dw_dtype == NRN_FP16 || dw_dtype == NRN_FP32, who + ": unknown type of dw");
    if (w->cols == 0) return NRN_OK;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (w->rows == 0) {
        NRN_CHECK_ARG(rows == 0 || dx, who + ": null array");
        if (rows) NRN_CUDA_TRY(cudaMemsetAsync(dx, 0, static_cast<size_t>(rows) * w->cols * (dx_dtype == NRN_FP32 ? 4 : 2), s));
        return NRN_OK;
    }
    NRN_CHECK_ARG((rows == 0 || (dy && x && dx)) && dw, who + ": null array");
    if (rows == 0) {
        NRN_CUDA_TRY(cudaMemsetAsync(dw, 0, static_cast<size_t>(w->rows) * w->cols * (dw_dtype == NRN_FP32 ? 4 : 2), s));
        return NRN_OK;
    }
    uint8_t* base = static_cast<uint8_t*>(workspace);
    const BackwardPlan p = backward_plan(rows, w, base);
    NRN_CHECK_ARG(workspace && workspace_bytes >= p.bytes, who + ": workspace too small");
    NRN_CHECK_ARG(reinterpret_cast<uintptr_t>(workspace) % 256 == 0, who + ": the workspace must be 256-byte aligned");
    const int64_t n = w->rows, k = w->cols;
    if (dtype == NRN_BF16) {
        NRN_TRY(quantize_both<__nv_bfloat16>(dy, rows, n, dy_stride, &p.dyt, &p.dy, s));
        NRN_TRY(quantize<__nv_bfloat16>(x, rows, k, x_stride, true, &p.xt, true, s));
    } else if (dtype == NRN_FP16) {
        NRN_TRY(quantize_both<__half>(dy, rows, n, dy_stride, &p.dyt, &p.dy, s));
        NRN_TRY(quantize<__half>(x, rows, k, x_stride, true, &p.xt, true, s));
    } else {
        NRN_TRY(quantize_both<float>(dy, rows, n, dy_stride, &p.dyt, &p.dy, s));
        NRN_TRY(quantize<float>(x, rows, k, x_stride, true, &p.xt, true, s));
    }
    NRN_TRY(run_transpose(w, &p.wt, true, s));
    NRN_TRY(run_product(&p.dy, &p.wt, dx, dx_dtype, k, workspace, p.product_bytes, err, true, s));
    return run_product(&p.dyt, &p.xt, dw, dw_dtype, k, workspace, p.product_bytes, err, true, s);
}

// block_matmul.cu -- 8-bit block quantiser and the product of block-scaled 8-bit operands.
#include <cuda_fp8.h>

#include <algorithm>
#include <type_traits>

#include "learn.cuh"
#include "provider.h"
#include "tma.cuh"

namespace pcu {

constexpr int kBlock = 128;  // elements of a scale's block along the inner dimension

// The smallest power of two, at least 2^-126, that brings amax (finite) to 448 = 1.75 * 2^8 or
// below: with amax = 1.f * 2^e it is 2^(e - 8) for 1.f <= 1.75 and 2^(e - 7) above.  1 for 0.
__device__ __forceinline__ float block_scale(float amax) {
    if (amax == 0.0f) return 1.0f;
    const unsigned bits = __float_as_uint(amax);
    const int e = (int)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u);
    return __uint_as_float((unsigned)max(e, 1) << 23);
}

__device__ __forceinline__ float from_e4m3(unsigned code) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)code, __NV_E4M3)));
}

// 16 elements from `from` on, `count` of them there, the others 0.  Whole 16-byte loads where the
// address allows it.
template <typename T> __device__ __forceinline__ void load_codes_input(const T *from, int count, float (&v)[16]) {
    if (count == 16 && (reinterpret_cast<uintptr_t>(from) & 15) == 0) {
        constexpr int V = 16 / sizeof(T);
#pragma unroll
        for (int i = 0; i < 16; i += V) {
            const uint4 raw = __ldg(reinterpret_cast<const uint4 *>(from + i));
            const T *t = reinterpret_cast<const T *>(&raw);
#pragma unroll
            for (int j = 0; j < V; ++j) v[i + j] = Elem<T>::load(t[j]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = i < count ? Elem<T>::load(from[i]) : 0.0f;
    }
}

// The largest magnitude's bits, which order as the magnitudes do; 0x7f800000 and above: an infinity
// or a NaN is among them.
__device__ __forceinline__ unsigned largest_bits(const float (&v)[16]) {
    unsigned most = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) most = max(most, __float_as_uint(v[i]) & 0x7fffffffu);
    return most;
}

// Values that are not finite: recorded, and made NaN.  Returns the largest bits of the others.
__device__ __forceinline__ unsigned settle(float (&v)[16], uint64_t event, unsigned long long *status) {
    unsigned most = 0;
    for (int i = 0; i < 16; ++i) {
        const unsigned bits = __float_as_uint(v[i]) & 0x7fffffffu;
        if (bits < 0x7f800000u) {
            most = max(most, bits);
        } else {
            record_fault(status, event + i, PCU_B200_KIND_INVALID);
            v[i] = NAN;
        }
    }
    return most;
}

// v * inverse as codes; exact up to the rounding to a code: the inverse of a power of two >= 2^-126
// is one <= 2^126.
__device__ __forceinline__ void store_codes(unsigned char *to, int count, const float (&v)[16], float inverse) {
    alignas(16) unsigned short pair[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
        pair[i] = __nv_cvt_float2_to_fp8x2(make_float2(v[2 * i] * inverse, v[2 * i + 1] * inverse), __NV_SATFINITE, __NV_E4M3);
    if (count == 16 && (reinterpret_cast<uintptr_t>(to) & 15) == 0) {
        *reinterpret_cast<uint4 *>(to) = *reinterpret_cast<const uint4 *>(pair);
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (i < count) to[i] = (unsigned char)(pair[i / 2] >> 8 * (i % 2));
    }
}

template <typename T> struct QuantizeParams {
    const T *input;
    uint64_t rows, columns, stride;
    unsigned char *codes;
    uint64_t codes_stride;
    float *scales;
    unsigned long long *status;
    ChainGuard guard;
};

// Eight threads take a row's 128 elements of a block, 16 each, and keep them in registers between
// the maximum and the codes, so the input is read once.  HIGH 1: a block is such a row, 32 blocks per
// CTA.  HIGH 128: a CTA takes a block, 4 rows per thread.
constexpr int kQuantizeThreads = 256;

template <typename T, int HIGH>
__global__ void __launch_bounds__(kQuantizeThreads) quantize_kernel(const QuantizeParams<T> p) {
    if (!chain_admits(p.guard)) return;
    constexpr int kRows = kQuantizeThreads / 8, PASSES = HIGH == 1 ? 1 : HIGH / kRows;
    const unsigned across = (unsigned)((p.columns + kBlock - 1) / kBlock);
    const unsigned block = HIGH == 1 ? blockIdx.x * kRows + threadIdx.x / 8 : blockIdx.x;
    const uint64_t column = (uint64_t)(block % across) * kBlock + threadIdx.x % 8 * 16;
    const uint64_t first = HIGH == 1 ? block / across : (uint64_t)(block / across) * HIGH + threadIdx.x / 8;
    const int count = column < p.columns ? (int)min((uint64_t)16, p.columns - column) : 0;
    float v[PASSES][16];
    unsigned most = 0;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const uint64_t row = first + i * kRows;
        load_codes_input(p.input + row * p.stride + column, row < p.rows ? count : 0, v[i]);
    }
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        unsigned here = largest_bits(v[i]);
        if (here >= 0x7f800000u) here = settle(v[i], (first + i * kRows) * p.columns + column, p.status);
        most = max(most, here);
    }
    for (int o = 4; o; o >>= 1) most = max(most, __shfl_xor_sync(~0u, most, o));
    if (HIGH > 1) {
        __shared__ unsigned scratch[kRows];
        if (threadIdx.x % 8 == 0) scratch[threadIdx.x / 8] = most;
        __syncthreads();
        most = scratch[threadIdx.x % 32];
        for (int o = 16; o; o >>= 1) most = max(most, __shfl_xor_sync(~0u, most, o));
    }
    const float scale = block_scale(__uint_as_float(most)), inverse = 1.0f / scale;
    if (first < p.rows && threadIdx.x % (HIGH == 1 ? 8 : kQuantizeThreads) == 0) p.scales[block] = scale;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const uint64_t row = first + i * kRows;
        if (row < p.rows && count) store_codes(p.codes + row * p.codes_stride + column, count, v[i], inverse);
    }
}

template <typename T> struct ProductParams {
    const unsigned char *left, *right;
    const float *left_scales, *right_scales;
    T *out;
    uint64_t rows, inner, columns, left_stride, right_stride, out_stride;
    unsigned long long *status;
    ChainGuard guard;
};

template <typename T> __device__ __forceinline__ void store_cell(const ProductParams<T> &p, uint64_t r, uint64_t c, float v) {
    const T y = Elem<T>::round(v);
    p.out[r * p.out_stride + c] = y;
    if (const unsigned kind = result_kind(Elem<T>::load(y))) record_fault(p.status, r * p.columns + c, kind);
}

// COLUMNS cells of one row from `column` on, in 16-byte pieces where the row allows it.
template <typename T, int COLUMNS>
__device__ __forceinline__ void store_row(const ProductParams<T> &p, uint64_t row, uint64_t column,
                                          const float (&v)[COLUMNS]) {
    constexpr int V = 16 / sizeof(T);
    T *to = p.out + row * p.out_stride + column;
    const bool whole = (reinterpret_cast<uintptr_t>(to) & 15) == 0;
#pragma unroll
    for (int i = 0; i < COLUMNS; i += V) {
        if (column + i >= p.columns) break;
        alignas(16) T y[V];
        bool fine = true;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            y[j] = Elem<T>::round(v[i + j]);
            fine &= isfinite(Elem<T>::load(y[j])) || column + i + j >= p.columns;
        }
        if (whole && column + i + V <= p.columns) {
            *reinterpret_cast<uint4 *>(to + i) = *reinterpret_cast<const uint4 *>(y);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (column + i + j < p.columns) to[i + j] = y[j];
        }
        if (!fine)
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (const unsigned kind = result_kind(Elem<T>::load(y[j])); kind && column + i + j < p.columns)
                    record_fault(p.status, row * p.columns + column + i + j, kind);
    }
}

// Any base and stride: 16 x 16 cells per CTA, one thread per cell.
template <typename T> __global__ void __launch_bounds__(256) product_plain_kernel(const ProductParams<T> p) {
    if (!chain_admits(p.guard)) return;
    __shared__ float sl[16][17], sr[16][17];
    const uint64_t tiles = (p.columns + 15) / 16;
    const uint64_t r0 = blockIdx.x / tiles * 16, c0 = blockIdx.x % tiles * 16;
    const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
    const uint64_t r = r0 + ty, c = c0 + tx, blocks = (p.inner + kBlock - 1) / kBlock;
    float acc = 0;
    for (uint64_t kb = 0; kb < blocks; ++kb) {
        float part = 0;
        for (int k0 = 0; k0 < kBlock; k0 += 16) {
            const uint64_t k = kb * kBlock + k0 + tx;
            sl[ty][tx] = r < p.rows && k < p.inner ? from_e4m3(p.left[r * p.left_stride + k]) : 0.0f;
            sr[ty][tx] = c0 + ty < p.columns && k < p.inner ? from_e4m3(p.right[(c0 + ty) * p.right_stride + k]) : 0.0f;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 16; ++i) part = fmaf(sl[ty][i], sr[tx][i], part);
            __syncthreads();
        }
        if (r < p.rows && c < p.columns)
            acc = fmaf(part, p.left_scales[r * blocks + kb] * p.right_scales[c / kBlock * blocks + kb], acc);
    }
    if (r < p.rows && c < p.columns) store_cell(p, r, c, acc);
}

// ------------------------------------------------------------------ tensor core product
//
// D = P . Q^T over blocks of 128 of the inner dimension, P's 128 rows and Q's BN rows per tile.  The
// tensor core cannot apply a scale that changes from block to block of its accumulator, so each
// block's product goes to a TMEM buffer of its own and the epilogue warps add it, scaled, to
// binary32 sums in registers while the next block's product runs.
//   * batch form: P = left, Q = right: a tile of 128 rows x 256 columns.
//   * row form (few rows): P = right, Q = left: 128 columns x BN rows, so that the weights, which
//     are all the traffic there is, fill the instruction's 128 rows.  The blocks of one tile are
//     split over a cluster's CTAs; the first CTA adds their sums, in rank order.
// Warp 0 issues the TMA loads, warp 1 the tcgen05.mma instructions, the others drain TMEM.
// All waits are bounded (mbar_wait); one that runs out records the watchdog kind, and the CTA still
// waits for its own copies and products before it frees TMEM and returns.

__device__ __forceinline__ uint64_t k_major_descriptor(uint32_t address) {
    // 128-byte swizzle, rows of 128 bytes, groups of 8 rows 1024 bytes apart, descriptor version 1
    return (uint64_t)(address >> 4) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

// D (binary32, TMEM) = or += A . B^T for 128 x N x 32 codes
__device__ __forceinline__ void mma_e4m3(uint32_t d, uint64_t a, uint64_t b, uint32_t shape, uint32_t add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(shape), "r"(add)
        : "memory");
}

// The barrier completes when all tensor core work issued before by this thread has.
__device__ __forceinline__ void mma_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar))
                 : "memory");
}

__device__ __forceinline__ void tmem_load16(uint32_t (&v)[16], uint32_t address) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(address));
}

// Waits for the loads issued so far; `v` is named so that nothing reads it earlier.
__device__ __forceinline__ void tmem_wait(uint32_t (&v)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]),
                   "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])
                 :
                 : "memory");
}

template <int BN_, bool ROWS_> struct ProductShape {
    static constexpr int BM = 128, BN = BN_;
    static constexpr bool ROWS = ROWS_;               // the row form
    static constexpr int EPILOGUE = BN == 256 ? 8 : 4;  // warps; warp w drains TMEM lanes 32 (w % 4)...
    static constexpr int COLUMNS = BN / (EPILOGUE / 4);  // accumulator columns per thread
    static constexpr int THREADS = (2 + EPILOGUE) * 32;
    static constexpr int BUFFERS = BN == 256 ? 2 : 4;
    static constexpr int TMEM_COLUMNS = BUFFERS * BN;
    static constexpr int P_BYTES = BM * kBlock, Q_BYTES = BN * kBlock, STAGE_BYTES = P_BYTES + Q_BYTES;
    static constexpr int STAGES = ROWS ? 5 : 4;
    static constexpr int PARTIAL_BYTES = BM * BN * 4;  // one CTA's sums, handed to the cluster's first
    static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + 1024;
    static_assert(!ROWS || BN <= 32, "the row form keeps a column's factor in a lane");
    static_assert(PARTIAL_BYTES <= STAGES * STAGE_BYTES || !ROWS, "the sums take the stages' place");
};

template <typename T> struct TileParams {
    ProductParams<T> out;
    uint64_t p_rows, q_rows;  // extents along the tile's rows and columns
    const float *p_scales, *q_scales;
    unsigned tiles_p, tiles_q, tiles;
    int blocks;  // of 128 along the inner dimension
};

template <typename T, typename S>
__global__ void __launch_bounds__(S::THREADS, 1)
    product_kernel(const __grid_constant__ CUtensorMap map_p, const __grid_constant__ CUtensorMap map_q,
                   const __grid_constant__ TileParams<T> t) {
    const ProductParams<T> &p = t.out;
    if (!chain_admits(p.guard)) return;  // the same answer in every CTA of the grid
    extern __shared__ unsigned char smem_raw[];
    unsigned char *const tiles = smem_raw + (1024 - (smem_addr(smem_raw) & 1023) & 1023);
    __shared__ uint64_t full[S::STAGES], empty[S::STAGES], ready[S::BUFFERS], drained[S::BUFFERS], finished;
    __shared__ uint32_t tmem_base;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

    // blocks [kb0, kb1) of the inner dimension: a cluster's share, all of them in the batch form
    uint32_t rank = 0, ranks = 1;
    if (S::ROWS) {
        asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
        asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
    }
    const int kb0 = (int)((int64_t)t.blocks * rank / ranks), kb1 = (int)((int64_t)t.blocks * (rank + 1) / ranks);
    const unsigned first = S::ROWS ? blockIdx.x / ranks : blockIdx.x, step = S::ROWS ? gridDim.x / ranks : gridDim.x;

    if (threadIdx.x == 0) {
        for (int i = 0; i < S::STAGES; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], 1);
        for (int i = 0; i < S::BUFFERS; ++i) mbar_init(&ready[i], 1), mbar_init(&drained[i], S::EPILOGUE);
        mbar_init(&finished, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_base)),
                     "r"(S::TMEM_COLUMNS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = tmem_base;

    // Tiles in groups of 8 tile rows, column by column inside a group, so that the tiles worked on at
    // once share a few panels of both operands in L2.
    auto place = [&](unsigned id, int &p0, int &q0) {
        const unsigned group = id / (8 * t.tiles_q) * 8, rows = min(8u, t.tiles_p - group), in = id - group * t.tiles_q;
        p0 = (int)((group + in % rows) * S::BM);
        q0 = (int)(in / rows * S::BN);
    };

    if (warp == 0) {
        if (lane == 0) {
            int it = 0;
            bool ok = true;
            for (unsigned id = first; ok && id < t.tiles; id += step) {
                int p0, q0;
                place(id, p0, q0);
                for (int kb = kb0; kb < kb1; ++kb, ++it) {
                    const int s = it % S::STAGES;
                    if (!(ok = mbar_wait(&empty[s], ((it / S::STAGES) & 1) ^ 1))) break;
                    unsigned char *to = tiles + s * S::STAGE_BYTES;
                    mbar_expect_tx(&full[s], S::STAGE_BYTES);
                    tma_load_2d(to, &map_p, &full[s], kb * kBlock, p0);
                    tma_load_2d(to + S::P_BYTES, &map_q, &full[s], kb * kBlock, q0);
                }
            }
            if (!ok) record_fault(p.status, 0, kWatchdog);
            // nothing is left in flight towards this CTA's shared memory when it ends
            for (int i = it > S::STAGES ? it - S::STAGES : 0; i < it; ++i)
                mbar_wait(&full[i % S::STAGES], (i / S::STAGES) & 1);
        }
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr uint32_t shape = 1u << 4 | (uint32_t)(S::BN / 8) << 17 | (uint32_t)(S::BM / 16) << 24;
            int it = 0;
            bool ok = true;
            for (unsigned id = first; ok && id < t.tiles; id += step)
                for (int kb = kb0; kb < kb1; ++kb, ++it) {
                    const int s = it % S::STAGES, b = it % S::BUFFERS;
                    if (!(ok = mbar_wait(&drained[b], ((it / S::BUFFERS) & 1) ^ 1) &&
                               mbar_wait(&full[s], (it / S::STAGES) & 1)))
                        break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t at = smem_addr(tiles + s * S::STAGE_BYTES);
                    const uint64_t pd = k_major_descriptor(at), qd = k_major_descriptor(at + S::P_BYTES);
#pragma unroll
                    for (int k = 0; k < kBlock / 32; ++k)  // 32 bytes further along the swizzled rows
                        mma_e4m3(tmem + b * S::BN, pd + 2 * k, qd + 2 * k, shape, k != 0);
                    mma_commit(&empty[s]);
                    mma_commit(&ready[b]);
                }
            if (!ok) record_fault(p.status, 0, kWatchdog);
            mma_commit(&finished);
            if (!mbar_wait(&finished, 0)) record_fault(p.status, 0, kWatchdog);
        }
    } else {
        const int quarter = warp % 4, half = (warp - 2) / 4;
        const int local = quarter * 32 + lane, from = half * S::COLUMNS;  // this thread's row and first column
        float sum[S::COLUMNS];
        int it = 0;
        bool ok = true;
        for (unsigned id = first; ok && id < t.tiles; id += step) {
            int p0, q0;
            place(id, p0, q0);
            const uint64_t row = (uint64_t)p0 + local, column = (uint64_t)q0 + from;
#pragma unroll
            for (int i = 0; i < S::COLUMNS; ++i) sum[i] = 0;
            // Batch form: one factor per thread and block, its columns being one block of 128 of the right
            // operand's.  Row form: lane c holds column c's.  Read one block ahead of its use.
            auto factor_of = [&](int kb) -> float {
                if (kb >= kb1) return 0.0f;
                if (!S::ROWS)
                    return row < t.p_rows && column < t.q_rows
                               ? t.p_scales[row * t.blocks + kb] * t.q_scales[column / kBlock * t.blocks + kb]
                               : 0.0f;
                return lane < S::BN && (uint64_t)q0 + lane < t.q_rows
                           ? t.q_scales[((uint64_t)q0 + lane) * t.blocks + kb] * t.p_scales[(uint64_t)p0 / kBlock * t.blocks + kb]
                           : 0.0f;
            };
            float next = factor_of(kb0);
            for (int kb = kb0; kb < kb1; ++kb, ++it) {
                const int b = it % S::BUFFERS;
                const float factor = next;
                next = factor_of(kb + 1);
                if (!(ok = __all_sync(~0u, mbar_wait(&ready[b], (it / S::BUFFERS) & 1)))) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t at = tmem + ((uint32_t)(quarter * 32) << 16) + b * S::BN + from;
                uint32_t v[2][16];
                tmem_load16(v[0], at);
#pragma unroll
                for (int c = 0; c < S::COLUMNS / 16; ++c) {
                    tmem_wait(v[c & 1]);
                    if (c + 1 < S::COLUMNS / 16) {
                        tmem_load16(v[(c + 1) & 1], at + (c + 1) * 16);
                    } else {  // the buffer has been read
                        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&drained[b]);
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float f = S::ROWS ? __shfl_sync(~0u, factor, c * 16 + i) : factor;
                        sum[c * 16 + i] = fmaf(__uint_as_float(v[c & 1][i]), f, sum[c * 16 + i]);
                    }
                }
            }
            if (!ok) break;
            if (!S::ROWS) {
                if (row < t.p_rows) store_row<T, S::COLUMNS>(p, row, column, sum);
            } else if (ranks == 1) {
#pragma unroll
                for (int i = 0; i < S::COLUMNS; ++i)
                    if (row < t.p_rows && column + i < t.q_rows) store_cell(p, column + i, row, sum[i]);
            } else {
                // to the cluster's first CTA, behind every CTA's last use of its stages (see below)
#pragma unroll
                for (int i = 0; i < S::COLUMNS; ++i) reinterpret_cast<float *>(tiles)[i * S::BM + local] = sum[i];
            }
        }
        if (!ok && lane == 0) record_fault(p.status, 0, kWatchdog);
    }

    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::TMEM_COLUMNS) : "memory");
    if (S::ROWS && ranks > 1) {
        // each CTA's sums are in its own shared memory: the first CTA reads them all
        asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
        if (rank == 0) {
            int p0, q0;
            place(first, p0, q0);
            for (int i = threadIdx.x; i < S::BM * S::BN; i += S::THREADS) {
                const uint64_t column = (uint64_t)p0 + i % S::BM, row = (uint64_t)q0 + i / S::BM;
                if (column >= t.p_rows || row >= t.q_rows) continue;
                float total = 0;
                for (uint32_t r = 0; r < ranks; ++r) {
                    uint32_t remote;
                    float v;
                    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_addr(tiles) + 4 * i), "r"(r));
                    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote) : "memory");
                    total += v;
                }
                store_cell(p, row, column, total);
            }
        }
        __syncwarp();
        asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
    }
}

template <typename T>
static int quantize_typed(const void *input, uint64_t rows, uint64_t columns, uint64_t stride, int high, void *codes,
                          uint64_t codes_stride, float *scales, uint64_t *status, cudaStream_t stream,
                          const ChainGuard &guard) {
    QuantizeParams<T> p{(const T *)input, rows, columns, stride, (unsigned char *)codes, codes_stride, scales,
                        reinterpret_cast<unsigned long long *>(status), guard};
    const uint64_t blocks = (rows + high - 1) / high * ((columns + kBlock - 1) / kBlock);
    constexpr int kRows = kQuantizeThreads / 8;
    if (high == 1)
        quantize_kernel<T, 1><<<(unsigned)((blocks + kRows - 1) / kRows), kQuantizeThreads, 0, stream>>>(p);
    else
        quantize_kernel<T, kBlock><<<(unsigned)blocks, kQuantizeThreads, 0, stream>>>(p);
    return pcu_host::launch_status();
}

// A map over rows x inner codes with boxes of one block of 128 by `high` rows.
static bool code_map(CUtensorMap *map, const unsigned char *base, uint64_t rows, uint64_t inner, uint64_t stride,
                     uint32_t high) {
    auto encode = pcu_host::tensor_map_encoder();
    if (!encode || !pcu_host::aligned(base, 16) || (rows > 1 && stride % 16 != 0)) return false;
    cuuint64_t dims[2] = {inner, rows}, strides[1] = {rows > 1 ? stride : (inner + 15) / 16 * 16};
    cuuint32_t box[2] = {kBlock, high}, steps[2] = {1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<unsigned char *>(base), dims, strides, box, steps,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, typename S>
static int launch_product(const ProductParams<T> &p, const CUtensorMap &map_p, const CUtensorMap &map_q, unsigned ranks,
                          cudaStream_t stream) {
    static std::mutex lock;
    static bool configured[64] = {false};
    int device = 0;
    if (cudaError_t e = cudaGetDevice(&device); e != cudaSuccess) return pcu_host::set_cuda_error(e);
    {
        std::lock_guard<std::mutex> guard(lock);
        if (device >= 64 || !configured[device]) {
            if (cudaError_t e = cudaFuncSetAttribute(product_kernel<T, S>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                     S::SMEM_BYTES);
                e != cudaSuccess)
                return pcu_host::set_cuda_error(e);
            if (device < 64) configured[device] = true;
        }
    }
    TileParams<T> t{};
    t.out = p;
    t.p_rows = S::ROWS ? p.columns : p.rows;
    t.q_rows = S::ROWS ? p.rows : p.columns;
    t.p_scales = S::ROWS ? p.right_scales : p.left_scales;
    t.q_scales = S::ROWS ? p.left_scales : p.right_scales;
    t.tiles_p = (unsigned)((t.p_rows + S::BM - 1) / S::BM);
    t.tiles_q = (unsigned)((t.q_rows + S::BN - 1) / S::BN);
    t.tiles = t.tiles_p * t.tiles_q;
    t.blocks = (int)((p.inner + kBlock - 1) / kBlock);
    cudaLaunchConfig_t config{};
    config.gridDim = S::ROWS ? t.tiles * ranks : std::min(t.tiles, (unsigned)pcu_host::sm_count());
    config.blockDim = S::THREADS;
    config.dynamicSmemBytes = S::SMEM_BYTES;
    config.stream = stream;
    cudaLaunchAttribute cluster{};
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim.x = ranks;
    cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
    config.attrs = &cluster;
    config.numAttrs = S::ROWS ? 1 : 0;
    if (cudaError_t e = cudaLaunchKernelEx(&config, product_kernel<T, S>, map_p, map_q, t); e != cudaSuccess) {
        (void)cudaGetLastError();
        return pcu_host::set_cuda_error(e);
    }
    return PCU_B200_OK;
}

template <typename T> static int product_typed(const ProductParams<T> &p, cudaStream_t stream) {
    CUtensorMap map_left, map_right;
    constexpr int kFew = 16;
    if (p.inner && p.rows <= kFew) {
        using S = ProductShape<kFew, true>;
        if (code_map(&map_right, p.right, p.columns, p.inner, p.right_stride, S::BM) &&
            code_map(&map_left, p.left, p.rows, p.inner, p.left_stride, S::BN)) {
            const uint64_t tiles = (p.columns + S::BM - 1) / S::BM, blocks = (p.inner + kBlock - 1) / kBlock;
            unsigned ranks = 1;
            while (ranks < 8 && tiles * ranks * 2 <= 2 * (uint64_t)pcu_host::sm_count() && blocks >= 8 * ranks) ranks *= 2;
            return launch_product<T, S>(p, map_right, map_left, ranks, stream);
        }
    } else if (p.inner) {
        using S = ProductShape<256, false>;
        if (code_map(&map_left, p.left, p.rows, p.inner, p.left_stride, S::BM) &&
            code_map(&map_right, p.right, p.columns, p.inner, p.right_stride, S::BN))
            return launch_product<T, S>(p, map_left, map_right, 1, stream);
    }
    const uint64_t tiles = (p.rows + 15) / 16 * ((p.columns + 15) / 16);
    product_plain_kernel<T><<<(unsigned)tiles, 256, 0, stream>>>(p);
    return pcu_host::launch_status();
}

}  // namespace pcu

using namespace pcu;

namespace {

constexpr uint64_t kMostExtent = 1ull << 31, kMostStride = 1ull << 40;

int quantize(int dtype, const void *input, uint64_t rows, uint64_t columns, uint64_t input_stride, int block_rows,
             void *codes, uint64_t codes_stride, float *scales, uint64_t *status, void *stream, const ChainGuard &guard) {
    if ((dtype != PCU_B200_F32 && dtype != PCU_B200_F16 && dtype != PCU_B200_BF16) || !status ||
        (block_rows != 1 && block_rows != kBlock))
        return PCU_B200_ERROR_INVALID_ARGUMENT;
    cudaStream_t s = pcu_host::as_stream(stream);
    if (rows == 0 || columns == 0) return chain_decide_only(guard, s);
    if (!input || !codes || !scales || (rows > 1 && (input_stride < columns || codes_stride < columns)))
        return PCU_B200_ERROR_INVALID_ARGUMENT;
    if (rows >= kMostExtent || columns >= kMostExtent || input_stride > kMostStride || codes_stride > kMostStride ||
        (rows + block_rows - 1) / block_rows * ((columns + kBlock - 1) / kBlock) >= kMostExtent)
        return PCU_B200_ERROR_SIZE_OVERFLOW;
    switch (dtype) {
    case PCU_B200_F32:
        return quantize_typed<float>(input, rows, columns, input_stride, block_rows, codes, codes_stride, scales, status, s, guard);
    case PCU_B200_F16:
        return quantize_typed<__half>(input, rows, columns, input_stride, block_rows, codes, codes_stride, scales, status, s, guard);
    default:
        return quantize_typed<__nv_bfloat16>(input, rows, columns, input_stride, block_rows, codes, codes_stride, scales, status, s, guard);
    }
}

int product(int out_dtype, const void *left, const float *left_scales, const void *right, const float *right_scales,
            void *out, uint64_t rows, uint64_t inner, uint64_t columns, uint64_t left_stride, uint64_t right_stride,
            uint64_t out_stride, uint64_t *status, void *stream, const ChainGuard &guard) {
    if ((out_dtype != PCU_B200_F32 && out_dtype != PCU_B200_F16 && out_dtype != PCU_B200_BF16) || !status)
        return PCU_B200_ERROR_INVALID_ARGUMENT;
    cudaStream_t s = pcu_host::as_stream(stream);
    if (rows == 0 || columns == 0) return chain_decide_only(guard, s);
    if (!out || (rows > 1 && out_stride < columns)) return PCU_B200_ERROR_INVALID_ARGUMENT;
    if (inner && (!left || !left_scales || !right || !right_scales || (rows > 1 && left_stride < inner) ||
                  (columns > 1 && right_stride < inner)))
        return PCU_B200_ERROR_INVALID_ARGUMENT;
    if (rows >= kMostExtent || inner >= kMostExtent || columns >= kMostExtent || left_stride > kMostStride ||
        right_stride > kMostStride || out_stride > kMostStride ||
        !pcu_host::multiply_fits((rows + 15) / 16, (columns + 15) / 16, kMostExtent - 1))
        return PCU_B200_ERROR_SIZE_OVERFLOW;
    auto fill = [&](auto *typed_out) {
        using T = std::remove_pointer_t<decltype(typed_out)>;
        return product_typed<T>(ProductParams<T>{(const unsigned char *)left, (const unsigned char *)right, left_scales,
                                                 right_scales, typed_out, rows, inner, columns, left_stride,
                                                 right_stride, out_stride,
                                                 reinterpret_cast<unsigned long long *>(status), guard},
                                s);
    };
    switch (out_dtype) {
    case PCU_B200_F32: return fill((float *)out);
    case PCU_B200_F16: return fill((__half *)out);
    default: return fill((__nv_bfloat16 *)out);
    }
}

}  // namespace

extern "C" int pcu_b200_block_quantize(int dtype, const void *input, uint64_t rows, uint64_t columns,
                                       uint64_t input_stride, int block_rows, void *codes, uint64_t codes_stride,
                                       float *scales, uint64_t *status, void *stream) {
    return quantize(dtype, input, rows, columns, input_stride, block_rows, codes, codes_stride, scales, status, stream,
                    ChainGuard{});
}

extern "C" int pcu_b200_block_matmul(int out_dtype, const void *left, const float *left_scales, const void *right,
                                     const float *right_scales, void *out, uint64_t rows, uint64_t inner,
                                     uint64_t columns, uint64_t left_stride, uint64_t right_stride,
                                     uint64_t out_stride, uint64_t *status, void *stream) {
    return product(out_dtype, left, left_scales, right, right_scales, out, rows, inner, columns, left_stride,
                   right_stride, out_stride, status, stream, ChainGuard{});
}

extern "C" int pcu_b200_guarded_block_quantize(int dtype, const void *input, uint64_t rows, uint64_t columns,
                                               uint64_t input_stride, int block_rows, void *codes,
                                               uint64_t codes_stride, float *scales, uint64_t *chain_records,
                                               uint32_t chain_stage, void *stream) {
    if (!chain_records) return PCU_B200_ERROR_INVALID_ARGUMENT;
    return quantize(dtype, input, rows, columns, input_stride, block_rows, codes, codes_stride, scales,
                    chain_records + 2ull * chain_stage, stream, pcu_host::slab_guard(chain_records, chain_stage));
}

extern "C" int pcu_b200_guarded_block_matmul(int out_dtype, const void *left, const float *left_scales,
                                             const void *right, const float *right_scales, void *out, uint64_t rows,
                                             uint64_t inner, uint64_t columns, uint64_t left_stride,
                                             uint64_t right_stride, uint64_t out_stride, uint64_t *chain_records,
                                             uint32_t chain_stage, void *stream) {
    if (!chain_records) return PCU_B200_ERROR_INVALID_ARGUMENT;
    return product(out_dtype, left, left_scales, right, right_scales, out, rows, inner, columns, left_stride,
                   right_stride, out_stride, chain_records + 2ull * chain_stage, stream,
                   pcu_host::slab_guard(chain_records, chain_stage));
}

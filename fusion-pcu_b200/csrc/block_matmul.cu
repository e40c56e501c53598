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
            const uint4 raw = *reinterpret_cast<const uint4 *>(from + i);
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

// Bound by memory: 16384 x 4096 F32 with blocks of 128 rows 53 us = 6.3 TB/s, 0.96 of a copy; 8192 x 4096 BF16 with
// blocks of one row 20 us = 5.0 TB/s.  Eight threads take a row's 128 elements of a block, 16 each, and keep them in registers between
// the maximum and the codes, so the input is read once.  HIGH 1: a block is such a row, 32 blocks per
// CTA.  HIGH 128: a CTA takes a block, 4 rows per thread.
constexpr int kQuantizeThreads = 256;

template <typename T, int HIGH>
__global__ void __launch_bounds__(kQuantizeThreads) quantize_kernel(const QuantizeParams<T> p) {
    in_stream_order();
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

// The factors of a block's product, scale x other scale = factor * rest: powers of two from 2^-126 on, so
// exponents add, and what binary32 has no exponent for stays in `rest`, 1 otherwise.  (Multiplied, 2^64 by
// 2^64 would be an infinity, and NaN with a product of 0.)  NaN for scales of any other kind.
struct BlockFactor {
    float factor, rest;
};
__device__ __forceinline__ BlockFactor block_factor(float scale, float other) {
    auto good = [](unsigned bits) { return (bits & 0x807fffffu) == 0 && bits >= 0x00800000u && bits < 0x7f800000u; };
    const unsigned a = __float_as_uint(scale), b = __float_as_uint(other);
    if (!good(a) || !good(b)) return {NAN, 1.0f};
    const int e = (int)(a >> 23) + (int)(b >> 23) - 127, near = min(max(e, 1), 254);
    return {__uint_as_float((unsigned)near << 23), __uint_as_float((unsigned)(e - near + 127) << 23)};
}

template <typename T> __device__ __forceinline__ void store_cell(const ProductParams<T> &p, uint64_t r, uint64_t c, float v) {
    const T y = Elem<T>::round(v);
    p.out[r * p.out_stride + c] = y;
    if (const unsigned kind = result_kind(Elem<T>::load(y))) record_fault(p.status, r * p.columns + c, kind);
}

// COLUMNS cells of one row from `column` on, which lies on a 32-byte boundary, in pieces of that size (whole
// sectors: a warp's lanes are in 32 rows).
template <typename T, int COLUMNS>
__device__ __forceinline__ void store_row(const ProductParams<T> &p, uint64_t row, uint64_t column,
                                          const uint32_t (&v)[COLUMNS]) {
    constexpr int V = 32 / sizeof(T);
    static_assert(COLUMNS % V == 0, "whole pieces");
    T *to = p.out + row * p.out_stride + column;
#pragma unroll
    for (int i = 0; i < COLUMNS; i += V) {
        if (column + i >= p.columns) break;
        alignas(32) T y[V];
        bool fine = true;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            y[j] = Elem<T>::round(__uint_as_float(v[i + j]));
            fine &= isfinite(Elem<T>::load(y[j]));
        }
        if (column + i + V <= p.columns) {
            const uint32_t *w = reinterpret_cast<const uint32_t *>(y);
            asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to + i), "r"(w[0]), "r"(w[1]),
                         "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                         : "memory");
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

// The same cells of a warp's 32 rows from `row` on (a lane's v: its row's), for a result whose rows lie anyhow: turned
// in registers, so that adjacent lanes store adjacent columns (5536 x 764 x 11555, F16 out: 614 us without).
template <typename T>
__device__ __forceinline__ void store_turned(const ProductParams<T> &p, uint64_t row, uint64_t column, uint32_t (&v)[32]) {
    const int lane = threadIdx.x % 32;
#pragma unroll
    for (int s = 16; s; s >>= 1)
#pragma unroll
        for (int j = 0; j < 32; ++j)
            if (!(j & s)) {
                const uint32_t got = __shfl_xor_sync(~0u, lane & s ? v[j] : v[j + s], s);
                if (lane & s) v[j] = got;
                else v[j + s] = got;
            }
    if (column + lane >= p.columns) return;
    T *to = p.out + row * p.out_stride + column + lane;
#pragma unroll
    for (int j = 0; j < 32; ++j) {
        if (row + j >= p.rows) break;
        const T y = Elem<T>::round(__uint_as_float(v[j]));
        to[j * p.out_stride] = y;
        if (const unsigned kind = result_kind(Elem<T>::load(y))) record_fault(p.status, (row + j) * p.columns + column + lane, kind);
    }
}

// Any base and stride: 16 x 16 cells per CTA, one thread per cell.
template <typename T> __global__ void __launch_bounds__(256) product_plain_kernel(const ProductParams<T> p) {
    in_stream_order();
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
        if (r < p.rows && c < p.columns) {
            const BlockFactor f = block_factor(p.left_scales[r * blocks + kb], p.right_scales[c / kBlock * blocks + kb]);
            acc = fmaf(part * f.factor, f.rest, acc);
        }
    }
    if (r < p.rows && c < p.columns) store_cell(p, r, c, acc);
}

// ------------------------------------------------------------------ tensor core product
//
// D = P . Q^T over blocks of 128 of the inner dimension.
//   * batch form (product_kernel): P = left, Q = right.  A pair of CTAs works on 256 x 256 cells, whose sums over
//     all blocks, scaled by the tensor cores, stay in TMEM.
//   * row form (product_rows_kernel), few rows: P = right, Q = left, 128 columns x BN rows, so that
//     the weights, which are all the traffic there is, fill the instruction's 128 rows.  The blocks
//     of one tile are split over a cluster's CTAs, which then add a share of the cells each, in rank order.  Each
//     block's product goes to a TMEM buffer of its own and is added, scaled, to sums in registers.
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

// True in one lane, always the same.  The warp that issues tensor core work runs its loop as a whole,
// so that descriptors stay in uniform registers, and elects a lane for the instructions themselves;
// a loop of one lane alone took 600 cycles to issue a block's eight products, which take 512.
__device__ __forceinline__ bool elect_one() {
    uint32_t elected;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(elected));
    return elected != 0;
}

// The barrier completes when all tensor core work issued before by this thread has.
__device__ __forceinline__ void mma_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar))
                 : "memory");
}

// This thread's lane and the columns from `address` on.
__device__ __forceinline__ void tmem_load(uint32_t (&v)[16], uint32_t address) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, "
        "%8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(address));
}
__device__ __forceinline__ void tmem_load(uint32_t (&v)[32], uint32_t address) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
          "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
          "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
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
__device__ __forceinline__ void tmem_wait(uint32_t (&v)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]),
                   "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]),
                   "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]),
                   "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31])
                 :
                 : "memory");
}

// A whole warp waits, with one answer.
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity) {
    return __all_sync(~0u, mbar_wait(bar, parity));
}

// What both forms take.  Tiles come in groups of 8 tile rows, column by column inside a group, so
// that the tiles worked on at once share a few panels of both operands in L2.
template <typename T> struct TileParams {
    ProductParams<T> out;
    uint64_t p_rows, q_rows;  // extents along the tile's rows and columns
    const float *p_scales, *q_scales;
    unsigned tiles_p, tiles_q, tiles;
    int blocks;  // of 128 along the inner dimension
};

template <typename T>
__device__ __forceinline__ void tile_place(const TileParams<T> &t, unsigned id, unsigned &p, unsigned &q) {
    const unsigned group = id / (8 * t.tiles_q) * 8, rows = min(8u, t.tiles_p - group), in = id - group * t.tiles_q;
    p = group + in % rows;
    q = in / rows;
}

// ---- batch form
//
// A pair of CTAs (a cluster of 2) owns 256 x 256 cells: each holds 128 rows of P and half of Q's rows,
// and one tcgen05.mma of the pair reads both, so each SM brings 32 KB per block of 128 from L2 where a
// CTA by itself, with 128 x 256 cells, brings 48 KB (and was bound by that, at 10 TB/s of L2 reads).  The
// scales are powers of two, so the tensor cores apply them (kind::mxf8f6f4, an exponent byte for each
// 32 codes: a block's byte four times) and sum over all blocks in TMEM.  Scales of any kind had to be
// applied in registers, a block's product at a time: that drained 256 KB of TMEM per pair and block, and
// ran at 36 % of the tensor cores' rate (165 us for 8192 x 4096 x 4096) however the drain was spread.
// 8192 x 4096 x 4096, BF16 out: 110 us = 2.5 PFLOP/s, tensor pipe 65 % busy; bound by the feed from L2 (every SM
// brings 32 KB per 512 cycles of products) and by the sums' way out, when the next tile's products wait for TMEM: the
// sums take half of it, two tiles' would leave no columns for the exponents.
// With few tiles, tiles of 256 x 64 (see product_typed).
// Warps: 0 TMA loads, 1 tcgen05.cp of the exponents and tcgen05.mma (first CTA only), 2 and 3 exponents
// into shared memory, 4 to 11 bring the sums to registers, 128 columns each, give TMEM back and store.
template <int BN_> struct Batch {
    static constexpr int HALF = 128, BM = 2 * HALF, BN = BN_;
    static constexpr int PIECES = (BN + 127) / 128;  // of 128 columns, or one of fewer
    static constexpr int EPILOGUE = 8, COLUMNS = BN / (EPILOGUE / 4), THREADS = (4 + EPILOGUE) * 32;
    static constexpr int P_BYTES = HALF * kBlock, Q_BYTES = BN / 2 * kBlock, STAGE_BYTES = P_BYTES + Q_BYTES;
    static constexpr int STAGES = 6;
    // exponents: 512 bytes per 128 rows and block, CHUNK blocks at a time, two chunks
    static constexpr int CHUNK = 8, EXPONENTS = 512 * (1 + PIECES);
    static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + 2 * CHUNK * EXPONENTS + 1024;
    // TMEM columns: the sums, then the exponents of four blocks (4 columns per 128 rows)
    static constexpr int TMEM_COLUMNS = 512, SCALES_AT = BN, SCALES_STEP = 16, SCALES = 4;
    static_assert(SCALES_AT + SCALES * SCALES_STEP <= TMEM_COLUMNS && 4 * (1 + PIECES) <= SCALES_STEP, "TMEM");
};

// A load by either CTA of a pair that signals the first CTA's barrier.
__device__ __forceinline__ void tma_load_pair(void *dst, const CUtensorMap *map, uint32_t bar, int x, int y) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 "
        "[%0], [%1, {%3, %4}], [%2];" ::"r"(smem_addr(dst)),
        "l"(map), "r"(bar), "r"(x), "r"(y)
        : "memory");
}

// D (binary32, TMEM of both CTAs) = or += A . B^T for 256 x N x 32 codes with their exponents in TMEM
__device__ __forceinline__ void mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t shape, uint32_t sa, uint32_t sb,
                                         uint32_t add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(shape), "r"(sa), "r"(sb), "r"(add)
        : "memory");
}

// 32 rows of 16 bytes (512 adjacent bytes) of each CTA's shared memory to 4 columns of its TMEM, to each
// quarter of the lanes.  In order with the products issued before and after it.
__device__ __forceinline__ void exponents_to_tmem(uint32_t to, uint32_t from) {
    // no swizzle, 8 x 16-byte pieces 128 bytes apart, descriptor version 1
    const uint64_t desc = (uint64_t)(from >> 4) | (uint64_t)(128 >> 4) << 16 | (uint64_t)(128 >> 4) << 32 | (uint64_t)1 << 46;
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(to), "l"(desc) : "memory");
}

// The barrier at this place in both CTAs completes when the pair's tensor core work issued before has.
__device__ __forceinline__ void mma_commit_pair(uint64_t *bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_addr(bar)),
        "h"((uint16_t)3)
        : "memory");
}

// An arrival at a barrier of any CTA of the cluster.  Relaxed for TMEM that has been read: nothing in memory
// is handed over (the loads have ended and tcgen05.fence orders them), and a release at cluster scope
// waits for all of the thread's memory accesses, 1,000 cycles here.
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_release_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// A scale's exponent byte, four times.  What is no power of two from 2^-126 on gives NaN.
__device__ __forceinline__ uint32_t exponent_word(float scale) {
    const uint32_t bits = __float_as_uint(scale), e = bits >> 23;
    return ((bits & 0x807fffffu) == 0 && e >= 1 && e <= 254 ? e : 0xffu) * 0x01010101u;
}

template <typename T, typename S>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(S::THREADS, 1)
    product_kernel(const __grid_constant__ CUtensorMap map_p, const __grid_constant__ CUtensorMap map_q,
                   const __grid_constant__ TileParams<T> t) {
    const ProductParams<T> &p = t.out;
    in_stream_order();
    if (!chain_admits(p.guard)) return;  // the same answer in every CTA of the grid
    extern __shared__ unsigned char smem_raw[];
    unsigned char *const tiles = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
    uint32_t *const exponents = reinterpret_cast<uint32_t *>(tiles + S::STAGES * S::STAGE_BYTES);
    __shared__ uint64_t full[S::STAGES], empty[S::STAGES], scaled[2], spent[2], ready, drained, finished;
    __shared__ uint32_t tmem_base;
    const int warp = __shfl_sync(~0u, threadIdx.x / 32, 0), lane = threadIdx.x % 32;  // uniform, for the compiler too
    const uint32_t rank = cluster_rank();
    const unsigned first = blockIdx.x / 2, step = gridDim.x / 2;
    const int KB = t.blocks;

    if (threadIdx.x == 0) {
        for (int i = 0; i < S::STAGES; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], 1);
        for (int i = 0; i < 2; ++i) mbar_init(&scaled[i], 4), mbar_init(&spent[i], 1);
        mbar_init(&ready, 1), mbar_init(&drained, 2 * S::EPILOGUE), mbar_init(&finished, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_base)),
                     "r"(S::TMEM_COLUMNS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    cluster_sync();  // the other CTA's barriers are initialised and its TMEM is allocated
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = __shfl_sync(~0u, tmem_base, 0);

    if (warp == 0) {
        if (lane == 0) {
            int it = 0;
            bool ok = true;
            for (unsigned id = first; ok && id < t.tiles; id += step) {
                unsigned tp, tq;
                tile_place(t, id, tp, tq);
                const int p0 = (int)(tp * S::BM + rank * S::HALF), q0 = (int)(tq * S::BN + rank * (S::BN / 2));
                for (int kb = 0; kb < KB; ++kb, ++it) {
                    const int s = it % S::STAGES;
                    if (!(ok = mbar_wait(&empty[s], ((it / S::STAGES) & 1) ^ 1))) break;
                    unsigned char *to = tiles + s * S::STAGE_BYTES;
                    const uint32_t bar = cluster_address(smem_addr(&full[s]), 0);
                    if (rank == 0) mbar_expect_tx(&full[s], 2 * S::STAGE_BYTES);  // both CTAs' loads
                    tma_load_pair(to, &map_p, bar, kb * kBlock, p0);
                    tma_load_pair(to + S::P_BYTES, &map_q, bar, kb * kBlock, q0);
                }
            }
            if (!ok) record_fault(p.status, 0, kWatchdog);
            // Nothing is left in flight towards either CTA's shared memory when the pair ends.
            if (rank == 0)
                for (int i = it > S::STAGES ? it - S::STAGES : 0; i < it; ++i)
                    mbar_wait(&full[i % S::STAGES], (i / S::STAGES) & 1);
        }
    } else if (warp == 1) {
        // The whole warp runs the loop, so that descriptors stay in uniform registers; one lane issues.
        if (rank == 0) {
            constexpr uint32_t shape = 1u << 23 | (uint32_t)(S::BN / 8) << 17 | (uint32_t)(S::BM / 16) << 24;
            const uint32_t stage0 = smem_addr(tiles), exponents0 = smem_addr(exponents);
            int it = 0, chunk = 0, tile = 0;
            bool ok = true;
            for (unsigned id = first; ok && id < t.tiles; id += step, ++tile) {
                ok = __all_sync(~0u, mbar_wait_cluster(&drained, (tile & 1) ^ 1));
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                for (int kb = 0; ok && kb < KB; ++kb, ++it) {
                    const int s = it % S::STAGES, in = kb % S::CHUNK, c = chunk & 1;
                    if (in == 0 && !(ok = __all_sync(~0u, mbar_acquire_cluster(&scaled[c], (chunk / 2) & 1)))) break;
                    if (!(ok = warp_wait(&full[s], (it / S::STAGES) & 1))) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint64_t pd = k_major_descriptor(stage0 + s * S::STAGE_BYTES), qd = pd + (S::P_BYTES >> 4);
                    const uint32_t scales = tmem + S::SCALES_AT + it % S::SCALES * S::SCALES_STEP;
                    const uint32_t from = exponents0 + (c * S::CHUNK + in) * S::EXPONENTS;
                    if (elect_one()) {
#pragma unroll
                        for (int i = 0; i < 1 + S::PIECES; ++i) exponents_to_tmem(scales + 4 * i, from + 512 * i);
#pragma unroll
                        for (int k = 0; k < kBlock / 32; ++k)  // 32 bytes further along the swizzled rows
                            mma_pair(tmem, pd + 2 * k, qd + 2 * k, shape, scales, scales + 4, kb > 0 || k > 0);
                        mma_commit_pair(&empty[s]);
                        if (in == S::CHUNK - 1 || kb == KB - 1) mma_commit_pair(&spent[c]);
                        if (kb == KB - 1) mma_commit_pair(&ready);
                    }
                    __syncwarp();
                    if (in == S::CHUNK - 1 || kb == KB - 1) ++chunk;
                }
            }
            if (elect_one()) mma_commit_pair(&finished);
            __syncwarp();
            ok = warp_wait(&finished, 0) && ok;
            if (!ok && lane == 0) record_fault(p.status, 0, kWatchdog);
        }
    } else if (warp < 4) {
        // Word (r % 32) * 4 + r / 32 of a piece is row r's exponent.  A warp takes half of this CTA's rows of P,
        // 4 rows by 8 adjacent blocks a load, and one piece of Q, whose rows share a scale.
        const int half = warp - 2, in = lane % S::CHUNK;
        const uint32_t scaled0 = cluster_address(smem_addr(&scaled[0]), 0);
        int chunk = 0;
        bool ok = true;
        for (unsigned id = first; ok && id < t.tiles; id += step) {
            unsigned tp, tq;
            tile_place(t, id, tp, tq);
            const uint64_t row0 = (uint64_t)tp * S::BM + rank * S::HALF + half * (S::HALF / 2);
            const uint64_t column_block = (uint64_t)tq * S::BN / 128 + half;
            for (int k0 = 0; k0 < KB; k0 += S::CHUNK, ++chunk) {
                const int c = chunk & 1, kb = k0 + in;
                if (!(ok = warp_wait(&spent[c], ((chunk / 2) & 1) ^ 1))) break;
                uint32_t *slot = exponents + (c * S::CHUNK + in) * (S::EXPONENTS / 4);
#pragma unroll
                for (int r = lane / S::CHUNK; r < S::HALF / 2; r += 32 / S::CHUNK) {
                    const int local = half * (S::HALF / 2) + r;
                    slot[local % 32 * 4 + local / 32] =
                        exponent_word(kb < KB && row0 + r < t.p_rows ? t.p_scales[(row0 + r) * KB + kb] : 1.0f);
                }
                const uint32_t word =
                    exponent_word(kb < KB && column_block * kBlock < t.q_rows ? t.q_scales[column_block * KB + kb] : 1.0f);
#pragma unroll
                for (int b = 0; b < S::CHUNK && half < S::PIECES; ++b) {
                    const uint32_t w = __shfl_sync(~0u, word, b);
                    uint32_t *piece = exponents + (c * S::CHUNK + b) * (S::EXPONENTS / 4) + 128 * (1 + half);
                    reinterpret_cast<uint4 *>(piece)[lane] = make_uint4(w, w, w, w);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // tcgen05.cp reads them
                __syncwarp();
                if (lane == 0) mbar_release_cluster(scaled0 + 8 * c);
            }
        }
        if (!ok && lane == 0) record_fault(p.status, 0, kWatchdog);
    } else {
        const int quarter = warp % 4, local = quarter * 32 + lane;  // this thread's row of the CTA's half
        const int from = (warp - 4) / 4 * S::COLUMNS;               // its first column
        const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16) + from;
        const uint32_t drained0 = cluster_address(smem_addr(&drained), 0);
        const bool pieces = ((reinterpret_cast<uintptr_t>(p.out) | p.out_stride * sizeof(T)) & 31) == 0;  // all rows alike
        int tile = 0;
        bool ok = true;
        for (unsigned id = first; id < t.tiles; id += step, ++tile) {
            if (!(ok = warp_wait(&ready, tile & 1))) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            uint32_t v[S::COLUMNS / 32][32];
#pragma unroll
            for (int i = 0; i < S::COLUMNS / 32; ++i) tmem_load(v[i], lanes + 32 * i);
#pragma unroll
            for (int i = 0; i < S::COLUMNS / 32; ++i) tmem_wait(v[i]);
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(drained0);  // the next tile's products may begin
            unsigned tp, tq;
            tile_place(t, id, tp, tq);
            const uint64_t row = (uint64_t)tp * S::BM + rank * S::HALF + local;
            if (!pieces) {
#pragma unroll
                for (int i = 0; i < S::COLUMNS / 32; ++i)
                    store_turned<T>(p, row - lane, (uint64_t)tq * S::BN + from + 32 * i, v[i]);
            } else if (row < t.p_rows) {
#pragma unroll
                for (int i = 0; i < S::COLUMNS / 32; ++i) store_row<T, 32>(p, row, (uint64_t)tq * S::BN + from + 32 * i, v[i]);
            }
        }
        if (!ok && lane == 0) record_fault(p.status, 0, kWatchdog);
    }

    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    cluster_sync();  // the pair's products and arrivals are done in both CTAs
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::TMEM_COLUMNS) : "memory");
}

// ---- row form
//
// 1 x 4096 x 16384 with its quantiser: 18.8 us for 64 MB of codes (17.2 behind other passes), 10.3 of them at a copy's
// rate; 32 rows 24.7 (21.3).  Two CTAs an SM with 5 blocks of 18 KB in flight each.  What is left is the way in and out
// (two launches, TMEM, the first loads, the cluster's sums): six stages, or three CTAs an SM with four, leave one row
// at 18.7 to 19.0 us.
template <int BN_> struct Rows {
    static constexpr int BM = 128, BN = BN_, BUFFERS = 4, EPILOGUE = 4, THREADS = (2 + EPILOGUE) * 32;
    static constexpr int TMEM_COLUMNS = BUFFERS * BN;
    static constexpr int P_BYTES = BM * kBlock, Q_BYTES = BN * kBlock, STAGE_BYTES = P_BYTES + Q_BYTES;
    static constexpr int STAGES = 5;
    static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + 1024;
    static_assert(BN <= 32, "a column's factor is kept in a lane");
    static_assert(BM * BN * 4 <= STAGES * STAGE_BYTES, "the sums take the stages' place");
};

template <typename T, typename S>
__global__ void __launch_bounds__(S::THREADS)
    product_rows_kernel(const __grid_constant__ CUtensorMap map_p, const __grid_constant__ CUtensorMap map_q,
                        const __grid_constant__ TileParams<T> t) {
    const ProductParams<T> &p = t.out;
    in_stream_order();
    if (!chain_admits(p.guard)) return;  // the same answer in every CTA of the grid
    extern __shared__ unsigned char smem_raw[];
    unsigned char *const tiles = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
    __shared__ uint64_t full[S::STAGES], empty[S::STAGES], ready[S::BUFFERS], drained[S::BUFFERS], finished;
    __shared__ uint32_t tmem_base;
    const int warp = __shfl_sync(~0u, threadIdx.x / 32, 0), lane = threadIdx.x % 32;  // uniform, for the compiler too
    // blocks [kb0, kb1) of the inner dimension: this CTA's share
    uint32_t ranks;
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
    const uint32_t rank = cluster_rank();
    const int kb0 = (int)((int64_t)t.blocks * rank / ranks), kb1 = (int)((int64_t)t.blocks * (rank + 1) / ranks);
    unsigned tp, tq;
    tile_place(t, blockIdx.x / ranks, tp, tq);
    const int p0 = (int)(tp * S::BM), q0 = (int)(tq * S::BN);

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
    const uint32_t tmem = __shfl_sync(~0u, tmem_base, 0);

    if (warp == 0) {
        if (lane == 0) {
            int it = 0;
            bool ok = true;
            for (int kb = kb0; kb < kb1; ++kb, ++it) {
                const int s = it % S::STAGES;
                if (!(ok = mbar_wait(&empty[s], ((it / S::STAGES) & 1) ^ 1))) break;
                unsigned char *to = tiles + s * S::STAGE_BYTES;
                mbar_expect_tx(&full[s], S::STAGE_BYTES);
                tma_load_2d(to, &map_p, &full[s], kb * kBlock, p0);
                tma_load_2d(to + S::P_BYTES, &map_q, &full[s], kb * kBlock, q0);
            }
            if (!ok) record_fault(p.status, 0, kWatchdog);
            // nothing is left in flight towards this CTA's shared memory when it ends
            for (int i = it > S::STAGES ? it - S::STAGES : 0; i < it; ++i)
                mbar_wait(&full[i % S::STAGES], (i / S::STAGES) & 1);
        }
    } else if (warp == 1) {
        constexpr uint32_t shape = 1u << 4 | (uint32_t)(S::BN / 8) << 17 | (uint32_t)(S::BM / 16) << 24;
        const uint32_t stage0 = smem_addr(tiles);
        int it = 0;
        bool ok = true;
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
            const int s = it % S::STAGES, b = it % S::BUFFERS;
            if (!(ok = warp_wait(&drained[b], ((it / S::BUFFERS) & 1) ^ 1) && warp_wait(&full[s], (it / S::STAGES) & 1)))
                break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint64_t pd = k_major_descriptor(stage0 + s * S::STAGE_BYTES), qd = pd + (S::P_BYTES >> 4);
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < kBlock / 32; ++k)  // 32 bytes further along the swizzled rows
                    mma_e4m3(tmem + b * S::BN, pd + 2 * k, qd + 2 * k, shape, k != 0);
                mma_commit(&empty[s]);
                mma_commit(&ready[b]);
            }
            __syncwarp();
        }
        if (elect_one()) mma_commit(&finished);
        __syncwarp();
        ok = warp_wait(&finished, 0) && ok;
        if (!ok && lane == 0) record_fault(p.status, 0, kWatchdog);
    } else {
        const int quarter = warp % 4, local = quarter * 32 + lane;  // this thread's row of the tile
        const uint64_t row = (uint64_t)p0 + local;
        // Lane c holds both operands' scales for the tile's column c, AHEAD blocks ahead: a load that misses
        // takes longer than a block.
        constexpr int AHEAD = 4;
        float sum[S::BN], p_scale[AHEAD], q_scale[AHEAD];
        const bool there = lane < S::BN && (uint64_t)q0 + lane < t.q_rows;
        auto fetch = [&](int kb, float &ps, float &qs) {
            ps = qs = 1.0f;
            if (kb < kb1 && there)
                ps = t.p_scales[(uint64_t)tp * t.blocks + kb], qs = t.q_scales[((uint64_t)q0 + lane) * t.blocks + kb];
        };
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) fetch(kb0 + i, p_scale[i], q_scale[i]);
#pragma unroll
        for (int i = 0; i < S::BN; ++i) sum[i] = 0;
        int it = 0;
        bool ok = true;
        static_assert(AHEAD == S::BUFFERS, "a block's place in the scales' ring is its buffer");
        for (int kb = kb0; ok && kb < kb1;) {
#pragma unroll
            for (int b = 0; b < S::BUFFERS; ++b) {
                if (!ok || kb >= kb1) break;
                const BlockFactor f = block_factor(q_scale[b], p_scale[b]);
                fetch(kb + AHEAD, p_scale[b], q_scale[b]);
                if (!(ok = warp_wait(&ready[b], (it / S::BUFFERS) & 1))) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                uint32_t v[S::BN];
                tmem_load(v, tmem + ((uint32_t)(quarter * 32) << 16) + b * S::BN);
                tmem_wait(v);
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&drained[b]);
                if (__any_sync(~0u, f.rest != 1.0f)) {
#pragma unroll
                    for (int i = 0; i < S::BN; ++i)
                        sum[i] = fmaf(__uint_as_float(v[i]) * __shfl_sync(~0u, f.factor, i), __shfl_sync(~0u, f.rest, i), sum[i]);
                } else {
#pragma unroll
                    for (int i = 0; i < S::BN; ++i)
                        sum[i] = fmaf(__uint_as_float(v[i]), __shfl_sync(~0u, f.factor, i), sum[i]);
                }
                ++kb, ++it;
            }
        }
        if (!ok) {
            if (lane == 0) record_fault(p.status, 0, kWatchdog);
        } else if (ranks == 1) {
#pragma unroll
            for (int i = 0; i < S::BN; ++i)
                if (row < t.p_rows && (uint64_t)q0 + i < t.q_rows) store_cell(p, (uint64_t)q0 + i, row, sum[i]);
        } else {  // for the cluster; every load and product of this CTA is done
#pragma unroll
            for (int i = 0; i < S::BN; ++i) reinterpret_cast<float *>(tiles)[i * S::BM + local] = sum[i];
        }
    }

    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::TMEM_COLUMNS) : "memory");
    if (ranks > 1) {
        cluster_sync();  // each CTA's sums are in its own shared memory
        // Every CTA adds a share of the cells, in rank order; the reads of a cell's sums go out together.
        for (int i = rank * S::THREADS + threadIdx.x; i < S::BM * S::BN; i += ranks * S::THREADS) {
            const uint64_t column = (uint64_t)p0 + i % S::BM, row = (uint64_t)q0 + i / S::BM;
            if (column >= t.p_rows || row >= t.q_rows) continue;
            float part[8], total = 0;
#pragma unroll
            for (uint32_t r = 0; r < 8; ++r) {
                part[r] = 0;
                if (r < ranks) cluster_read(part[r], smem_addr(tiles) + 4 * i, r);
            }
#pragma unroll
            for (uint32_t r = 0; r < 8; ++r) total += part[r];
            store_cell(p, row, column, total);
        }
        __syncwarp();
        cluster_sync();  // and stay until they have been read
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
        return pcu_host::launch_grid(quantize_kernel<T, 1>, (unsigned)((blocks + kRows - 1) / kRows), kQuantizeThreads, stream, p);
    return pcu_host::launch_grid(quantize_kernel<T, kBlock>, (unsigned)blocks, kQuantizeThreads, stream, p);
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

template <typename T> static TileParams<T> tile_params(const ProductParams<T> &p, bool row_form, int bm, int bn) {
    TileParams<T> t{};
    t.out = p;
    t.p_rows = row_form ? p.columns : p.rows;
    t.q_rows = row_form ? p.rows : p.columns;
    t.p_scales = row_form ? p.right_scales : p.left_scales;
    t.q_scales = row_form ? p.left_scales : p.right_scales;
    t.tiles_p = (unsigned)((t.p_rows + bm - 1) / bm);
    t.tiles_q = (unsigned)((t.q_rows + bn - 1) / bn);
    t.tiles = t.tiles_p * t.tiles_q;
    t.blocks = (int)((p.inner + kBlock - 1) / kBlock);
    return t;
}

template <typename T, typename S>
static int launch_batch(const ProductParams<T> &p, const CUtensorMap &left, const CUtensorMap &right, cudaStream_t stream) {
    if (const int rc = pcu_host::allow_shared<product_kernel<T, S>>(S::SMEM_BYTES)) return rc;
    const TileParams<T> t = tile_params(p, false, S::BM, S::BN);
    const unsigned pairs = std::min(t.tiles, (unsigned)std::max(1, pcu_host::sm_count() / 2));
    return pcu_host::launch_cluster(product_kernel<T, S>, 2 * pairs, S::THREADS, S::SMEM_BYTES, 0, stream, left, right, t);
}

template <typename T, typename S>
static int launch_rows(const ProductParams<T> &p, const CUtensorMap &left, const CUtensorMap &right, cudaStream_t stream) {
    if (const int rc = pcu_host::allow_shared<product_rows_kernel<T, S>>(S::SMEM_BYTES)) return rc;
    const TileParams<T> t = tile_params(p, true, S::BM, S::BN);
    unsigned ranks = 1;
    while (ranks < 8 && t.tiles * ranks * 2 <= 2 * (uint64_t)pcu_host::sm_count() && (unsigned)t.blocks >= 8 * ranks) ranks *= 2;
    return pcu_host::launch_cluster(product_rows_kernel<T, S>, t.tiles * ranks, S::THREADS, S::SMEM_BYTES, ranks, stream,
                                    right, left, t);
}

template <typename T> static int product_typed(const ProductParams<T> &p, cudaStream_t stream) {
    CUtensorMap left, right;
    if (p.inner && p.rows <= 32) {
        const bool few = p.rows <= 16;
        if (code_map(&right, p.right, p.columns, p.inner, p.right_stride, 128) &&
            code_map(&left, p.left, p.rows, p.inner, p.left_stride, few ? 16 : 32))
            return few ? launch_rows<T, Rows<16>>(p, left, right, stream) : launch_rows<T, Rows<32>>(p, left, right, stream);
    } else if (p.inner) {
        // Tiles of 256 x 64 while all of them run at once: each takes some 0.6 of a 256 x 256 tile's time.
        const uint64_t narrow = (p.rows + 255) / 256 * ((p.columns + 63) / 64);
        const bool few = narrow <= (uint64_t)pcu_host::sm_count() / 2;
        if (code_map(&left, p.left, p.rows, p.inner, p.left_stride, 128) &&
            code_map(&right, p.right, p.columns, p.inner, p.right_stride, few ? 32 : 128))
            return few ? launch_batch<T, Batch<64>>(p, left, right, stream) : launch_batch<T, Batch<256>>(p, left, right, stream);
    }
    const uint64_t tiles = (p.rows + 15) / 16 * ((p.columns + 15) / 16);
    return pcu_host::launch_grid(product_plain_kernel<T>, (unsigned)tiles, 256, stream, p);
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
    if (!pcu_host::aligned(input, pcu_host::element_bytes(dtype)) || !pcu_host::aligned(scales, 4) || !pcu_host::aligned(status, 8))
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
    if (!pcu_host::aligned(out, pcu_host::element_bytes(out_dtype)) || !pcu_host::aligned(left_scales, 4) ||
        !pcu_host::aligned(right_scales, 4) || !pcu_host::aligned(status, 8))
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

// block_matmul.cu -- 8-bit block quantiser and the product of block-scaled 8-bit operands.
#include <cuda_fp8.h>

#include "learn.cuh"
#include "provider.h"

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

// value * (1 / scale), exact: the reciprocal of a power of two >= 2^-126 is one <= 2^126
__device__ __forceinline__ unsigned to_e4m3(float v, float inverse) {
    return isfinite(v) ? (unsigned)__nv_cvt_float_to_fp8(v * inverse, __NV_SATFINITE, __NV_E4M3) : 0x7fu;
}

template <typename T> struct QuantizeParams {
    const T *input;
    uint64_t rows, columns, stride;
    int high;
    unsigned char *codes;
    uint64_t codes_stride;
    float *scales;
    unsigned long long *status;
    ChainGuard guard;
};

// One CTA per block.
template <typename T> __global__ void __launch_bounds__(kBlock) quantize_kernel(const QuantizeParams<T> p) {
    if (!chain_admits(p.guard)) return;
    __shared__ float scratch[kBlock / 32];
    const uint64_t kb = blockIdx.x % ((p.columns + kBlock - 1) / kBlock), rb = blockIdx.x / ((p.columns + kBlock - 1) / kBlock);
    const uint64_t c = kb * kBlock + threadIdx.x, r0 = rb * p.high, r1 = min(r0 + p.high, p.rows);
    float amax = 0;
    if (c < p.columns)
        for (uint64_t r = r0; r < r1; ++r) {
            const float v = fabsf(Elem<T>::load(p.input[r * p.stride + c]));
            if (isfinite(v)) amax = fmaxf(amax, v);
            else record_fault(p.status, r * p.columns + c, PCU_B200_KIND_INVALID);
        }
    for (int o = 16; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, o));
    if (threadIdx.x % 32 == 0) scratch[threadIdx.x / 32] = amax;
    __syncthreads();
    const float scale = block_scale(fmaxf(fmaxf(scratch[0], scratch[1]), fmaxf(scratch[2], scratch[3])));
    if (threadIdx.x == 0) p.scales[blockIdx.x] = scale;
    if (c < p.columns)
        for (uint64_t r = r0; r < r1; ++r)
            p.codes[r * p.codes_stride + c] =
                (unsigned char)to_e4m3(Elem<T>::load(p.input[r * p.stride + c]), 1.0f / scale);
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

template <typename T>
static int quantize_typed(const void *input, uint64_t rows, uint64_t columns, uint64_t stride, int high, void *codes,
                          uint64_t codes_stride, float *scales, uint64_t *status, cudaStream_t stream,
                          const ChainGuard &guard) {
    QuantizeParams<T> p{(const T *)input, rows, columns, stride, high, (unsigned char *)codes, codes_stride, scales,
                        reinterpret_cast<unsigned long long *>(status), guard};
    const uint64_t blocks = (rows + high - 1) / high * ((columns + kBlock - 1) / kBlock);
    quantize_kernel<T><<<(unsigned)blocks, kBlock, 0, stream>>>(p);
    return pcu_host::launch_status();
}

template <typename T> static int product_typed(ProductParams<T> p, cudaStream_t stream) {
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

// learn.cuh -- element types and small helpers shared by the learning operators (distill.cu,
// group_norm.cu, block_matmul.cu).
//
// These operators take binary16 and bfloat16 beside the strict path's binary32 and binary64.
// All arithmetic on the three narrow types is in binary32 and rounds once, where a result is
// stored; binary64 stays binary64 throughout.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>

#include "common.cuh"
#include "pcu_b200_learn.h"

namespace pcu {

template <typename T> struct Elem;
template <> struct Elem<float> {
    using Wide = float;
    static __device__ __forceinline__ float load(float v) { return v; }
    static __device__ __forceinline__ float round(float v) { return v; }
};
template <> struct Elem<double> {
    using Wide = double;
    static __device__ __forceinline__ double load(double v) { return v; }
    static __device__ __forceinline__ double round(double v) { return v; }
};
template <> struct Elem<__half> {
    using Wide = float;
    static __device__ __forceinline__ float load(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half round(float v) { return __float2half_rn(v); }
};
template <> struct Elem<__nv_bfloat16> {
    using Wide = float;
    static __device__ __forceinline__ float load(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 round(float v) { return __float2bfloat16_rn(v); }
};
template <typename T> using WideOf = typename Elem<T>::Wide;

// 2^x.  binary32: the hardware's approximation (2 ulp), results below 2^-126 flushed to zero --
// these are softmax terms, summed with one that is 1.  binary64: the library function.
__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ double fast_exp2(double x) { return exp2(x); }

// The fault kind of a result that has to be finite: 0, Overflow (infinity) or Invalid (NaN).
template <typename W> __device__ __forceinline__ unsigned result_kind(W v) {
    return isfinite(v) ? 0u : (isnan(v) ? (unsigned)PCU_B200_KIND_INVALID : (unsigned)PCU_B200_KIND_OVERFLOW);
}

}  // namespace pcu

namespace pcu_host {

inline size_t element_bytes(int dtype) {
    switch (dtype) {
    case PCU_B200_F32: return 4;
    case PCU_B200_F64: return 8;
    case PCU_B200_F16:
    case PCU_B200_BF16: return 2;
    default: return 0;
    }
}

inline bool multiply_fits(uint64_t a, uint64_t b, uint64_t limit) { return a == 0 || b <= limit / a; }

}  // namespace pcu_host

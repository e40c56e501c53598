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
#include <type_traits>

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

// 16 bytes of elements to wide values and back, two to a word where the types are 16 bits wide.
template <typename T> __device__ __forceinline__ void unpack(uint4 raw, WideOf<T> (&v)[16 / sizeof(T)]) {
#pragma unroll
    for (int i = 0; i < (int)(16 / sizeof(T)); ++i) v[i] = Elem<T>::load(reinterpret_cast<const T *>(&raw)[i]);
}
template <> __device__ __forceinline__ void unpack<__nv_bfloat16>(uint4 raw, float (&v)[8]) {
    const unsigned w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
}
template <> __device__ __forceinline__ void unpack<__half>(uint4 raw, float (&v)[8]) {
    const unsigned w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
        v[2 * i] = f.x, v[2 * i + 1] = f.y;
    }
}

template <typename T> __device__ __forceinline__ uint4 pack(const WideOf<T> (&v)[16 / sizeof(T)]) {
    alignas(16) T r[16 / sizeof(T)];
#pragma unroll
    for (int i = 0; i < (int)(16 / sizeof(T)); ++i) r[i] = Elem<T>::round(v[i]);
    return *reinterpret_cast<const uint4 *>(r);
}
template <> __device__ __forceinline__ uint4 pack<__nv_bfloat16>(const float (&v)[8]) {
    __nv_bfloat162 r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    return *reinterpret_cast<const uint4 *>(r);
}
template <> __device__ __forceinline__ uint4 pack<__half>(const float (&v)[8]) {
    __half2 r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    return *reinterpret_cast<const uint4 *>(r);
}

// The largest of 16 bytes of elements; NaN loses against a number.
template <typename T> __device__ __forceinline__ WideOf<T> largest(uint4 raw, const WideOf<T> (&v)[16 / sizeof(T)]) {
    WideOf<T> top = v[0];
#pragma unroll
    for (int i = 1; i < (int)(16 / sizeof(T)); ++i) top = fmax(top, v[i]);
    return top;
}
template <> __device__ __forceinline__ float largest<__nv_bfloat16>(uint4 raw, const float (&)[8]) {
    const __nv_bfloat162 *w = reinterpret_cast<const __nv_bfloat162 *>(&raw);
    const __nv_bfloat162 m = __hmax2(__hmax2(w[0], w[1]), __hmax2(w[2], w[3]));
    return fmaxf(__low2float(m), __high2float(m));
}
template <> __device__ __forceinline__ float largest<__half>(uint4 raw, const float (&)[8]) {
    const __half2 *w = reinterpret_cast<const __half2 *>(&raw);
    const __half2 m = __hmax2(__hmax2(w[0], w[1]), __hmax2(w[2], w[3]));
    return fmaxf(__low2float(m), __high2float(m));
}

// Not 0 where an element of the 16 bytes is an infinity or a NaN: a full exponent field, the largest,
// carries into the sign's place when one is added to it.
template <typename T> __device__ __forceinline__ unsigned not_finite(uint4 raw) {
    constexpr unsigned field = sizeof(T) == 2 ? (std::is_same<T, __half>::value ? 0x7c007c00u : 0x7f807f80u)
                               : sizeof(T) == 4 ? 0x7f800000u : 0x7ff00000u;
    constexpr unsigned one = sizeof(T) == 2 ? (std::is_same<T, __half>::value ? 0x04000400u : 0x00800080u)
                             : sizeof(T) == 4 ? 0x00800000u : 0x00100000u;
    constexpr unsigned sign = sizeof(T) == 2 ? 0x80008000u : 0x80000000u;
    unsigned bad = ((raw.y & field) + one) | ((raw.w & field) + one);
    if (sizeof(T) < 8) bad |= ((raw.x & field) + one) | ((raw.z & field) + one);
    return bad & sign;
}

// First in each kernel: waits for the grids before it in the stream (all of them, with what they wrote), and
// lets the next one's CTAs be placed when all of this grid's are, so that a call's way in runs while the
// call before it finishes.  Every thread passes here, whatever it does next.  What calls read is loaded with
// coherent loads (no __ldg): a kernel is there before its predecessor has written, so its inputs are not constant
// for as long as it runs, which non-coherent loads want.
__device__ __forceinline__ void in_stream_order() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

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

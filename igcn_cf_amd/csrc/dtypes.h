// float32, bfloat16 and float16 values in kernels that take all three (IGCN_DTYPE_*).
#pragma once
#include "common.h"
#include <hip/hip_fp16.h>
#include <hip/hip_bf16.h>

namespace igcn {

template <typename T> __device__ __forceinline__ float to_float(T x);
template <> __device__ __forceinline__ float to_float(float x) { return x; }
template <> __device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_float(__hip_bfloat16 x) { return __uint_as_float((uint32_t)__builtin_bit_cast(uint16_t, x) << 16); }

// to nearest even.  The float32 value is rounded first and for all types alike: left to itself the compiler folds the last product or
// sum into the conversion to float16 (v_fma_mixlo_f16), here and there but not everywhere, and two kernels of one result would differ.
template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float(float x) { return x; }
template <> __device__ __forceinline__ __half from_float(float x) { asm("" : "+v"(x)); return __float2half_rn(x); }
template <> __device__ __forceinline__ __hip_bfloat16 from_float(float x) { return __builtin_bit_cast(__hip_bfloat16, static_cast<__bf16>(x)); }

// N values at once, from and to any address (the hardware moves 16 bytes anywhere); spelled out as vectors, or the compiler takes them apart
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef i32x4 i32x4_any __attribute__((aligned(1)));
typedef i32x2 i32x2_any __attribute__((aligned(1)));
template <typename T, int N> __device__ __forceinline__ void load_vector(T (&x)[N], const T *__restrict__ p)
{
    static_assert(sizeof(x) % 16 == 0 || sizeof(x) == 8, "whole vectors");
    if constexpr (sizeof(x) == 8) {
        const i32x2 w = *reinterpret_cast<const i32x2_any *>(p);
        __builtin_memcpy(x, &w, 8);
    } else {
#pragma unroll
        for (unsigned i = 0; i < sizeof(x) / 16; ++i) {
            const i32x4 w = reinterpret_cast<const i32x4_any *>(p)[i];
            __builtin_memcpy(reinterpret_cast<char *>(x) + 16 * i, &w, 16);
        }
    }
}
template <typename T, int N> __device__ __forceinline__ void store_vector(T *__restrict__ p, const T (&x)[N])
{
    static_assert(sizeof(x) % 16 == 0 || sizeof(x) == 8, "whole vectors");
    if constexpr (sizeof(x) == 8) {
        i32x2 w;
        __builtin_memcpy(&w, x, 8);
        *reinterpret_cast<i32x2_any *>(p) = w;
    } else {
#pragma unroll
        for (unsigned i = 0; i < sizeof(x) / 16; ++i) {
            i32x4 w;
            __builtin_memcpy(&w, reinterpret_cast<const char *>(x) + 16 * i, 16);
            reinterpret_cast<i32x4_any *>(p)[i] = w;
        }
    }
}

// host side: is d a dtype / does p miss the alignment of one value of it
inline bool dtype_ok(int32_t d) { return d == IGCN_DTYPE_F32 || d == IGCN_DTYPE_BF16 || d == IGCN_DTYPE_F16; }
inline bool misaligned(const void *p, int32_t d) { return (reinterpret_cast<uintptr_t>(p) & (d == IGCN_DTYPE_F32 ? 3 : 1)) != 0; }

}  // namespace igcn

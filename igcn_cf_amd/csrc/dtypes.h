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

// host side: is d a dtype / does p miss the alignment of one value of it
inline bool dtype_ok(int32_t d) { return d == IGCN_DTYPE_F32 || d == IGCN_DTYPE_BF16 || d == IGCN_DTYPE_F16; }
inline bool misaligned(const void *p, int32_t d) { return (reinterpret_cast<uintptr_t>(p) & (d == IGCN_DTYPE_F32 ? 3 : 1)) != 0; }

}  // namespace igcn

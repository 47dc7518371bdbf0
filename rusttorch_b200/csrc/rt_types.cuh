// rt_types.cuh — the storage types of the token operators: conversions to and
// from f32; and token ids.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

namespace rt {

using bf16 = __nv_bfloat16;
using f16 = __half;

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(bf16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(f16 x) { return __half2float(x); }

// Rounded to nearest, ties to even (f16: to infinity beyond 65504).
template <class T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ bf16 from_f32<bf16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ f16 from_f32<f16>(float x) { return __float2half_rn(x); }

// Ids and targets: 32- or 64-bit integers, read as 64.
struct IndexArray {
  const void* p;
  bool wide;   // int64
  __device__ __forceinline__ long long operator[](size_t i) const {
    return wide ? static_cast<const long long*>(p)[i]
                : (long long)static_cast<const int*>(p)[i];
  }
};

}  // namespace rt

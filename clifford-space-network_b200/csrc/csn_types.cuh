// csn_types.cuh -- element types of the kernels that take fp32, bf16 or fp16 tensors.
//
// Values are read and written in their own type and computed in float32; a 16-bit pair is one
// 32-bit access.  A store rounds to nearest even once.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace csn {

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }

template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// V neighbouring elements of type T as they lie in memory: one access
template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
  T v[V];
};

// min(sigmoid(z), sigmoid(-z)) = e / (1 + e) with e = exp(-|z|), to full relative precision; the other of the two is
// one minus it.  The fast exponential rounds its argument: off by (4 + 2 |z|) 2^-24 relative, and the quotient by
// 2^-22, which a recurrence sees at random and not as a drift.
__device__ __forceinline__ float sigmoid_small(float z) {
  const float e = __expf(-fabsf(z));
  return __fdividef(e, 1.0f + e);
}

// sigmoid(z); 0 where exp(-z) is too large for float32
__device__ __forceinline__ float sigmoid(float z) { return __fdividef(1.0f, 1.0f + __expf(-z)); }

}  // namespace csn

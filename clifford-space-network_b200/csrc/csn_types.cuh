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

// two floats rounded to a pair of 16-bit numbers, the first in the low half
template <typename T>
__device__ __forceinline__ uint32_t pack(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack<float>(float a, float) { return __float_as_uint(a); }
template <>
__device__ __forceinline__ uint32_t pack<__nv_bfloat16>(float a, float b) {
  __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack<__half>(float a, float b) {
  __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&v);
}

// V neighbouring elements of type T as they lie in memory: one access
template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
  T v[V];
};

// ------------------------------------------------------------- V float32 values
// One or two channels of a lane.
template <int V>
struct Vals {
  float v[V];
  __device__ __forceinline__ float get(int i) const { return v[i]; }
  static __device__ __forceinline__ Vals make(float a, float b) {
    Vals r;
    r.v[0] = a;
    if (V > 1) r.v[V - 1] = b;
    return r;
  }
};
template <int V>
__device__ __forceinline__ Vals<V> splat(float a) { return Vals<V>::make(a, a); }
template <int V>
__device__ __forceinline__ Vals<V> fma(Vals<V> a, Vals<V> b, Vals<V> c) {
#pragma unroll
  for (int i = 0; i < V; ++i) c.v[i] = fmaf(a.v[i], b.v[i], c.v[i]);
  return c;
}
template <int V>
__device__ __forceinline__ Vals<V> operator*(Vals<V> a, Vals<V> b) {
#pragma unroll
  for (int i = 0; i < V; ++i) a.v[i] *= b.v[i];
  return a;
}
template <int V>
__device__ __forceinline__ Vals<V> operator+(Vals<V> a, Vals<V> b) {
#pragma unroll
  for (int i = 0; i < V; ++i) a.v[i] += b.v[i];
  return a;
}
template <int V>
__device__ __forceinline__ Vals<V> operator-(Vals<V> a, Vals<V> b) {
#pragma unroll
  for (int i = 0; i < V; ++i) a.v[i] -= b.v[i];
  return a;
}

// two float32 products, or fused sums of products, or sums in one instruction
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 w, x, y, z;\n\tmov.b64 w, {%2, %3};\n\tmov.b64 x, {%4, %5};\n\tmov.b64 y, {%6, %7};\n\tfma.rn.f32x2 z, w, x, y;\n\t"
      "mov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 twice(float a) { return make_float2(a, a); }

__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float inverse_fast(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
constexpr float LOG2E = 1.4426950408889634f;

// a = sigmoid(z) and q = sigmoid(-z) = 1 / (1 + e) with e = exp(z), which is off by a few units of its own and, since its
// argument is rounded, 2 |z| 2^-24 relative.  The smaller of the two takes that error relative to itself: q as it is, and
// for z < 0 a = e q, so that what a closed gate leaves of a state and its gradients keep their precision (1 - q would
// be off by 2^-25 whatever a is, and 0 from z = -17 on).  For z >= 0 a = 1 - q, rounded once: the long memory of a near 1
// decays without a drift.  exp(z) too large for float32: q = 0, a = 1.
template <int V>
__device__ __forceinline__ void sigmoid_pair(Vals<V> z, Vals<V>& a, Vals<V>& q) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float e = exp2_fast(LOG2E * z.v[i]);
    q.v[i] = inverse_fast(1.0f + e);
    a.v[i] = e < 1.0f ? e * q.v[i] : 1.0f - q.v[i];
  }
}

// sigmoid(z), with the same error; 0 where exp(-z) is too large for float32
__device__ __forceinline__ float sigmoid(float z) { return inverse_fast(1.0f + exp2_fast(-LOG2E * z)); }
template <int V>
__device__ __forceinline__ Vals<V> sigmoid(Vals<V> z) {
#pragma unroll
  for (int i = 0; i < V; ++i) z.v[i] = sigmoid(z.v[i]);
  return z;
}

}  // namespace csn

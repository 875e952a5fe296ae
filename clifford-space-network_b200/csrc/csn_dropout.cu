// csn_dropout.cu -- dropout with the residual add, from a counter-based generator.
//
//   y = residual + keep * x * 65536 / (65536 - cut),   keep = (16 random bits >= cut)
// The bits come from Philox4x32-10 (J. K. Salmon et al., "Parallel random numbers: as easy as 1, 2, 3", SC 2011):
// block j = element / 8 of the flattened tensor is enciphered from the counter (j, offset) under the key `seed`, and
// its 128 bits serve 8 elements with 16 bits each.  A place's bits depend on nothing else, so the backward pass draws
// the mask again (dx = keep * dy * scale is the same kernel without a residual) and no mask is stored.  16 bits an
// element give steps of 2^-16 for the probability, and the scale is that of the probability actually drawn, so the
// mean is exact.
//
// A thread takes whole blocks of 8, in 16-byte accesses.  Bound by memory: 32768 x 2048 bf16 with residual and backward
// 131 us, 5.1 TB/s.
#include <cstdint>

#include "csn_internal.h"
#include "csn_types.cuh"

namespace csn {
namespace {

__device__ __forceinline__ uint4 philox4x32(uint4 c, uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint32_t h0 = __umulhi(0xD2511F53u, c.x), l0 = 0xD2511F53u * c.x;
    const uint32_t h1 = __umulhi(0xCD9E8D57u, c.z), l1 = 0xCD9E8D57u * c.z;
    c = make_uint4(h1 ^ c.y ^ k0, l1, h0 ^ c.w ^ k1, l0);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return c;
}

// 8 neighbouring elements, as the words that they lie in
template <typename T>
struct Block8 {
  static constexpr int N = 2 * (int)sizeof(T);
  uint32_t w[N];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const uint4 q = __ldg(reinterpret_cast<const uint4*>(p) + i / 4);
      w[i] = q.x, w[i + 1] = q.y, w[i + 2] = q.z, w[i + 3] = q.w;
    }
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < N; i += 4)
      reinterpret_cast<uint4*>(p)[i / 4] = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
  }
  // elements 2 i and 2 i + 1
  __device__ __forceinline__ float2 get(int i) const;
  __device__ __forceinline__ void set(int i, float a, float b) {
    if (sizeof(T) == 4) w[N / 4 * i] = __float_as_uint(a), w[N / 4 * i + N / 4 - 1] = __float_as_uint(b);
    else w[i] = pack<T>(a, b);
  }
};
template <>
__device__ __forceinline__ float2 Block8<float>::get(int i) const {
  return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
}
template <>
__device__ __forceinline__ float2 Block8<__nv_bfloat16>::get(int i) const {
  return make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 Block8<__half>::get(int i) const {
  return __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
}

// x * scale where the place is kept; a dropped one is 0 whatever stood there, an infinity or a NaN too
__device__ __forceinline__ float kept(uint32_t bits, uint32_t cut, float x, float scale) {
  return bits >= cut ? x * scale : 0.0f;
}

template <typename T, bool RES>
__global__ void __launch_bounds__(256) dropout_add_kernel(const T* __restrict__ x, const T* __restrict__ res,
                                                          const int64_t* __restrict__ rng, T* __restrict__ y,
                                                          int64_t n, uint32_t cut, float scale) {
  const uint64_t seed = (uint64_t)rng[0], off = (uint64_t)rng[1];
  auto draw = [&](int64_t j) {
    return philox4x32(make_uint4((uint32_t)j, (uint32_t)((uint64_t)j >> 32), (uint32_t)off, (uint32_t)(off >> 32)),
                      (uint32_t)seed, (uint32_t)(seed >> 32));
  };
  const int64_t whole = n / 8;
  for (int64_t j = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; j < whole; j += (int64_t)gridDim.x * blockDim.x) {
    Block8<T> xv, rv;
    xv.load(x + j * 8);
    if (RES) rv.load(res + j * 8);
    const uint4 w = draw(j);
    const uint32_t word[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = xv.get(i), r = RES ? rv.get(i) : make_float2(0.0f, 0.0f);
      const float a = kept(word[i] & 0xffffu, cut, v.x, scale), b = kept(word[i] >> 16, cut, v.y, scale);
      xv.set(i, RES ? r.x + a : a, RES ? r.y + b : b);
    }
    xv.store(y + j * 8);
  }
  if (blockIdx.x == 0 && threadIdx.x < n % 8) {  // the last, short block
    const int e = threadIdx.x;
    const uint4 w = draw(whole);
    const uint32_t u = e < 2 ? w.x : e < 4 ? w.y : e < 6 ? w.z : w.w;
    const float v = kept(e & 1 ? u >> 16 : u & 0xffffu, cut, to_float(x[whole * 8 + e]), scale);
    y[whole * 8 + e] = from_float<T>(RES ? to_float(res[whole * 8 + e]) + v : v);
  }
}

template <typename T>
void launch_dropout(const void* x, const void* res, const int64_t* rng, void* y, int64_t n, int cut, cudaStream_t st) {
  const int64_t ctas = ((n + 7) / 8 + 255) / 256;
  const unsigned grid = (unsigned)(ctas < 148 * 8 ? ctas : 148 * 8);  // 8 fit on an SM
  const float scale = cut < 65536 ? 65536.0f / (float)(65536 - cut) : 0.0f;
  const T* xt = static_cast<const T*>(x);
  const T* rt = static_cast<const T*>(res);
  T* yt = static_cast<T*>(y);
  if (res) dropout_add_kernel<T, true><<<grid, 256, 0, st>>>(xt, rt, rng, yt, n, (uint32_t)cut, scale);
  else dropout_add_kernel<T, false><<<grid, 256, 0, st>>>(xt, rt, rng, yt, n, (uint32_t)cut, scale);
}

}  // namespace
}  // namespace csn

using namespace csn;

extern "C" int csn_dropout_add(const void* x, const void* residual, const int64_t* rng, void* y, int64_t n, int cut,
                               int dtype, void* stream) {
  if (n < 0 || cut < 0 || cut > 65536) return set_error(CSN_ERR_INVALID, "csn_dropout_add: needs n >= 0 and 0 <= cut <= 65536");
  if (dtype != CSN_F32 && dtype != CSN_BF16 && dtype != CSN_F16)
    return set_error(CSN_ERR_UNSUPPORTED, "csn_dropout_add: dtype is float32, bfloat16 or float16");
  if (n == 0) return CSN_OK;
  auto al = [](const void* p, int b) { return (reinterpret_cast<uintptr_t>(p) % b) == 0; };
  if (!x || !rng || !y || !al(x, 16) || !al(residual, 16) || !al(y, 16) || !al(rng, 8))
    return set_error(CSN_ERR_INVALID, "csn_dropout_add: missing or misaligned pointer");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  KernelTimer kt("dropout_add", st);
  if (dtype == CSN_F32) launch_dropout<float>(x, residual, rng, y, n, cut, st);
  else if (dtype == CSN_BF16) launch_dropout<__nv_bfloat16>(x, residual, rng, y, n, cut, st);
  else launch_dropout<__half>(x, residual, rng, y, n, cut, st);
  return check_launch("csn_dropout_add");
}

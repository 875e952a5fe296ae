// csn_dropout.cu -- dropout with the residual add, from a counter-based generator.
//
//   y = residual + keep * x * 65536 / (65536 - cut),   keep = (16 random bits >= cut)
// The bits come from Philox4x32-10 (J. K. Salmon et al., "Parallel random numbers: as easy as 1, 2, 3", SC 2011):
// block j = element / 8 of the flattened tensor is enciphered from the counter (j, offset) under the key `seed`, and
// its 128 bits serve 8 elements with 16 bits each.  A place's bits depend on nothing else, so the backward pass draws
// the mask again (dx = keep * dy * scale is the same kernel without a residual) and no mask is stored.  16 bits an
// element give steps of 2^-16 for the probability, and the scale is that of the probability actually drawn, so the
// mean is exact.
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

template <typename T, bool RES>
__global__ void __launch_bounds__(256) dropout_add_kernel(const T* __restrict__ x, const T* __restrict__ res,
                                                          const int64_t* __restrict__ rng, T* __restrict__ y,
                                                          int64_t n, uint32_t cut, float scale) {
  const uint64_t seed = (uint64_t)rng[0], off = (uint64_t)rng[1];
  const int64_t blocks = (n + 7) / 8;
  for (int64_t j = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; j < blocks; j += (int64_t)gridDim.x * blockDim.x) {
    T xv[8], rv[8];
    const int64_t i0 = j * 8;
    const bool whole = i0 + 8 <= n;
    if (whole) {
      *reinterpret_cast<Pack<T, 16 / sizeof(T)>*>(xv) = *reinterpret_cast<const Pack<T, 16 / sizeof(T)>*>(x + i0);
      if (sizeof(T) == 4)
        *reinterpret_cast<Pack<T, 4>*>(xv + 4) = *reinterpret_cast<const Pack<T, 4>*>(x + i0 + 4);
      if (RES) {
        *reinterpret_cast<Pack<T, 16 / sizeof(T)>*>(rv) = *reinterpret_cast<const Pack<T, 16 / sizeof(T)>*>(res + i0);
        if (sizeof(T) == 4)
          *reinterpret_cast<Pack<T, 4>*>(rv + 4) = *reinterpret_cast<const Pack<T, 4>*>(res + i0 + 4);
      }
    } else {
      for (int e = 0; e < 8; ++e)
        if (i0 + e < n) {
          xv[e] = x[i0 + e];
          if (RES) rv[e] = res[i0 + e];
        }
    }
    const uint4 w = philox4x32(make_uint4((uint32_t)j, (uint32_t)((uint64_t)j >> 32), (uint32_t)off, (uint32_t)(off >> 32)),
                               (uint32_t)seed, (uint32_t)(seed >> 32));
    const uint32_t word[4] = {w.x, w.y, w.z, w.w};
    T out[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t bits = e & 1 ? word[e / 2] >> 16 : word[e / 2] & 0xffffu;
      // a dropped place is 0 whatever stood there, an infinity or a NaN too
      const float v = bits >= cut ? to_float(xv[e]) * scale : 0.0f;
      out[e] = from_float<T>(RES ? to_float(rv[e]) + v : v);
    }
    if (whole) {
      *reinterpret_cast<Pack<T, 16 / sizeof(T)>*>(y + i0) = *reinterpret_cast<Pack<T, 16 / sizeof(T)>*>(out);
      if (sizeof(T) == 4) *reinterpret_cast<Pack<T, 4>*>(y + i0 + 4) = *reinterpret_cast<Pack<T, 4>*>(out + 4);
    } else {
      for (int e = 0; e < 8; ++e)
        if (i0 + e < n) y[i0 + e] = out[e];
    }
  }
}

template <typename T>
void launch_dropout(const void* x, const void* res, const int64_t* rng, void* y, int64_t n, int cut, cudaStream_t st) {
  const int64_t ctas = ((n + 7) / 8 + 255) / 256;
  const unsigned grid = (unsigned)(ctas < 148 * 64 ? ctas : 148 * 64);
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

// csn_layer_norm.cu -- layer norm of 16-bit rows of any width, and its adjoint.
//
//   m = mean(x),  r = 1 / sqrt(mean((x - m)^2) + eps),  h = (x - m) r,  y = h w + b
// Adjoint, with g = dy w:
//   dx = r (g - mean(g) - h mean(g h)),  dw = sum over rows of dy h,  db = sum over rows of dy
// Rows are read and written in their own type and computed in float32 (csn_block.cu has the float32 rows); w and b are
// of the rows' type or float32.
#include <algorithm>
#include <cstdint>

#include "csn_internal.h"
#include "csn_types.cuh"

namespace csn {
namespace {

constexpr int THREADS = 256;

template <typename T, int N>
__device__ __forceinline__ void load(const T* p, float (&v)[N]) {
  const Pack<T, N> x = *reinterpret_cast<const Pack<T, N>*>(p);
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = to_float(x.v[i]);
}
template <typename T, int N>
__device__ __forceinline__ void store(T* p, const float (&v)[N]) {
  Pack<T, N> x;
#pragma unroll
  for (int i = 0; i < N; ++i) x.v[i] = from_float<T>(v[i]);
  *reinterpret_cast<Pack<T, N>*>(p) = x;
}

// Sum over a CTA, in a fixed order; every thread gets it.
__device__ __forceinline__ float cta_sum(float v, float* room) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) room[threadIdx.x / 32] = v;
  __syncthreads();
  v = 0.0f;
#pragma unroll
  for (int i = 0; i < THREADS / 32; ++i) v += room[i];
  return v;
}

// A row to a CTA, read three times.
template <typename T, typename W>
__global__ void __launch_bounds__(THREADS) forward_kernel(const T* __restrict__ x, int64_t ld, const W* __restrict__ w,
                                                          const W* __restrict__ b, T* __restrict__ y, float* mean, float* rstd,
                                                          int64_t R, int C, float eps) {
  __shared__ float room[THREADS / 32];
  for (int64_t r = blockIdx.x; r < R; r += gridDim.x) {
    const T* p = x + r * ld;
    float s = 0.0f;
    for (int c = threadIdx.x; c < C; c += THREADS) s += to_float(p[c]);
    const float m = cta_sum(s, room) / C;
    s = 0.0f;
    for (int c = threadIdx.x; c < C; c += THREADS) {
      const float d = to_float(p[c]) - m;
      s = fmaf(d, d, s);
    }
    const float k = 1.0f / sqrtf(cta_sum(s, room) / C + eps);
    for (int c = threadIdx.x; c < C; c += THREADS)
      y[r * C + c] = from_float<T>(fmaf((to_float(p[c]) - m) * k, to_float(w[c]), to_float(b[c])));
    if (threadIdx.x == 0 && mean) mean[r] = m, rstd[r] = k;
  }
}

template <typename T, typename W>
__global__ void __launch_bounds__(THREADS) backward_kernel(const T* __restrict__ dy, int64_t ldy, const T* __restrict__ x,
                                                           int64_t ld, const float* __restrict__ mean,
                                                           const float* __restrict__ rstd, const W* __restrict__ w,
                                                           T* __restrict__ dx, int64_t R, int C) {
  __shared__ float room[THREADS / 32];
  for (int64_t r = blockIdx.x; r < R; r += gridDim.x) {
    const T *p = x + r * ld, *q = dy + r * ldy;
    const float m = mean[r], k = rstd[r];
    float s = 0.0f, t = 0.0f;
    for (int c = threadIdx.x; c < C; c += THREADS) {
      const float g = to_float(q[c]) * to_float(w[c]);
      s += g;
      t = fmaf(g, (to_float(p[c]) - m) * k, t);
    }
    s = cta_sum(s, room) / C;
    t = cta_sum(t, room) / C;
    for (int c = threadIdx.x; c < C; c += THREADS) {
      const float h = (to_float(p[c]) - m) * k;
      dx[r * C + c] = from_float<T>(k * (to_float(q[c]) * to_float(w[c]) - s - h * t));
    }
  }
}

// part[i][0 and 1][C]: the sums of dy h and dy over the rows i, i + gridDim.y, ...
template <typename T>
__global__ void __launch_bounds__(THREADS) weights_kernel(const T* __restrict__ dy, int64_t ldy, const T* __restrict__ x,
                                                          int64_t ld, const float* __restrict__ mean,
                                                          const float* __restrict__ rstd, float* part, int64_t R, int C) {
  const int c = blockIdx.x * THREADS + threadIdx.x;
  if (c >= C) return;
  float s = 0.0f, t = 0.0f;
  for (int64_t r = blockIdx.y; r < R; r += gridDim.y) {
    const float d = to_float(dy[r * ldy + c]);
    s = fmaf(d, (to_float(x[r * ld + c]) - mean[r]) * rstd[r], s);
    t += d;
  }
  part[(int64_t)blockIdx.y * 2 * C + c] = s;
  part[((int64_t)blockIdx.y * 2 + 1) * C + c] = t;
}

template <typename W>
__global__ void __launch_bounds__(THREADS) finish_kernel(const float* __restrict__ part, int n, int C, W* dw, W* db) {
  const int c = blockIdx.x * THREADS + threadIdx.x;
  if (c >= C) return;
  float s = 0.0f, t = 0.0f;
  for (int i = 0; i < n; ++i) {
    s += part[(int64_t)i * 2 * C + c];
    t += part[((int64_t)i * 2 + 1) * C + c];
  }
  if (dw) dw[c] = from_float<W>(s);
  if (db) db[c] = from_float<W>(t);
}

int parts(int64_t R) { return (int)std::min<int64_t>(std::max<int64_t>(R, 1), 148 * 2); }
bool aligned(const void* p, int n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

int check_rows(int64_t R, int64_t C, int dtype, int wtype) {
  if (R < 0 || C < 1 || C > (1 << 30)) return set_error(CSN_ERR_INVALID, "csn_layer_norm_rows: R >= 0 rows of 1 to 2^30 places expected");
  if ((dtype != CSN_BF16 && dtype != CSN_F16) || (wtype != dtype && wtype != CSN_F32))
    return set_error(CSN_ERR_UNSUPPORTED, "csn_layer_norm_rows: bfloat16 or float16 rows, weights of the rows' type or float32");
  return CSN_OK;
}

struct Back {
  const void *dy, *x, *w;
  int64_t ldy, ld;
  const float *mean, *rstd;
  void *dx, *dw, *db;
  float* part;
  int64_t R;
  int C;
};
template <typename T, typename W>
void backward(const Back& A, cudaStream_t st) {
  const unsigned grid = (unsigned)std::min<int64_t>(A.R, 148 * 8);
  const T *dy = static_cast<const T*>(A.dy), *x = static_cast<const T*>(A.x);
  if (A.R && A.dx)
    backward_kernel<T, W><<<grid, THREADS, 0, st>>>(dy, A.ldy, x, A.ld, A.mean, A.rstd, static_cast<const W*>(A.w), static_cast<T*>(A.dx), A.R, A.C);
  if (!A.dw && !A.db) return;
  const int n = parts(A.R);
  const unsigned tiles = (unsigned)((A.C + THREADS - 1) / THREADS);
  weights_kernel<T><<<dim3(tiles, (unsigned)n), THREADS, 0, st>>>(dy, A.ldy, x, A.ld, A.mean, A.rstd, A.part, A.R, A.C);
  finish_kernel<W><<<tiles, THREADS, 0, st>>>(A.part, n, A.C, static_cast<W*>(A.dw), static_cast<W*>(A.db));
}
template <typename T, typename W>
void forward(const void* x, int64_t ld, const void* w, const void* b, void* y, float* mean, float* rstd, int64_t R, int C, float eps,
             cudaStream_t st) {
  const unsigned grid = (unsigned)std::min<int64_t>(R, 148 * 8);
  forward_kernel<T, W><<<grid, THREADS, 0, st>>>(static_cast<const T*>(x), ld, static_cast<const W*>(w), static_cast<const W*>(b),
                                                 static_cast<T*>(y), mean, rstd, R, C, eps);
}

}  // namespace
}  // namespace csn

using namespace csn;

extern "C" int csn_layer_norm_rows_fwd(const void* x, int64_t ldx, const void* weight, const void* bias, void* y, float* mean,
                                       float* rstd, int64_t R, int64_t C, float eps, int dtype, int weight_dtype, void* stream) {
  if (int rc = check_rows(R, C, dtype, weight_dtype)) return rc;
  if (R == 0) return CSN_OK;
  const int ws = weight_dtype == CSN_F32 ? 4 : 2;
  if (!x || !weight || !bias || !y || !mean != !rstd || !aligned(x, 2) || !aligned(y, 16) || !aligned(weight, ws) || !aligned(bias, ws))
    return set_error(CSN_ERR_INVALID, "csn_layer_norm_rows_fwd: missing or misaligned pointer");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  KernelTimer kt("layer_norm_rows_fwd", st);
  auto* f = dtype == CSN_BF16 ? (weight_dtype == CSN_F32 ? forward<__nv_bfloat16, float> : forward<__nv_bfloat16, __nv_bfloat16>)
                              : (weight_dtype == CSN_F32 ? forward<__half, float> : forward<__half, __half>);
  f(x, ldx, weight, bias, y, mean, rstd, R, (int)C, eps, st);
  return check_launch("csn_layer_norm_rows_fwd");
}

extern "C" size_t csn_layer_norm_rows_bwd_workspace_bytes(int64_t R, int64_t C) {
  if (R < 0 || C < 1) return 0;
  return (size_t)parts(R) * 2 * (size_t)C * sizeof(float);
}

extern "C" int csn_layer_norm_rows_bwd(const void* dy, int64_t ldy, const void* x, int64_t ldx, const float* mean, const float* rstd,
                                       const void* weight, void* dx, void* dweight, void* dbias, int64_t R, int64_t C, int dtype,
                                       int weight_dtype, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_rows(R, C, dtype, weight_dtype)) return rc;
  const int ws = weight_dtype == CSN_F32 ? 4 : 2;
  if ((R && (!dy || !x || !mean || !rstd || !weight)) || !aligned(dy, 2) || !aligned(x, 2) || !aligned(dx, 16) || !aligned(weight, ws) ||
      !aligned(dweight, ws) || !aligned(dbias, ws))
    return set_error(CSN_ERR_INVALID, "csn_layer_norm_rows_bwd: missing or misaligned pointer");
  if ((dweight || dbias) && (!workspace || !aligned(workspace, 16) || workspace_bytes < csn_layer_norm_rows_bwd_workspace_bytes(R, C)))
    return set_error(CSN_ERR_INVALID, "csn_layer_norm_rows_bwd: workspace smaller than csn_layer_norm_rows_bwd_workspace_bytes");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  KernelTimer kt("layer_norm_rows_bwd", st);
  const Back A = {dy, x, weight, ldy, ldx, mean, rstd, dx, dweight, dbias, static_cast<float*>(workspace), R, (int)C};
  auto* f = dtype == CSN_BF16 ? (weight_dtype == CSN_F32 ? backward<__nv_bfloat16, float> : backward<__nv_bfloat16, __nv_bfloat16>)
                              : (weight_dtype == CSN_F32 ? backward<__half, float> : backward<__half, __half>);
  f(A, st);
  return check_launch("csn_layer_norm_rows_bwd");
}

// csn_ffn.cu -- the gated feed-forward product of 16-bit tensors and its adjoint.
//
//   g = x Wg^T,  u = x Wu^T,  y = silu(g) * u          x [R, C], Wg, Wu [F, C], y [R, F]
// Adjoint, with w = sigmoid(g):
//   dg = dy u w (1 + g (1 - w)),  du = dy g w,  dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x
// The backward pass forms g and u again in float32 (they are never stored): keeping them would cost 8 bytes written
// and read an element in float32, or, rounded to 16 bits, a third of the gradients' precision.
// dg and du are rounded to the tensors' own type once, as the operands of the products that follow.
#include <cstdint>

#include "csn_internal.h"
#include "csn_types.cuh"

namespace csn {
namespace {

constexpr int TILE = 64, KT = 16;

// A matrix as products read it: element (i, k) at p + i * si + k * sk
template <typename T>
struct Mat2 {
  const T* p;
  int64_t si, sk;
};

// acc += rows of A times rows of B over k, for the 64 x 64 tile at (m0, n0); 256 threads with 4 x 4 values each
template <typename T>
__device__ __forceinline__ void tile_product(const Mat2<T>& A, const Mat2<T>& B, int64_t M, int64_t N, int64_t K,
                                             int64_t m0, int64_t n0, float (*as)[TILE + 4], float (*bs)[TILE + 4],
                                             float (*acc)[4]) {
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  for (int64_t k0 = 0; k0 < K; k0 += KT) {
    for (int i = threadIdx.x; i < TILE * KT; i += 256) {
      // neighbouring threads take neighbouring elements of whichever axis is contiguous
      const int ak = A.sk == 1 ? i % KT : i / TILE, am = A.sk == 1 ? i / KT : i % TILE;
      const int bk = B.sk == 1 ? i % KT : i / TILE, bn = B.sk == 1 ? i / KT : i % TILE;
      as[ak][am] = m0 + am < M && k0 + ak < K ? to_float(A.p[(m0 + am) * A.si + (k0 + ak) * A.sk]) : 0.0f;
      bs[bk][bn] = n0 + bn < N && k0 + bk < K ? to_float(B.p[(n0 + bn) * B.si + (k0 + bk) * B.sk]) : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < KT; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(as[k][ty * 4 + i], bs[k][tx * 4 + j], acc[i][j]);
    __syncthreads();
  }
}

template <typename T>
__global__ void __launch_bounds__(256) gate_kernel(Mat2<T> x, Mat2<T> wg, Mat2<T> wu, const T* dy, int64_t ldy, T* y,
                                                   T* dg, T* du, int64_t R, int64_t C, int64_t F) {
  __shared__ float as[KT][TILE + 4], bs[KT][TILE + 4];
  const int64_t m0 = (int64_t)blockIdx.y * TILE, n0 = (int64_t)blockIdx.x * TILE;
  float g[4][4] = {}, u[4][4] = {};
  tile_product(x, wg, R, F, C, m0, n0, as, bs, g);
  tile_product(x, wu, R, F, C, m0, n0, as, bs, u);
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int64_t r = m0 + threadIdx.x / 16 * 4 + i, c = n0 + threadIdx.x % 16 * 4 + j;
      if (r >= R || c >= F) continue;
      float w, wn;
      sigmoid_pair(g[i][j], w, wn);
      if (y) y[r * F + c] = from_float<T>(g[i][j] * w * u[i][j]);
      if (dy) {
        const float d = to_float(dy[r * ldy + c]);
        dg[r * F + c] = from_float<T>(d * u[i][j] * (w * fmaf(g[i][j], wn, 1.0f)));
        du[r * F + c] = from_float<T>(d * g[i][j] * w);
      }
    }
}

// out[m, n] = sum_k A(m, k) B(n, k) + A2(m, k) B2(n, k)
template <typename T>
__global__ void __launch_bounds__(256) product_kernel(Mat2<T> a, Mat2<T> b, Mat2<T> a2, Mat2<T> b2, T* out, int64_t M,
                                                      int64_t N, int64_t K) {
  __shared__ float as[KT][TILE + 4], bs[KT][TILE + 4];
  const int64_t m0 = (int64_t)blockIdx.y * TILE, n0 = (int64_t)blockIdx.x * TILE;
  float acc[4][4] = {};
  tile_product(a, b, M, N, K, m0, n0, as, bs, acc);
  if (a2.p) tile_product(a2, b2, M, N, K, m0, n0, as, bs, acc);
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int64_t r = m0 + threadIdx.x / 16 * 4 + i, c = n0 + threadIdx.x % 16 * 4 + j;
      if (r < M && c < N) out[r * N + c] = from_float<T>(acc[i][j]);
    }
}

dim3 tiles(int64_t M, int64_t N) { return dim3((unsigned)((N + TILE - 1) / TILE), (unsigned)((M + TILE - 1) / TILE)); }

template <typename T>
void forward(const void* x, int64_t ldx, const void* wg, int64_t ldg, const void* wu, int64_t ldu, void* y, int64_t R,
             int64_t C, int64_t F, cudaStream_t st) {
  gate_kernel<T><<<tiles(R, F), 256, 0, st>>>({static_cast<const T*>(x), ldx, 1}, {static_cast<const T*>(wg), ldg, 1},
                                              {static_cast<const T*>(wu), ldu, 1}, nullptr, 0, static_cast<T*>(y),
                                              nullptr, nullptr, R, C, F);
}

template <typename T>
void backward(const void* x, int64_t ldx, const void* wg, int64_t ldg, const void* wu, int64_t ldu, const void* dy,
              int64_t ldy, void* dx, void* dwg, void* dwu, int64_t R, int64_t C, int64_t F, void* ws, cudaStream_t st) {
  const T *xt = static_cast<const T*>(x), *gt = static_cast<const T*>(wg), *ut = static_cast<const T*>(wu);
  T* dg = static_cast<T*>(ws);
  T* du = dg + R * F;
  gate_kernel<T><<<tiles(R, F), 256, 0, st>>>({xt, ldx, 1}, {gt, ldg, 1}, {ut, ldu, 1}, static_cast<const T*>(dy), ldy,
                                              nullptr, dg, du, R, C, F);
  if (dx)
    product_kernel<T><<<tiles(R, C), 256, 0, st>>>({dg, F, 1}, {gt, 1, ldg}, {du, F, 1}, {ut, 1, ldu},
                                                   static_cast<T*>(dx), R, C, F);
  const Mat2<T> none = {nullptr, 0, 0};
  if (dwg) product_kernel<T><<<tiles(F, C), 256, 0, st>>>({dg, 1, F}, {xt, 1, ldx}, none, none, static_cast<T*>(dwg), F, C, R);
  if (dwu) product_kernel<T><<<tiles(F, C), 256, 0, st>>>({du, 1, F}, {xt, 1, ldx}, none, none, static_cast<T*>(dwu), F, C, R);
}

bool al16b(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int check_ffn(const char* who, int64_t R, int64_t C, int64_t F, int dtype) {
  // rows, channels and hidden units are 32-bit coordinates of the tiles
  if (R < 0 || C < 0 || F < 0 || R > (1 << 21) || C > (1 << 21) || F > (1 << 21)) return set_error(CSN_ERR_INVALID, who);
  if (dtype != CSN_BF16 && dtype != CSN_F16) return set_error(CSN_ERR_UNSUPPORTED, who);
  return CSN_OK;
}

}  // namespace
}  // namespace csn

using namespace csn;

extern "C" size_t csn_silu_gated_linear_workspace_bytes(int64_t R, int64_t C, int64_t F, int backward) {
  if (R <= 0 || C <= 0 || F <= 0) return 0;
  return backward ? (size_t)R * F * 4 : 0;
}

extern "C" int csn_silu_gated_linear_fwd(const void* x, int64_t ldx, const void* w_gate, int64_t ld_gate,
                                         const void* w_up, int64_t ld_up, void* y, int64_t R, int64_t C, int64_t F,
                                         int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_ffn("csn_silu_gated_linear_fwd: needs 0 <= R, C, F <= 2^21 and dtype bfloat16 or float16", R, C, F, dtype))
    return rc;
  if (R == 0 || F == 0) return CSN_OK;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (!y || (C > 0 && (!x || !w_gate || !w_up)) || !al16b(y))
    return set_error(CSN_ERR_INVALID, "csn_silu_gated_linear_fwd: missing or misaligned pointer");
  if (C == 0)
    return cudaMemsetAsync(y, 0, (size_t)R * F * 2, st) == cudaSuccess
               ? CSN_OK : set_error(CSN_ERR_CUDA, "csn_silu_gated_linear_fwd: cudaMemsetAsync");
  const size_t need = csn_silu_gated_linear_workspace_bytes(R, C, F, 0);
  if (need && (!workspace || !al16b(workspace) || workspace_bytes < need))
    return set_error(CSN_ERR_INVALID, "csn_silu_gated_linear_fwd: workspace smaller than csn_silu_gated_linear_workspace_bytes");
  KernelTimer kt("silu_gated_linear_fwd", st);
  if (dtype == CSN_BF16) forward<__nv_bfloat16>(x, ldx, w_gate, ld_gate, w_up, ld_up, y, R, C, F, st);
  else forward<__half>(x, ldx, w_gate, ld_gate, w_up, ld_up, y, R, C, F, st);
  return check_launch("csn_silu_gated_linear_fwd");
}

extern "C" int csn_silu_gated_linear_bwd(const void* x, int64_t ldx, const void* w_gate, int64_t ld_gate,
                                         const void* w_up, int64_t ld_up, const void* dy, int64_t ld_dy, void* dx,
                                         void* dw_gate, void* dw_up, int64_t R, int64_t C, int64_t F, int dtype,
                                         void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_ffn("csn_silu_gated_linear_bwd: needs 0 <= R, C, F <= 2^21 and dtype bfloat16 or float16", R, C, F, dtype))
    return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (R == 0 || C == 0 || F == 0) {  // sums over nothing
    const size_t bytes[3] = {(size_t)R * C * 2, (size_t)F * C * 2, (size_t)F * C * 2};
    void* outs[3] = {dx, dw_gate, dw_up};
    for (int i = 0; i < 3; ++i)
      if (outs[i] && bytes[i] && cudaMemsetAsync(outs[i], 0, bytes[i], st) != cudaSuccess)
        return set_error(CSN_ERR_CUDA, "csn_silu_gated_linear_bwd: cudaMemsetAsync");
    return CSN_OK;
  }
  if (!x || !w_gate || !w_up || !dy || !al16b(dx) || !al16b(dw_gate) || !al16b(dw_up))
    return set_error(CSN_ERR_INVALID, "csn_silu_gated_linear_bwd: missing or misaligned pointer");
  const size_t need = csn_silu_gated_linear_workspace_bytes(R, C, F, 1);
  if (need && (!workspace || !al16b(workspace) || workspace_bytes < need))
    return set_error(CSN_ERR_INVALID, "csn_silu_gated_linear_bwd: workspace smaller than csn_silu_gated_linear_workspace_bytes");
  KernelTimer kt("silu_gated_linear_bwd", st);
  if (dtype == CSN_BF16)
    backward<__nv_bfloat16>(x, ldx, w_gate, ld_gate, w_up, ld_up, dy, ld_dy, dx, dw_gate, dw_up, R, C, F, workspace, st);
  else
    backward<__half>(x, ldx, w_gate, ld_gate, w_up, ld_up, dy, ld_dy, dx, dw_gate, dw_up, R, C, F, workspace, st);
  return check_launch("csn_silu_gated_linear_bwd");
}

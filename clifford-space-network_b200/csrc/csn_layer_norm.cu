// csn_layer_norm.cu -- layer norm of 16-bit rows of any width, and its adjoint.
//
//   m = mean(x),  r = 1 / sqrt(mean((x - m)^2) + eps),  h = (x - m) r,  y = h w + b
// Adjoint, with g = dy w:
//   dx = r (g - mean(g) - h mean(g h)),  dw = sum over rows of dy h,  db = sum over rows of dy
// Rows are read and written in their own type and computed in float32 (csn_block.cu has the float32 rows); w and b are
// of the rows' type or float32.
//
// x - m is formed before anything else: r x - m r instead would put half a step of |m| r into h, which is 1 for a float16 row of one
// value near 60000.  m is a quotient, and where C > 2^13, so that 24 bits do not hold the sum of C places of 11 bits, it
// is corrected by the mean of x - m.  So rows of one value give h = 0 to the bit, whatever their width.
#include <algorithm>
#include <cmath>
#include <cstdint>

#include "csn_internal.h"
#include "csn_types.cuh"

namespace csn {
namespace {

constexpr int THREADS = 256;

// V neighbouring places in float32.  The arithmetic of 8 goes in pairs, one instruction each: one by one, with each place taken
// out of its word and put back by itself, the kernels executed 20 and 40 instructions an element and were bound by them.
template <int V>
struct Floats {
  float v[V];
};
template <int V>
__device__ __forceinline__ Floats<V> all(float a) {
  Floats<V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) r.v[i] = a;
  return r;
}
template <int V>
__device__ __forceinline__ Floats<V> fma(const Floats<V>& a, const Floats<V>& b, const Floats<V>& c) {
  Floats<V> r;
  if constexpr (V % 2 == 0) {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      const float2 x = fma2(make_float2(a.v[i], a.v[i + 1]), make_float2(b.v[i], b.v[i + 1]), make_float2(c.v[i], c.v[i + 1]));
      r.v[i] = x.x, r.v[i + 1] = x.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = fmaf(a.v[i], b.v[i], c.v[i]);
  }
  return r;
}
template <int V>
__device__ __forceinline__ Floats<V> mul(const Floats<V>& a, const Floats<V>& b) {
  Floats<V> r;
  if constexpr (V % 2 == 0) {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      const float2 x = mul2(make_float2(a.v[i], a.v[i + 1]), make_float2(b.v[i], b.v[i + 1]));
      r.v[i] = x.x, r.v[i + 1] = x.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = a.v[i] * b.v[i];
  }
  return r;
}
template <int V>
__device__ __forceinline__ Floats<V> add(const Floats<V>& a, const Floats<V>& b) {
  Floats<V> r;
  if constexpr (V % 2 == 0) {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      const float2 x = add2(make_float2(a.v[i], a.v[i + 1]), make_float2(b.v[i], b.v[i + 1]));
      r.v[i] = x.x, r.v[i + 1] = x.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = a.v[i] + b.v[i];
  }
  return r;
}
template <int V>
__device__ __forceinline__ float sum(const Floats<V>& a) {
  float r = a.v[0];
#pragma unroll
  for (int i = 1; i < V; ++i) r += a.v[i];
  return r;
}

__device__ __forceinline__ float2 pair(uint32_t w, __nv_bfloat16) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
__device__ __forceinline__ float2 pair(uint32_t w, __half) { return __half22float2(*reinterpret_cast<__half2*>(&w)); }

// V places as they lie in memory
template <typename T, int V>
struct Piece {
  Pack<T, V> p;
};
template <typename T>
struct Piece<T, 8> {
  uint4 p;
};
template <typename T, int V>
__device__ __forceinline__ Floats<V> floats(const Piece<T, V>& x) {
  Floats<V> r;
  if constexpr (V == 8) {
    const uint32_t w[4] = {x.p.x, x.p.y, x.p.z, x.p.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = pair(w[i], T{});
      r.v[2 * i] = f.x, r.v[2 * i + 1] = f.y;
    }
  } else {
    r.v[0] = to_float(x.p.v[0]);
  }
  return r;
}
template <typename T, int V>
__device__ __forceinline__ void store(T* to, const Floats<V>& a) {
  if constexpr (V == 8)
    *reinterpret_cast<uint4*>(to) = make_uint4(pack<T>(a.v[0], a.v[1]), pack<T>(a.v[2], a.v[3]), pack<T>(a.v[4], a.v[5]), pack<T>(a.v[6], a.v[7]));
  else
    to[0] = from_float<T>(a.v[0]);
}
// V neighbouring weights
template <int V>
__device__ __forceinline__ Floats<V> weights(const float* p) {
  Floats<V> r;
  if constexpr (V == 8) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    r.v[0] = a.x, r.v[1] = a.y, r.v[2] = a.z, r.v[3] = a.w, r.v[4] = b.x, r.v[5] = b.y, r.v[6] = b.z, r.v[7] = b.w;
  } else {
    r.v[0] = __ldg(p);
  }
  return r;
}
template <int V, typename T>
__device__ __forceinline__ Floats<V> weights(const T* p) { return floats<T, V>(*reinterpret_cast<const Piece<T, V>*>(p)); }

// Sums of n values over the TPR threads that share a row, in a fixed order; each of them gets them.  Rows of more than a
// warp meet in `room`, whose two halves take turns, so that one barrier a call is enough.
template <int TPR, int n>
__device__ __forceinline__ void row_sums(float (&v)[n], float* room, int& turn) {
#pragma unroll
  for (int o = (TPR < 32 ? TPR : 32) / 2; o; o >>= 1)
#pragma unroll
    for (int i = 0; i < n; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  if constexpr (TPR > 32) {
    constexpr int WARPS = TPR / 32;
    using Sums = Pack<float, n>;
    Sums* mine = reinterpret_cast<Sums*>(room) + turn * (blockDim.x / 32);
    turn ^= 1;
    const int warp = threadIdx.x / 32, first = warp / WARPS * WARPS;
    if ((threadIdx.x & 31) == 0) {
      Sums own;
#pragma unroll
      for (int i = 0; i < n; ++i) own.v[i] = v[i];
      mine[warp] = own;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < n; ++i) v[i] = 0.0f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const Sums other = mine[first + w];
#pragma unroll
      for (int i = 0; i < n; ++i) v[i] += other.v[i];
    }
  }
}

// s / C, which is exact where float32 has it, as the product with 1 / C is not (Markstein's remainder step)
__device__ __forceinline__ float mean_of(float s, float n, float over) {
  const float m = s * over;
  return fmaf(fmaf(-m, n, s), over, m);
}
// The mean m of a row corrected by that of x - m, whose part of the mean square of x - m is taken out.
__device__ __forceinline__ void correct(float d, float& m, float& square) {
  m += d;
  const float var = fmaf(-d, d, square);
  // a NaN stays one, and squares past float32's range an infinity
  square = var < 0.0f ? 0.0f : square < INFINITY ? var : square;
}

// TPR threads take a row, NV pieces of V neighbouring places each, and ROWS rows at a time, to have enough loads in flight: a row
// is read once and stays in registers, in its own type.  V = 8 where rows start on 16 bytes and C is a multiple of 8, else 1.
// A warp takes rows of up to 2048 places: two reductions without a barrier.
// bf16 on a B200: R32768 C2048 51 us (5.3 TB/s), R524288 C128 59 (4.6), R8192 C8192 51 (5.2), R4096 C16384 76 (3.5; the second
// mean is 10 of it), where a CTA to a row that read it three times took 93, 812 and 88 for the first three.  Bound by memory
// and, where rows are short, by the instructions that rows cost besides their places.  Slower: C2048 with a CTA to a row 80 us
// (barriers), with 173 registers a thread 64 (8 warps an SM).
template <typename T, typename W, int TPR, int NV, int V, int ROWS>
__global__ void __launch_bounds__(TPR > THREADS ? TPR : THREADS, TPR > THREADS ? 1 : NV * V >= 64 ? 3 : 4)
    forward_kernel(const T* __restrict__ x, int64_t ld, const W* __restrict__ w, const W* __restrict__ b, T* __restrict__ y, float* mean,
                   float* rstd, int64_t R, int C, float eps) {
  constexpr int N = TPR > THREADS ? TPR : THREADS, GROUPS = N / TPR;
  constexpr bool FAR = TPR * NV * V > 8192;  // (all of them have C > 8192)
  __shared__ __align__(16) float room[2 * (TPR > 32 ? N / 32 : 1) * (FAR ? 2 : 1) * ROWS];
  const int t = threadIdx.x % TPR;
  const float n = C, over = 1.0f / n;
  int turn = 0;
  for (int64_t r0 = blockIdx.x * (int64_t)(GROUPS * ROWS); r0 < R; r0 += (int64_t)gridDim.x * (GROUPS * ROWS)) {
    Piece<T, V> p[ROWS][NV];
    float m[ROWS], s[ROWS], q[FAR ? 2 * ROWS : ROWS];  // q: the sums of (x - m)^2, and of x - m
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
      const int64_t r = r0 + j * GROUPS + threadIdx.x / TPR;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = (k * TPR + t) * V;
        if (r < R && c < C) p[j][k] = *reinterpret_cast<const Piece<T, V>*>(x + r * ld + c);
        else p[j][k] = {};
      }
    }
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
      Floats<V> a = floats<T, V>(p[j][0]);
#pragma unroll
      for (int k = 1; k < NV; ++k) a = add<V>(a, floats<T, V>(p[j][k]));
      s[j] = sum<V>(a);
    }
    row_sums<TPR>(s, room, turn);
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
      m[j] = mean_of(s[j], n, over);
      Floats<V> a = all<V>(0.0f), b = a;
#pragma unroll
      for (int k = 0; k < NV; ++k)
        if ((k * TPR + t) * V < C) {
          const Floats<V> d = add<V>(floats<T, V>(p[j][k]), all<V>(-m[j]));
          if (FAR) b = add<V>(b, d);
          a = fma<V>(d, d, a);
        }
      q[j] = sum<V>(a);
      if (FAR) q[FAR ? ROWS + j : 0] = sum<V>(b);
    }
    row_sums<TPR>(q, room, turn);
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
      float square = q[j] * over;
      if (FAR) correct(mean_of(q[FAR ? ROWS + j : 0], n, over), m[j], square);
      s[j] = 1.0f / sqrtf(square + eps);
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * TPR + t) * V;
      if (c >= C) continue;
      const Floats<V> wv = weights<V>(w + c), bv = weights<V>(b + c);
#pragma unroll
      for (int j = 0; j < ROWS; ++j) {
        const int64_t r = r0 + j * GROUPS + threadIdx.x / TPR;
        if (r >= R) continue;
        const Floats<V> h = mul<V>(add<V>(floats<T, V>(p[j][k]), all<V>(-m[j])), all<V>(s[j]));
        store<T, V>(y + r * C + c, fma<V>(h, wv, bv));
      }
    }
    if (t == 0 && mean) {
#pragma unroll
      for (int j = 0; j < ROWS; ++j) {
        const int64_t r = r0 + j * GROUPS + threadIdx.x / TPR;
        if (r < R) mean[r] = m[j], rstd[r] = s[j];
      }
    }
  }
}

// Rows too long for that: a CTA to a row, which is read three times.
template <typename T, typename W>
__global__ void __launch_bounds__(1024) long_forward_kernel(const T* __restrict__ x, int64_t ld, const W* __restrict__ w,
                                                            const W* __restrict__ b, T* __restrict__ y, float* mean, float* rstd,
                                                            int64_t R, int C, float eps) {
  __shared__ __align__(16) float room[128];
  const float n = C, over = 1.0f / n;
  int turn = 0;
  for (int64_t r = blockIdx.x; r < R; r += gridDim.x) {
    const T* p = x + r * ld;
    float s[1] = {0.0f};
    for (int c = threadIdx.x; c < C; c += 1024) s[0] += to_float(p[c]);
    row_sums<1024>(s, room, turn);
    float m = mean_of(s[0], n, over), q[2] = {0.0f, 0.0f};
    for (int c = threadIdx.x; c < C; c += 1024) {
      const float d = to_float(p[c]) - m;
      q[0] = fmaf(d, d, q[0]);
      q[1] += d;
    }
    row_sums<1024>(q, room, turn);
    float square = q[0] * over;
    correct(mean_of(q[1], n, over), m, square);
    const float k = 1.0f / sqrtf(square + eps);
    for (int c = threadIdx.x; c < C; c += 1024)
      y[r * C + c] = from_float<T>(fmaf((to_float(p[c]) - m) * k, to_float(w[c]), to_float(b[c])));
    if (threadIdx.x == 0 && mean) mean[r] = m, rstd[r] = k;
  }
}

// The adjoint.  TPR threads take a row, NV pieces of V neighbouring places each.  A thread's places are the same in every row,
// so it also gathers their sums of dy h and dy, which the CTA adds up at the end: part[CTA][0 and 1][C].  For V = 8 each
// thread copies its own pieces of x and dy into shared memory DEPTH - 1 rows ahead (cp.async; no other thread reads them, so
// that no barrier is needed): the registers that loads in flight would take leave room for more warps.
// bf16 on a B200, with the sums: R32768 C2048 91 us (4.4 TB/s), R524288 C128 76 (5.3), R8192 C8192 109 (3.7), R1048576 C64 83 (4.8).
// Neither memory nor issue is full (an SM issues in 42 to 68 % of its cycles, with 15 to 21 of 64 warps): a row's meeting at its barrier and the chain from
// its sums to its gradient are what a few warps wait for.  Slower: 8 places to a thread 108 us for C2048 (shuffles, the meeting
// and addresses cost a row 130 instructions a thread, whatever it has of it), loads into registers 160, mean and rstd
// read when a row's turn comes 140 for C8192, more CTAs than the SMs hold at a time.
template <typename T, typename W, int TPR, int NV, int V, int DEPTH>
__global__ void __launch_bounds__(TPR > THREADS ? TPR : THREADS, TPR > THREADS ? 1 : NV > 1 ? 2 : 4)
    backward_kernel(const T* __restrict__ dy, int64_t ldy, const T* __restrict__ x, int64_t ld, const float* __restrict__ mean,
                    const float* __restrict__ rstd, const W* __restrict__ w, T* __restrict__ dx, float* __restrict__ part, int64_t R,
                    int C) {
  constexpr int N = TPR > THREADS ? TPR : THREADS, GROUPS = N / TPR;
  using Piece = Piece<T, V>;
  extern __shared__ __align__(16) char ring_bytes[];  // [DEPTH][2][NV][N] pieces, [DEPTH][2][N] mean and rstd; at the end the sums of the groups
  Piece* const ring = reinterpret_cast<Piece*>(ring_bytes) + threadIdx.x;
  float* const stats = reinterpret_cast<float*>(ring_bytes + DEPTH * 2 * NV * N * sizeof(Piece)) + threadIdx.x;
  __shared__ __align__(16) float room[2 * (TPR > 32 ? N / 32 : 1) * 2];
  const int t = threadIdx.x % TPR;
  const float over = 1.0f / C;
  const int64_t step = (int64_t)gridDim.x * GROUPS, first = blockIdx.x * (int64_t)GROUPS;
  Piece ahead[V == 8 ? 1 : 2 * NV] = {};  // V = 1: cp.async takes 4 bytes at least
  float ahead_mean = 0.0f, ahead_rstd = 0.0f;
  auto fetch = [&](int64_t r0, int slot) {  // the pieces of a row
    const int64_t r = r0 + threadIdx.x / TPR;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * TPR + t) * V;
      if (r < R && c < C) {
        Piece* const to = ring + (slot * 2 * NV + k) * N;
        if constexpr (V == 8) {
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(x + r * ld + c) : "memory");
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to + NV * N)), "l"(dy + r * ldy + c)
                       : "memory");
        } else {
          ahead[k] = *reinterpret_cast<const Piece*>(x + r * ld + c);
          ahead[NV + k] = *reinterpret_cast<const Piece*>(dy + r * ldy + c);
        }
      }
    }
    if (r < R) {
      float* const to = stats + slot * 2 * N;
      if constexpr (V == 8) {
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(mean + r) : "memory");
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"((uint32_t)__cvta_generic_to_shared(to + N)), "l"(rstd + r) : "memory");
      } else {
        ahead_mean = __ldg(mean + r), ahead_rstd = __ldg(rstd + r);
      }
    }
    if constexpr (V == 8) asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < DEPTH - 1; ++i) fetch(first + i * step, i);
  Floats<V> dw[NV] = {}, db[NV] = {}, wv[NV] = {};
#pragma unroll
  for (int k = 0; k < NV; ++k)
    if ((k * TPR + t) * V < C) wv[k] = weights<V>(w + (k * TPR + t) * V);
  int turn = 0, slot = 0;
  for (int64_t r0 = first; r0 < R; r0 += step) {
    const int64_t r = r0 + threadIdx.x / TPR;
    const bool there = r < R;
    Piece now[V == 8 ? 1 : 2 * NV];
    float k1 = ahead_rstd, m = ahead_mean;
    if constexpr (V == 1) {
#pragma unroll
      for (int k = 0; k < 2 * NV; ++k) now[k] = ahead[k];
    }
    fetch(r0 + (DEPTH - 1) * step, slot == 0 ? DEPTH - 1 : slot - 1);
    if constexpr (V == 8) {
      asm volatile("cp.async.wait_group %0;" ::"n"(DEPTH - 1) : "memory");
      m = stats[slot * 2 * N], k1 = stats[(slot * 2 + 1) * N];
    }
    if (!there) m = k1 = 0.0f;
    const Piece* const mine = ring + slot * 2 * NV * N;
    auto of_x = [&](int k) { return floats<T, V>(V == 8 ? mine[k * N] : now[V == 8 ? 0 : k]); };
    auto of_dy = [&](int k) { return floats<T, V>(V == 8 ? mine[(NV + k) * N] : now[V == 8 ? 0 : NV + k]); };
    Floats<V> s0 = all<V>(0.0f), s1 = s0;
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (there && (k * TPR + t) * V < C) {
        const Floats<V> d = of_dy(k), h = mul<V>(add<V>(of_x(k), all<V>(-m)), all<V>(k1));
        const Floats<V> g = mul<V>(d, wv[k]);
        s0 = add<V>(s0, g);
        s1 = fma<V>(g, h, s1);
        dw[k] = fma<V>(d, h, dw[k]);
        db[k] = add<V>(db[k], d);
      }
    if (dx) {
      float s[2] = {sum<V>(s0), sum<V>(s1)};
      row_sums<TPR>(s, room, turn);
      const float a = -k1 * s[0] * over, b = -k1 * s[1] * over;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = (k * TPR + t) * V;
        if (!there || c >= C) continue;
        const Floats<V> h = mul<V>(add<V>(of_x(k), all<V>(-m)), all<V>(k1));
        const Floats<V> g = mul<V>(of_dy(k), wv[k]);
        store<T, V>(dx + r * C + c, fma<V>(g, all<V>(k1), fma<V>(h, all<V>(b), all<V>(a))));
      }
    }
    slot = slot == DEPTH - 1 ? 0 : slot + 1;
  }
  if (!part) return;
  float* const to = part + blockIdx.x * (int64_t)2 * C;
  float* const gathered = reinterpret_cast<float*>(ring_bytes);
  if constexpr (V == 8) asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (GROUPS > 1) {
      __syncthreads();
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e) gathered[(threadIdx.x / TPR * NV + k) * TPR * V + t * V + e] = i ? db[k].v[e] : dw[k].v[e];
      __syncthreads();
      for (int c = threadIdx.x; c < C; c += N) {
        float v = 0.0f;
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) v += gathered[g * NV * TPR * V + c];
        to[i * C + c] = v;
      }
    } else {
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e)
          if ((k * TPR + t) * V + e < C) to[i * C + (k * TPR + t) * V + e] = i ? db[k].v[e] : dw[k].v[e];
    }
  }
}

template <typename T, typename W>
__global__ void __launch_bounds__(1024) long_backward_kernel(const T* __restrict__ dy, int64_t ldy, const T* __restrict__ x, int64_t ld,
                                                             const float* __restrict__ mean, const float* __restrict__ rstd,
                                                             const W* __restrict__ w, T* __restrict__ dx, int64_t R, int C) {
  __shared__ __align__(16) float room[128];
  const float over = 1.0f / C;
  int turn = 0;
  for (int64_t r = blockIdx.x; r < R; r += gridDim.x) {
    const T *p = x + r * ld, *q = dy + r * ldy;
    const float m = mean[r], k = rstd[r];
    float s[2] = {0.0f, 0.0f};
    for (int c = threadIdx.x; c < C; c += 1024) {
      const float g = to_float(q[c]) * to_float(w[c]);
      s[0] += g;
      s[1] = fmaf(g, (to_float(p[c]) - m) * k, s[1]);
    }
    row_sums<1024>(s, room, turn);
    const float a = s[0] * over, b = s[1] * over;
    for (int c = threadIdx.x; c < C; c += 1024)
      dx[r * C + c] = from_float<T>(k * (fmaf(to_float(q[c]), to_float(w[c]), -a) - (to_float(p[c]) - m) * k * b));
  }
}

// part[i][0 and 1][C]: the sums of dy h and dy over the rows i, i + gridDim.y, ...
template <typename T>
__global__ void __launch_bounds__(THREADS) long_weights_kernel(const T* __restrict__ dy, int64_t ldy, const T* __restrict__ x,
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

// The sums over the n parts: 32 columns of dw, then of db, to a CTA, its warps taking parts in turn, in a fixed order.
template <typename W>
__global__ void __launch_bounds__(512) finish_kernel(const float* __restrict__ part, int n, int C, W* dw, W* db) {
  __shared__ float sums[16][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
  const int64_t c = blockIdx.x * (int64_t)32 + lane;
  float s = 0.0f;
  if (c < 2 * (int64_t)C) {
#pragma unroll 8
    for (int i = warp; i < n; i += 16) s += __ldg(part + (int64_t)i * 2 * C + c);
  }
  sums[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && c < 2 * (int64_t)C) {
    s = 0.0f;
#pragma unroll
    for (int w = 0; w < 16; ++w) s += sums[w][lane];
    W* to = c < C ? dw : db;
    if (to) to[c < C ? c : c - C] = from_float<W>(s);
  }
}

// CTAs of the backward pass at most, and so partial sums of the weights' gradients
int parts(int64_t R, int64_t C) { return (int)std::min<int64_t>(std::max<int64_t>(R, 1), C > 8192 ? 148 : 148 * 4); }
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
struct Front {
  const T* x;
  int64_t ld;
  const W *w, *b;
  T* y;
  float *mean, *rstd;
  int64_t R;
  int C;
  float eps;
  cudaStream_t st;

  template <int TPR, int NV, int V>
  void run() const {
    constexpr int N = TPR > THREADS ? TPR : THREADS, ROWS = TPR > THREADS ? 2 : NV * V >= 32 ? 1 : NV * V >= 16 ? 2 : 4;
    const int64_t ctas = (R + N / TPR * ROWS - 1) / (N / TPR * ROWS);
    forward_kernel<T, W, TPR, NV, V, ROWS><<<(unsigned)std::min<int64_t>(ctas, 148 * 16), N, 0, st>>>(x, ld, w, b, y, mean, rstd, R, C, eps);
  }
  // A warp takes rows of up to 2048 places: it needs no barrier.
  void lay_out(bool vec) const {
    const int n = C / 8;
    if (!vec) narrow();
    else if (n <= 8) run<8, 1, 8>();
    else if (n <= 16) run<16, 1, 8>();
    else if (n <= 32) run<32, 1, 8>();
    else if (n <= 64) run<32, 2, 8>();
    else if (n <= 128) run<32, 4, 8>();
    else if (n <= 256) run<32, 8, 8>();
    else if (n <= 512) run<256, 2, 8>();
    else if (n <= 1024) run<256, 4, 8>();
    else if (n <= 2048) run<512, 4, 8>();
    else run_long();
  }
  void narrow() const {
    if (C <= 32) run<32, 1, 1>();
    else if (C <= 128) run<32, 4, 1>();
    else if (C <= 512) run<32, 16, 1>();
    else if (C <= 1024) run<32, 32, 1>();
    else if (C <= 4096) run<256, 16, 1>();
    else if (C <= 8192) run<512, 16, 1>();
    else run_long();
  }
  void run_long() const {
    long_forward_kernel<T, W><<<(unsigned)std::min<int64_t>(R, 148 * 4), 1024, 0, st>>>(x, ld, w, b, y, mean, rstd, R, C, eps);
  }
};
template <typename T, typename W>
struct BackOf : Back {
  cudaStream_t st;
  template <int TPR, int NV, int V>
  void run() const {
    constexpr int N = TPR > THREADS ? TPR : THREADS, GROUPS = N / TPR, DEPTH = V == 8 ? (NV > 2 ? 3 : NV > 1 ? 5 : 6) : 2;
    constexpr int ring = V == 8 ? DEPTH * (2 * NV * N * V * 2 + 2 * N * 4) : 0, sums = GROUPS > 1 ? N * NV * V * 4 : 0, smem = ring > sums ? ring : sums;
    // That an SM holds at a time; more of them start a second, mostly empty round.  C <= 64: 3 of 6 rows' depth, R1048576 C64 88 us with
    // events around the call; 4 CTAs of that depth 92, 4 of a depth of 5, which do fit, 96.
    constexpr int CTAS = TPR > THREADS ? 1 : NV > 1 ? 2 : V == 8 ? 3 : 4;
    static_assert((smem + 2048) * CTAS <= 228 * 1024, "1 KB of an SM's shared memory goes to each CTA, and some to its static part");
    constexpr auto kernel = backward_kernel<T, W, TPR, NV, V, DEPTH>;
    if (smem > 32 * 1024 && allow_smem<kernel>(smem) != cudaSuccess) return;  // its error is found after the call
    const int n = (int)std::min<int64_t>((R + GROUPS - 1) / GROUPS, 148 * CTAS);
    kernel<<<n, N, smem, st>>>(static_cast<const T*>(dy), ldy, static_cast<const T*>(x), ld, mean, rstd, static_cast<const W*>(w),
                               static_cast<T*>(dx), dw || db ? part : nullptr, R, C);
    finish(n);
  }
  // What a thread has of a row grows only where a CTA's threads do not reach: it keeps two sums for each of its places.
  void lay_out(bool vec) const {
    const int n = C / 8;
    if (!vec) narrow();
    else if (n <= 8) run<8, 1, 8>();
    else if (n <= 16) run<8, 2, 8>();
    else if (n <= 32) run<16, 2, 8>();
    else if (n <= 64) run<32, 2, 8>();
    else if (n <= 128) run<64, 2, 8>();
    else if (n <= 256) run<128, 2, 8>();
    else if (n <= 512) run<256, 2, 8>();
    else if (n <= 1024) run<512, 2, 8>();
    else if (n <= 2048) run<512, 4, 8>();
    else run_long();
  }
  void narrow() const {
    if (C <= 32) run<32, 1, 1>();
    else if (C <= 128) run<32, 4, 1>();
    else if (C <= 512) run<128, 4, 1>();
    else if (C <= 1024) run<256, 4, 1>();
    else if (C <= 4096) run<512, 8, 1>();
    else if (C <= 8192) run<512, 16, 1>();
    else run_long();
  }
  void run_long() const {
    if (dx)
      long_backward_kernel<T, W><<<(unsigned)std::min<int64_t>(R, 148 * 4), 1024, 0, st>>>(
          static_cast<const T*>(dy), ldy, static_cast<const T*>(x), ld, mean, rstd, static_cast<const W*>(w), static_cast<T*>(dx), R, C);
    const int n = parts(R, C);
    if (dw || db)
      long_weights_kernel<T><<<dim3((unsigned)((C + THREADS - 1) / THREADS), (unsigned)n), THREADS, 0, st>>>(
          static_cast<const T*>(dy), ldy, static_cast<const T*>(x), ld, mean, rstd, part, R, C);
    finish(n);
  }
  void finish(int n) const {
    if (dw || db) finish_kernel<W><<<(unsigned)((2 * (int64_t)C + 31) / 32), 512, 0, st>>>(part, n, C, static_cast<W*>(dw), static_cast<W*>(db));
  }
};

bool eights(const void* p, int64_t ld, int64_t R, int C) { return C % 8 == 0 && aligned(p, 16) && (R <= 1 || ld % 8 == 0); }

template <typename T, typename W>
void backward(const Back& A, cudaStream_t st) {
  const BackOf<T, W> f = {A, st};
  f.lay_out(eights(A.dy, A.ldy, A.R, A.C) && eights(A.x, A.ld, A.R, A.C) && aligned(A.w, 16));
}
template <typename T, typename W>
void forward(const void* x, int64_t ld, const void* w, const void* b, void* y, float* mean, float* rstd, int64_t R, int C, float eps,
             cudaStream_t st) {
  const Front<T, W> f = {static_cast<const T*>(x), ld, static_cast<const W*>(w), static_cast<const W*>(b), static_cast<T*>(y), mean, rstd, R, C, eps, st};
  f.lay_out(eights(x, ld, R, C) && aligned(w, 16) && aligned(b, 16));
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
  return (size_t)parts(R, C) * 2 * (size_t)C * sizeof(float);
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
  if (R == 0) {  // nothing is read: the weight may be missing
    for (void* to : {dweight, dbias})
      if (to)
        if (cudaError_t e = cudaMemsetAsync(to, 0, (size_t)C * ws, st)) return set_cuda_error(e, "csn_layer_norm_rows_bwd");
    return CSN_OK;
  }
  KernelTimer kt("layer_norm_rows_bwd", st);
  const Back A = {dy, x, weight, ldy, ldx, mean, rstd, dx, dweight, dbias, static_cast<float*>(workspace), R, (int)C};
  auto* f = dtype == CSN_BF16 ? (weight_dtype == CSN_F32 ? backward<__nv_bfloat16, float> : backward<__nv_bfloat16, __nv_bfloat16>)
                              : (weight_dtype == CSN_F32 ? backward<__half, float> : backward<__half, __half>);
  f(A, st);
  return check_launch("csn_layer_norm_rows_bwd");
}

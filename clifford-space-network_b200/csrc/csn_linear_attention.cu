// csn_linear_attention.cu -- linear attention with a decay for each head, its adjoint and its step.
#include "csn_linear_attention.cuh"

#include <algorithm>
#include <cstdio>

namespace csn {
namespace {

using namespace la;

constexpr int MAX_D = 128;
constexpr int BLOCK = 16;  // steps that are worked on together

// n steps from X, in their order of processing (BACK: time runs down; X carried is Y, after its fade):
//   out_i = so (l^(i+1) X^T a_i + sum over j <= i of l^(i-j) sb (a_i . b_j) v_j),   X <- l^n X + sum of l^(n-1-j) sb b_j v_j^T
// (one power of l less before the first product and one more in the last sum where time runs down).  A thread has one
// place of v and the K entries of the state beside it in registers: one packed pair of FMA an entry and step for each of the two
// products, the products a . b shared by all threads.  The state is rounded once a block: step by step, a memory of
// thousands of steps costs it a digit.
// The rows come DEPTH - 1 blocks ahead by cp.async, 16 bytes at a time where they are aligned (`wide`).  What it does most is load a
// and b from shared memory, which every thread needs, one load for two packed FMA: at B32 T2048 H4 D32 that pipe is busy for 48 to
// 64 % of the time and issue for 41 to 53 %, with 2 to 3 warps a scheduler, which wait for such loads.  At B8 T1024 H4 D32, 2 warps an
// SM, it is 13 % and 25 %: there a single warp's chain is the time.  Forward, with the first pass, B32 T2048 H4 D32
// 161 us, B8 T4096 H16 D64 780, B2 T2048 H16 D128 386.  Slower: step by step (three roundings a step, too) and rows loaded when
// their turn comes, 706 us for the first; half as many segments 158, 874 and 457.
// OUT: false for the first pass.
constexpr int MAX_PASSES = 3;
struct Passes {
  Pass pass[MAX_PASSES];
};
constexpr int DEPTH = 3;
__host__ __device__ constexpr int line(int places) { return places + 4; }  // aligned, and rows spread over the banks
__host__ __device__ constexpr int stage_floats(int kp, int vp, bool out) { return BLOCK * ((out ? 2 : 1) * line(kp) + line(vp)); }

__device__ __forceinline__ void copy_async(float* to, const float* from, bool wide) {
  const uint32_t at = (uint32_t)__cvta_generic_to_shared(to);
  if (wide) asm volatile("cp.async.ca.shared.global [%0], [%1], 16;" ::"r"(at), "l"(from) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(at), "l"(from) : "memory");
}

template <int KP, int VP, bool OUT>
__global__ void __launch_bounds__(VP) blocks_kernel(const Batch B, const __grid_constant__ Passes passes, bool wide) {
  const Pass& P = passes.pass[blockIdx.z];
  const Unit U(B, blockIdx.x, !OUT, P.back);
  if (U.s < 0 || (!OUT && U.ends(P.back))) return;
  constexpr int NJ = BLOCK * BLOCK / VP, LK = line(KP), LV = line(VP), STAGE = stage_floats(KP, VP, OUT);
  const int h = blockIdx.y, c = threadIdx.x, late = P.back ? 1 : 0;
  const bool mine = c < P.V;
  extern __shared__ __align__(16) float stages[];  // [DEPTH][b, v, a][BLOCK][places]
  __shared__ __align__(16) float prod[OUT ? BLOCK : 1][BLOCK + 4];
  __shared__ float power[BLOCK + 2];
  if (c < BLOCK + 2) power[c] = fade(B.log_decay[h], c);
  for (int i = c; i < DEPTH * STAGE; i += VP) stages[i] = 0.0f;
  const int64_t size = (int64_t)P.K * P.V;
  float2 x[KP / 2];
#pragma unroll
  for (int i = 0; i < KP / 2; ++i) x[i] = make_float2(0.0f, 0.0f);
  const bool cut = U.len > B.seg;
  const float* const enters = cut ? P.made : P.state;
  if (OUT && enters && mine) {
    const float* p = enters + ((cut ? U.unit : U.s) * B.H + h) * size + c * P.sc;
#pragma unroll
    for (int i = 0; i < KP / 2; ++i) {
      if (2 * i < P.K) x[i].x = p[2 * i * P.sr];
      if (2 * i + 1 < P.K) x[i].y = p[(2 * i + 1) * P.sr];
    }
  }
  const float* a = static_cast<const float*>(P.a.p) + U.start(B, P.a) + h / P.a.shared * P.a.head;
  const float* b = static_cast<const float*>(P.b.p) + U.start(B, P.b) + h / P.b.shared * P.b.head;
  const float* v = static_cast<const float*>(P.v.p) + U.start(B, P.v) + h / P.v.shared * P.v.head;
  const int steps = U.to - U.from;
  // the rows of a block, in their order of processing; what lies behind the last is left as it is
  auto fetch = [&](int done) {
    const int n = min(BLOCK, steps - done);
    float* const to = stages + done / BLOCK % DEPTH * STAGE;
    auto rows = [&](const float* from, int64_t pitch, int places, int l, float* at) {
      const int w = wide ? 4 : 1, pieces = (places + w - 1) / w;
      for (int i = c; i < n * pieces; i += VP) {
        const int r = i / pieces, d = (i - r * pieces) * w;
        copy_async(at + r * l + d, from + (P.back ? U.to - 1 - done - r : U.from + done + r) * pitch + d, wide);
      }
    };
    if (n > 0) {
      rows(b, P.b.row, P.K, LK, to);
      rows(v, P.v.row, P.V, LV, to + BLOCK * LK);
      if (OUT) rows(a, P.a.row, P.K, LK, to + BLOCK * (LK + LV));
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  __syncthreads();
  for (int i = 0; i < DEPTH - 1; ++i) fetch(i * BLOCK);
  for (int done = 0; done < steps; done += BLOCK) {
    const int n = min(BLOCK, steps - done);
    asm volatile("cp.async.wait_group %0;" ::"n"(DEPTH - 2) : "memory");
    __syncthreads();
    fetch(done + (DEPTH - 1) * BLOCK);  // over the block before, which every thread is done with
    const float* const bs = stages + done / BLOCK % DEPTH * STAGE;
    const float *const vb = bs + BLOCK * LK, *const as = bs + BLOCK * (LK + LV);
    if (OUT) {
      const int i = c % BLOCK, j0 = c / BLOCK * NJ;
      float2 r[NJ];
#pragma unroll
      for (int j = 0; j < NJ; ++j) r[j] = make_float2(0.0f, 0.0f);
#pragma unroll 4
      for (int d = 0; d < KP; d += 4) {
        const float4 a4 = *reinterpret_cast<const float4*>(as + i * LK + d);
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          const float4 b4 = *reinterpret_cast<const float4*>(bs + (j0 + j) * LK + d);
          r[j] = fma2(make_float2(a4.x, a4.y), make_float2(b4.x, b4.y), r[j]);
          r[j] = fma2(make_float2(a4.z, a4.w), make_float2(b4.z, b4.w), r[j]);
        }
      }
#pragma unroll
      for (int j = 0; j < NJ; ++j) prod[OUT ? i : 0][j0 + j] = j0 + j <= i ? (r[j].x + r[j].y) * power[i - j0 - j] : 0.0f;
    }
    float2 o[OUT ? BLOCK : 1];
    float vs[BLOCK];
#pragma unroll
    for (int i = 0; i < BLOCK; ++i) {
      vs[i] = i < n && mine ? vb[i * LV + c] * P.sb : 0.0f;
      if (OUT) o[OUT ? i : 0] = make_float2(0.0f, 0.0f);
    }
    const float whole = power[n];
    // what rows behind the last hold does not count
    float w[BLOCK];
#pragma unroll
    for (int i = 0; i < BLOCK; ++i) w[i] = i < n ? vs[i] * power[n - 1 - i + late] : 0.0f;
#pragma unroll
    for (int d = 0; d < KP; d += 4) {
      float2 t0 = make_float2(0.0f, 0.0f), t1 = t0;
#pragma unroll
      for (int i = 0; i < BLOCK; ++i) {
        const float4 b4 = *reinterpret_cast<const float4*>(bs + i * LK + d);
        t0 = fma2(make_float2(b4.x, b4.y), twice(w[i]), t0);
        t1 = fma2(make_float2(b4.z, b4.w), twice(w[i]), t1);
        if (OUT) {
          const float4 a4 = *reinterpret_cast<const float4*>(as + i * LK + d);
          o[OUT ? i : 0] = fma2(make_float2(a4.x, a4.y), x[d / 2], o[OUT ? i : 0]);
          o[OUT ? i : 0] = fma2(make_float2(a4.z, a4.w), x[d / 2 + 1], o[OUT ? i : 0]);
        }
      }
      x[d / 2] = fma2(twice(whole), x[d / 2], t0);
      x[d / 2 + 1] = fma2(twice(whole), x[d / 2 + 1], t1);
    }
    if (!OUT) continue;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < BLOCK; ++i) {
      float r = 0.0f;
#pragma unroll
      for (int j = 0; j <= i; j += 4) {
        const float4 p4 = *reinterpret_cast<const float4*>(&prod[OUT ? i : 0][j]);
        const float pv[4] = {p4.x, p4.y, p4.z, p4.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (j + e <= i) r = fmaf(pv[e], vs[j + e], r);  // a later step's infinity has to stay out
      }
      if (i >= n || !mine) continue;
      r = fmaf(power[i + 1 - late], o[OUT ? i : 0].x + o[OUT ? i : 0].y, r) * P.so;
      const int64_t t = U.row0 + (P.back ? U.to - 1 - done - i : U.from + done + i), at = (t * B.H + h) * P.V + c;
      static_cast<float*>(P.out)[at] = r;
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  float* to = OUT ? (P.last && U.ends(P.back) ? P.last + (U.s * B.H + h) * size : nullptr) : P.made + (U.unit * B.H + h) * size;
  if (to && mine) {
#pragma unroll
    for (int i = 0; i < KP / 2; ++i) {
      if (2 * i < P.K) to[2 * i * P.sr + c * P.sc] = x[i].x;
      if (2 * i + 1 < P.K) to[(2 * i + 1) * P.sr + c * P.sc] = x[i].y;
    }
  }
}

// What enters each segment of the sequences that are cut, in place of what it made: made[u] holds the sum of a unit's own steps.
__global__ void __launch_bounds__(256) join_kernel(const Batch B, const float* __restrict__ enters, float* made, int size, bool back) {
  const int64_t s = blockIdx.x;
  const int h = blockIdx.y, i = blockIdx.z * 256 + threadIdx.x;
  const int64_t row0 = B.cu ? Unit::border(B, s) : s * B.T;
  const int64_t len = B.cu ? max(Unit::border(B, s + 1), row0) - row0 : B.T;
  const int64_t first = B.cu ? row0 / B.seg + s : s * B.segs, n = (len + B.seg - 1) / B.seg;
  if (n < 2) return;
  __shared__ float fades[2];  // of a whole segment and of the last one
  if (threadIdx.x < 2) fades[threadIdx.x] = fade(B.log_decay[h], threadIdx.x == 0 ? B.seg : (int)(len - (n - 1) * B.seg));
  __syncthreads();
  if (i >= size) return;
  const float whole = fades[0], rest = fades[1];
  float x = enters ? enters[(s * B.H + h) * size + i] : 0.0f;
  const int64_t step = (back ? -1 : 1) * (int64_t)B.H * size;
  float* p = made + ((first + (back ? n - 1 : 0)) * B.H + h) * size + i;
  constexpr int N = 8;  // loads in flight
  for (int64_t j0 = 0; j0 < n; j0 += N) {
    float own[N];
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j0 + j + 1 < n) own[j] = p[j * step];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (j0 + j >= n) break;
      p[j * step] = x;
      if (j0 + j + 1 < n) x = fmaf(back && j0 + j == 0 ? rest : whole, x, own[j]);  // only the last segment in time may be short
    }
    p += N * step;
  }
}

// [rows][H][D] float32 to [rows][H / shared][D] of type T; N places to a thread
template <typename T, int N>
__global__ void __launch_bounds__(256) gather_kernel(const float* __restrict__ part, T* out, int64_t n, int D, int shared) {
  const int per = D / N;
  for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    // (a 64-bit division costs as much as the loads)
    const int64_t row = i <= 0x7fffffff ? (int64_t)((uint32_t)i / (uint32_t)per) : i / per;
    const float* p = part + row * shared * D + (i - row * per) * N;
    Pack<float, N> v = *reinterpret_cast<const Pack<float, N>*>(p);
    for (int j = 1; j < shared; ++j) {
      const Pack<float, N> w = *reinterpret_cast<const Pack<float, N>*>(p + (int64_t)j * D);
#pragma unroll
      for (int e = 0; e < N; ++e) v.v[e] += w.v[e];
    }
    Pack<T, N> o;
#pragma unroll
    for (int e = 0; e < N; ++e) o.v[e] = from_float<T>(v.v[e]);
    reinterpret_cast<Pack<T, N>*>(out)[i] = o;
  }
}
template <typename T>
void gather(const float* part, void* out, int64_t n, int D, int shared, cudaStream_t st) {
  const int N = D % 4 ? 1 : 4;
  const unsigned grid = (unsigned)std::min((n / N + 255) / 256, (int64_t)148 * 16);
  if (N == 4) gather_kernel<T, 4><<<grid, 256, 0, st>>>(part, static_cast<T*>(out), n / 4, D, shared);
  else gather_kernel<T, 1><<<grid, 256, 0, st>>>(part, static_cast<T*>(out), n, D, shared);
}

// Rows of no sequence are 0: those before the first border and from the last one on.
__global__ void __launch_bounds__(256) outside_kernel(const Batch B, uint16_t* out, int64_t row) {
  const int64_t a = Unit::border(B, 0) * row, b = max(Unit::border(B, B.S) * row, a), n = a + B.T * row - b;
  for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256)
    out[i < a ? i : i - a + b] = 0;
}

// ------------------------------------------------------------------------- step
struct StepArgs {
  const void *q, *k, *v;
  int64_t qs, qh, ks, kh, vs, vh;  // strides of stream and head
  const float* log_decay;
  float* s;
  void* o;
  int H, shared, Dk, Dv;
  float scale;
};

// A CTA has one head of one stream.  VEC neighbouring entries of a row of the state belong to a thread, 1 << WIDE threads
// take a row and the others the rows that follow, ROWS of them in flight.  Bound by the states' bytes: B256 H16 D128 bf16 85 us,
// 6.3 TB/s.
constexpr int STEP_THREADS = 256;
template <typename T, int VEC, int ROWS>
__global__ void __launch_bounds__(STEP_THREADS) step_kernel(const StepArgs A, int wide) {
  __shared__ float qs[MAX_D], ks[MAX_D], vs[MAX_D];
  __shared__ float part[STEP_THREADS * VEC];
  const int h = blockIdx.x % A.H, tid = threadIdx.x;
  const int64_t b = blockIdx.x / A.H;
  const int c = (tid & ((1 << wide) - 1)) * VEC, r0 = tid >> wide, step = STEP_THREADS >> wide;
  float* s = A.s + (b * A.H + h) * (int64_t)A.Dk * A.Dv + c;
  const bool mine = c < A.Dv;
  using Row = Pack<float, VEC>;
  Row x[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i)
    if (mine && r0 + i * step < A.Dk) x[i] = *reinterpret_cast<const Row*>(s + (int64_t)(r0 + i * step) * A.Dv);
  if (tid < A.Dk) {
    qs[tid] = to_float(static_cast<const T*>(A.q)[b * A.qs + h * A.qh + tid]) * A.scale;
    ks[tid] = to_float(static_cast<const T*>(A.k)[b * A.ks + h / A.shared * A.kh + tid]);
  }
  if (tid < A.Dv) vs[tid] = to_float(static_cast<const T*>(A.v)[b * A.vs + h / A.shared * A.vh + tid]);
  const float l = expf(A.log_decay[h]);
  __syncthreads();
  float o[VEC] = {}, v[VEC] = {};
  if (mine) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = vs[c + e];
    for (int r = r0;;) {
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        const int k = r + i * step;
        if (k >= A.Dk) break;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          x[i].v[e] = fmaf(ks[k], v[e], l * x[i].v[e]);
          o[e] = fmaf(qs[k], x[i].v[e], o[e]);
        }
        *reinterpret_cast<Row*>(s + (int64_t)k * A.Dv) = x[i];
      }
      r += ROWS * step;
      if (r >= A.Dk) break;
#pragma unroll
      for (int i = 0; i < ROWS; ++i)
        if (r + i * step < A.Dk) x[i] = *reinterpret_cast<const Row*>(s + (int64_t)(r + i * step) * A.Dv);
    }
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e) part[tid * VEC + e] = o[e];
  __syncthreads();
  if (tid < A.Dv) {
    float r = 0.0f;
    for (int i = 0; i < step; ++i) r += part[(i << wide) * VEC + tid];
    static_cast<T*>(A.o)[(b * A.H + h) * A.Dv + tid] = from_float<T>(r);
  }
}

// ------------------------------------------------------------------------- host
int width_of(int dtype) { return dtype == CSN_F32 ? 4 : dtype == CSN_BF16 || dtype == CSN_F16 ? 2 : 0; }
bool aligned(const void* p, int n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b; }

// The steps of a segment, a multiple of 128.  float32: enough segments for 24 warps on each SM.  16 bits, one CTA an SM: what
// takes the least time by these, measured with 128 x 128 states in bf16, in units of 0.1 us: a block of 128 steps 39, the start and end
// of a CTA 90; where sequences are cut, in the first pass 27 and 70, and join_kernel 50, 5 a segment and its states' bytes.  Other
// passes are taken to have these times in the same proportion (a block of 64 places takes about 0.7 of them, one of float16 1.2), and
// a packed batch to be one sequence, since its borders are not known here: none may be as long as a segment, and the first
// pass and join_kernel find nothing to do (3 x 15 us of 664 for L20011 H12 Dk72 Dv104 float16 and 37 sequences).
void cut(Batch& B, int Dk, int Dv, int passes, bool packed, bool half) {
  const int64_t rows = up(B.T, 128), heads = (int64_t)B.H * (packed ? 1 : B.S), ways = std::min(passes, 2);
  int64_t best = 1;
  if (half) {
    int64_t least = INT64_MAX;
    for (int64_t n = 1; n <= std::min(rows, (int64_t)64); ++n) {
      const int64_t blocks = up(rows, n);
      int64_t cost = up(heads * passes * n, 148) * (39 * blocks + 90);
      if (n > 1) cost += up(heads * ways * n, 148) * (27 * blocks + 70) + ways * (50 + 5 * n + heads * n * Dk * Dv / 50000);
      if (cost < least) least = cost, best = n;
    }
  } else {
    best = std::min(rows, up(148 * 24, heads * passes * up(std::min(Dk, Dv), 32)));
  }
  B.seg = (int)(std::max(up(rows, std::max(best, (int64_t)1)), (int64_t)1) * 128);
  B.segs = packed ? 0 : (int)std::max(up(B.T, B.seg), (int64_t)1);
  B.units = packed ? B.T / B.seg + B.S : B.S * B.segs;
}
bool is_cut(const Batch& B, bool packed) { return packed ? B.T > B.seg : B.segs > 1; }

Batch batch(int64_t S, int64_t T, int H, int Dk, int Dv, const int32_t* cu, bool packed, const float* log_decay, bool backward, int dtype) {
  Batch B = {cu, S, T, H, 0, 0, 0, log_decay};
  cut(B, Dk, Dv, backward ? 3 : 1, packed, dtype != CSN_F32);
  return B;
}

size_t copy_floats(int64_t rows, int64_t heads, int64_t D) { return (size_t)up(rows * heads * up(D, 8) * 8 * 2, 16) * 4; }
struct Room {  // in floats
  int64_t states, dk, dv, copies;
  size_t bytes(bool backward) const { return sizeof(float) * (size_t)((backward ? 2 : 1) * states + dk + dv + copies); }
};
Room room(const Batch& B, int Hk, int Dk, int Dv, bool packed, bool backward, int mask) {
  const int64_t rows = packed ? B.T : B.S * B.T;
  const bool shared = backward && Hk < B.H;
  int64_t copies = 0;
  const int64_t heads[4] = {B.H, Hk, Hk, B.H}, D[4] = {Dk, Dk, Dv, Dv};
  for (int i = 0; i < 4; ++i)
    if (mask >> i & 1) copies += copy_floats(rows, heads[i], D[i]);
  // each part in whole sectors of 32 bytes, which the rows of the partial gradients are written in
  return {is_cut(B, packed) ? up(B.units * B.H * Dk * Dv, 8) * 8 : 0, shared ? up(rows * B.H * Dk, 8) * 8 : 0,
          shared ? up(rows * B.H * Dv, 8) * 8 : 0, copies};
}

template <int KP, int VP, bool OUT>
cudaError_t launch_blocks(const Batch& B, const Passes& P, int count, bool wide, cudaStream_t st) {
  constexpr int smem = DEPTH * stage_floats(KP, VP, OUT) * 4;
  if (smem > 32 * 1024)
    if (cudaError_t e = allow_smem<blocks_kernel<KP, VP, OUT>>(smem)) return e;
  blocks_kernel<KP, VP, OUT><<<dim3((unsigned)unit_grid(B, !OUT), (unsigned)B.H, (unsigned)count), VP, smem, st>>>(B, P, wide);
  return cudaSuccess;
}
template <int KP>
cudaError_t launch_blocks(const Batch& B, const Passes& P, int count, int V, bool first, bool wide, cudaStream_t st) {
  if (V <= 32) return first ? launch_blocks<KP, 32, false>(B, P, count, wide, st) : launch_blocks<KP, 32, true>(B, P, count, wide, st);
  if (V <= 64) return first ? launch_blocks<KP, 64, false>(B, P, count, wide, st) : launch_blocks<KP, 64, true>(B, P, count, wide, st);
  return first ? launch_blocks<KP, 128, false>(B, P, count, wide, st) : launch_blocks<KP, 128, true>(B, P, count, wide, st);
}

int run(const Batch& B, const Pass* passes, int count, bool first, int dtype, cudaStream_t st) {
  if (dtype != CSN_F32 && B.T > 0) return tensor_passes(B, passes, count, first, dtype == CSN_BF16, st);
  auto wide = [](const Stream& x, int places) {
    return places % 4 == 0 && aligned(x.p, 16) && x.seq % 4 == 0 && x.row % 4 == 0 && x.head % 4 == 0;
  };
  bool done[MAX_PASSES] = {};
  for (int i = 0; i < count; ++i) {  // passes of the same sizes run side by side in one launch
    if (done[i]) continue;
    Passes P;
    int n = 0;
    bool all_wide = true;
    for (int j = i; j < count; ++j) {
      const Pass& p = passes[j];
      if (done[j] || p.K != passes[i].K || p.V != passes[i].V) continue;
      done[j] = true;
      P.pass[n++] = p;
      all_wide = all_wide && wide(p.a, p.K) && wide(p.b, p.K) && wide(p.v, p.V);
    }
    KernelTimer kt(first ? "linear_attention_first" : "linear_attention", st);
    const int K = passes[i].K, V = passes[i].V;
    const cudaError_t e = K <= 32   ? launch_blocks<32>(B, P, n, V, first, all_wide, st)
                          : K <= 64 ? launch_blocks<64>(B, P, n, V, first, all_wide, st)
                                    : launch_blocks<128>(B, P, n, V, first, all_wide, st);
    if (e != cudaSuccess) return set_cuda_error(e, "csn_linear_attention: shared memory");
  }
  return CSN_OK;
}

// Rows of 16-bit streams that TMA cannot read, copied to rows that it can: [rows][heads][D up to a multiple of 8].
struct Copy {
  const uint16_t* from;
  uint16_t* to;
  int64_t seq, row, head, T, n;  // n: places in all
  int heads, D, pitch;
};
struct Copies {
  Copy copy[4];
};
__global__ void __launch_bounds__(256) copy_kernel(const __grid_constant__ Copies copies) {
  const Copy& C = copies.copy[blockIdx.y];
  for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < C.n; i += (int64_t)gridDim.x * 256) {
    const int d = (int)(i % C.D), h = (int)(i / C.D % C.heads);
    const int64_t r = i / C.D / C.heads;
    C.to[(r * C.heads + h) * C.pitch + d] = C.from[r / C.T * C.seq + r % C.T * C.row + h * C.head + d];
  }
}
bool tma_reads(const void* p, const int64_t* st, int64_t S, int64_t T, int64_t heads) {
  auto step = [](int64_t n, int64_t stride) { return n <= 1 || (stride > 0 && stride % 8 == 0 && stride < (1ll << 38)); };
  return aligned(p, 16) && step(S, st[0]) && step(T, st[1]) && step(heads, st[2]);
}
// Puts copies of the streams of `mask` at `to` and the streams' new places into them.
void copy_streams(Stream* const* streams, const int64_t* heads, const int64_t* D, int count, int mask, int64_t S, int64_t T, bool packed,
                  float* to, cudaStream_t st) {
  Copies C;
  int n = 0;
  int64_t most = 0;
  for (int i = 0; i < count; ++i) {
    if (!(mask >> i & 1)) continue;
    Stream& x = *streams[i];
    const int64_t rows = packed ? T : S * T, pitch = up(D[i], 8) * 8;
    C.copy[n++] = {static_cast<const uint16_t*>(x.p), reinterpret_cast<uint16_t*>(to), x.seq, x.row, x.head, T, rows * heads[i] * D[i],
                   (int)heads[i], (int)D[i], (int)pitch};
    most = std::max(most, C.copy[n - 1].n);
    x = {to, T * heads[i] * pitch, heads[i] * pitch, pitch, x.shared};
    to += copy_floats(rows, heads[i], D[i]);
  }
  if (!n) return;
  KernelTimer kt("linear_attention_copies", st);
  copy_kernel<<<dim3((unsigned)std::min(up(most, 256), (int64_t)148 * 8), (unsigned)n), 256, 0, st>>>(C);
}

void join(const Batch& B, const float* enters, float* made, int size, bool back, cudaStream_t st) {
  KernelTimer kt("linear_attention_join", st);
  join_kernel<<<dim3((unsigned)B.S, (unsigned)B.H, (unsigned)up(size, 256)), 256, 0, st>>>(B, enters, made, size, back);
}

void clear_outside(const Batch& B, void* out, int64_t row_bytes, cudaStream_t st) {
  if (B.cu) outside_kernel<<<64, 256, 0, st>>>(B, static_cast<uint16_t*>(out), row_bytes / 2);
}

int check_sizes(const char* name, int64_t S, int64_t T, int64_t H, int64_t Hk, int64_t Dk, int64_t Dv, int dtype) {
  static thread_local char text[160];
  const char* wrong = S < 0 || T < 0 || H < 0 || Hk < 0 ? "negative size" : nullptr;
  if (!wrong && (H > 0 && (Hk < 1 || H % Hk))) wrong = "the heads of k and v have to divide those of q";
  if (!wrong && S * std::max(H, (int64_t)1) > (1 << 28)) wrong = "at most 2^28 heads in all";
  if (!wrong && (S > (1 << 30) || T > (1 << 30) || H > 65535)) wrong = "at most 2^30 sequences and steps and 65535 heads";
  int code = CSN_ERR_INVALID;
  if (!wrong && (Dk < 1 || Dv < 1 || Dk > MAX_D || Dv > MAX_D)) wrong = "head sizes of 1 to 128", code = CSN_ERR_UNSUPPORTED;
  if (!wrong && !width_of(dtype)) wrong = "dtype is float32, bfloat16 or float16", code = CSN_ERR_UNSUPPORTED;
  if (!wrong) return CSN_OK;
  snprintf(text, sizeof text, "%s: %s", name, wrong);
  return set_error(code, text);
}

Stream stream_of(const void* p, const int64_t* st, int shared) { return {p, st[0], st[1], st[2], shared}; }

}  // namespace
}  // namespace csn

using namespace csn;
using namespace csn::la;

extern "C" int csn_linear_attention_copies(const void* q, const void* k, const void* v, const void* d_o, const int64_t* strides, int64_t S,
                                           int64_t T, int64_t H, int64_t Hk, int64_t Dk, int64_t Dv, int packed, int dtype) {
  if (dtype == CSN_F32 || !strides || T <= 0) return 0;
  const int64_t n = packed ? 1 : S;
  return (tma_reads(q, strides, n, T, H) ? 0 : 1) | (tma_reads(k, strides + 3, n, T, Hk) ? 0 : 2) |
         (tma_reads(v, strides + 6, n, T, Hk) ? 0 : 4) | (!d_o || tma_reads(d_o, strides + 9, n, T, H) ? 0 : 8);
}

extern "C" size_t csn_linear_attention_workspace_bytes(int64_t S, int64_t T, int64_t H, int64_t Hk, int64_t Dk, int64_t Dv,
                                                       int packed, int dtype, int copies, int backward) {
  if (S <= 0 || T <= 0 || H <= 0 || Hk <= 0 || check_sizes("csn_linear_attention_workspace_bytes", S, T, H, Hk, Dk, Dv, dtype) != CSN_OK)
    return 0;
  const Batch B = batch(S, T, (int)H, (int)Dk, (int)Dv, nullptr, packed != 0, nullptr, backward != 0, dtype);
  return room(B, (int)Hk, (int)Dk, (int)Dv, packed != 0, backward != 0, dtype == CSN_F32 ? 0 : copies).bytes(backward != 0);
}

extern "C" int csn_linear_attention_fwd(const void* q, const void* k, const void* v, const int64_t* strides, const float* log_decay,
                                        const float* s0, const int32_t* cu_seqlens, void* o, float* s_last, int64_t S, int64_t T,
                                        int64_t H, int64_t Hk, int64_t Dk, int64_t Dv, float scale, int dtype, void* workspace,
                                        size_t workspace_bytes, void* stream) {
  if (int rc = check_sizes("csn_linear_attention_fwd", S, T, H, Hk, Dk, Dv, dtype)) return rc;
  if (S == 0 || H == 0) return CSN_OK;
  const int size = width_of(dtype);
  const bool packed = cu_seqlens != nullptr, rows = T > 0;
  if (!log_decay || !aligned(s0, 16) || !aligned(s_last, 16) ||
      (rows && (!q || !k || !v || !strides || !o || !aligned(q, size) || !aligned(k, size) || !aligned(v, size) || !aligned(o, 16))))
    return set_error(CSN_ERR_INVALID, "csn_linear_attention_fwd: missing or misaligned pointer");
  const Batch B = batch(S, T, (int)H, (int)Dk, (int)Dv, cu_seqlens, packed, log_decay, false, dtype);
  const int mask = csn_linear_attention_copies(q, k, v, nullptr, strides, S, T, H, Hk, Dk, Dv, packed, dtype);
  const Room R = room(B, (int)Hk, (int)Dk, (int)Dv, packed, false, mask);
  if (R.bytes(false) && (!workspace || workspace_bytes < R.bytes(false) || !aligned(workspace, 16)))
    return set_error(CSN_ERR_INVALID, "csn_linear_attention_fwd: workspace smaller than csn_linear_attention_workspace_bytes");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int shared = (int)(H / Hk), entries = (int)(Dk * Dv);
  static const int64_t none[9] = {};
  const int64_t* ss = strides ? strides : none;
  Pass P = {stream_of(q, ss, 1), stream_of(k, ss + 3, shared), stream_of(v, ss + 6, shared), o, s0, s_last, nullptr, Dv, 1,
            (int)Dk, (int)Dv, scale, 1.0f, false, false};
  Stream* const streams[3] = {&P.a, &P.b, &P.v};
  const int64_t heads[3] = {H, Hk, Hk}, places[3] = {Dk, Dk, Dv};
  copy_streams(streams, heads, places, 3, mask, S, T, packed, static_cast<float*>(workspace) + R.states, st);
  if (R.states) {
    P.made = static_cast<float*>(workspace);
    if (int rc = run(B, &P, 1, true, dtype, st)) return rc;
    join(B, s0, P.made, entries, false, st);
  }
  if (int rc = run(B, &P, 1, false, dtype, st)) return rc;
  if (rows) clear_outside(B, o, H * Dv * size, st);
  return check_launch("csn_linear_attention_fwd");
}

extern "C" int csn_linear_attention_bwd(const void* q, const void* k, const void* v, const void* d_o, const int64_t* strides,
                                        const float* log_decay, const float* s0, const int32_t* cu_seqlens, const float* ds_last,
                                        void* dq, void* dk, void* dv, float* ds0, int64_t S, int64_t T, int64_t H, int64_t Hk,
                                        int64_t Dk, int64_t Dv, float scale, int dtype, void* workspace, size_t workspace_bytes,
                                        void* stream) {
  if (int rc = check_sizes("csn_linear_attention_bwd", S, T, H, Hk, Dk, Dv, dtype)) return rc;
  if (S == 0 || H == 0) return CSN_OK;
  const int size = width_of(dtype);
  const bool packed = cu_seqlens != nullptr, rows = T > 0;
  if (!log_decay || !aligned(s0, 16) || !aligned(ds_last, 16) || !aligned(ds0, 16) ||
      (rows && (!q || !k || !v || !d_o || !strides || (ds0 && !dv) || !aligned(q, size) || !aligned(k, size) || !aligned(v, size) ||
                !aligned(d_o, size) || !aligned(dq, 16) || !aligned(dk, 16) || !aligned(dv, 16))))
    return set_error(CSN_ERR_INVALID, "csn_linear_attention_bwd: missing or misaligned pointer");
  const Batch B = batch(S, T, (int)H, (int)Dk, (int)Dv, cu_seqlens, packed, log_decay, true, dtype);
  const int mask = csn_linear_attention_copies(q, k, v, d_o, strides, S, T, H, Hk, Dk, Dv, packed, dtype);
  const Room R = room(B, (int)Hk, (int)Dk, (int)Dv, packed, true, mask);
  if (R.bytes(true) && (!workspace || workspace_bytes < R.bytes(true) || !aligned(workspace, 16)))
    return set_error(CSN_ERR_INVALID, "csn_linear_attention_bwd: workspace smaller than csn_linear_attention_workspace_bytes");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int shared = (int)(H / Hk), entries = (int)(Dk * Dv);
  static const int64_t none[12] = {};
  const int64_t* ss = strides ? strides : none;
  Stream Q = stream_of(q, ss, 1), K = stream_of(k, ss + 3, shared), V = stream_of(v, ss + 6, shared), O = stream_of(d_o, ss + 9, 1);
  float* ws = static_cast<float*>(workspace);
  float *made = ws, *back = ws + R.states, *dk32 = back + R.states, *dv32 = dk32 + R.dk;
  Stream* const streams[4] = {&Q, &K, &V, &O};
  const int64_t heads[4] = {H, Hk, Hk, H}, places[4] = {Dk, Dk, Dv, Dv};
  copy_streams(streams, heads, places, 4, mask, S, T, packed, dv32 + R.dv, st);
  Pass P[3] = {
      {O, V, K, dq, s0, nullptr, nullptr, 1, Dv, (int)Dv, (int)Dk, scale, 1.0f, false, false},
      {V, O, Q, shared > 1 ? dk32 : dk, ds_last, nullptr, nullptr, 1, Dv, (int)Dv, (int)Dk, 1.0f, scale, shared > 1, true},
      {K, Q, O, shared > 1 ? dv32 : dv, ds_last, ds0, nullptr, Dv, 1, (int)Dk, (int)Dv, 1.0f, scale, shared > 1, true}};
  if (R.states) {
    P[0].made = made, P[1].made = P[2].made = back;
    // the states of the forward direction are those that dq needs
    const Pass firsts[2] = {dq ? P[0] : P[2], P[2]};
    if (int rc = run(B, firsts, dq && (dk || dv) ? 2 : 1, true, dtype, st)) return rc;
    if (dq) join(B, s0, made, entries, false, st);
    if (dk || dv) join(B, ds_last, back, entries, true, st);
  }
  Pass wanted[3];
  int count = 0;
  if (dq) wanted[count++] = P[0];
  if (dk) wanted[count++] = P[1];
  if (dv || ds0) wanted[count++] = P[2];
  if (int rc = run(B, wanted, count, false, dtype, st)) return rc;
  if (rows) {
    const int64_t n = packed ? T : S * T;
    if (shared > 1) {
      KernelTimer kt("linear_attention_gather", st);
      auto* add = dtype == CSN_F32 ? gather<float> : dtype == CSN_BF16 ? gather<__nv_bfloat16> : gather<__half>;
      if (dk) add(dk32, dk, n * Hk * Dk, (int)Dk, shared, st);
      if (dv) add(dv32, dv, n * Hk * Dv, (int)Dv, shared, st);
    }
    if (dq) clear_outside(B, dq, H * Dk * size, st);
    if (dk) clear_outside(B, dk, Hk * Dk * size, st);
    if (dv) clear_outside(B, dv, Hk * Dv * size, st);
  }
  return check_launch("csn_linear_attention_bwd");
}

namespace csn {
namespace {
// whether [p, p + its last element] meets the states
bool shares(const float* s, int64_t states, const void* p, int64_t B, int64_t bs, int64_t H, int64_t hs, int64_t D, int size) {
  const char *a = reinterpret_cast<const char*>(s), *b = reinterpret_cast<const char*>(s + states);
  const int64_t first = std::min((B - 1) * bs, (int64_t)0) + std::min((H - 1) * hs, (int64_t)0);
  const int64_t last = std::max((B - 1) * bs, (int64_t)0) + std::max((H - 1) * hs, (int64_t)0) + D;
  const char* c = static_cast<const char*>(p);
  return c + first * size < b && c + last * size > a;
}

template <typename T>
void launch_step(const StepArgs& A, int64_t ctas, cudaStream_t st) {
  const bool four = A.Dv % 4 == 0;
  int wide = 0;
  while ((four ? 4 : 1) << wide < A.Dv) ++wide;
  if (four) step_kernel<T, 4, 8><<<(unsigned)ctas, STEP_THREADS, 0, st>>>(A, wide);
  else step_kernel<T, 1, 8><<<(unsigned)ctas, STEP_THREADS, 0, st>>>(A, wide);
}
}  // namespace
}  // namespace csn

extern "C" int csn_linear_attention_step(const void* q, const void* k, const void* v, const int64_t* strides, const float* log_decay,
                                         float* s, void* o, int64_t B, int64_t H, int64_t Hk, int64_t Dk, int64_t Dv, float scale,
                                         int dtype, void* stream) {
  if (int rc = check_sizes("csn_linear_attention_step", B, 1, H, Hk, Dk, Dv, dtype)) return rc;
  if (B == 0 || H == 0) return CSN_OK;
  const int size = width_of(dtype);
  if (!q || !k || !v || !strides || !log_decay || !s || !o || !aligned(q, size) || !aligned(k, size) || !aligned(v, size) ||
      !aligned(s, 16) || !aligned(o, 16))
    return set_error(CSN_ERR_INVALID, "csn_linear_attention_step: missing or misaligned pointer");
  if (B * H > 0x7fffffff) return set_error(CSN_ERR_UNSUPPORTED, "csn_linear_attention_step: at most 2^31 - 1 heads in all");
  const int64_t states = B * H * Dk * Dv;
  if (shares(s, states, q, B, strides[0], H, strides[1], Dk, size) || shares(s, states, k, B, strides[2], Hk, strides[3], Dk, size) ||
      shares(s, states, v, B, strides[4], Hk, strides[5], Dv, size) || shares(s, states, o, B, H * Dv, H, Dv, Dv, size) ||
      shares(s, states, log_decay, 1, 0, 1, 0, H, 4))
    return set_error(CSN_ERR_INVALID, "csn_linear_attention_step: s shares memory with an input or the result");
  const StepArgs A = {q, k, v, strides[0], strides[1], strides[2], strides[3], strides[4], strides[5], log_decay, s, o,
                      (int)H, (int)(H / Hk), (int)Dk, (int)Dv, scale};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  KernelTimer kt("linear_attention_step", st);
  if (dtype == CSN_F32) launch_step<float>(A, B * H, st);
  else if (dtype == CSN_BF16) launch_step<__nv_bfloat16>(A, B * H, st);
  else launch_step<__half>(A, B * H, st);
  return check_launch("csn_linear_attention_step");
}

// csn_gated_scan.cu -- the gated linear recurrence over channels, its adjoint and its step.
//
//   a_t = sigmoid(f_t),  q_t = 1 - a_t,  h_t = a_t h_{t-1} + q_t x_t,  y_t = h_t silu(g_t)   (y_t = h_t without g)
// Adjoint, with D_t = h_{t-1} - x_t, dh_t = dy_t silu(g_t) and lam_t = dh_t + a_{t+1} lam_{t+1} (the gradient of
// the last state enters at the end):
//   dx = q lam,  df = lam D a q,  dg = dy h silu'(g),  dh0 = a_0 lam_0
// Each step is the affine map h -> a h + b, and maps compose: (A2, B2) o (A1, B1) = (A2 A1, A2 B1 + B2).  A warp
// takes STEPS neighbouring steps of 32 * V neighbouring channels (a lane keeps V channels; a row of a warp is one
// 128-byte access for 16-bit pairs and for float32), composes its steps in registers, the warps of a CTA pass their
// composed maps through shared memory, and every step is then finished from the state that enters its warp.  So the
// inputs are read once.  All sums, products and states are float32.
//
// The forward pass keeps the float32 state before every MARK-th step ("marks") where a backward pass will follow:
// the adjoint forms the states between two marks again instead of reading rounded outputs (y is not h where there is
// a gate, and a 16-bit h would cost df its precision where h is close to x).
#include <cstdint>

#include "csn_internal.h"
#include "csn_types.cuh"

namespace csn {
namespace {

constexpr int WARPS = 8;
constexpr int STEPS = 8;              // steps of one warp
constexpr int MARK = WARPS * STEPS;   // steps of one CTA pass, and the distance of the kept states

struct Rows {  // rows of an input: element (sequence s, step t, channel c) at p + s * seq + t * row + c
  const void* p;
  int64_t seq, row;
};

struct ScanArgs {
  Rows f, x, g, dy;
  const float* h0;
  const int32_t* cu;  // packed: sequence s has the rows cu[s] .. cu[s + 1] - 1
  void* y;
  float* h_last;
  float* marks;
  const float* dh_last;
  void *df, *dx, *dg;
  float* dh0;
  int64_t S, T, C;
  int tiles;
};

// The rows of sequence s.  Borders outside 0..T, or falling ones, are cut to what is there.
struct Seq {
  int64_t row0;  // its first row in the outputs
  int64_t len;
  int64_t mark0;  // its first mark: room for ceil(len / MARK) of them whatever the other lengths are
  __device__ __forceinline__ Seq(const ScanArgs& A, int64_t s) {
    if (A.cu) {
      const int64_t b = min(max((int64_t)A.cu[s], (int64_t)0), A.T);
      const int64_t e = min(max((int64_t)A.cu[s + 1], b), A.T);
      row0 = b;
      len = e - b;
    } else {
      row0 = s * A.T;
      len = A.T;
    }
    mark0 = row0 / MARK + s;
  }
  template <typename T>
  __device__ __forceinline__ const T* in(const Rows& r, const ScanArgs& A, int64_t s) const {
    return static_cast<const T*>(r.p) + (A.cu ? row0 * r.row : s * r.seq);
  }
};

template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load(const T* p) {
  return *reinterpret_cast<const Pack<T, V>*>(p);
}
template <typename T, int V>
__device__ __forceinline__ void store(T* p, const float* v) {
  Pack<T, V> o;
#pragma unroll
  for (int i = 0; i < V; ++i) o.v[i] = from_float<T>(v[i]);
  *reinterpret_cast<Pack<T, V>*>(p) = o;
}

// Rows that belong to no sequence (before the first, behind the last) are written as 0.
template <typename T, int V>
__device__ void clear_outside(const ScanArgs& A, const Seq& q, int64_t s, int64_t c, bool live, int warp,
                              T* o0, T* o1, T* o2) {
  if (!A.cu || !live) return;
  const float zero[V] = {};
  auto clear = [&](int64_t from, int64_t to) {
    for (int64_t r = from + warp; r < to; r += WARPS) {
      if (o0) store<T, V>(o0 + r * A.C + c, zero);
      if (o1) store<T, V>(o1 + r * A.C + c, zero);
      if (o2) store<T, V>(o2 + r * A.C + c, zero);
    }
  };
  if (s == 0) clear(0, q.row0);
  if (s == A.S - 1) clear(q.row0 + q.len, A.T);
}

template <typename T, int V, bool GATE>
__global__ void __launch_bounds__(WARPS * 32) gated_scan_fwd_kernel(const ScanArgs A) {
  __shared__ float2 maps[2][WARPS][32 * V];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t s = blockIdx.x / A.tiles;
  const int64_t c = (int64_t)(blockIdx.x % A.tiles) * (32 * V) + lane * V;
  const bool live = c < A.C;
  const Seq q(A, s);
  const T* f = q.in<T>(A.f, A, s) + c;
  const T* x = q.in<T>(A.x, A, s) + c;
  const T* g = GATE ? q.in<T>(A.g, A, s) + c : nullptr;
  T* y = static_cast<T*>(A.y);
  float carry[V];
#pragma unroll
  for (int v = 0; v < V; ++v) carry[v] = A.h0 && live ? A.h0[s * A.C + c + v] : 0.0f;

  int half = 0;
  for (int64_t t0 = 0; t0 < q.len; t0 += MARK, half ^= 1) {
    const int64_t t1 = t0 + warp * STEPS;
    // P, H: the composed map from the state that enters this warp to the state after each step
    float P[STEPS][V], H[STEPS][V];
    Pack<T, V> gr[STEPS];
    {
      Pack<T, V> fr[STEPS], xr[STEPS];
#pragma unroll
      for (int l = 0; l < STEPS; ++l)
        if (live && t1 + l < q.len) {
          fr[l] = load<T, V>(f + (t1 + l) * A.f.row);
          xr[l] = load<T, V>(x + (t1 + l) * A.x.row);
          if (GATE) gr[l] = load<T, V>(g + (t1 + l) * A.g.row);
        }
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float p = 1.0f, h = 0.0f;
#pragma unroll
        for (int l = 0; l < STEPS; ++l) {
          if (live && t1 + l < q.len) {
            float a, b;
            sigmoid_pair(to_float(fr[l].v[v]), a, b);
            p *= a;
            h = fmaf(a, h, b * to_float(xr[l].v[v]));
          }
          P[l][v] = p;
          H[l][v] = h;
        }
      }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) maps[half][warp][lane * V + v] = make_float2(P[STEPS - 1][v], H[STEPS - 1][v]);
    __syncthreads();
    float in[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float h = carry[v];
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        if (w == warp) in[v] = h;
        const float2 m = maps[half][w][lane * V + v];
        h = fmaf(m.x, h, m.y);
      }
      carry[v] = h;
    }
    if (A.marks && warp == 0 && live) store<float, V>(A.marks + (q.mark0 + t0 / MARK) * A.C + c, in);
#pragma unroll
    for (int l = 0; l < STEPS; ++l)
      if (live && t1 + l < q.len) {
        float o[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
          o[v] = fmaf(P[l][v], in[v], H[l][v]);
          if (GATE) {
            float z = to_float(gr[l].v[v]), sg, sn;
            sigmoid_pair(z, sg, sn);
            o[v] *= z * sg;
          }
        }
        store<T, V>(y + (q.row0 + t1 + l) * A.C + c, o);
      }
  }
  if (warp == 0 && live && A.h_last) store<float, V>(A.h_last + s * A.C + c, carry);
  clear_outside<T, V>(A, q, s, c, live, warp, y, static_cast<T*>(nullptr), static_cast<T*>(nullptr));
}

template <typename T, int V, bool GATE>
__global__ void __launch_bounds__(WARPS * 32) gated_scan_bwd_kernel(const ScanArgs A) {
  __shared__ float2 maps[2][WARPS][32 * V];  // the forward map of a warp's steps
  __shared__ float back[2][WARPS][32 * V];   // what leaves a warp's first step when nothing enters its last
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t s = blockIdx.x / A.tiles;
  const int64_t c = (int64_t)(blockIdx.x % A.tiles) * (32 * V) + lane * V;
  const bool live = c < A.C;
  const Seq q(A, s);
  const T* f = q.in<T>(A.f, A, s) + c;
  const T* x = q.in<T>(A.x, A, s) + c;
  const T* g = GATE ? q.in<T>(A.g, A, s) + c : nullptr;
  const T* dy = A.dy.p ? q.in<T>(A.dy, A, s) + c : nullptr;
  T *df = static_cast<T*>(A.df), *dx = static_cast<T*>(A.dx), *dg = static_cast<T*>(A.dg);
  float mu[V];  // the gradient that enters the pass from behind: a lam of the step after it
#pragma unroll
  for (int v = 0; v < V; ++v) mu[v] = A.dh_last && live ? A.dh_last[s * A.C + c + v] : 0.0f;

  int half = 0;
  for (int64_t t0 = (q.len - 1) / MARK * MARK; t0 >= 0 && q.len > 0; t0 -= MARK, half ^= 1) {
    const int64_t t1 = t0 + warp * STEPS;
    float a[STEPS][V], b[STEPS][V], xs[STEPS][V], e[STEPS][V], sg[STEPS][V];
    Pack<T, V> gr[STEPS], dr[STEPS];
    {
      Pack<T, V> fr[STEPS], xr[STEPS];
#pragma unroll
      for (int l = 0; l < STEPS; ++l)
        if (live && t1 + l < q.len) {
          fr[l] = load<T, V>(f + (t1 + l) * A.f.row);
          xr[l] = load<T, V>(x + (t1 + l) * A.x.row);
          if (dy) dr[l] = load<T, V>(dy + (t1 + l) * A.dy.row);
          if (GATE) gr[l] = load<T, V>(g + (t1 + l) * A.g.row);
        }
#pragma unroll
      for (int l = 0; l < STEPS; ++l) {
        const bool in = live && t1 + l < q.len;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          a[l][v] = 1.0f;  // a step behind the end passes state and gradient on
          b[l][v] = xs[l][v] = e[l][v] = sg[l][v] = 0.0f;
          if (in) {
            sigmoid_pair(to_float(fr[l].v[v]), a[l][v], b[l][v]);
            xs[l][v] = to_float(xr[l].v[v]);
            e[l][v] = dy ? to_float(dr[l].v[v]) : 0.0f;
            if (GATE) {
              float sn;
              sigmoid_pair(to_float(gr[l].v[v]), sg[l][v], sn);
              e[l][v] *= to_float(gr[l].v[v]) * sg[l][v];
            }
          }
        }
      }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float p = 1.0f, h = 0.0f, r = 0.0f;
#pragma unroll
      for (int l = 0; l < STEPS; ++l) {
        p *= a[l][v];
        h = fmaf(a[l][v], h, b[l][v] * xs[l][v]);
      }
#pragma unroll
      for (int l = STEPS - 1; l >= 0; --l) r = a[l][v] * (e[l][v] + r);
      maps[half][warp][lane * V + v] = make_float2(p, h);
      back[half][warp][lane * V + v] = r;
    }
    __syncthreads();
    float h[V], m[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      h[v] = live ? A.marks[(q.mark0 + t0 / MARK) * A.C + c + v] : 0.0f;
#pragma unroll
      for (int w = 0; w < WARPS - 1; ++w)
        if (w < warp) {
          const float2 k = maps[half][w][lane * V + v];
          h[v] = fmaf(k.x, h[v], k.y);
        }
      float r = mu[v];
#pragma unroll
      for (int w = WARPS - 1; w >= 0; --w) {
        if (w == warp) m[v] = r;
        r = fmaf(maps[half][w][lane * V + v].x, r, back[half][w][lane * V + v]);
      }
      mu[v] = r;
    }
    // forward over the steps: xs becomes D_t = h_{t-1} - x_t, and dg is done
#pragma unroll
    for (int l = 0; l < STEPS; ++l) {
      float o[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float hn = fmaf(a[l][v], h[v], b[l][v] * xs[l][v]);
        xs[l][v] = h[v] - xs[l][v];
        h[v] = hn;
        if (GATE) {
          const float z = to_float(gr[l].v[v]), w = sg[l][v];
          o[v] = dy ? to_float(dr[l].v[v]) * hn * (w * fmaf(z, 1.0f - w, 1.0f)) : 0.0f;
        }
      }
      if (GATE && dg && live && t1 + l < q.len) store<T, V>(dg + (q.row0 + t1 + l) * A.C + c, o);
    }
    // and back: lam_t = dh_t + a_{t+1} lam_{t+1}
#pragma unroll
    for (int l = STEPS - 1; l >= 0; --l) {
      float of[V], ox[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float lam = e[l][v] + m[v];
        m[v] = a[l][v] * lam;
        ox[v] = b[l][v] * lam;
        of[v] = ox[v] * a[l][v] * xs[l][v];
      }
      if (live && t1 + l < q.len) {
        if (dx) store<T, V>(dx + (q.row0 + t1 + l) * A.C + c, ox);
        if (df) store<T, V>(df + (q.row0 + t1 + l) * A.C + c, of);
      }
    }
  }
  if (warp == 0 && live && A.dh0) store<float, V>(A.dh0 + s * A.C + c, mu);
  clear_outside<T, V>(A, q, s, c, live, warp, df, dx, dg);
}

struct StepArgs {
  const void *f, *x, *g;
  int64_t fr, xr, gr;
  float* h;
  void* y;
  int64_t n, C;  // n = packs in all
};

template <typename T, int V, bool GATE>
__global__ void __launch_bounds__(256) gated_step_kernel(const StepArgs A) {
  const int64_t per = A.C / V;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < A.n; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / per, c = (i - r * per) * V;
    const Pack<T, V> f = load<T, V>(static_cast<const T*>(A.f) + r * A.fr + c);
    const Pack<T, V> x = load<T, V>(static_cast<const T*>(A.x) + r * A.xr + c);
    Pack<T, V> g;
    if (GATE) g = load<T, V>(static_cast<const T*>(A.g) + r * A.gr + c);
    const Pack<float, V> h = load<float, V>(A.h + r * A.C + c);
    float hn[V], o[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float a, b;
      sigmoid_pair(to_float(f.v[v]), a, b);
      o[v] = hn[v] = fmaf(a, h.v[v], b * to_float(x.v[v]));
      if (GATE) {
        float z = to_float(g.v[v]), sg, sn;
        sigmoid_pair(z, sg, sn);
        o[v] *= z * sg;
      }
    }
    store<float, V>(A.h + r * A.C + c, hn);
    store<T, V>(static_cast<T*>(A.y) + r * A.C + c, o);
  }
}

int width_of(int dtype) { return dtype == CSN_F32 ? 4 : dtype == CSN_BF16 || dtype == CSN_F16 ? 2 : 0; }

bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) % bytes) == 0; }

// Two channels a lane need even strides and 4-byte aligned rows; otherwise a lane takes one.
bool pairs(const Rows& r) { return !r.p || (r.seq % 2 == 0 && r.row % 2 == 0 && aligned(r.p, 4)); }

template <typename T, int V>
void launch_scan(ScanArgs A, bool bwd, cudaStream_t st) {
  A.tiles = (int)((A.C + 32 * V - 1) / (32 * V));
  const unsigned grid = (unsigned)(A.S * A.tiles);
  if (!bwd) {
    if (A.g.p) gated_scan_fwd_kernel<T, V, true><<<grid, WARPS * 32, 0, st>>>(A);
    else gated_scan_fwd_kernel<T, V, false><<<grid, WARPS * 32, 0, st>>>(A);
  } else {
    if (A.g.p) gated_scan_bwd_kernel<T, V, true><<<grid, WARPS * 32, 0, st>>>(A);
    else gated_scan_bwd_kernel<T, V, false><<<grid, WARPS * 32, 0, st>>>(A);
  }
}

void dispatch_scan(const ScanArgs& A, int dtype, bool bwd, cudaStream_t st) {
  const bool two = A.C % 2 == 0 && pairs(A.f) && pairs(A.x) && pairs(A.g) && pairs(A.dy);
  if (dtype == CSN_F32) launch_scan<float, 1>(A, bwd, st);
  else if (dtype == CSN_BF16 && two) launch_scan<__nv_bfloat16, 2>(A, bwd, st);
  else if (dtype == CSN_BF16) launch_scan<__nv_bfloat16, 1>(A, bwd, st);
  else if (two) launch_scan<__half, 2>(A, bwd, st);
  else launch_scan<__half, 1>(A, bwd, st);
}

int check_scan(const char* who, const ScanArgs& A, int dtype) {
  if (A.S < 0 || A.T < 0 || A.C < 0) return set_error(CSN_ERR_INVALID, who);
  if (!width_of(dtype)) return set_error(CSN_ERR_UNSUPPORTED, who);
  // the grid has one CTA for each 32 channels of a sequence at most
  if (A.S > 0 && A.C > 0 && (A.C + 31) / 32 > (int64_t)0x7fffffff / A.S) return set_error(CSN_ERR_INVALID, who);
  return CSN_OK;
}

}  // namespace
}  // namespace csn

using namespace csn;

extern "C" int64_t csn_gated_scan_marks(int64_t S, int64_t T, int64_t C, int packed) {
  if (S <= 0 || T < 0 || C <= 0) return 0;
  return ((packed ? T : S * T) / MARK + S) * C;
}

extern "C" int csn_gated_scan_fwd(const void* f, const void* x, const void* gate, const int64_t* strides,
                                  const float* h0, const int32_t* cu_seqlens, void* y, float* h_last, float* marks,
                                  int64_t S, int64_t T, int64_t C, int dtype, void* stream) {
  ScanArgs A = {};
  A.S = S, A.T = T, A.C = C;
  if (int rc = check_scan("csn_gated_scan_fwd: needs S, T, C >= 0, dtype float32, bfloat16 or float16, and at most "
                          "2^31 - 1 tiles of 32 channels", A, dtype))
    return rc;
  if (S == 0 || C == 0) return CSN_OK;
  const int size = width_of(dtype);
  if (T > 0 && (!f || !x || !y || !strides || !aligned(f, size) || !aligned(x, size) || !aligned(gate, size)))
    return set_error(CSN_ERR_INVALID, "csn_gated_scan_fwd: f, x, strides and y are required, aligned to their type");
  if (!aligned(h0, 16) || !aligned(y, 16) || !aligned(h_last, 16) || !aligned(marks, 16) || !aligned(cu_seqlens, 4))
    return set_error(CSN_ERR_INVALID, "csn_gated_scan_fwd: h0, y, h_last and marks must be 16-byte aligned");
  if (strides) {
    A.f = {f, strides[0], strides[1]};
    A.x = {x, strides[2], strides[3]};
    A.g = {gate, gate ? strides[4] : 0, gate ? strides[5] : 0};
  }
  A.h0 = h0, A.cu = cu_seqlens, A.y = y, A.h_last = h_last, A.marks = marks;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  KernelTimer kt("gated_scan_fwd", st);
  dispatch_scan(A, dtype, false, st);
  return check_launch("csn_gated_scan_fwd");
}

extern "C" int csn_gated_scan_bwd(const void* f, const void* x, const void* gate, const void* dy,
                                  const int64_t* strides, const int32_t* cu_seqlens, const float* marks,
                                  const float* dh_last, void* df, void* dx, void* dgate, float* dh0, int64_t S,
                                  int64_t T, int64_t C, int dtype, void* stream) {
  ScanArgs A = {};
  A.S = S, A.T = T, A.C = C;
  if (int rc = check_scan("csn_gated_scan_bwd: needs S, T, C >= 0, dtype float32, bfloat16 or float16, and at most "
                          "2^31 - 1 tiles of 32 channels", A, dtype))
    return rc;
  if (S == 0 || C == 0) return CSN_OK;
  const int size = width_of(dtype);
  if (T > 0 && (!f || !x || !marks || !strides || !aligned(f, size) || !aligned(x, size) || !aligned(gate, size) ||
                !aligned(dy, size)))
    return set_error(CSN_ERR_INVALID, "csn_gated_scan_bwd: f, x, marks and strides are required, aligned to their type");
  if (!aligned(marks, 16) || !aligned(dh_last, 16) || !aligned(df, 16) || !aligned(dx, 16) || !aligned(dgate, 16) ||
      !aligned(dh0, 16) || !aligned(cu_seqlens, 4))
    return set_error(CSN_ERR_INVALID, "csn_gated_scan_bwd: marks, dh_last and the gradients must be 16-byte aligned");
  if (strides) {
    A.f = {f, strides[0], strides[1]};
    A.x = {x, strides[2], strides[3]};
    A.g = {gate, gate ? strides[4] : 0, gate ? strides[5] : 0};
    A.dy = {dy, dy ? strides[6] : 0, dy ? strides[7] : 0};
  }
  A.cu = cu_seqlens, A.marks = const_cast<float*>(marks), A.dh_last = dh_last;
  A.df = df, A.dx = dx, A.dg = gate ? dgate : nullptr, A.dh0 = dh0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  KernelTimer kt("gated_scan_bwd", st);
  dispatch_scan(A, dtype, true, st);
  return check_launch("csn_gated_scan_bwd");
}

namespace csn {
namespace {
template <typename T, int V>
void launch_step(StepArgs A, int64_t B, cudaStream_t st) {
  A.n = B * (A.C / V);
  const int64_t ctas = (A.n + 255) / 256;
  const unsigned grid = (unsigned)(ctas < 148 * 64 ? ctas : 148 * 64);
  if (A.g) gated_step_kernel<T, V, true><<<grid, 256, 0, st>>>(A);
  else gated_step_kernel<T, V, false><<<grid, 256, 0, st>>>(A);
}
}  // namespace
}  // namespace csn

extern "C" int csn_gated_step(const void* f, const void* x, const void* gate, const int64_t* strides, float* h,
                              void* y, int64_t B, int64_t C, int dtype, void* stream) {
  if (B < 0 || C < 0) return set_error(CSN_ERR_INVALID, "csn_gated_step: negative size");
  if (!width_of(dtype)) return set_error(CSN_ERR_UNSUPPORTED, "csn_gated_step: dtype is float32, bfloat16 or float16");
  if (B == 0 || C == 0) return CSN_OK;
  const int size = width_of(dtype);
  if (!f || !x || !strides || !h || !y || !aligned(f, size) || !aligned(x, size) || !aligned(gate, size) ||
      !aligned(h, 16) || !aligned(y, 16))
    return set_error(CSN_ERR_INVALID, "csn_gated_step: missing or misaligned pointer");
  StepArgs A = {f, x, gate, strides[0], strides[1], gate ? strides[2] : 0, h, y, 0, C};
  const bool two = C % 2 == 0 && strides[0] % 2 == 0 && strides[1] % 2 == 0 && A.gr % 2 == 0 && aligned(f, 4) &&
                   aligned(x, 4) && aligned(gate, 4);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  KernelTimer kt("gated_step", st);
  if (dtype == CSN_F32) launch_step<float, 1>(A, B, st);
  else if (dtype == CSN_BF16 && two) launch_step<__nv_bfloat16, 2>(A, B, st);
  else if (dtype == CSN_BF16) launch_step<__nv_bfloat16, 1>(A, B, st);
  else if (two) launch_step<__half, 2>(A, B, st);
  else launch_step<__half, 1>(A, B, st);
  return check_launch("csn_gated_step");
}

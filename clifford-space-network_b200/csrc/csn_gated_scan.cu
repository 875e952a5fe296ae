// csn_gated_scan.cu -- the gated linear recurrence over channels, its adjoint and its step.
//
//   a_t = sigmoid(f_t),  q_t = 1 - a_t,  h_t = a_t h_{t-1} + q_t x_t,  y_t = h_t silu(g_t)   (y_t = h_t without g)
// Adjoint, with D_t = h_{t-1} - x_t, dh_t = dy_t silu(g_t) and lam_t = dh_t + a_{t+1} lam_{t+1} (the gradient of
// the last state enters at the end):
//   dx = q lam,  df = lam D a q,  dg = dy h silu'(g),  dh0 = a_0 lam_0
//
// With s = min(a, q), exact in its relative precision, a step is h + s (x - h) or x + s (h - x): rounding a itself
// near 1 would drift a long memory, rounding h does not.  c = s, or -s where q is the larger, keeps both.
//
// Each step is an affine map h -> A h + B, and maps compose: (A2, B2) o (A1, B1) = (A2 A1, A2 B1 + B2).  A warp takes
// STEPS neighbouring steps of 32 * V neighbouring channels (a lane keeps V channels; a row of a warp is one 128-byte
// access for 16-bit pairs and for float32) and composes them in registers; the warps of a CTA pass their maps through
// shared memory, the CTAs of a cluster, which take neighbouring MARK-step pieces of one sequence, through distributed
// shared memory; then every warp runs its steps again from the state that enters them.  So inputs are read once,
// one pass ahead of their use, and sums, products and states are float32 and in a fixed order.
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
__device__ void clear_outside(const ScanArgs& A, const Seq& q, int64_t s, int64_t c, bool live, int warp, int warps,
                              T* o0, T* o1, T* o2) {
  if (!A.cu || !live) return;
  const float zero[V] = {};
  auto clear = [&](int64_t from, int64_t to) {
    for (int64_t r = from + warp; r < to; r += warps) {
      if (o0) store<T, V>(o0 + r * A.C + c, zero);
      if (o1) store<T, V>(o1 + r * A.C + c, zero);
      if (o2) store<T, V>(o2 + r * A.C + c, zero);
    }
  };
  if (s == 0) clear(0, q.row0);
  if (s == A.S - 1) clear(q.row0 + q.len, A.T);
}

// ------------------------------------------------------------------------ one step
__device__ __forceinline__ bool keeps(float c) { return __float_as_int(c) >= 0; }  // a >= q
__device__ __forceinline__ float coefficient(float f) {
  const float s = sigmoid_small(f);
  return f >= 0.0f ? s : -s;
}
__device__ __forceinline__ float step(float c, float h, float x) { return fmaf(c, x - h, keeps(c) ? h : x); }
__device__ __forceinline__ float times_a(float c, float v) { return fmaf(-c, v, keeps(c) ? v : 0.0f); }
__device__ __forceinline__ float times_q(float c, float v) { return fmaf(c, v, keeps(c) ? 0.0f : v); }

// -------------------------------------------------------------------- the cluster
struct Cluster {
  uint32_t rank, size;
  __device__ __forceinline__ Cluster() {
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(size));
  }
  // *p of CTA `to` = v
  __device__ __forceinline__ void put(float2* p, uint32_t to, float2 v) const {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(to));
    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(a), "f"(v.x), "f"(v.y) : "memory");
  }
  __device__ __forceinline__ void sync() const {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
};
constexpr int MOST_CTAS = 16;  // of a cluster

// The raw inputs of a warp's steps.  Steps behind the end read the last row, channels behind the last read the last
// ones: every address is inside, and what does not count is left out where it is used.
template <typename T, int V, int N>
struct Raw {
  Pack<T, V> v[N][STEPS];
  __device__ __forceinline__ void read(int i, const T* p, int64_t row, int64_t t1, int64_t len) {
#pragma unroll
    for (int l = 0; l < STEPS; ++l) v[i][l] = load<T, V>(p + min(t1 + l, len - 1) * row);
  }
};

template <typename T, int V, bool GATE>
__global__ void __launch_bounds__(WARPS * 32, 2) gated_scan_fwd_kernel(const ScanArgs A) {
  __shared__ float2 maps[2][WARPS][32 * V];
  __shared__ float2 peers[2][MOST_CTAS][32 * V];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Cluster K;
  const int64_t unit = blockIdx.x / K.size;
  const int64_t s = unit / A.tiles;
  const int64_t c0 = (unit % A.tiles) * (32 * V) + lane * V;
  const bool live = c0 < A.C;
  const int64_t c = live ? c0 : A.C - V;
  const Seq q(A, s);
  const T* f = q.in<T>(A.f, A, s) + c;
  const T* x = q.in<T>(A.x, A, s) + c;
  const T* g = GATE ? q.in<T>(A.g, A, s) + c : nullptr;
  T* y = static_cast<T*>(A.y);
  float carry[V];
#pragma unroll
  for (int v = 0; v < V; ++v) carry[v] = A.h0 ? A.h0[s * A.C + c + v] : 0.0f;

  const int64_t pass = (int64_t)K.size * MARK;
  int64_t t1 = K.rank * MARK + warp * STEPS;
  Raw<T, V, GATE ? 3 : 2> next;
  auto fetch = [&](int64_t t) {
    next.read(0, f, A.f.row, t, q.len);
    next.read(1, x, A.x.row, t, q.len);
    if (GATE) next.read(2, g, A.g.row, t, q.len);
  };
  if (q.len > 0) fetch(t1);
  if (K.size > 1) K.sync();  // shared memory of a CTA is there once it has started
  int half = 0;
  for (int64_t t0 = 0; t0 < q.len; t0 += pass, t1 += pass, half ^= 1) {
    const int n = (int)max((int64_t)0, min((int64_t)STEPS, q.len - t1));
    float cs[STEPS][V];
    Pack<T, V> xr[STEPS], gr[STEPS];
#pragma unroll
    for (int l = 0; l < STEPS; ++l) {
      xr[l] = next.v[1][l];
      if (GATE) gr[l] = next.v[GATE ? 2 : 0][l];
#pragma unroll
      for (int v = 0; v < V; ++v) cs[l][v] = coefficient(to_float(next.v[0][l].v[v]));
    }
    if (t0 + pass < q.len) fetch(t1 + pass);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float p = 1.0f, h = 0.0f;
      auto compose = [&](int l) {
        p = times_a(cs[l][v], p);
        h = step(cs[l][v], h, to_float(xr[l].v[v]));
      };
      if (n == STEPS) {
#pragma unroll
        for (int l = 0; l < STEPS; ++l) compose(l);
      } else {
#pragma unroll
        for (int l = 0; l < STEPS; ++l)
          if (l < n) compose(l);
      }
      maps[half][warp][lane * V + v] = make_float2(p, h);
    }
    __syncthreads();
    // (p, b) of this thread: the warps before its own; then of the whole CTA
    float p[V], b[V], in[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float tp = 1.0f, tb = 0.0f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        if (w == warp) p[v] = tp, b[v] = tb;
        const float2 m = maps[half][w][lane * V + v];
        tb = fmaf(m.x, tb, m.y);
        tp *= m.x;
      }
      if (K.size > 1) {
        for (uint32_t r = warp; r < K.size; r += WARPS) K.put(&peers[half][K.rank][lane * V + v], r, make_float2(tp, tb));
      } else {
        in[v] = fmaf(p[v], carry[v], b[v]);
        carry[v] = fmaf(tp, carry[v], tb);
      }
    }
    if (K.size > 1) {
      K.sync();
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float h = carry[v];
        for (uint32_t r = 0; r < K.size; ++r) {
          if (r == K.rank) in[v] = fmaf(p[v], h, b[v]);
          const float2 m = peers[half][r][lane * V + v];
          h = fmaf(m.x, h, m.y);
        }
        carry[v] = h;
      }
    }
    if (A.marks && warp == 0 && live && t1 < q.len) store<float, V>(A.marks + (q.mark0 + t1 / MARK) * A.C + c, in);
    T* out = y + (q.row0 + t1) * A.C + c;
    auto finish = [&](int l) {
      float o[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        o[v] = in[v] = step(cs[l][v], in[v], to_float(xr[l].v[v]));
        if (GATE) {
          const float z = to_float(gr[l].v[v]);
          o[v] *= z * sigmoid(z);
        }
      }
      if (live) store<T, V>(out + l * A.C, o);
    };
    if (n == STEPS) {
#pragma unroll
      for (int l = 0; l < STEPS; ++l) finish(l);
    } else {
#pragma unroll
      for (int l = 0; l < STEPS; ++l)
        if (l < n) finish(l);
    }
  }
  if (K.rank == 0 && warp == 0 && live && A.h_last) store<float, V>(A.h_last + s * A.C + c, carry);
  clear_outside<T, V>(A, q, s, c, live, K.rank * WARPS + warp, K.size * WARPS, y, static_cast<T*>(nullptr),
                      static_cast<T*>(nullptr));
}

template <typename T, int V, bool GATE>
__global__ void __launch_bounds__(WARPS * 32, 2) gated_scan_bwd_kernel(const ScanArgs A) {
  __shared__ float2 maps[2][WARPS][32 * V];  // the forward map of a warp's steps
  __shared__ float back[2][WARPS][32 * V];   // what leaves a warp's first step when nothing enters its last
  __shared__ float2 peers[2][MOST_CTAS][32 * V];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Cluster K;
  const int64_t unit = blockIdx.x / K.size;
  const int64_t s = unit / A.tiles;
  const int64_t c0 = (unit % A.tiles) * (32 * V) + lane * V;
  const bool live = c0 < A.C;
  const int64_t c = live ? c0 : A.C - V;
  const Seq q(A, s);
  const T* f = q.in<T>(A.f, A, s) + c;
  const T* x = q.in<T>(A.x, A, s) + c;
  const T* g = GATE ? q.in<T>(A.g, A, s) + c : nullptr;
  const T* dy = A.dy.p ? q.in<T>(A.dy, A, s) + c : nullptr;
  T *df = static_cast<T*>(A.df), *dx = static_cast<T*>(A.dx), *dg = static_cast<T*>(A.dg);
  float mu[V];  // the gradient that enters the pass from behind: a lam of the step after it
#pragma unroll
  for (int v = 0; v < V; ++v) mu[v] = A.dh_last ? A.dh_last[s * A.C + c + v] : 0.0f;

  const int64_t pass = (int64_t)K.size * MARK;
  const int64_t last = q.len > 0 ? (q.len - 1) / pass * pass : -pass;
  int64_t t1 = last + K.rank * MARK + warp * STEPS;
  Raw<T, V, GATE ? 4 : 3> next;
  auto fetch = [&](int64_t t) {
    next.read(0, f, A.f.row, t, q.len);
    next.read(1, x, A.x.row, t, q.len);
    if (dy) next.read(2, dy, A.dy.row, t, q.len);
    if (GATE) next.read(GATE ? 3 : 0, g, A.g.row, t, q.len);
  };
  if (q.len > 0) fetch(t1);
  if (K.size > 1) K.sync();  // shared memory of a CTA is there once it has started
  int half = 0;
  for (int64_t t0 = last; t0 >= 0; t0 -= pass, t1 -= pass, half ^= 1) {
    const int n = (int)max((int64_t)0, min((int64_t)STEPS, q.len - t1));
    float cs[STEPS][V], e[STEPS][V];  // e = dh
    Pack<T, V> xr[STEPS], dr[STEPS], gr[STEPS];
#pragma unroll
    for (int l = 0; l < STEPS; ++l) {
      xr[l] = next.v[1][l];
      dr[l] = next.v[2][l];
      if (GATE) gr[l] = next.v[GATE ? 3 : 0][l];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        cs[l][v] = coefficient(to_float(next.v[0][l].v[v]));
        e[l][v] = dy ? to_float(dr[l].v[v]) : 0.0f;
        if (GATE && dy) {
          const float z = to_float(gr[l].v[v]);
          e[l][v] *= z * sigmoid(z);
        }
      }
    }
    // the state that enters this CTA's steps
    float h[V];
#pragma unroll
    for (int v = 0; v < V; ++v)
      h[v] = t0 + K.rank * MARK < q.len ? A.marks[(q.mark0 + t0 / MARK + K.rank) * A.C + c + v] : 0.0f;
    if (t0 > 0) fetch(t1 - pass);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float p = 1.0f, b = 0.0f, r = 0.0f;
      auto compose = [&](int l) {
        p = times_a(cs[l][v], p);
        b = step(cs[l][v], b, to_float(xr[l].v[v]));
      };
      auto onward = [&](int l) { r = times_a(cs[l][v], e[l][v] + r); };
      if (n == STEPS) {
#pragma unroll
        for (int l = 0; l < STEPS; ++l) compose(l);
#pragma unroll
        for (int l = STEPS - 1; l >= 0; --l) onward(l);
      } else {
#pragma unroll
        for (int l = 0; l < STEPS; ++l)
          if (l < n) compose(l);
#pragma unroll
        for (int l = STEPS - 1; l >= 0; --l)
          if (l < n) onward(l);
      }
      maps[half][warp][lane * V + v] = make_float2(p, b);
      back[half][warp][lane * V + v] = r;
    }
    __syncthreads();
    // (p, b) of this thread: the warps behind its own, in the direction of the gradient; then of the whole CTA
    float p[V], b[V], m[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float tp = 1.0f, tb = 0.0f;
#pragma unroll
      for (int w = WARPS - 1; w >= 0; --w) {
        if (w == warp) p[v] = tp, b[v] = tb;
        const float k = maps[half][w][lane * V + v].x;
        tb = fmaf(k, tb, back[half][w][lane * V + v]);
        tp *= k;
      }
#pragma unroll
      for (int w = 0; w < WARPS - 1; ++w)
        if (w < warp) {
          const float2 k = maps[half][w][lane * V + v];
          h[v] = fmaf(k.x, h[v], k.y);
        }
      if (K.size > 1) {
        for (uint32_t r = warp; r < K.size; r += WARPS) K.put(&peers[half][K.rank][lane * V + v], r, make_float2(tp, tb));
      } else {
        m[v] = fmaf(p[v], mu[v], b[v]);
        mu[v] = fmaf(tp, mu[v], tb);
      }
    }
    if (K.size > 1) {
      K.sync();
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float r = mu[v];
        for (int k = (int)K.size - 1; k >= 0; --k) {
          if (k == (int)K.rank) m[v] = fmaf(p[v], r, b[v]);
          const float2 w = peers[half][k][lane * V + v];
          r = fmaf(w.x, r, w.y);
        }
        mu[v] = r;
      }
    }
    const int64_t at = (q.row0 + t1) * A.C + c;
    float D[STEPS][V];
    // forward over the steps: D_t = h_{t-1} - x_t, and dg is done
    auto ahead = [&](int l) {
      float o[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float xv = to_float(xr[l].v[v]);
        D[l][v] = h[v] - xv;
        h[v] = step(cs[l][v], h[v], xv);
        if (GATE) {
          const float z = to_float(gr[l].v[v]), w = sigmoid(z);
          o[v] = dy ? to_float(dr[l].v[v]) * h[v] * (w * fmaf(z, 1.0f - w, 1.0f)) : 0.0f;
        }
      }
      if (GATE && dg && live) store<T, V>(dg + at + l * A.C, o);
    };
    // and back: lam_t = dh_t + a_{t+1} lam_{t+1}
    auto finish = [&](int l) {
      float of[V], ox[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float lam = e[l][v] + m[v], sm = fabsf(cs[l][v]);
        m[v] = times_a(cs[l][v], lam);
        ox[v] = times_q(cs[l][v], lam);
        of[v] = lam * D[l][v] * fmaf(-sm, sm, sm);
      }
      if (dx && live) store<T, V>(dx + at + l * A.C, ox);
      if (df && live) store<T, V>(df + at + l * A.C, of);
    };
    if (n == STEPS) {
#pragma unroll
      for (int l = 0; l < STEPS; ++l) ahead(l);
#pragma unroll
      for (int l = STEPS - 1; l >= 0; --l) finish(l);
    } else {
#pragma unroll
      for (int l = 0; l < STEPS; ++l)
        if (l < n) ahead(l);
#pragma unroll
      for (int l = STEPS - 1; l >= 0; --l)
        if (l < n) finish(l);
    }
  }
  if (K.rank == 0 && warp == 0 && live && A.dh0) store<float, V>(A.dh0 + s * A.C + c, mu);
  clear_outside<T, V>(A, q, s, c, live, K.rank * WARPS + warp, K.size * WARPS, df, dx, dg);
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
      o[v] = hn[v] = step(coefficient(to_float(f.v[v])), h.v[v], to_float(x.v[v]));
      if (GATE) {
        const float z = to_float(g.v[v]);
        o[v] *= z * sigmoid(z);
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

// CTAs of a cluster: the time axis is split until the GPU has enough CTAs to hide its memory's latency, as far as the
// (mean) length has pieces for them.  Packed sequences are split further, since a few of them may hold most rows.
int cluster_size(const ScanArgs& A) {
  const int64_t units = A.S * A.tiles, len = A.cu ? A.T / 4 : A.T;
  int k = 1;
  while (k < MOST_CTAS && units * k < 3 * 148 && len > (int64_t)k * MARK) k *= 2;
  return k;
}

template <typename T, int V>
cudaError_t launch_scan(ScanArgs A, bool bwd, cudaStream_t st) {
  A.tiles = (int)((A.C + 32 * V - 1) / (32 * V));
  void (*kernel)(const ScanArgs) = bwd ? (A.g.p ? gated_scan_bwd_kernel<T, V, true> : gated_scan_bwd_kernel<T, V, false>)
                                       : (A.g.p ? gated_scan_fwd_kernel<T, V, true> : gated_scan_fwd_kernel<T, V, false>);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = cluster_size(A), at.val.clusterDim.y = 1, at.val.clusterDim.z = 1;
  if (at.val.clusterDim.x > 8)  // 8 is the size that every GPU takes; sm_100a takes 16 when asked to
    if (cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                             cudaFuncAttributeNonPortableClusterSizeAllowed, 1))
      return e;
  cfg.gridDim = dim3((unsigned)(A.S * A.tiles * at.val.clusterDim.x));
  cfg.blockDim = dim3(WARPS * 32);
  cfg.stream = st;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, (const ScanArgs)A);
}

int dispatch_scan(const ScanArgs& A, int dtype, bool bwd, cudaStream_t st, const char* who) {
  const bool two = A.C % 2 == 0 && pairs(A.f) && pairs(A.x) && pairs(A.g) && pairs(A.dy);
  cudaError_t e;
  if (dtype == CSN_F32) e = launch_scan<float, 1>(A, bwd, st);
  else if (dtype == CSN_BF16 && two) e = launch_scan<__nv_bfloat16, 2>(A, bwd, st);
  else if (dtype == CSN_BF16) e = launch_scan<__nv_bfloat16, 1>(A, bwd, st);
  else if (two) e = launch_scan<__half, 2>(A, bwd, st);
  else e = launch_scan<__half, 1>(A, bwd, st);
  if (e != cudaSuccess) return set_cuda_error(e, who);
  return check_launch(who);
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
  return dispatch_scan(A, dtype, false, st, "csn_gated_scan_fwd");
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
  return dispatch_scan(A, dtype, true, st, "csn_gated_scan_bwd");
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

// csn_gated_scan.cu -- the gated linear recurrence over channels, its adjoint and its step.
//
//   a_t = sigmoid(f_t),  q_t = 1 - a_t,  h_t = a_t h_{t-1} + q_t x_t,  y_t = h_t silu(g_t)   (y_t = h_t without g)
// Adjoint, with D_t = h_{t-1} - x_t, dh_t = dy_t silu(g_t) and lam_t = dh_t + a_{t+1} lam_{t+1} (the gradient of
// the last state enters at the end):
//   dx = q lam,  df = lam D a q,  dg = dy h silu'(g),  dh0 = a_0 lam_0
//
// Each step is an affine map h -> a h + b, and maps compose: (a2, b2) o (a1, b1) = (a2 a1, a2 b1 + b2).  A warp takes
// STEPS neighbouring steps of 128 bytes of neighbouring channels (two to a lane in 16 bits, one in float32) and
// composes them in registers; the warps of a CTA pass their maps through
// shared memory, the CTAs of a cluster, which take neighbouring MARK-step pieces of one sequence, through distributed
// shared memory; then every warp runs its steps again from the state that enters them.  So inputs are read once: each
// warp copies its rows into shared memory with cp.async one pass ahead of their use.  Sums, products and states are
// float32 and in a fixed order.
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
  bool wide;  // every row starts on 16 bytes and holds multiples of 16
};

// The rows of sequence s.  Borders outside 0..T, or falling ones, are cut to what is there.
struct Seq {
  int64_t row0;  // its first row in the outputs
  int len;
  int64_t mark0;  // its first mark: room for ceil(len / MARK) of them whatever the other lengths are
  __device__ __forceinline__ Seq(const ScanArgs& A, int64_t s) {
    if (A.cu) {
      const int64_t b = min(max((int64_t)A.cu[s], (int64_t)0), A.T);
      const int64_t e = min(max((int64_t)A.cu[s + 1], b), A.T);
      row0 = b;
      len = (int)(e - b);
    } else {
      row0 = s * A.T;
      len = (int)A.T;
    }
    mark0 = row0 / MARK + s;
  }
};

constexpr int ROW = 144;            // bytes of a tile's row in shared memory: 128, and a word more where rows are odd
constexpr int PIECE = MARK * ROW;   // of one tensor's rows of one CTA pass

template <typename T>
struct Lane {
  static constexpr int V = sizeof(T) == 4 ? 1 : 2;  // channels of a lane
  using F = Vals<V>;
  static constexpr int CHANNELS = 32 * V;           // of a tile
};

template <typename T>
__device__ __forceinline__ Vals<Lane<T>::V> unpack(uint32_t v);
template <>
__device__ __forceinline__ Vals<1> unpack<float>(uint32_t v) { return Vals<1>::make(__uint_as_float(v), 0.0f); }
template <>
__device__ __forceinline__ Vals<2> unpack<__nv_bfloat16>(uint32_t v) {
  return Vals<2>::make(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
template <>
__device__ __forceinline__ Vals<2> unpack<__half>(uint32_t v) {
  const float2 f = __half22float2(*reinterpret_cast<__half2*>(&v));
  return Vals<2>::make(f.x, f.y);
}

// V states at p, of which `have` are there
template <int V>
__device__ __forceinline__ Vals<V> load_state(const float* p, int have) {
  return Vals<V>::make(have > 0 ? p[0] : 0.0f, V > 1 && have > 1 ? p[V - 1] : 0.0f);
}
template <int V>
__device__ __forceinline__ void store_state(float* p, Vals<V> h, int have) {
  if (have > 0) p[0] = h.get(0);
  if (V > 1 && have > 1) p[V - 1] = h.get(V - 1);
}

// Rows of one input as a warp copies and reads them.  ODD: 16-bit rows that do not all start on 4 bytes; such a row is
// copied in the whole words that hold it and shifted when it is read.
template <typename T, bool ODD>
struct Input {
  const char* p;  // this lane's first bytes of the warp's first row of the next pass
  int64_t row;    // bytes
  int left;       // ODD: bytes of the tile

  __device__ __forceinline__ Input(const Rows& r, const ScanArgs& A, const Seq& q, int64_t s, int64_t tile, int t1) {
    p = nullptr;
    row = r.row * (int64_t)sizeof(T);
    left = (int)min((int64_t)32 * Lane<T>::V, A.C - tile) * (int)sizeof(T);
    if (!r.p) return;
    const int lane = threadIdx.x & 31;
    p = static_cast<const char*>(r.p) + ((A.cu ? q.row0 * r.row : s * r.seq) + tile) * (int64_t)sizeof(T) + t1 * row;
    if (!ODD) p += A.wide ? (lane >> 3) * row + (lane & 7) * 16 : lane * 4;
  }
  // the warp's n rows into shared memory at `to`, then `step` rows on
  __device__ __forceinline__ void copy(char* to, int n, bool wide, int step) {
    const int lane = threadIdx.x & 31;
    const uint32_t at = (uint32_t)__cvta_generic_to_shared(to);
    if (ODD) {
#pragma unroll
      for (int l = 0; l < STEPS; ++l)
        if (l < n) {
          const char* w = p + l * row;
          const int skew = (int)(reinterpret_cast<uintptr_t>(w) & 2);
          w -= skew;
          if (lane * 4 < left + skew) copy4(at + l * ROW + lane * 4, w + lane * 4);
          if (lane == 0 && 128 < left + skew) copy4(at + l * ROW + 128, w + 128);
        }
    } else if (wide) {
      const int l = lane >> 3;
      if ((lane & 7) * 16 < left) {
#pragma unroll
        for (int i = 0; i < STEPS / 4; ++i)
          if (l + i * 4 < n)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at + (l + i * 4) * ROW + (lane & 7) * 16),
                         "l"(p + i * 4 * row)
                         : "memory");
      }
    } else if (lane * 4 < left) {
#pragma unroll
      for (int l = 0; l < STEPS; ++l)
        if (l < n) copy4(at + l * ROW + lane * 4, p + l * row);
    }
    p += step * row;
  }
  static __device__ __forceinline__ void copy4(uint32_t to, const char* from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory");
  }
  // how far (in bits) the lanes' words of row l lie beyond the words' start; `p` as it was when the rows were copied
  __device__ __forceinline__ static uint32_t skew(const char* p, int64_t row, int l) {
    return (uint32_t)(reinterpret_cast<uintptr_t>(p + l * row) & 2) * 8;
  }
};

// a lane's channels of a row in shared memory
template <typename T, bool ODD>
__device__ __forceinline__ Vals<Lane<T>::V> read(const char* row, uint32_t skew) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(row) + (threadIdx.x & 31);
  return unpack<T>(ODD ? __funnelshift_r(w[0], w[1], skew) : w[0]);
}

// a lane's channels of one output row
template <typename T, bool ODD>
__device__ __forceinline__ void store_row(T* p, Vals<Lane<T>::V> o, int have) {
  constexpr int V = Lane<T>::V;
  if (!ODD) {
    if (have) *reinterpret_cast<uint32_t*>(p) = pack<T>(o.get(0), o.get(V - 1));
  } else {
    if (have > 0) p[0] = from_float<T>(o.get(0));
    if (have > 1) p[V - 1] = from_float<T>(o.get(V - 1));
  }
}

// Rows that belong to no sequence (before the first, behind the last) are written as 0.
template <typename T, bool ODD>
__device__ __noinline__ void clear_outside(const ScanArgs& A, const Seq& q, int64_t s, int64_t c, int have, int first,
                                           int step, T* o) {
  const Vals<Lane<T>::V> zero = splat<Lane<T>::V>(0.0f);
  if (s == 0)
    for (int64_t r = first; r < q.row0; r += step) store_row<T, ODD>(o + r * A.C + c, zero, have);
  if (s == A.S - 1)
    for (int64_t r = q.row0 + q.len + first; r < A.T; r += step) store_row<T, ODD>(o + r * A.C + c, zero, have);
}

__device__ __forceinline__ void copies_queued() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void copies_done() {
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncwarp();
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ int cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return (int)r;
}
__device__ __forceinline__ int cluster_ranks() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return (int)r;
}

// A map h -> p h + b of V channels, and its copy in another CTA's shared memory
template <int V>
struct alignas(8 * V) Map {
  Vals<V> p, b;
  __device__ __forceinline__ void put(Map* to, int cta) const {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(to)), "r"(cta));
    if (V == 1)
      asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(a), "f"(p.get(0)), "f"(b.get(0)) : "memory");
    else
      asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(a), "f"(p.get(0)), "f"(p.get(V - 1)),
                   "f"(b.get(0)), "f"(b.get(V - 1))
                   : "memory");
  }
};
constexpr int MOST_CTAS = 16;  // of a cluster

template <typename T, bool GATE, bool ODD>
__global__ void __launch_bounds__(WARPS * 32, 3) gated_scan_fwd_kernel(const __grid_constant__ ScanArgs A) {
  using F = typename Lane<T>::F;
  constexpr int V = Lane<T>::V, N = GATE ? 3 : 2;
  extern __shared__ __align__(128) char ring[];  // [2][N][MARK rows]
  __shared__ Map<V> maps[2][WARPS][32], peers[2][MOST_CTAS][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = cluster_rank(), ranks = cluster_ranks();
  const int unit = blockIdx.x / ranks;
  const int64_t s = unit / A.tiles, tile = (int64_t)(unit % A.tiles) * Lane<T>::CHANNELS, c = tile + lane * V;
  const int have = (int)max((int64_t)0, min((int64_t)V, A.C - c));
  const Seq q(A, s);
  T* y = static_cast<T*>(A.y);
  F carry = A.h0 ? load_state<V>(A.h0 + s * A.C + c, have) : splat<V>(0.0f);
  const int pass = ranks * MARK;
  int t1 = rank * MARK + warp * STEPS;
  char* mine = ring + warp * STEPS * ROW;
  Input<T, ODD> f(A.f, A, q, s, tile, t1), x(A.x, A, q, s, tile, t1), g(A.g, A, q, s, tile, t1);
  auto fetch = [&](int half, int n) {
    char* to = mine + half * N * PIECE;
    f.copy(to, n, A.wide, pass);
    x.copy(to + PIECE, n, A.wide, pass);
    if (GATE) g.copy(to + 2 * PIECE, n, A.wide, pass);
    copies_queued();
  };
  const char *f0 = f.p, *x0 = x.p, *g0 = g.p;  // ODD: MARK rows are whole words, so the first pass's skews are every pass's
  fetch(0, q.len - t1);
  T* out = y + (q.row0 + t1) * A.C + c;
  if (ranks > 1) cluster_sync();  // shared memory of a CTA is there once it has started
  int half = 0;
  for (int t0 = 0; t0 < q.len; t0 += pass, t1 += pass, out += pass * A.C, half ^= 1) {
    const int n = q.len - t1;  // steps left
    copies_done();
    if (t0 + pass < q.len) fetch(half ^ 1, n - pass);
    const char* in = mine + half * N * PIECE;
    F a[STEPS], b[STEPS];
#pragma unroll
    for (int l = 0; l < STEPS; ++l) {
      F w;
      sigmoid_pair(read<T, ODD>(in + l * ROW, f.skew(f0, f.row, l)), a[l], w);
      b[l] = w * read<T, ODD>(in + PIECE + l * ROW, x.skew(x0, x.row, l));
    }
    if (n < STEPS) {
#pragma unroll
      for (int l = 0; l < STEPS; ++l)
        if (l >= n) a[l] = splat<V>(1.0f), b[l] = splat<V>(0.0f);  // a step behind the end passes the state on
    }
    Map<V> m = {a[0], b[0]};
#pragma unroll
    for (int l = 1; l < STEPS; ++l) {
      m.p = a[l] * m.p;
      m.b = fma(a[l], m.b, b[l]);
    }
    maps[half][warp][lane] = m;
    __syncthreads();
    F h;
    if (ranks == 1) {
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        if (w == warp) h = carry;
        const Map<V> k = maps[half][w][lane];
        carry = fma(k.p, carry, k.b);
      }
    } else {
      // the warps before this one, and then the whole CTA
      Map<V> before, all = {splat<V>(1.0f), splat<V>(0.0f)};
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        if (w == warp) before = all;
        const Map<V> k = maps[half][w][lane];
        all.b = fma(k.p, all.b, k.b);
        all.p = k.p * all.p;
      }
      for (int r = warp; r < ranks; r += WARPS) all.put(&peers[half][rank][lane], r);
      cluster_sync();
#pragma unroll 4
      for (int r = 0; r < ranks; ++r) {
        if (r == rank) h = fma(before.p, carry, before.b);
        const Map<V> k = peers[half][r][lane];
        carry = fma(k.p, carry, k.b);
      }
    }
    if (A.marks && warp == 0 && n > 0) store_state<V>(A.marks + (q.mark0 + t1 / MARK) * A.C + c, h, have);
    auto finish = [&](int l) {
      h = fma(a[l], h, b[l]);
      F o = h;
      if (GATE) {
        const F z = read<T, ODD>(in + 2 * PIECE + l * ROW, g.skew(g0, g.row, l));
        o = h * (z * sigmoid(z));
      }
      store_row<T, ODD>(out + l * A.C, o, have);
    };
    if (n >= STEPS) {
#pragma unroll
      for (int l = 0; l < STEPS; ++l) finish(l);
    } else {
#pragma unroll
      for (int l = 0; l < STEPS; ++l)
        if (l < n) finish(l);
    }
  }
  if (rank == 0 && warp == 0 && A.h_last) store_state<V>(A.h_last + s * A.C + c, carry, have);
  if (A.cu) clear_outside<T, ODD>(A, q, s, c, have, rank * WARPS + warp, ranks * WARPS, y);
}

template <typename T, bool GATE, bool ODD>
__global__ void __launch_bounds__(WARPS * 32, 2) gated_scan_bwd_kernel(const __grid_constant__ ScanArgs A) {
  using F = typename Lane<T>::F;
  constexpr int V = Lane<T>::V, N = GATE ? 4 : 3;
  extern __shared__ __align__(128) char ring[];  // [2][N][MARK rows]
  // a warp's steps forward, and back: what leaves its first step when nothing enters its last
  __shared__ Map<V> maps[2][WARPS][32], peers[2][MOST_CTAS][32];
  __shared__ F back[2][WARPS][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = cluster_rank(), ranks = cluster_ranks();
  const int unit = blockIdx.x / ranks;
  const int64_t s = unit / A.tiles, tile = (int64_t)(unit % A.tiles) * Lane<T>::CHANNELS, c = tile + lane * V;
  const int have = (int)max((int64_t)0, min((int64_t)V, A.C - c));
  const Seq q(A, s);
  // the gradient that enters the pass from behind: a lam of the step after it
  F mu = A.dh_last ? load_state<V>(A.dh_last + s * A.C + c, have) : splat<V>(0.0f);
  const int pass = ranks * MARK;
  const int last = q.len > 0 ? (q.len - 1) / pass * pass : -pass;
  int t1 = last + rank * MARK + warp * STEPS;
  char* mine = ring + warp * STEPS * ROW;
  Input<T, ODD> f(A.f, A, q, s, tile, t1), x(A.x, A, q, s, tile, t1), d(A.dy, A, q, s, tile, t1), g(A.g, A, q, s, tile, t1);
  auto fetch = [&](int half, int n) {
    char* to = mine + half * N * PIECE;
    f.copy(to, n, A.wide, -pass);
    x.copy(to + PIECE, n, A.wide, -pass);
    d.copy(to + 2 * PIECE, n, A.wide, -pass);
    if (GATE) g.copy(to + 3 * PIECE, n, A.wide, -pass);
    copies_queued();
  };
  const char *f0 = f.p, *x0 = x.p, *d0 = d.p, *g0 = g.p;  // ODD: as above
  if (last >= 0) fetch(0, q.len - t1);
  int64_t at = (q.row0 + t1) * A.C + c;
  const float* mark = A.marks + (q.mark0 + last / MARK + rank) * A.C + c;
  if (ranks > 1) cluster_sync();  // shared memory of a CTA is there once it has started
  int half = 0;
  for (int t0 = last; t0 >= 0; t0 -= pass, t1 -= pass, at -= pass * A.C, mark -= ranks * A.C, half ^= 1) {
    const int n = q.len - t1;  // steps left
    // the state that enters this CTA's steps
    F h = t0 + rank * MARK < q.len ? load_state<V>(mark, have) : splat<V>(0.0f);
    copies_done();
    if (t0 > 0) fetch(half ^ 1, n + pass);
    const char* in = mine + half * N * PIECE;
    auto x_of = [&](int l) { return read<T, ODD>(in + PIECE + l * ROW, x.skew(x0, x.row, l)); };
    auto d_of = [&](int l) { return read<T, ODD>(in + 2 * PIECE + l * ROW, d.skew(d0, d.row, l)); };
    auto g_of = [&](int l) { return read<T, ODD>(in + 3 * PIECE + l * ROW, g.skew(g0, g.row, l)); };
    F a[STEPS], w[STEPS], e[STEPS];  // w = 1 - a, e = dh
    Map<V> m = {splat<V>(1.0f), splat<V>(0.0f)};
    F r = splat<V>(0.0f);
    auto take = [&](int l) {
      sigmoid_pair(read<T, ODD>(in + l * ROW, f.skew(f0, f.row, l)), a[l], w[l]);
      e[l] = d_of(l);
      if (GATE) {
        const F z = g_of(l);
        e[l] = e[l] * (z * sigmoid(z));
      }
      m.p = a[l] * m.p;
      m.b = fma(a[l], m.b, w[l] * x_of(l));
    };
    if (n >= STEPS) {
#pragma unroll
      for (int l = 0; l < STEPS; ++l) take(l);
    } else {
#pragma unroll
      for (int l = 0; l < STEPS; ++l) {
        a[l] = splat<V>(1.0f), w[l] = e[l] = splat<V>(0.0f);  // behind the end: passes state and gradient on
        if (l < n) take(l);
      }
    }
#pragma unroll
    for (int l = STEPS - 1; l >= 0; --l) r = a[l] * (e[l] + r);
    maps[half][warp][lane] = m;
    back[half][warp][lane] = r;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < WARPS - 1; ++k)
      if (k < warp) {
        const Map<V> u = maps[half][k][lane];
        h = fma(u.p, h, u.b);
      }
    if (ranks == 1) {
#pragma unroll
      for (int k = WARPS - 1; k >= 0; --k) {
        if (k == warp) r = mu;
        mu = fma(maps[half][k][lane].p, mu, back[half][k][lane]);
      }
    } else {
      // the warps behind this one, in the direction of the gradient, and then the whole CTA
      Map<V> before, all = {splat<V>(1.0f), splat<V>(0.0f)};
#pragma unroll
      for (int k = WARPS - 1; k >= 0; --k) {
        if (k == warp) before = all;
        const F u = maps[half][k][lane].p;
        all.b = fma(u, all.b, back[half][k][lane]);
        all.p = u * all.p;
      }
      for (int k = warp; k < ranks; k += WARPS) all.put(&peers[half][rank][lane], k);
      cluster_sync();
#pragma unroll 4
      for (int k = ranks - 1; k >= 0; --k) {
        if (k == rank) r = fma(before.p, mu, before.b);
        const Map<V> u = peers[half][k][lane];
        mu = fma(u.p, mu, u.b);
      }
    }
    // forward over the steps: D_t = h_{t-1} - x_t, and dg is done
    F D[STEPS];
    auto ahead = [&](int l) {
      const F xv = x_of(l);
      D[l] = h - xv;
      h = fma(a[l], h, w[l] * xv);
      if (GATE) {
        const F z = g_of(l), v = sigmoid(z);
        const F slope = v * fma(z, splat<V>(1.0f) - v, splat<V>(1.0f));
        store_row<T, ODD>(static_cast<T*>(A.dg) + at + l * A.C, d_of(l) * h * slope, have);
      }
    };
    // and back: lam_t = dh_t + a_{t+1} lam_{t+1}
    auto finish = [&](int l) {
      const F lam = e[l] + r, o = w[l] * lam;
      r = a[l] * lam;
      store_row<T, ODD>(static_cast<T*>(A.dx) + at + l * A.C, o, have);
      store_row<T, ODD>(static_cast<T*>(A.df) + at + l * A.C, o * a[l] * D[l], have);
    };
    if (n >= STEPS) {
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
  if (rank == 0 && warp == 0 && A.dh0) store_state<V>(A.dh0 + s * A.C + c, mu, have);
  if (A.cu) {
    const int first = rank * WARPS + warp, step = ranks * WARPS;
    clear_outside<T, ODD>(A, q, s, c, have, first, step, static_cast<T*>(A.df));
    clear_outside<T, ODD>(A, q, s, c, have, first, step, static_cast<T*>(A.dx));
    if (GATE) clear_outside<T, ODD>(A, q, s, c, have, first, step, static_cast<T*>(A.dg));
  }
}

// ---------------------------------------------------------------------------- step
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
      Vals<1> a, q;
      sigmoid_pair(Vals<1>{{to_float(f.v[v])}}, a, q);
      o[v] = hn[v] = fmaf(a.get(0), h.v[v], q.get(0) * to_float(x.v[v]));
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

bool rows_align(const Rows& r, int size, int bytes) {
  return !r.p || (r.seq * size % bytes == 0 && r.row * size % bytes == 0 && aligned(r.p, bytes));
}

// CTAs of a cluster: the time axis is split until the GPU has enough CTAs to hide its memory's latency, as far as the
// (mean) length has pieces for them.  Packed sequences are split further, since a few of them may hold most rows.
int cluster_size(const ScanArgs& A) {
  const int64_t units = A.S * A.tiles, len = A.cu ? A.T / 4 : A.T;
  int k = 1;
  while (k < MOST_CTAS && units * k < 3 * 148 && len > (int64_t)k * MARK) k *= 2;
  return k;
}

template <typename T, bool ODD>
cudaError_t launch_scan(ScanArgs A, bool bwd, cudaStream_t st) {
  A.tiles = (int)((A.C + Lane<T>::CHANNELS - 1) / Lane<T>::CHANNELS);
  const bool gate = A.g.p;
  void (*kernel)(const ScanArgs) =
      bwd ? (gate ? gated_scan_bwd_kernel<T, true, ODD> : gated_scan_bwd_kernel<T, false, ODD>)
          : (gate ? gated_scan_fwd_kernel<T, true, ODD> : gated_scan_fwd_kernel<T, false, ODD>);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = cluster_size(A), at.val.clusterDim.y = 1, at.val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)(A.S * A.tiles * at.val.clusterDim.x));
  cfg.blockDim = dim3(WARPS * 32);
  cfg.dynamicSmemBytes = 2 * ((bwd ? 3 : 2) + gate) * PIECE;
  cfg.stream = st;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  const void* k = reinterpret_cast<const void*>(kernel);
  if (cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)cfg.dynamicSmemBytes)) return e;
  if (at.val.clusterDim.x > 8)  // 8 is the size that every GPU takes; sm_100a takes 16 when asked to
    if (cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeNonPortableClusterSizeAllowed, 1)) return e;
  return cudaLaunchKernelEx(&cfg, kernel, (const ScanArgs)A);
}

int dispatch_scan(ScanArgs A, int dtype, bool bwd, cudaStream_t st, const char* who) {
  const int size = width_of(dtype);
  auto all = [&](int bytes) {
    return A.C * size % bytes == 0 && rows_align(A.f, size, bytes) && rows_align(A.x, size, bytes) &&
           rows_align(A.g, size, bytes) && rows_align(A.dy, size, bytes);
  };
  A.wide = all(16);
  const bool odd = !all(4);
  const cudaError_t e = dtype == CSN_F32 ? launch_scan<float, false>(A, bwd, st)
                        : dtype == CSN_BF16
                            ? (odd ? launch_scan<__nv_bfloat16, true>(A, bwd, st) : launch_scan<__nv_bfloat16, false>(A, bwd, st))
                            : (odd ? launch_scan<__half, true>(A, bwd, st) : launch_scan<__half, false>(A, bwd, st));
  if (e != cudaSuccess) return set_cuda_error(e, who);
  return check_launch(who);
}

int check_scan(const char* who, const ScanArgs& A, int dtype) {
  if (A.S < 0 || A.T < 0 || A.C < 0 || A.T > (1 << 30)) return set_error(CSN_ERR_INVALID, who);
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
  if (int rc = check_scan("csn_gated_scan_fwd: needs S, T, C >= 0, T <= 2^30, dtype float32, bfloat16 or float16, and at most "
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
  if (int rc = check_scan("csn_gated_scan_bwd: needs S, T, C >= 0, T <= 2^30, dtype float32, bfloat16 or float16, and at most "
                          "2^31 - 1 tiles of 32 channels", A, dtype))
    return rc;
  if (S == 0 || C == 0) return CSN_OK;
  const int size = width_of(dtype);
  if (T > 0 && (!f || !x || !dy || !marks || !strides || !df || !dx || (gate && !dgate) || !aligned(f, size) ||
                !aligned(x, size) || !aligned(gate, size) || !aligned(dy, size)))
    return set_error(CSN_ERR_INVALID, "csn_gated_scan_bwd: f, x, dy, marks, strides, df, dx and (with a gate) dgate are "
                                      "required, inputs aligned to their type");
  if (!aligned(marks, 16) || !aligned(dh_last, 16) || !aligned(df, 16) || !aligned(dx, 16) || !aligned(dgate, 16) ||
      !aligned(dh0, 16) || !aligned(cu_seqlens, 4))
    return set_error(CSN_ERR_INVALID, "csn_gated_scan_bwd: marks, dh_last and the gradients must be 16-byte aligned");
  if (strides) {
    A.f = {f, strides[0], strides[1]};
    A.x = {x, strides[2], strides[3]};
    A.g = {gate, gate ? strides[4] : 0, gate ? strides[5] : 0};
    A.dy = {dy, strides[6], strides[7]};
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

// csn_gated_scan.cu -- the gated linear recurrence over channels, its adjoint and its step.
//
//   a_t = sigmoid(f_t),  q_t = 1 - a_t,  h_t = a_t h_{t-1} + q_t x_t,  y_t = h_t silu(g_t)   (y_t = h_t without g)
// Adjoint, with D_t = h_{t-1} - x_t, dh_t = dy_t silu(g_t) and lam_t = dh_t + a_{t+1} lam_{t+1} (the gradient of
// the last state enters at the end):
//   dx = q lam,  df = lam D a q,  dg = dy h silu'(g),  dh0 = a_0 lam_0
//
// Each step is an affine map h -> a h + b, and maps compose: (a2, b2) o (a1, b1) = (a2 a1, a2 b1 + b2).  A warp takes
// STEPS neighbouring steps of 128 bytes of neighbouring channels (two to a lane in 16 bits, one in float32) and
// composes them in registers; the warps of a CTA, which take neighbouring steps, pass their maps through shared
// memory; then every warp runs its steps again from the state that enters them.  So the inputs are read once: each
// warp copies its rows into shared memory with cp.async one pass (MARK steps) ahead of their use.
//
// Sequences of at most 32 steps need fewer warps than a CTA has: it then takes 2, 4 or 8 of them.
//
// Where there are too few sequences and channels to fill the GPU, sequences are cut into chunks: reduce_kernel composes
// the map of every chunk that another follows (it reads f and x once more, which the scan then finds in L2 where they
// fit), and the CTA of a chunk composes those before it into the state that enters it.  All sums, products and states
// are float32 and in an order that the sizes alone fix.
//
// What bounds it: the latency of a pass, not memory.  An element costs about 40 instructions forward (two of them on
// the MUFU for the decay, two for the gate) and 73 back (two and four: the gate's sigmoid twice), and with 256 CTAs of
// 8 warps the schedulers issue in 60 to 64 % of the cycles, MUFU 42 to 48 %, HBM 0.58 of its rate: nothing is full, and
// a warp waits for fixed latencies, shared memory and MUFU results.  bf16 with a gate on a B200: B8 T2048 C2048 forward
// 71 us (3.8 TB/s of what has to move), backward 124 us (3.8 TB/s); B24 T2048 C2048 181 us (4.5 TB/s) and 346 us (4.1
// TB/s); one sequence of 65536 x 1024 50 us for the reduce pass (5.4 TB/s) and 114 us for the scan (4.7 TB/s).  Slower:
// steps of 4 or 16 a warp, 4 or 16 warps a CTA, 2 or 4 CTAs an SM forward and 1 or 3 back, packed float32 pairs (the
// same instruction count, in moves), and the time axis split over clusters that pass maps every MARK steps (prompt 319
// us with st.async, 419 with barrier.cluster).
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
  float2* maps;  // [units][C]: the maps of chunks that another follows (backward: that follow another)
  int tiles;
  int chunk;     // steps of a chunk, a multiple of MARK
  int chunks;    // of a sequence, where all have one length
  int group;     // warps that share a sequence; the others of a CTA have sequences of their own
  bool wide;  // every row starts on 16 bytes and holds multiples of 16
};

// The part of a sequence that a CTA works on.  Unit u is chunk u % chunks of sequence u / chunks, or, in a packed
// batch, where sequence s begins with unit cu[s] / chunk + s (room for its chunks whatever the other lengths are), the
// one that the borders give; some units are empty.  Borders outside 0..T, or falling ones, are cut to what is there.
struct Part {
  int64_t s;      // sequence; -1: none
  int64_t row0;   // its first row in the outputs
  int64_t unit;
  int len;        // its steps
  int k;          // chunk of the sequence
  int from, to;   // steps of the chunk
  int64_t mark0;  // the sequence's first mark: room for ceil(len / MARK) of them

  __device__ __forceinline__ int64_t border(const ScanArgs& A, int64_t i) const {
    return min(max((int64_t)A.cu[i], (int64_t)0), A.T);
  }
  __device__ __forceinline__ Part(const ScanArgs& A, int64_t u) : unit(u) {
    if (A.cu) {
      // the last s that begins at unit u or before: each round, 32 lanes look at 32 places of what is left
      int64_t lo = 0, n = A.S;
      while (n > 0) {
        const int64_t step = (n + 31) / 32, i = lo + (threadIdx.x & 31) * step;
        const bool yes = i < lo + n && border(A, i) / A.chunk + i <= u;
        const int c = __popc(__ballot_sync(0xffffffffu, yes));
        if (c == 0) break;
        lo += (c - 1) * step;
        n = step == 1 ? 0 : min(step, A.S - lo);
      }
      s = border(A, lo) / A.chunk + lo <= u ? lo : -1;
      if (s < 0) return;
      row0 = border(A, s);
      len = (int)(max(border(A, s + 1), row0) - row0);
      k = (int)(u - (row0 / A.chunk + s));
    } else {
      s = u / A.chunks;
      row0 = s * A.T;
      len = (int)A.T;
      k = (int)(u - s * A.chunks);
    }
    mark0 = row0 / MARK + s;
    const int64_t first = (int64_t)k * A.chunk;
    from = (int)min(first, (int64_t)len);
    to = (int)min(first + A.chunk, (int64_t)len);
    if (k > 0 && from >= len) s = -1;
  }
};

constexpr int ROW = 128;           // bytes of a tile's row in shared memory
constexpr int PIECE = MARK * ROW;  // of one tensor's rows of one CTA pass

template <typename T>
struct Lane {
  static constexpr int V = sizeof(T) == 4 ? 1 : 2;  // channels of a lane
  using F = Vals<V>;
};
// channels of a tile: 32 words' worth, less a pair where rows are odd, so that 32 words hold them at either shift
__host__ __device__ constexpr int channels(int size, bool odd) { return size == 4 ? 32 : odd ? 62 : 64; }

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
// copied in the whole words that hold it and shifted when it is read.  A warp's rows lie an even number of rows from
// where they lay in its last pass, so only a row's place among the warp's, even or odd, says how far it is shifted.
template <typename T, bool ODD>
struct Input {
  const char* p;  // this lane's first bytes of the warp's first row of the next pass (ODD: word of the second row: q)
  const char* q;
  int64_t row;    // bytes
  int left;       // bytes of the tile
  int skew[2];    // ODD: bits

  __device__ __forceinline__ Input(const Rows& r, const ScanArgs& A, const Part& part, int64_t tile, int t1) {
    p = q = nullptr;
    row = r.row * (int64_t)sizeof(T);
    left = (int)min((int64_t)channels(sizeof(T), ODD), A.C - tile) * (int)sizeof(T);
    skew[0] = skew[1] = 0;
    if (!r.p) return;
    const int lane = threadIdx.x & 31;
    p = static_cast<const char*>(r.p) + ((A.cu ? part.row0 * r.row : part.s * r.seq) + tile) * (int64_t)sizeof(T) + t1 * row;
    if (ODD) {
      q = p + row;
      skew[0] = (int)(reinterpret_cast<uintptr_t>(p) & 2) * 8;
      skew[1] = (int)(reinterpret_cast<uintptr_t>(q) & 2) * 8;
      p += lane * 4 - skew[0] / 8;
      q += lane * 4 - skew[1] / 8;
    } else {
      p += A.wide ? (lane >> 3) * row + (lane & 7) * 16 : lane * 4;
    }
  }
  // the warp's n rows into shared memory at `to`, then `step` rows on
  __device__ __forceinline__ void copy(char* to, int n, bool wide, int step) {
    const int lane = threadIdx.x & 31;
    const uint32_t at = (uint32_t)__cvta_generic_to_shared(to);
    if (ODD) {
#pragma unroll
      for (int o = 0; o < 2; ++o) {
        const char* w = o ? q : p;
        if (lane * 4 < left + skew[o] / 8) {
#pragma unroll
          for (int l = o; l < STEPS; l += 2)
            if (l < n) copy4(at + l * ROW + lane * 4, w + (l - o) * row);
        }
      }
      q += step * row;
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
  // this lane's channels of the warp's row l, which was copied to `at`
  __device__ __forceinline__ Vals<Lane<T>::V> read(const char* at, int l) const {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(at + l * ROW) + (threadIdx.x & 31);
    // ODD: the last lane has no channels, and reads its own word twice
    return unpack<T>(ODD ? __funnelshift_r(w[0], w[(threadIdx.x & 31) < 31], skew[l & 1]) : w[0]);
  }
};

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
__device__ __noinline__ void clear_outside(const ScanArgs& A, const Part& q, int64_t c, int have, void* out) {
  T* o = static_cast<T*>(out);
  const Vals<Lane<T>::V> zero = splat<Lane<T>::V>(0.0f);
  const int warp = threadIdx.x >> 5;
  if (q.s == 0)
    for (int64_t r = warp; r < q.row0; r += WARPS) store_row<T, ODD>(o + r * A.C + c, zero, have);
  if (q.s == A.S - 1)
    for (int64_t r = q.row0 + q.len + warp; r < A.T; r += WARPS) store_row<T, ODD>(o + r * A.C + c, zero, have);
}

__device__ __forceinline__ void copies_queued() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void copies_done() {
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncwarp();
}

// The scan of a chunked batch is launched while its reduce pass runs (programmatic dependent launch): it has its rows
// under way when it waits here for what that pass leaves in A.maps.
__device__ __forceinline__ void others_done() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void others_may_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// A map h -> p h + b of V channels
template <int V>
struct alignas(8 * V) Map {
  Vals<V> p, b;
  __device__ __forceinline__ Vals<V> of(Vals<V> h) const { return fma(p, h, b); }
  __device__ __forceinline__ Map after(const Map& m) const { return {p * m.p, fma(p, m.b, b)}; }
  static __device__ __forceinline__ Map none() { return {splat<V>(1.0f), splat<V>(0.0f)}; }
};

// A chunk's map in memory
template <int V>
__device__ __forceinline__ Map<V> load_map(const float2* p, int have) {
  const float2 u = have > 0 ? p[0] : make_float2(1.0f, 0.0f), w = V > 1 && have > 1 ? p[V - 1] : u;
  return {Vals<V>::make(u.x, w.x), Vals<V>::make(u.y, w.y)};
}
template <int V>
__device__ __forceinline__ void store_map(float2* p, const Map<V>& m, int have) {
  if (have > 0) p[0] = make_float2(m.p.get(0), m.b.get(0));
  if (V > 1 && have > 1) p[V - 1] = make_float2(m.p.get(V - 1), m.b.get(V - 1));
}

// The value that enters a chunk: `v` through the maps of n chunks from unit u on, each `step` units further.  The warps
// compose n / WARPS neighbouring ones each.
template <int V>
__device__ __forceinline__ Vals<V> enter(const ScanArgs& A, Map<V> (*maps)[32], Vals<V> v, int64_t u, int n, int step,
                                         int64_t c, int have) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  Map<V> m = Map<V>::none();
#pragma unroll 4
  for (int j = n * warp / WARPS; j < n * (warp + 1) / WARPS; ++j) m = load_map<V>(A.maps + (u + j * step) * A.C + c, have).after(m);
  maps[warp][lane] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WARPS; ++w) v = maps[w][lane].of(v);
  return v;
}

// The map of a chunk that another follows; BACK: of the gradient, through a chunk that follows another.  Each warp
// composes a contiguous eighth of the chunk.
template <typename T, bool GATE, bool ODD, bool BACK>
__global__ void __launch_bounds__(WARPS * 32, 3) reduce_kernel(const __grid_constant__ ScanArgs A) {
  using F = typename Lane<T>::F;
  constexpr int V = Lane<T>::V, N = BACK && GATE ? 3 : 2;
  extern __shared__ __align__(128) char ring[];  // [2][N][MARK rows]
  __shared__ Map<V> maps[WARPS][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  others_may_start();
  const Part q(A, blockIdx.x / A.tiles);
  if (q.s < 0 || (BACK ? q.k == 0 : q.to == q.len)) return;
  const int64_t tile = (int64_t)(blockIdx.x % A.tiles) * channels(sizeof(T), ODD), c = tile + lane * V;
  const int have = (int)max((int64_t)0, min((int64_t)V, min(A.C, tile + channels(sizeof(T), ODD)) - c));
  const int share = A.chunk / WARPS, first = q.from + warp * share, past = min(first + share, q.to);
  char* mine = ring + warp * STEPS * ROW;
  // BACK goes from the last steps to the first
  int t = BACK ? first + (max(past - first, 1) - 1) / STEPS * STEPS : first;
  const int step = BACK ? -STEPS : STEPS;
  Input<T, ODD> f(A.f, A, q, tile, t), x(BACK ? A.dy : A.x, A, q, tile, t), g(A.g, A, q, tile, t);
  auto fetch = [&](int half, int n) {
    char* to = mine + half * N * PIECE;
    f.copy(to, n, A.wide, step);
    x.copy(to + PIECE, n, A.wide, step);
    if (N > 2) g.copy(to + 2 * PIECE, n, A.wide, step);
    copies_queued();
  };
  Map<V> m = Map<V>::none();
  if (past > first) fetch(0, past - t);
  for (int half = 0; BACK ? t >= first && past > first : t < past; t += step, half ^= 1) {
    copies_done();
    const int u = t + step;
    if (BACK ? u >= first : u < past) fetch(half ^ 1, past - u);
    const char* in = mine + half * N * PIECE;
    const int n = past - t;
    auto take = [&](int l) {
      F a, w;
      sigmoid_pair(f.read(in, l), a, w);
      F v = x.read(in + PIECE, l);
      if (BACK) {
        if (GATE) {
          const F z = g.read(in + 2 * PIECE, l);
          v = v * (z * sigmoid(z));
        }
        m.b = a * (v + m.b);
      } else {
        m.b = fma(a, m.b, w * v);
      }
      m.p = a * m.p;
    };
    if (n >= STEPS) {
#pragma unroll
      for (int l = 0; l < STEPS; ++l) take(BACK ? STEPS - 1 - l : l);
    } else {
#pragma unroll
      for (int l = 0; l < STEPS; ++l)
        if ((BACK ? STEPS - 1 - l : l) < n) take(BACK ? STEPS - 1 - l : l);
    }
  }
  maps[warp][lane] = m;
  __syncthreads();
  if (warp == 0) {
    m = Map<V>::none();
#pragma unroll
    for (int w = 0; w < WARPS; ++w) m = maps[BACK ? WARPS - 1 - w : w][lane].after(m);
    store_map<V>(A.maps + q.unit * A.C + c, m, have);
  }
}

template <typename T, bool GATE, bool ODD>
__global__ void __launch_bounds__(WARPS * 32, 3) gated_scan_fwd_kernel(const __grid_constant__ ScanArgs A) {
  using F = typename Lane<T>::F;
  constexpr int V = Lane<T>::V, N = GATE ? 3 : 2;
  extern __shared__ __align__(128) char ring[];  // [2][N][MARK rows]
  __shared__ Map<V> maps[2][WARPS][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int among = warp % A.group, head = warp - among;  // place in the sequence's warps, and the first of them
  const int64_t unit = (int64_t)(blockIdx.x / A.tiles) * (WARPS / A.group) + head / A.group;
  const bool spare = A.group < WARPS && unit >= A.S;  // goes through the motions of the last sequence
  const Part q(A, spare ? A.S - 1 : unit);
  if (q.s < 0) return;
  const int64_t tile = (int64_t)(blockIdx.x % A.tiles) * channels(sizeof(T), ODD), c = tile + lane * V;
  const int have = spare ? 0 : (int)max((int64_t)0, min((int64_t)V, min(A.C, tile + channels(sizeof(T), ODD)) - c));
  int t1 = q.from + among * STEPS;
  char* mine = ring + warp * STEPS * ROW;
  Input<T, ODD> f(A.f, A, q, tile, t1), x(A.x, A, q, tile, t1), g(A.g, A, q, tile, t1);
  auto fetch = [&](int half, int n) {
    char* to = mine + half * N * PIECE;
    f.copy(to, n, A.wide, MARK);
    x.copy(to + PIECE, n, A.wide, MARK);
    if (GATE) g.copy(to + 2 * PIECE, n, A.wide, MARK);
    copies_queued();
  };
  fetch(0, q.to - t1);
  others_done();
  F carry = A.h0 ? load_state<V>(A.h0 + q.s * A.C + c, have) : splat<V>(0.0f);
  if (q.k > 0) carry = enter<V>(A, maps[1], carry, q.unit - q.k, q.k, 1, c, have);
  T* out = static_cast<T*>(A.y) + (q.row0 + t1) * A.C + c;
  float* mark = A.marks + (q.mark0 + q.from / MARK) * A.C + c;
  int half = 0;
  for (int t0 = q.from; t0 < q.to; t0 += MARK, t1 += MARK, out += MARK * A.C, half ^= 1) {
    const int n = q.to - t1;  // steps left
    copies_done();
    if (t0 + MARK < q.to) fetch(half ^ 1, n - MARK);
    const char* in = mine + half * N * PIECE;
    F a[STEPS], b[STEPS];
#pragma unroll
    for (int l = 0; l < STEPS; ++l) {
      F w;
      sigmoid_pair(f.read(in, l), a[l], w);
      b[l] = w * x.read(in + PIECE, l);
    }
    if (n < STEPS) {
#pragma unroll
      for (int l = 0; l < STEPS; ++l)
        if (l >= n) a[l] = splat<V>(1.0f), b[l] = splat<V>(0.0f);  // a step behind the end passes the state on
    }
    Map<V> m = {a[0], b[0]};
#pragma unroll
    for (int l = 1; l < STEPS; ++l) m = Map<V>{a[l], b[l]}.after(m);
    maps[half][warp][lane] = m;
    __syncthreads();
    F h;
    if (A.group == WARPS) {
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        if (w == warp) h = carry;
        carry = maps[half][w][lane].of(carry);
      }
    } else {
      for (int w = 0; w < A.group; ++w) {
        if (w == among) h = carry;
        carry = maps[half][head + w][lane].of(carry);
      }
    }
    if (A.marks) {
      if (among == 0) store_state<V>(mark, h, have);
      mark += A.C;
    }
    auto finish = [&](int l) {
      h = fma(a[l], h, b[l]);
      F o = h;
      if (GATE) {
        const F z = g.read(in + 2 * PIECE, l);
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
  if (q.to == q.len && among == 0 && A.h_last) store_state<V>(A.h_last + q.s * A.C + c, carry, have);
  if (A.cu && q.k == 0) clear_outside<T, ODD>(A, q, c, have, A.y);
}

template <typename T, bool GATE, bool ODD>
__global__ void __launch_bounds__(WARPS * 32, 2) gated_scan_bwd_kernel(const __grid_constant__ ScanArgs A) {
  using F = typename Lane<T>::F;
  constexpr int V = Lane<T>::V, N = GATE ? 4 : 3;
  extern __shared__ __align__(128) char ring[];  // [2][N][MARK rows]
  // a warp's steps forward, and back: what leaves its first step when nothing enters its last
  __shared__ Map<V> maps[2][WARPS][32];
  __shared__ F back[2][WARPS][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int among = warp % A.group, head = warp - among;  // place in the sequence's warps, and the first of them
  const int64_t unit = (int64_t)(blockIdx.x / A.tiles) * (WARPS / A.group) + head / A.group;
  const bool spare = A.group < WARPS && unit >= A.S;  // goes through the motions of the last sequence
  const Part q(A, spare ? A.S - 1 : unit);
  if (q.s < 0) return;
  const int64_t tile = (int64_t)(blockIdx.x % A.tiles) * channels(sizeof(T), ODD), c = tile + lane * V;
  const int have = spare ? 0 : (int)max((int64_t)0, min((int64_t)V, min(A.C, tile + channels(sizeof(T), ODD)) - c));
  const int last = q.to > q.from ? q.from + (q.to - q.from - 1) / MARK * MARK : q.from - MARK;
  int t1 = last + among * STEPS;
  char* mine = ring + warp * STEPS * ROW;
  Input<T, ODD> f(A.f, A, q, tile, t1), x(A.x, A, q, tile, t1), d(A.dy, A, q, tile, t1), g(A.g, A, q, tile, t1);
  auto fetch = [&](int half, int n) {
    char* to = mine + half * N * PIECE;
    f.copy(to, n, A.wide, -MARK);
    x.copy(to + PIECE, n, A.wide, -MARK);
    d.copy(to + 2 * PIECE, n, A.wide, -MARK);
    if (GATE) g.copy(to + 3 * PIECE, n, A.wide, -MARK);
    copies_queued();
  };
  if (last >= q.from) fetch(0, q.to - t1);
  others_done();
  // the gradient that enters from behind: a lam of the step after
  F mu = A.dh_last ? load_state<V>(A.dh_last + q.s * A.C + c, have) : splat<V>(0.0f);
  if (q.to < q.len) {
    const int behind = (q.len - 1) / A.chunk - q.k;
    mu = enter<V>(A, maps[1], mu, q.unit + behind, behind, -1, c, have);
  }
  int64_t at = (q.row0 + t1) * A.C + c;
  const float* mark = A.marks + (q.mark0 + last / MARK) * A.C + c;
  int half = 0;
  for (int t0 = last; t0 >= q.from; t0 -= MARK, t1 -= MARK, at -= MARK * A.C, mark -= A.C, half ^= 1) {
    const int n = q.to - t1;  // steps left
    F h = load_state<V>(mark, have);  // the state that enters the pass
    copies_done();
    if (t0 > q.from) fetch(half ^ 1, n + MARK);
    const char* in = mine + half * N * PIECE;
    auto x_of = [&](int l) { return x.read(in + PIECE, l); };
    auto d_of = [&](int l) { return d.read(in + 2 * PIECE, l); };
    auto g_of = [&](int l) { return g.read(in + 3 * PIECE, l); };
    F a[STEPS], w[STEPS], e[STEPS];  // w = 1 - a, e = dh
    Map<V> m = Map<V>::none();
    F r = splat<V>(0.0f);
    auto take = [&](int l) {
      sigmoid_pair(f.read(in, l), a[l], w[l]);
      e[l] = d_of(l);
      if (GATE) {
        const F z = g_of(l);
        e[l] = e[l] * (z * sigmoid(z));
      }
      m = Map<V>{a[l], w[l] * x_of(l)}.after(m);
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
    if (A.group == WARPS) {
#pragma unroll
      for (int k = 0; k < WARPS - 1; ++k)
        if (k < warp) h = maps[half][k][lane].of(h);
#pragma unroll
      for (int k = WARPS - 1; k >= 0; --k) {
        if (k == warp) r = mu;
        mu = fma(maps[half][k][lane].p, mu, back[half][k][lane]);
      }
    } else {
      for (int k = head; k < warp; ++k) h = maps[half][k][lane].of(h);
      for (int k = head + A.group - 1; k >= head; --k) {
        if (k == warp) r = mu;
        mu = fma(maps[half][k][lane].p, mu, back[half][k][lane]);
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
  if (q.k == 0 && among == 0 && A.dh0) store_state<V>(A.dh0 + q.s * A.C + c, mu, have);
  if (A.cu && q.k == 0) {
    clear_outside<T, ODD>(A, q, c, have, A.df);
    clear_outside<T, ODD>(A, q, c, have, A.dx);
    if (GATE) clear_outside<T, ODD>(A, q, c, have, A.dg);
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

// How sequences are cut.  The GPU holds 148 x per_sm CTAs at a time.  Where sequences and tiles alone do not fill half
// of them, each sequence gets as many chunks as fit at one time; packed sequences, whose lengths are not known here and
// may be anything, are cut at an even share of all rows.  Chunks have 4 passes at least: below that the second
// reading and its launch cost more than they bring.
struct Cut {
  int tiles, chunk, chunks, group;
  int64_t units, ctas;  // pieces of work; those of a tile that a CTA takes at a time
  Cut(int64_t S, int64_t T, int64_t C, bool packed, int dtype, bool odd, bool bwd) {
    const int wide = channels(dtype == CSN_F32 ? 4 : 2, odd);
    const int64_t slots = 148 * (bwd ? 2 : 3);
    tiles = (int)((C + wide - 1) / wide);
    int64_t n = packed ? 1 : slots / (S * tiles);
    int64_t len = packed ? T * tiles / slots : n > 1 ? T / n : T;
    len = (len + MARK - 1) / MARK * MARK;
    if (len < 4 * MARK) len = 4 * MARK;
    chunk = (int)(len < T ? len : (T + MARK - 1) / MARK * MARK);
    if (chunk == 0) chunk = MARK;
    chunks = (int)((T + chunk - 1) / chunk);
    if (chunks == 0) chunks = 1;
    units = packed ? T / chunk + S : S * chunks;
    group = packed || T > 32 ? WARPS : T > 16 ? 4 : T > 8 ? 2 : 1;
    ctas = (units * group + WARPS - 1) / WARPS;
  }
  bool split(int64_t T) const { return T > chunk; }
};

template <auto KERNEL>
cudaError_t launch_part(int64_t grid, int smem, const ScanArgs& A, bool early, cudaStream_t st) {
  if (cudaError_t e = allow_smem<KERNEL>(smem)) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(WARPS * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = early ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, KERNEL, A);
}

template <typename T, bool GATE, bool ODD>
cudaError_t launch_scan(const ScanArgs& A, bool bwd, const Cut& cut, cudaStream_t st) {
  const int64_t grid = cut.ctas * cut.tiles;
  constexpr int piece = 2 * PIECE;
  const bool split = cut.split(A.T);
  if (split) {
    const cudaError_t e = bwd ? launch_part<reduce_kernel<T, GATE, ODD, true>>(grid, (GATE ? 3 : 2) * piece, A, false, st)
                              : launch_part<reduce_kernel<T, false, ODD, false>>(grid, 2 * piece, A, false, st);
    if (e != cudaSuccess) return e;
  }
  return bwd ? launch_part<gated_scan_bwd_kernel<T, GATE, ODD>>(grid, (GATE ? 4 : 3) * piece, A, split, st)
             : launch_part<gated_scan_fwd_kernel<T, GATE, ODD>>(grid, (GATE ? 3 : 2) * piece, A, split, st);
}
template <typename T, bool ODD>
cudaError_t launch_scan(const ScanArgs& A, bool bwd, const Cut& cut, cudaStream_t st) {
  return A.g.p ? launch_scan<T, true, ODD>(A, bwd, cut, st) : launch_scan<T, false, ODD>(A, bwd, cut, st);
}

int dispatch_scan(ScanArgs A, int dtype, bool bwd, void* workspace, size_t bytes, cudaStream_t st, const char* who) {
  const int size = width_of(dtype);
  auto all = [&](int to) {
    return A.C * size % to == 0 && rows_align(A.f, size, to) && rows_align(A.x, size, to) && rows_align(A.g, size, to) &&
           rows_align(A.dy, size, to);
  };
  A.wide = all(16);
  const bool odd = !all(4);
  const Cut cut(A.S, A.T, A.C, A.cu != nullptr, dtype, odd, bwd);
  A.tiles = cut.tiles, A.chunk = cut.chunk, A.chunks = cut.chunks, A.group = cut.group, A.maps = static_cast<float2*>(workspace);
  if (cut.units * cut.tiles > 0x7fffffff) return set_error(CSN_ERR_INVALID, "csn_gated_scan: more than 2^31 - 1 tiles of work");
  if (cut.split(A.T) && (!workspace || !aligned(workspace, 16) || bytes < (size_t)cut.units * A.C * sizeof(float2)))
    return set_error(CSN_ERR_INVALID, "csn_gated_scan: workspace smaller than csn_gated_scan_workspace_bytes");
  const cudaError_t e =
      dtype == CSN_F32 ? launch_scan<float, false>(A, bwd, cut, st)
      : dtype == CSN_BF16
          ? (odd ? launch_scan<__nv_bfloat16, true>(A, bwd, cut, st) : launch_scan<__nv_bfloat16, false>(A, bwd, cut, st))
          : (odd ? launch_scan<__half, true>(A, bwd, cut, st) : launch_scan<__half, false>(A, bwd, cut, st));
  return e == cudaSuccess ? CSN_OK : set_cuda_error(e, who);
}

int check_scan(const char* who, const ScanArgs& A, int dtype) {
  if (A.S < 0 || A.T < 0 || A.C < 0 || A.T > (1 << 30)) return set_error(CSN_ERR_INVALID, who);
  if (!width_of(dtype)) return set_error(CSN_ERR_UNSUPPORTED, who);
  // a CTA for each 32 channels of a sequence at least
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

extern "C" size_t csn_gated_scan_workspace_bytes(int64_t S, int64_t T, int64_t C, int packed, int dtype, int backward) {
  ScanArgs A = {};
  A.S = S, A.T = T, A.C = C;
  if (S <= 0 || T <= 0 || C <= 0 || check_scan("", A, dtype)) return 0;
  size_t most = 0;  // whichever way the rows turn out to lie
  for (int odd = 0; odd < 2; ++odd) {
    const Cut cut(S, T, C, packed != 0, dtype, odd != 0, backward != 0);
    const size_t n = cut.split(T) ? (size_t)cut.units * C * sizeof(float2) : 0;
    if (n > most) most = n;
  }
  return most;
}

extern "C" int csn_gated_scan_fwd(const void* f, const void* x, const void* gate, const int64_t* strides,
                                  const float* h0, const int32_t* cu_seqlens, void* y, float* h_last, float* marks,
                                  int64_t S, int64_t T, int64_t C, int dtype, void* workspace, size_t workspace_bytes,
                                  void* stream) {
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
  return dispatch_scan(A, dtype, false, workspace, workspace_bytes, st, "csn_gated_scan_fwd");
}

extern "C" int csn_gated_scan_bwd(const void* f, const void* x, const void* gate, const void* dy,
                                  const int64_t* strides, const int32_t* cu_seqlens, const float* marks,
                                  const float* dh_last, void* df, void* dx, void* dgate, float* dh0, int64_t S,
                                  int64_t T, int64_t C, int dtype, void* workspace, size_t workspace_bytes,
                                  void* stream) {
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
  return dispatch_scan(A, dtype, true, workspace, workspace_bytes, st, "csn_gated_scan_bwd");
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

// whether the bytes of B rows of C elements at p reach into h
bool shares(const StepArgs& A, const void* p, int64_t row, int64_t B, int size) {
  if (!p) return false;
  const intptr_t first = reinterpret_cast<intptr_t>(p), last = first + (B - 1) * row * size, h = reinterpret_cast<intptr_t>(A.h);
  return (first < last ? first : last) < h + B * A.C * 4 && h < (first < last ? last : first) + A.C * size;
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
  if (shares(A, f, A.fr, B, size) || shares(A, x, A.xr, B, size) || shares(A, gate, A.gr, B, size) || shares(A, y, C, B, size))
    return set_error(CSN_ERR_INVALID, "csn_gated_step: h shares memory with an input or the result");
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

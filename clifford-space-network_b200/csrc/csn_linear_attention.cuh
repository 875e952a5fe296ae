// csn_linear_attention.cuh -- what the step-by-step and the tensor-core kernels of linear attention share.
//
//   S_t = l S_{t-1} + k_t v_t^T,   o_t = c S_t^T q_t,   l = exp(log_decay)     (one head; S is Dk x Dv)
// Adjoint, with D_t = c q_t do_t^T + l D_{t+1} (at the end plus the gradient of the last state):
//   dq_t = c S_t do_t,  dk_t = D_t v_t,  dv_t = D_t^T k_t,  dS_{-1} = l D_0
// So each of o, dq, dk and dv is one pass of a single form over three streams a, b, v of rows, and only the direction
// of time, the places of the two scales and the way a state lies in memory (S or S^T) differ:
//   X_t = l X_{t-1} + sb b_t v_t^T,   out_t = so X_t^T a_t
//     o: (q, k, v)   dq: (do, v, k), X = S^T      sb = 1, so = c, forward
//     dv: (k, q, do) dk: (v, do, q), X = D^T      sb = c, so = 1, backward, where Y_t = l X_t is what is carried
//
// Where there are too few sequences and heads to fill the GPU, sequences are cut into segments of `seg` steps.  A first
// pass leaves the state that each segment makes of nothing (only b and v are read), join_kernel runs over these in
// the order of time and puts in their place the state that enters each segment, and the segments then run side by
// side from there.  A sequence of a packed batch begins with unit cu[s] / seg + s, which leaves room for its segments
// whatever the other lengths are; some units are empty.
#pragma once

#include <cstdint>

#include "csn_internal.h"
#include "csn_types.cuh"

namespace csn {
namespace la {

struct Stream {  // element (sequence s, step t, head h, place d) at p + s * seq + t * row + h * head + d
  const void* p;
  int64_t seq, row, head;  // in elements
  int shared;              // heads of the pass that read one head of the stream
};

struct Batch {
  const int32_t* cu;  // packed: sequence s has the rows cu[s] .. cu[s + 1] - 1 of T; NULL: S sequences of T steps
  int64_t S, T;
  int H, seg, segs;   // segs: of a sequence, where all have one length
  int64_t units;
  const float* log_decay;
};

struct Pass {
  Stream a, b, v;
  void* out;             // [rows][H][V] contiguous; float32 where `wide`, the tensors' type elsewhere
  const float* state;    // [S][H][K V] float32: what enters each sequence, NULL for 0
  float* last;           // [S][H][K V]: what leaves it, NULL: not wanted
  float* made;           // [units][H][K V], of cut sequences: what the first pass leaves, and then what enters each segment
  int64_t sr, sc;        // entry (place of b, place of v) of a state at sr, sc
  int K, V;              // places of b and of v
  float so, sb;
  bool wide, back;
};

// The part of a sequence that a unit has: steps from .. to - 1 of len.
struct Unit {
  int64_t s, row0, unit;  // s = -1: none
  int len, from, to;

  static __device__ __forceinline__ int64_t border(const Batch& B, int64_t i) {
    return min(max((int64_t)B.cu[i], (int64_t)0), B.T);
  }
  // Unit u; or, `first`, in a packed batch the unit that row u seg lies in, and the next one where time runs down: each whole
  // segment has one such row, so that the first pass, which is for these (those behind them) alone, need not start a CTA for
  // every short sequence.
  __device__ __forceinline__ Unit(const Batch& B, int64_t u, bool first, bool back) : unit(u) {
    int64_t m;
    if (B.cu) {
      const int64_t at = first ? u * B.seg : u;
      int64_t lo = 0, n = B.S;  // the last s that begins at `at` or before lies in lo .. lo + n - 1
      while (n > 1) {
        const int64_t half = n / 2, i = lo + half, row = border(B, i);
        if ((first ? row : row / B.seg + i) <= at) lo = i, n -= half;
        else n = half;
      }
      s = lo;
      row0 = border(B, s);
      len = (int)(max(border(B, s + 1), row0) - row0);
      const int64_t base = row0 / B.seg + s;
      if (first) unit = row0 <= at ? base + (at - row0) / B.seg + (back ? 1 : 0) : -1;
      m = unit - base;
    } else {
      s = u / B.segs;
      row0 = s * B.T;
      len = (int)B.T;
      m = u - s * B.segs;
    }
    if (m < 0 || (m > 0 && m * B.seg >= len)) {
      s = -1;
      from = to = 0;
      return;
    }
    from = (int)(m * B.seg);
    to = (int)min((int64_t)from + B.seg, (int64_t)len);
  }
  __device__ __forceinline__ bool ends(bool back) const { return back ? from == 0 : to == len; }
  // elements from a stream's p to step 0 of the sequence
  __device__ __forceinline__ int64_t start(const Batch& B, const Stream& x) const { return B.cu ? row0 * x.row : s * x.seq; }
};

// CTAs along the units: all of them, or what the first pass needs
inline int64_t unit_grid(const Batch& B, bool first) { return first && B.cu ? (B.T + B.seg - 1) / B.seg : B.units; }

// l^n without the rounding of log_decay * n (a product of 1000 would cost exp its last 10 bits); l^0 = 1 for l = 0 too
__device__ __forceinline__ float fade(float log_decay, int n) { return n == 0 ? 1.0f : (float)exp((double)log_decay * n); }

// Passes over 16-bit rows on the tensor cores; `first`: only the states that units make of nothing.  Rows of the streams start on
// 16 bytes, their strides are multiples of that and not 0 where an axis has more than one place.  seg is a multiple of 128.
int tensor_passes(const Batch& B, const Pass* passes, int count, bool first, bool bf16, cudaStream_t st);

}  // namespace la
}  // namespace csn

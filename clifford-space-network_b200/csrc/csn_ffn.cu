// csn_ffn.cu -- the gated feed-forward product of 16-bit tensors and its adjoint, on the tensor cores.
//
//   g = x Wg^T,  u = x Wu^T,  y = silu(g) * u          x [R, C], Wg, Wu [F, C], y [R, F]
// Adjoint, with w = sigmoid(g):
//   dg = dy u w (1 + g (1 - w)),  du = dy g w,  dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x
// The backward pass takes g and u in float32 from what the forward pass kept ([2, R, F]), or forms them again.  Keeping
// them costs 8 bytes an element written and read, forming them 4 C operations: at 6.5 TB/s and 1.4 PFLOP/s the two are
// even near C = 1000, and the caller of these entry points decides (the PyTorch functions keep them from C = 1536 on; rounded to
// 16 bits they would cost a third of the gradients' precision).
// dg and du are rounded to the tensors' own type once, as the operands of the products that follow.  In float16,
// whose numbers end at 65504 and lose bits below 2^-14, they are first scaled by the power of two that brings the largest
// finite |dy| into [2^10, 2^11), and the products are scaled back in float32.  So a row whose dy is 2^-24 of the largest
// keeps its precision, and |dg / dy| and |du / dy| up to 32 fit.  The pass also notes the largest |dg| and |du|: where they do
// not fit after all, it runs again with the scale that brings these into [2^14, 2^15).  This second pass is launched each
// time, while the first runs, and ends at once where they do fit: at most 2 us (launched after the first: 6 to 8).
//
// mm_kernel is one persistent kernel for the four products (Mode).  A pair of CTAs on two SMs (cta_group::2) makes a
// tile of 256 x BN: each loads 128 rows of A and half of B, so a k block of 64 moves 32 KB into an SM for the products
// that take 48 KB when it works alone.  In each CTA a warp feeds a ring of shared-memory stages by TMA, a warp of the
// pair issues tcgen05.mma into one of two accumulators in tensor memory, and for each accumulator eight warps finish it,
// so that loads, products and both epilogues overlap across tiles (all sixteen on one accumulator after the other:
// R65536 C128 F256 forward 26.6 us against 20.8).  For the gate, BN = 2 FN: CTA 0 loads FN rows of Wg and CTA 1 the same
// FN rows of Wu as the halves of one operand, so g and u of a place sit in one tensor-memory lane and the gate is a
// per-lane epilogue.  The transposed products read the same row-major tensors with an MN-major operand: nothing is
// transposed in memory.
//
// What bounds it, bf16 on a B200: large products the tensor pipe, 94 to 98 % active.  R2048 C4096 F8192 forward 174 us,
// 1.58 PFLOP/s, 0.94 of what the library's product of 8192^3 reaches; training R8192 C4096 F8192 2.75 ms, 1.2 PFLOP/s of
// the 12 R C F that it cannot do without, under the power cap.  With few channels the gate's epilogue does, two MUFU
// operations and about 35 instructions an element: R65536 C128 F256 forward 22 us against 7.7 us for its bytes.  Rows
// that start on 16 but not on 128 bytes cost the loads a third (R1021 C1032 F2744 22 us, R1024 C1024 F2752 16).
//
// few_rows_kernel takes R <= 64 rows (generation): there the weights are what is read, so they take the 128-row side
// of the product (64 rows of Wg and 64 of Wu) and x the narrow side, and a cluster splits C where F alone gives too
// few CTAs, its partial sums joined through distributed shared memory in a fixed order.  Bound by the weights' bytes and
// by the start and end of a short kernel: R4 C2048 F8192 15 us of 10.3 with the weights in HBM, R2 C256 F512 4.6 us.
#include <cstdint>

#include "csn_internal.h"
#include "csn_tc.cuh"
#include "csn_types.cuh"

namespace csn {
namespace {

using namespace tc;

enum Mode { GATE, GATE_BWD, DX, DW };

constexpr int BM = 128, BK = 64;                    // rows of a CTA (a pair has 2 BM), k of a stage
constexpr int EPI_WARPS = 16;                       // 8 for each accumulator
constexpr int THREADS = (EPI_WARPS + 2) * 32;
constexpr int STAGE_ROW = 80;                       // a lane's 64 bytes, padded against bank conflicts
constexpr int STAGING = EPI_WARPS * 32 * STAGE_ROW;
constexpr int PAIRS = 74;                           // of SMs: what the work is cut up for

__host__ __device__ constexpr int stage_bytes(int bn) { return (BM + bn / 2) * BK * 2; }
__host__ __device__ constexpr int stages(int bn) { return bn == 256 ? 5 : 7; }
constexpr int smem_bytes(int bn) { return stages(bn) * stage_bytes(bn) + STAGING + 1024; }

struct Maps {
  CUtensorMap a[2], b[2];
};

struct Args {
  int m, n;           // the output's rows and columns (of one half, for DW)
  int mt, nt;         // its tiles
  int kb;             // k blocks of one half
  int halves_m;       // 2 for DW: dWg, then dWu
  int halves_k;       // 2 for DX: dg Wg, then du Wu
  int splits, kper;   // k blocks are cut into `splits` ranges of kper
  void* out[2];       // y; dg, du; dx; dWg, dWu
  int64_t ldo;
  const void* dy;
  int64_t ldy;
  float* part;        // splits > 1: [splits][halves_m][m][n]
  float* pre;         // GATE: g and u are kept here, [2][m][n]
  uint32_t* range;  // float16 backward: what scales dg and du
  bool again;       // GATE_BWD: the pass that runs where the first scale was too large
};

// The scale of float16's dg and du.  range[0]: bits of the largest finite |dy|, range[1]: of the largest finite |dg| or
// |du| under the first scale, where that is above 65504 (0: none).
constexpr uint32_t HALF_MAX = 0x477fe000;  // bits of 65504

__device__ __forceinline__ bool too_large(const uint32_t* range) { return range[1] != 0; }
// its exponent as a float32 has it, and that of its inverse is 254 less this: |dy| is 0 or 2^-24 to 2^16, so the first is
// 122 to 161, and the second 9 at least.
__device__ __forceinline__ uint32_t scale_exponent(const uint32_t* range, bool again) {
  if (range[0] == 0) return 127;
  const uint32_t first = 127 + 10 + 127 - (range[0] >> 23);
  return again ? first + 14 + 127 - (range[1] >> 23) : first;
}
// for dg and du
__device__ __forceinline__ float scale_up(const uint32_t* range, bool again) {
  return range ? __uint_as_float(scale_exponent(range, again) << 23) : 1.0f;
}
// for the products of dg and du
__device__ __forceinline__ float scale_down(const uint32_t* range) {
  return range ? __uint_as_float((254 - scale_exponent(range, too_large(range))) << 23) : 1.0f;
}
// the larger of `top` and what is finite of the larger of |a| and |b| (a NaN counts as nothing)
__device__ __forceinline__ float finite_max(float top, float a, float b) {
  const float m = fmaxf(fabsf(a), fabsf(b));
  return fmaxf(top, m < __int_as_float(0x7f800000) ? m : 0.0f);
}
// A warp's maximum into the bits of *to, where the order does not matter, if it is above `floor`: when all warps of a grid add
// theirs, they stand in line for one address (gate_back_kernel, 33.5 million elements in 38 thousand warps: 90 us against 65).
__device__ __forceinline__ void note_max(uint32_t* to, float top, uint32_t floor) {
  const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
  if ((threadIdx.x & 31) == 0 && bits > floor) atomicMax(to, bits);
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if (BF16) {
    __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&v);
  }
  __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&v);
}
template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
  if (BF16) return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&v));
  return __half22float2(*reinterpret_cast<__half2*>(&v));
}

// A warp's 32 rows x 64 bytes pass between a lane's own row in `stage` and memory in whole row pieces (4 lanes a row,
// 8 rows an access); `vec`: rows start on 16 bytes and hold multiples of 16.
__device__ __forceinline__ void put_rows(const char* stage, int lane, char* out, int64_t row_bytes, int rows, int bytes,
                                         bool vec) {
  __syncwarp();
  if (vec) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = i * 8 + lane / 4, at = lane % 4 * 16;
      if (r < rows && at < bytes)
        *reinterpret_cast<uint4*>(out + r * row_bytes + at) = *reinterpret_cast<const uint4*>(stage + r * STAGE_ROW + at);
    }
  } else if (lane * 2 < bytes) {
    for (int r = 0; r < rows; ++r)
      *reinterpret_cast<uint16_t*>(out + r * row_bytes + lane * 2) =
          *reinterpret_cast<const uint16_t*>(stage + r * STAGE_ROW + lane * 2);
  }
  __syncwarp();
}
// what lies outside comes as 0
__device__ __forceinline__ void get_rows(char* stage, int lane, const char* in, int64_t row_bytes, int rows, int bytes,
                                         bool vec) {
  if (vec) {
    uint4 got[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = i * 8 + lane / 4, at = lane % 4 * 16;
      got[i] = r < rows && at < bytes ? *reinterpret_cast<const uint4*>(in + r * row_bytes + at) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *reinterpret_cast<uint4*>(stage + (i * 8 + lane / 4) * STAGE_ROW + lane % 4 * 16) = got[i];
  } else {
    for (int r = 0; r < 32; ++r)
      *reinterpret_cast<uint16_t*>(stage + r * STAGE_ROW + lane * 2) =
          r < rows && lane * 2 < bytes ? *reinterpret_cast<const uint16_t*>(in + r * row_bytes + lane * 2) : (uint16_t)0;
  }
  __syncwarp();
}
// 8 words (32 bytes) of a lane's own row
__device__ __forceinline__ void put8(char* p, const uint32_t* v) {
  reinterpret_cast<uint4*>(p)[0] = make_uint4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<uint4*>(p)[1] = make_uint4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void get8(const char* p, uint32_t* v) {
  const uint4 a = reinterpret_cast<const uint4*>(p)[0], b = reinterpret_cast<const uint4*>(p)[1];
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}

// Tiles are walked in groups of 16 rows of tiles, column by column: the operands of the tiles under way at one time
// (16 x 5 pairs') are read from HBM once and stay in L2.
struct Tile {
  int m, n, half, split;
  __device__ __forceinline__ Tile(const Args& P, int t) {
    const int per_unit = P.mt * P.nt;
    const int unit = t / per_unit;
    t -= unit * per_unit;
    half = unit % P.halves_m;
    split = unit / P.halves_m;
    const int per = 16 * P.nt, g = t / per, rem = t - g * per;
    const int gm = min(16, P.mt - g * 16);
    m = g * 16 + rem % gm;
    n = rem / gm;
  }
};

template <Mode MODE, bool BF16, int BN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
    mm_kernel(const __grid_constant__ Maps maps, const Args P) {
  constexpr int ST = stages(BN), SB = stage_bytes(BN);
  constexpr bool A_MN = MODE == DW, B_MN = MODE == DX || MODE == DW;
  constexpr int FN = BN / 2;
  extern __shared__ char raw[];
  // full, acc_empty: those of CTA 0 count for the pair; empty, acc_full: each CTA's own
  __shared__ uint64_t full[ST], empty[ST], acc_full[2], acc_empty[2], drained;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile uint32_t gave_up;
  char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = (int)cluster_rank();
  const int tiles = P.mt * P.nt * P.halves_m * P.splits, first = blockIdx.x / 2, step = gridDim.x / 2;
  constexpr bool SCALED = MODE == GATE_BWD && !BF16;
  if (SCALED && P.again) {  // launched early (programmatic dependent launch): what the first pass leaves is awaited
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (!too_large(P.range)) return;
  } else if (SCALED) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  }

  if (threadIdx.x == 0) {
    for (int i = 0; i < ST; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], 1);
    for (int i = 0; i < 2; ++i) mbar_init(&acc_full[i], 1), mbar_init(&acc_empty[i], EPI_WARPS);
    mbar_init(&drained, 1);
    mbar_init_fence();
    gave_up = 0;
  }
  if (warp == EPI_WARPS) tmem_alloc_pair<2 * BN>(&tmem_slot);
  fence_before();
  __syncthreads();
  cluster_sync();  // the other CTA's barriers are there
  fence_after();
  const uint32_t tmem = tmem_slot;

  if (warp == EPI_WARPS) {  // TMA
    int s = 0, it = 0;
    uint32_t parity = 1;
    bool ok = true;
    for (int t = first; t < tiles && ok; t += step) {
      const Tile T(P, t);
      const int k0 = T.split * P.kper, k1 = min(k0 + P.kper, P.kb * P.halves_k);
      const int m = (T.m * 2 + rank) * BM;
      for (int k = k0; k < k1; ++k, ++it) {
        if (!(ok = __all_sync(0xffffffffu, mbar_wait(&empty[s], parity, &gave_up)))) break;
        if (elect_one()) {
          if (rank == 0) mbar_expect(&full[s], 2 * SB);
          const uint32_t bar = peer_addr(&full[s], 0);
          char* a = smem + s * SB;
          char* b = a + BM * BK * 2;
          if (MODE == GATE || MODE == GATE_BWD) {
            tma_load_pair(a, &maps.a[0], k * BK, m, bar);
            tma_load_pair(b, &maps.b[rank], k * BK, T.n * FN, bar);
          } else if (MODE == DX) {
            const int h = k >= P.kb, kk = (k - h * P.kb) * BK;
            tma_load_pair(a, &maps.a[h], kk, m, bar);
#pragma unroll
            for (int j = 0; j < FN / 64; ++j)
              tma_load_pair(b + j * 8192, &maps.b[h], T.n * BN + rank * FN + j * 64, kk, bar);
          } else {
#pragma unroll
            for (int j = 0; j < BM / 64; ++j) tma_load_pair(a + j * 8192, &maps.a[T.half], m + j * 64, k * BK, bar);
#pragma unroll
            for (int j = 0; j < FN / 64; ++j)
              tma_load_pair(b + j * 8192, &maps.b[0], T.n * BN + rank * FN + j * 64, k * BK, bar);
          }
        }
        __syncwarp();
        if (++s == ST) s = 0, parity ^= 1;
      }
    }
    if (ok) {  // the pair's last commits arrive before this CTA leaves
      for (int j = it > ST ? it - ST : 0; j < it; ++j) mbar_wait(&empty[j % ST], (j / ST) & 1, &gave_up);
    } else if (rank == 0) {  // copies in flight end before the shared memory does (CTA 0's barriers count both CTAs')
      for (int j = it > ST ? it - ST : 0; j < it; ++j)
        for (uint32_t i = 0; i < POLLS && !mbar_try(&full[j % ST], (j / ST) & 1); ++i) {}
    }
  } else if (warp == EPI_WARPS + 1) {
    if (rank == 0) {  // MMA
      constexpr uint32_t IDESC = instruction(BF16, A_MN, B_MN, 2 * BM, BN);
      const uint64_t desc0 = operand(smem_addr(smem), 8192);
      int s = 0, n = 0;
      uint32_t parity = 0;
      bool ok = true;
      for (int t = first; t < tiles && ok; t += step, ++n) {
        const Tile T(P, t);
        const int k0 = T.split * P.kper, k1 = min(k0 + P.kper, P.kb * P.halves_k);
        const uint32_t d = tmem + (n & 1) * BN;
        if (!(ok = __all_sync(0xffffffffu, mbar_wait(&acc_empty[n & 1], ((n >> 1) + 1) & 1, &gave_up)))) break;
        fence_after();
        for (int k = k0; k < k1; ++k) {
          if (!(ok = __all_sync(0xffffffffu, mbar_wait(&full[s], parity, &gave_up)))) break;
          fence_after();
          if (elect_one()) {
            const uint64_t ad = desc0 + (uint32_t)(s * SB >> 4), bd = ad + (BM * BK * 2 >> 4);
#pragma unroll
            for (int j = 0; j < BK / 16; ++j)
              mma_pair(d, ad + j * (A_MN ? 2048 >> 4 : 32 >> 4), bd + j * (B_MN ? 2048 >> 4 : 32 >> 4), IDESC, k > k0 || j > 0);
            mma_commit_pair(&empty[s]);
            if (k == k1 - 1) mma_commit_pair(&acc_full[n & 1]);
          }
          __syncwarp();
          if (++s == ST) s = 0, parity ^= 1;
        }
      }
      if (!ok) {
        if (elect_one()) mma_commit_pair(&drained);
        __syncwarp();
        for (uint32_t i = 0; i < POLLS && !mbar_try(&drained, 0); ++i) {}
      }
    }
  } else {
    // epilogue: warp w finishes accumulator w / 8, reads the tensor-memory lanes of quarter w % 4 and half of the columns
    char* stage = smem + ST * SB + warp * 32 * STAGE_ROW;
    char* own = stage + lane * STAGE_ROW;
    const int acc = warp / 8, quarter = warp % 4, side = warp / 4 % 2;
    const float up = SCALED ? scale_up(P.range, P.again) : 1.0f;
    const float down = (MODE == DX || MODE == DW) && !BF16 ? scale_down(P.range) : 1.0f;
    float top = 0.0f;  // SCALED: the largest finite |dg| and |du|
    const uint32_t d = tmem + acc * BN + ((uint32_t)(quarter * 32) << 16), release = peer_addr(&acc_empty[acc], 0);
    const bool vec = (MODE == DX || MODE == DW) && P.splits > 1 ? P.n % 4 == 0 : P.ldo % 8 == 0;
    const bool vec_dy = MODE == GATE_BWD && P.ldy % 8 == 0 && (reinterpret_cast<uintptr_t>(P.dy) & 15) == 0 && P.n % 8 == 0;
    const bool vec_pre = P.n % 4 == 0;
    uint32_t parity = 0;
    for (int t = first + acc * step; t < tiles; t += 2 * step, parity ^= 1) {
      const Tile T(P, t);
      const int64_t row0 = (int64_t)(T.m * 2 + rank) * BM + quarter * 32;
      const int rows = (int)min((int64_t)32, P.m - row0);
      const bool ok = mbar_wait(&acc_full[acc], parity, &gave_up);
      __syncwarp();
      fence_after();
      const float nan = __int_as_float(0x7fffffff);
#pragma unroll 1
      for (int c = side * (MODE <= GATE_BWD ? FN / 2 : FN); c < (side + 1) * (MODE <= GATE_BWD ? FN / 2 : FN); c += 32) {
        const int64_t col = (int64_t)T.n * (MODE <= GATE_BWD ? FN : BN) + c;
        const int cols = (int)min((int64_t)32, P.n - col);
        if (rows <= 0 || cols <= 0) continue;
        if (MODE == GATE || MODE == GATE_BWD) {
          const int64_t at = (row0 * P.ldo + col) * 2;
          if (MODE == GATE_BWD)
            get_rows(stage, lane, static_cast<const char*>(P.dy) + (row0 * P.ldy + col) * 2, P.ldy * 2, rows, cols * 2, vec_dy);
          uint32_t du[2][8];  // GATE: y
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float g[16], u[16];
            tmem_load16(d + c + h * 16, g);
            tmem_load16(d + FN + c + h * 16, u);
            uint32_t dy[8], o[8];
            if (MODE == GATE_BWD) get8(own + h * 32, dy);
            tmem_load_wait();
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              float r0[2], r1[2];
              const float2 dv = MODE == GATE_BWD ? unpack2<BF16>(dy[i]) : make_float2(0.0f, 0.0f);
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                const float gv = ok ? g[2 * i + j] : nan, uv = u[2 * i + j];
                const float w = sigmoid(gv);
                if (MODE == GATE) {
                  r0[j] = gv * w * uv;
                } else {
                  const float e = (j ? dv.y : dv.x) * up;
                  r0[j] = e * uv * (w * fmaf(gv, 1.0f - w, 1.0f));
                  r1[j] = e * gv * w;
                  if (SCALED) top = finite_max(top, r0[j], r1[j]);
                }
              }
              if (MODE == GATE_BWD) {
                o[i] = pack2<BF16>(r0[0], r0[1]);
                du[h][i] = pack2<BF16>(r1[0], r1[1]);
              } else {
                du[h][i] = pack2<BF16>(r0[0], r0[1]);
              }
            }
            if (MODE == GATE_BWD) put8(own + h * 32, o);  // where this half's dy was
            if (MODE == GATE && P.pre && h * 16 < cols) {
              float* pre = P.pre + row0 * P.n + col + h * 16;
              const int part = min(cols - h * 16, 16) * 4;
              if (!ok) {
#pragma unroll
                for (int i = 0; i < 16; ++i) g[i] = u[i] = nan;
              }
              put8(own, reinterpret_cast<uint32_t*>(g));
              put8(own + 32, reinterpret_cast<uint32_t*>(g) + 8);
              put_rows(stage, lane, reinterpret_cast<char*>(pre), (int64_t)P.n * 4, rows, part, vec_pre);
              put8(own, reinterpret_cast<uint32_t*>(u));
              put8(own + 32, reinterpret_cast<uint32_t*>(u) + 8);
              put_rows(stage, lane, reinterpret_cast<char*>(pre + (int64_t)P.m * P.n), (int64_t)P.n * 4, rows, part, vec_pre);
            }
          }
          if (MODE == GATE_BWD)
            put_rows(stage, lane, static_cast<char*>(P.out[0]) + at, P.ldo * 2, rows, cols * 2, vec);
          put8(own, du[0]);
          put8(own + 32, du[1]);
          put_rows(stage, lane, static_cast<char*>(MODE == GATE ? P.out[0] : P.out[1]) + at, P.ldo * 2, rows, cols * 2, vec);
        } else {
          void* to = T.half ? P.out[1] : P.out[0];
          if (!to) continue;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float v[16];
            tmem_load16(d + c + h * 16, v);
            tmem_load_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (!ok) v[i] = nan;
            if (P.splits > 1) {
              if (h * 16 >= cols) continue;
              put8(own, reinterpret_cast<uint32_t*>(v));
              put8(own + 32, reinterpret_cast<uint32_t*>(v) + 8);
              char* out = reinterpret_cast<char*>(P.part) +
                          ((((int64_t)T.split * P.halves_m + T.half) * P.m + row0) * P.n + col + h * 16) * 4;
              put_rows(stage, lane, out, (int64_t)P.n * 4, rows, min(cols - h * 16, 16) * 4, vec);
            } else {
              uint32_t o[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) o[i] = pack2<BF16>(v[2 * i] * down, v[2 * i + 1] * down);
              put8(own + h * 32, o);
            }
          }
          if (P.splits == 1)
            put_rows(stage, lane, static_cast<char*>(to) + (row0 * P.ldo + col) * 2, P.ldo * 2, rows, cols * 2, vec);
        }
      }
      fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(release);
    }
    if (SCALED && !P.again) note_max(&P.range[1], top, HALF_MAX);
  }
  fence_before();
  __syncthreads();
  cluster_sync();  // nothing of the pair is on its way to a CTA that has left
  fence_after();
  if (warp == EPI_WARPS) tmem_free_pair<2 * BN>(tmem);
}

// Sums of the k ranges, in their order: element i of half h is out[h][i].
template <bool BF16>
__global__ void __launch_bounds__(128) join_kernel(const float* __restrict__ part, void* out0, void* out1, int64_t n,
                                                   int halves, int splits, const uint32_t* range) {
  const float down = BF16 ? 1.0f : scale_down(range);
  const int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x, stride = n * halves;
  if (i >= stride) return;
  const bool second = i >= n;
  void* out = second ? out1 : out0;
  if (!out) return;
  float v = 0.0f;
#pragma unroll 16
  for (int s = 0; s < splits; ++s) v += part[s * stride + i];
  v *= down;
  const int64_t at = second ? i - n : i;
  if (BF16) static_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(v);
  else static_cast<__half*>(out)[at] = __float2half_rn(v);
}

// dg and du from the g and u that were kept: element (r, c) of g at r * F + c, of u R * F further.  A thread has 8
// neighbouring elements where rows allow it (VEC), else one.  Memory bound: 14 bytes an element.
template <bool BF16, bool VEC>
__global__ void __launch_bounds__(256) gate_back_kernel(const float* __restrict__ pre, const uint16_t* __restrict__ dy, int64_t ldy,
                                                        uint16_t* dg, uint16_t* du, int64_t ld, int64_t R, int64_t F,
                                                        uint32_t* range, bool again) {
  constexpr int N = VEC ? 8 : 1;
  if (!BF16 && again && !too_large(range)) return;
  const float up = BF16 ? 1.0f : scale_up(range, again);
  float top = 0.0f;  // float16: the largest finite |dg| and |du|
  const int64_t per = F / N, n = R * per;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / per, c = (i - r * per) * N;
    float g[N], u[N], d[N], a[N], b[N];
    const float* p = pre + r * F + c;
    if (VEC) {
#pragma unroll
      for (int j = 0; j < N; j += 4) {
        const float4 x = __ldg(reinterpret_cast<const float4*>(p + j)), y = __ldg(reinterpret_cast<const float4*>(p + R * F + j));
        g[j] = x.x, g[j + 1] = x.y, g[j + 2] = x.z, g[j + 3] = x.w, u[j] = y.x, u[j + 1] = y.y, u[j + 2] = y.z, u[j + 3] = y.w;
      }
      const uint4 q = __ldg(reinterpret_cast<const uint4*>(dy + r * ldy + c));
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 v = unpack2<BF16>(w[j]);
        d[2 * j] = v.x, d[2 * j + 1] = v.y;
      }
    } else {
      g[0] = p[0], u[0] = p[R * F];
      d[0] = unpack2<BF16>(dy[r * ldy + c]).x;
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float w = sigmoid(g[j]), e = d[j] * up;
      a[j] = e * u[j] * (w * fmaf(g[j], 1.0f - w, 1.0f));
      b[j] = e * g[j] * w;
      if (!BF16) top = finite_max(top, a[j], b[j]);
    }
    if (VEC) {
      *reinterpret_cast<uint4*>(dg + r * ld + c) =
          make_uint4(pack2<BF16>(a[0], a[1]), pack2<BF16>(a[2], a[3]), pack2<BF16>(a[4], a[5]), pack2<BF16>(a[6], a[7]));
      *reinterpret_cast<uint4*>(du + r * ld + c) =
          make_uint4(pack2<BF16>(b[0], b[1]), pack2<BF16>(b[2], b[3]), pack2<BF16>(b[4], b[5]), pack2<BF16>(b[6], b[7]));
    } else {
      dg[r * ld + c] = (uint16_t)pack2<BF16>(a[0], 0.0f);
      du[r * ld + c] = (uint16_t)pack2<BF16>(b[0], 0.0f);
    }
  }
  if (!BF16 && !again) note_max(&range[1], top, HALF_MAX);
}

// range[0] (0 before): bits of the largest finite |dy|.  A thread has 8 neighbouring elements of a row; `vec`: in one access.
// A CTA adds one maximum: R1024 F2752 4 us, with one a warp 9.
__global__ void __launch_bounds__(256) amax_kernel(const __half* __restrict__ dy, int64_t ld, int64_t R, int64_t F, bool vec,
                                                   uint32_t* range) {
  float top = 0.0f;
  const int64_t per = (F + 7) / 8, n = R * per;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / per, c = (i - r * per) * 8;
    const __half* p = dy + r * ld + c;
    if (vec) {
      const uint4 q = __ldg(reinterpret_cast<const uint4*>(p));
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 v = unpack2<false>(w[j]);
        top = finite_max(top, v.x, v.y);
      }
    } else {
      for (int j = 0; j < 8 && c + j < F; ++j) top = finite_max(top, __half2float(p[j]), 0.0f);
    }
  }
  __shared__ uint32_t tops[8];
  const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
  if ((threadIdx.x & 31) == 0) tops[threadIdx.x / 32] = bits;
  __syncthreads();
  if (threadIdx.x < 32) note_max(range, threadIdx.x < 8 ? __uint_as_float(tops[threadIdx.x]) : 0.0f, 0);
}

// ------------------------------------------------------------------------ few rows
constexpr int FEW = 64, HALF_ROWS = 64, FEW_THREADS = 6 * 32;

__host__ __device__ constexpr int few_stage(int nr) { return (2 * HALF_ROWS + nr) * BK * 2; }
__host__ __device__ constexpr int few_stages(int nr) { return nr == 64 ? 4 : 5; }
constexpr int few_smem(int nr) { return few_stages(nr) * few_stage(nr) + 1024; }

struct FewArgs {
  int R, F, kb;
  void* y;
};

__device__ __forceinline__ float4 peer_float4(uint32_t addr, uint32_t rank) {
  uint32_t a;
  float4 v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
  return v;
}

template <bool BF16, int NR>
__global__ void __launch_bounds__(FEW_THREADS) few_rows_kernel(const __grid_constant__ Maps maps, const FewArgs P) {
  constexpr int ST = few_stages(NR), SB = few_stage(NR), COLS = NR < 32 ? 32 : NR;
  extern __shared__ char raw[];
  __shared__ uint64_t full[ST], empty[ST], done;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile uint32_t gave_up;
  char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  uint32_t ranks;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
  const int f0 = blockIdx.x / ranks * HALF_ROWS;
  const int k0 = P.kb * (int)rank / (int)ranks, k1 = P.kb * ((int)rank + 1) / (int)ranks;  // none is empty: kb >= 4 ranks

  if (threadIdx.x == 0) {
    for (int i = 0; i < ST; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], 1);
    mbar_init(&done, 1);
    mbar_init_fence();
    gave_up = 0;
  }
  if (warp == 4) tmem_alloc<COLS>(&tmem_slot);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_slot;
  // [NR][128], in the stages once they are done with: neighbouring lanes write and read neighbouring places, which
  // matters for what other CTAs read (in the other order a read took 32 trips: 20 thousand cycles for 41 rows)
  float* sums = reinterpret_cast<float*>(smem);

  bool ok = true;
  if (warp == 4) {
    int k = k0;
    for (; k < k1; ++k) {
      const int it = k - k0, s = it % ST;
      if (!__all_sync(0xffffffffu, mbar_wait(&empty[s], (it / ST + 1) & 1, &gave_up))) break;
      if (elect_one()) {
        mbar_expect(&full[s], SB);
        char* a = smem + s * SB;
        tma_load(a, &maps.a[0], k * BK, f0, &full[s]);
        tma_load(a + HALF_ROWS * BK * 2, &maps.a[1], k * BK, f0, &full[s]);
        tma_load(a + 2 * HALF_ROWS * BK * 2, &maps.b[0], k * BK, 0, &full[s]);
      }
      __syncwarp();
    }
    if (k < k1)
      for (int j = max(0, k - k0 - ST); j < k - k0; ++j)
        for (uint32_t i = 0; i < POLLS && !mbar_try(&full[j % ST], (j / ST) & 1); ++i) {}
  } else if (warp == 5) {
    constexpr uint32_t IDESC = instruction(BF16, false, false, 128, NR);
    const uint64_t desc0 = operand(smem_addr(smem), 0);
    for (int k = k0; k < k1; ++k) {
      const int it = k - k0, s = it % ST;
      if (!__all_sync(0xffffffffu, mbar_wait(&full[s], (it / ST) & 1, &gave_up))) break;
      fence_after();
      if (elect_one()) {
        const uint64_t ad = desc0 + (uint32_t)(s * SB >> 4), bd = ad + (2 * HALF_ROWS * BK * 2 >> 4);
#pragma unroll
        for (int j = 0; j < BK / 16; ++j) mma(tmem, ad + j * 2, bd + j * 2, IDESC, k > k0 || j > 0);
        mma_commit(&empty[s]);
      }
      __syncwarp();
    }
    if (elect_one()) mma_commit(&done);
    __syncwarp();
  } else {
    // `done` counts the products issued: complete, unless a wait gave up
    ok = mbar_wait(&done, 0, &gave_up);
    __syncwarp();
    fence_after();
    const int row = warp * 32 + lane;
#pragma unroll
    for (int c = 0; c < NR; c += 16) {
      float v[16];
      tmem_load16(tmem + ((uint32_t)(warp * 32) << 16) + c, v);
      tmem_load_wait();
#pragma unroll
      for (int i = 0; i < 16; ++i) sums[(c + i) * 2 * HALF_ROWS + row] = ok && !gave_up ? v[i] : __int_as_float(0x7fffffff);
    }
    fence_before();
  }
  __syncthreads();
  cluster_sync();
  const uint32_t base = smem_addr(sums);
  // a thread has 4 neighbouring hidden units of a row
  for (int i = rank * FEW_THREADS + threadIdx.x; i < P.R * (HALF_ROWS / 4); i += ranks * FEW_THREADS) {
    const int r = i / (HALF_ROWS / 4), f = i % (HALF_ROWS / 4) * 4, left = P.F - f0 - f;
    if (left <= 0) continue;
    float4 g = make_float4(0.0f, 0.0f, 0.0f, 0.0f), u = g;
#pragma unroll 4
    for (uint32_t k = 0; k < ranks; ++k) {
      const float4 a = peer_float4(base + (r * 2 * HALF_ROWS + f) * 4, k);
      const float4 b = peer_float4(base + (r * 2 * HALF_ROWS + HALF_ROWS + f) * 4, k);
      g.x += a.x, g.y += a.y, g.z += a.z, g.w += a.w;
      u.x += b.x, u.y += b.y, u.z += b.z, u.w += b.w;
    }
    const uint32_t lo = pack2<BF16>(g.x * sigmoid(g.x) * u.x, g.y * sigmoid(g.y) * u.y);
    const uint32_t hi = pack2<BF16>(g.z * sigmoid(g.z) * u.z, g.w * sigmoid(g.w) * u.w);
    uint16_t* y = static_cast<uint16_t*>(P.y) + (int64_t)r * P.F + f0 + f;
    if (P.F % 4 == 0) {
      *reinterpret_cast<uint2*>(y) = make_uint2(lo, hi);
    } else {
      y[0] = (uint16_t)lo;
      if (left > 1) y[1] = (uint16_t)(lo >> 16);
      if (left > 2) y[2] = (uint16_t)hi;
      if (left > 3) y[3] = (uint16_t)(hi >> 16);
    }
  }
  cluster_sync();  // the peers have read this CTA's sums
  if (warp == 4) {
    fence_after();
    tmem_free<COLS>(tmem);
  }
}

// ---------------------------------------------------------------------- padded copies
// Rows that do not start on 16 bytes cannot be read by TMA: they are copied to rows that do, all operands in one launch,
// 16 bytes a thread, in the widest loads that the source allows (N bytes).
struct PadArgs {
  const char* src[3];
  char* dst[3];
  int64_t end[3];  // 16-byte pieces up to and with this operand
  int64_t ld[3];   // bytes of a source row
  int pieces, bytes;  // of a row
};

template <int N>
__device__ __forceinline__ void pad_piece(const char* p, int have, uint16_t* v) {
#pragma unroll
  for (int i = 0; i < 16; i += N) {
    if (i + N <= have) {
      if (N == 8) *reinterpret_cast<uint2*>(v + i / 2) = __ldg(reinterpret_cast<const uint2*>(p + i));
      else if (N == 4) *reinterpret_cast<uint32_t*>(v + i / 2) = __ldg(reinterpret_cast<const uint32_t*>(p + i));
      else v[i / 2] = __ldg(reinterpret_cast<const uint16_t*>(p + i));
    } else {
      for (int j = i; j < i + N; j += 2) v[j / 2] = j < have ? __ldg(reinterpret_cast<const uint16_t*>(p + j)) : (uint16_t)0;
    }
  }
}

__global__ void __launch_bounds__(256) pad_kernel(const PadArgs P) {
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < P.end[2]; i += (int64_t)gridDim.x * blockDim.x) {
    const int o = i < P.end[0] ? 0 : i < P.end[1] ? 1 : 2;
    const char* src = o == 0 ? P.src[0] : o == 1 ? P.src[1] : P.src[2];
    char* dst = o == 0 ? P.dst[0] : o == 1 ? P.dst[1] : P.dst[2];
    const int64_t ld = o == 0 ? P.ld[0] : o == 1 ? P.ld[1] : P.ld[2];
    const int64_t k = i - (o == 0 ? 0 : o == 1 ? P.end[0] : P.end[1]), r = k / P.pieces;
    const int at = (int)(k - r * P.pieces) * 16, have = min(16, P.bytes - at);
    const char* p = src + r * ld + at;
    uint4 v;
    uint16_t* w = reinterpret_cast<uint16_t*>(&v);
    const uintptr_t a = reinterpret_cast<uintptr_t>(src) | (uintptr_t)ld;
    if (a % 8 == 0) pad_piece<8>(p, have, w);
    else if (a % 4 == 0) pad_piece<4>(p, have, w);
    else pad_piece<2>(p, have, w);
    *reinterpret_cast<uint4*>(dst + k * 16) = v;
  }
}

// ---------------------------------------------------------------------------- host
int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to; }

// How a product of m x n over k blocks is cut up: into tiles 256 or 128 columns wide, whichever takes less time when
// PAIRS of them run at a time.  A k block of a wide tile counts 1 and of a narrow one 0.7 (it moves 24 KB an SM for half
// the products of 32 KB), what a tile costs besides 8 and 4.  Forward, wide / narrow, us: R6509 C1152 F3440 71 / 86, R3000
// C768 F1536 15.2 / 17.2, R178 C1736 F4112 17.6 / 14.1, R512 C256 F1024 8.0 / 6.3.  Where tiles leave more than half of the SMs
// idle and k has 32 blocks or more, k is cut into ranges of at least 8, whose sums a second kernel adds (shorter sums
// take less time than that kernel's launch).
struct Plan {
  int bn, mt, nt, splits, kper;
  Plan(int64_t m, int64_t n, int64_t blocks, int halves, bool gate) {
    mt = (int)up(m, 2 * BM);
    const int64_t wide = mt * up(n, gate ? 128 : 256) * halves, narrow = mt * up(n, gate ? 64 : 128) * halves;
    bn = up(wide, PAIRS) * (blocks + 8.0) <= up(narrow, PAIRS) * (0.7 * blocks + 4.0) ? 256 : 128;
    nt = (int)up(n, gate ? bn / 2 : bn);
    splits = 1;
    const int64_t tiles = (int64_t)mt * nt * halves;
    if (!gate && tiles * 2 <= PAIRS && blocks >= 32) {
      const int64_t s = PAIRS / tiles;
      splits = (int)(s < blocks / 8 ? s : blocks / 8);
    }
    kper = (int)up(blocks, splits);
    splits = (int)up(blocks, kper);
  }
};

size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

// A pass's scratch: padded copies of the operands that need one (bits of `copies`: x, w_gate, w_up), and for the backward
// pass dg, du [R, ld], the scale of float16 ones, and the partial sums of split products.
struct Scratch {
  int64_t ld;
  size_t pad[3], dg, du, range, part, total;
  Scratch(int64_t R, int64_t C, int64_t F, int copies, bool bwd) {
    size_t n = 0;
    for (int i = 0; i < 3; ++i) {
      pad[i] = n;
      if (copies >> i & 1) n += align256((size_t)(i ? F : R) * up(C, 8) * 16);
    }
    total = n;
    ld = up(F, 8) * 8;
    if (!bwd) return;
    const Plan px(R, C, 2 * up(F, BK), 1, false), pw(F, C, up(R, BK), 2, false);
    const size_t sx = px.splits > 1 ? (size_t)px.splits * R * C * 4 : 0;
    const size_t sw = pw.splits > 1 ? (size_t)pw.splits * 2 * F * C * 4 : 0;
    dg = n;
    du = dg + align256((size_t)R * ld * 2);
    range = du + align256((size_t)R * ld * 2);
    part = range + 256;
    total = part + align256(sx > sw ? sx : sw);
  }
};

template <Mode MODE, bool BF16, int BN>
int run_mm(const Maps& maps, const Args& P, cudaStream_t st, const char* who) {
  if (cudaError_t e = allow_smem<mm_kernel<MODE, BF16, BN>>(smem_bytes(BN))) return set_cuda_error(e, who);
  const int64_t tiles = (int64_t)P.mt * P.nt * P.halves_m * P.splits;
  const int64_t pairs = sm_count() / 2;
  const unsigned grid = 2 * (unsigned)(tiles < pairs ? tiles : pairs);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem_bytes(BN);
  cfg.stream = st;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = P.again ? 1 : 0;
  if (cudaError_t e = cudaLaunchKernelEx(&cfg, mm_kernel<MODE, BF16, BN>, maps, P)) return set_cuda_error(e, who);
  return check_launch(who);
}

template <bool BF16>
int run_gate(const void* x, int64_t ldx, const void* wg, int64_t ldg, const void* wu, int64_t ldu, const void* dy,
             int64_t ldy, void* o0, void* o1, int64_t ldo, float* pre, uint32_t* range, int64_t R, int64_t C, int64_t F,
             cudaStream_t st, const char* who) {
  const Plan p(R, F, up(C, BK), 1, true);
  Maps maps;
  if (!make_map(&maps.a[0], x, R, C, ldx, BM, BF16) || !make_map(&maps.b[0], wg, F, C, ldg, p.bn / 2, BF16) ||
      !make_map(&maps.b[1], wu, F, C, ldu, p.bn / 2, BF16))
    return set_error(CSN_ERR_CUDA, "silu_gated_linear: cuTensorMapEncodeTiled");
  maps.a[1] = maps.a[0];
  Args P = {};
  P.m = (int)R, P.n = (int)F, P.mt = p.mt, P.nt = p.nt, P.kb = (int)up(C, BK), P.halves_m = P.halves_k = 1;
  P.splits = p.splits, P.kper = p.kper, P.out[0] = o0, P.out[1] = o1, P.ldo = ldo, P.dy = dy, P.ldy = ldy, P.pre = pre, P.range = range;
  if (dy) {
    int rc = p.bn == 256 ? run_mm<GATE_BWD, BF16, 256>(maps, P, st, who) : run_mm<GATE_BWD, BF16, 128>(maps, P, st, who);
    P.again = true;
    if (!BF16 && !rc) rc = p.bn == 256 ? run_mm<GATE_BWD, BF16, 256>(maps, P, st, who) : run_mm<GATE_BWD, BF16, 128>(maps, P, st, who);
    return rc;
  }
  return p.bn == 256 ? run_mm<GATE, BF16, 256>(maps, P, st, who) : run_mm<GATE, BF16, 128>(maps, P, st, who);
}

template <bool BF16, int NR>
int run_few(const Maps& maps, const FewArgs& P, int ranks, cudaStream_t st, const char* who) {
  if (cudaError_t e = allow_smem<few_rows_kernel<BF16, NR>>(few_smem(NR))) return set_cuda_error(e, who);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(up(P.F, HALF_ROWS) * ranks));
  cfg.blockDim = dim3(FEW_THREADS);
  cfg.dynamicSmemBytes = few_smem(NR);
  cfg.stream = st;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = ranks, at.val.clusterDim.y = 1, at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  if (cudaError_t e = cudaLaunchKernelEx(&cfg, few_rows_kernel<BF16, NR>, maps, P)) return set_cuda_error(e, who);
  return check_launch(who);
}

template <bool BF16>
int forward(const void* x, int64_t ldx, const void* wg, int64_t ldg, const void* wu, int64_t ldu, void* y, float* pre, int64_t R,
            int64_t C, int64_t F, cudaStream_t st) {
  const char* who = "csn_silu_gated_linear_fwd";
  if (R > FEW || pre)
    return run_gate<BF16>(x, ldx, wg, ldg, wu, ldu, nullptr, 0, y, nullptr, F, pre, nullptr, R, C, F, st, who);
  const int nr = R <= 16 ? 16 : R <= 32 ? 32 : 64;
  Maps maps;
  if (!make_map(&maps.a[0], wg, F, C, ldg, HALF_ROWS, BF16) || !make_map(&maps.a[1], wu, F, C, ldu, HALF_ROWS, BF16) ||
      !make_map(&maps.b[0], x, R, C, ldx, nr, BF16))
    return set_error(CSN_ERR_CUDA, "silu_gated_linear: cuTensorMapEncodeTiled");
  maps.b[1] = maps.b[0];
  const FewArgs P = {(int)R, (int)F, (int)up(C, BK), y};
  // Ranges of C, at least 4 blocks each, until there are one and a half CTAs an SM.  Two fit, but clusters do not fill
  // every SM: R9 C1824 F4736 took 17.3 us with 296 CTAs and takes 10.0 with 148.
  int ranks = 1;
  while (ranks < 8 && up(F, HALF_ROWS) * ranks * 2 <= 3 * PAIRS && P.kb >= ranks * 2 * 4) ranks *= 2;
  return nr == 16 ? run_few<BF16, 16>(maps, P, ranks, st, who)
                  : nr == 32 ? run_few<BF16, 32>(maps, P, ranks, st, who) : run_few<BF16, 64>(maps, P, ranks, st, who);
}

template <Mode MODE, bool BF16>
int run_product(const Maps& maps, Args P, int64_t blocks, const Plan& p, float* part, cudaStream_t st,
                const char* who) {
  P.mt = p.mt, P.nt = p.nt, P.kb = (int)(blocks / P.halves_k), P.splits = p.splits, P.kper = p.kper, P.part = part;
  int rc = p.bn == 256 ? run_mm<MODE, BF16, 256>(maps, P, st, who) : run_mm<MODE, BF16, 128>(maps, P, st, who);
  if (rc || p.splits == 1) return rc;
  const int64_t n = (int64_t)P.m * P.n;
  join_kernel<BF16><<<(unsigned)up(n * P.halves_m, 128), 128, 0, st>>>(part, P.out[0], P.out[1], n, P.halves_m, p.splits, P.range);
  return check_launch(who);
}

template <bool BF16>
int backward(const void* x, int64_t ldx, const void* wg, int64_t ldg, const void* wu, int64_t ldu, const void* dy,
             int64_t ldy, const float* pre, void* dx, void* dwg, void* dwu, int64_t R, int64_t C, int64_t F, const Scratch& s,
             void* ws, cudaStream_t st) {
  const char* who = "csn_silu_gated_linear_bwd";
  char* base = static_cast<char*>(ws);
  void *dg = base + s.dg, *du = base + s.du;
  float* part = reinterpret_cast<float*>(base + s.part);
  uint32_t* range = nullptr;
  const bool vec = F % 8 == 0 && ldy % 8 == 0 && (reinterpret_cast<uintptr_t>(dy) & 15) == 0;
  if (!BF16) {
    range = reinterpret_cast<uint32_t*>(base + s.range);
    if (cudaError_t e = cudaMemsetAsync(range, 0, 8, st)) return set_cuda_error(e, who);
    const int64_t ctas = up(R * up(F, 8), 256);
    amax_kernel<<<(unsigned)(ctas < 16 * PAIRS ? ctas : 16 * PAIRS), 256, 0, st>>>(static_cast<const __half*>(dy), ldy, R, F, vec, range);
    if (int rc = check_launch(who)) return rc;
  }
  if (pre) {
    const int64_t ctas = up(R * (vec ? F / 8 : F), 256);
    const unsigned grid = (unsigned)(ctas < 64 * PAIRS ? ctas : 64 * PAIRS);
    const uint16_t* d = static_cast<const uint16_t*>(dy);
    uint16_t *a = static_cast<uint16_t*>(dg), *b = static_cast<uint16_t*>(du);
    for (int again = 0; again < (BF16 ? 1 : 2); ++again) {
      if (vec) gate_back_kernel<BF16, true><<<grid, 256, 0, st>>>(pre, d, ldy, a, b, s.ld, R, F, range, again != 0);
      else gate_back_kernel<BF16, false><<<grid, 256, 0, st>>>(pre, d, ldy, a, b, s.ld, R, F, range, again != 0);
      if (int rc = check_launch(who)) return rc;
    }
  } else if (int rc = run_gate<BF16>(x, ldx, wg, ldg, wu, ldu, dy, ldy, dg, du, s.ld, nullptr, range, R, C, F, st, who)) {
    return rc;
  }
  if (dx) {
    const Plan p(R, C, 2 * up(F, BK), 1, false);
    Maps maps;
    if (!make_map(&maps.a[0], dg, R, F, s.ld, BM, BF16) || !make_map(&maps.a[1], du, R, F, s.ld, BM, BF16) ||
        !make_map(&maps.b[0], wg, F, C, ldg, BK, BF16) || !make_map(&maps.b[1], wu, F, C, ldu, BK, BF16))
      return set_error(CSN_ERR_CUDA, "silu_gated_linear: cuTensorMapEncodeTiled");
    Args P = {};
    P.m = (int)R, P.n = (int)C, P.halves_m = 1, P.halves_k = 2, P.out[0] = dx, P.ldo = C, P.range = range;
    if (int rc = run_product<DX, BF16>(maps, P, 2 * up(F, BK), p, part, st, who)) return rc;
  }
  if (dwg || dwu) {
    const Plan p(F, C, up(R, BK), 2, false);
    Maps maps;
    if (!make_map(&maps.a[0], dg, R, F, s.ld, BK, BF16) || !make_map(&maps.a[1], du, R, F, s.ld, BK, BF16) ||
        !make_map(&maps.b[0], x, R, C, ldx, BK, BF16))
      return set_error(CSN_ERR_CUDA, "silu_gated_linear: cuTensorMapEncodeTiled");
    maps.b[1] = maps.b[0];
    Args P = {};
    P.m = (int)F, P.n = (int)C, P.halves_m = 2, P.halves_k = 1, P.out[0] = dwg, P.out[1] = dwu, P.ldo = C, P.range = range;
    if (int rc = run_product<DW, BF16>(maps, P, up(R, BK), p, part, st, who)) return rc;
  }
  return CSN_OK;
}

bool al16b(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool even(const void* p) { return p && (reinterpret_cast<uintptr_t>(p) & 1) == 0; }

// whether TMA reads a matrix in place: its rows start on 16 bytes
bool tiled(const void* p, int64_t rows, int64_t cols, int64_t ld) {
  return al16b(p) && ld % 8 == 0 && (rows == 1 || ld >= cols) && ld > 0 && ld < ((int64_t)1 << 38);
}

// The operands as TMA reads them: themselves, or their copies in the workspace.
struct Operands {
  const void* p[3];
  int64_t ld[3];
  int copies = 0;
  Operands(const void* x, int64_t ldx, const void* wg, int64_t ldg, const void* wu, int64_t ldu, int64_t R, int64_t C, int64_t F)
      : p{x, wg, wu}, ld{ldx, ldg, ldu} {
    for (int i = 0; i < 3; ++i) {
      const int64_t rows = i ? F : R;
      if (rows == 1) ld[i] = up(C, 8) * 8;  // the stride of one row says nothing
      if (!tiled(p[i], rows, C, ld[i])) copies |= 1 << i;
    }
  }
  int copy(int64_t R, int64_t C, int64_t F, const Scratch& s, void* ws, cudaStream_t st) {
    if (!copies) return CSN_OK;
    PadArgs A = {};
    A.pieces = (int)up(C, 8), A.bytes = (int)C * 2;
    int64_t n = 0;
    for (int i = 0; i < 3; ++i) {
      if (copies >> i & 1) {
        A.src[i] = static_cast<const char*>(p[i]), A.dst[i] = static_cast<char*>(ws) + s.pad[i], A.ld[i] = ld[i] * 2;
        n += (i ? F : R) * A.pieces;
        p[i] = A.dst[i], ld[i] = up(C, 8) * 8;
      }
      A.end[i] = n;
    }
    const int64_t ctas = up(n, 256);
    pad_kernel<<<(unsigned)(ctas < 32 * PAIRS ? ctas : 32 * PAIRS), 256, 0, st>>>(A);
    return check_launch("csn_silu_gated_linear: padded copies");
  }
};

int check_ffn(const char* who, int64_t R, int64_t C, int64_t F, int dtype) {
  // tile coordinates and counts are 32-bit
  if (R < 0 || C < 0 || F < 0 || R > (1 << 21) || C > (1 << 21) || F > (1 << 21)) return set_error(CSN_ERR_INVALID, who);
  if (dtype != CSN_BF16 && dtype != CSN_F16) return set_error(CSN_ERR_UNSUPPORTED, who);
  return CSN_OK;
}

}  // namespace
}  // namespace csn

using namespace csn;

extern "C" int csn_silu_gated_linear_copies(const void* x, int64_t ldx, const void* w_gate, int64_t ld_gate, const void* w_up,
                                            int64_t ld_up, int64_t R, int64_t C, int64_t F) {
  return Operands(x, ldx, w_gate, ld_gate, w_up, ld_up, R, C, F).copies;
}

extern "C" size_t csn_silu_gated_linear_workspace_bytes(int64_t R, int64_t C, int64_t F, int copies, int backward) {
  if (R <= 0 || C <= 0 || F <= 0 || R > (1 << 21) || C > (1 << 21) || F > (1 << 21)) return 0;
  return Scratch(R, C, F, copies, backward != 0).total;
}

extern "C" int csn_silu_gated_linear_fwd(const void* x, int64_t ldx, const void* w_gate, int64_t ld_gate,
                                         const void* w_up, int64_t ld_up, void* y, float* pre, int64_t R, int64_t C, int64_t F,
                                         int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_ffn("csn_silu_gated_linear_fwd: needs 0 <= R, C, F <= 2^21 and dtype bfloat16 or float16", R, C, F, dtype))
    return rc;
  if (R == 0 || F == 0) return CSN_OK;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (!y || !al16b(y) || !al16b(pre)) return set_error(CSN_ERR_INVALID, "csn_silu_gated_linear_fwd: y missing, or y or pre misaligned");
  if (C == 0) {
    cudaError_t e = cudaMemsetAsync(y, 0, (size_t)R * F * 2, st);
    if (e == cudaSuccess && pre) e = cudaMemsetAsync(pre, 0, (size_t)R * F * 8, st);
    return e == cudaSuccess ? CSN_OK : set_cuda_error(e, "csn_silu_gated_linear_fwd");
  }
  if (!even(x) || !even(w_gate) || !even(w_up))
    return set_error(CSN_ERR_INVALID, "csn_silu_gated_linear_fwd: x, w_gate and w_up are required, aligned to their type");
  Operands o(x, ldx, w_gate, ld_gate, w_up, ld_up, R, C, F);
  const Scratch s(R, C, F, o.copies, false);
  if (s.total && (!workspace || !al16b(workspace) || workspace_bytes < s.total))
    return set_error(CSN_ERR_INVALID, "csn_silu_gated_linear_fwd: workspace smaller than csn_silu_gated_linear_workspace_bytes");
  KernelTimer kt("silu_gated_linear_fwd", st);
  if (int rc = o.copy(R, C, F, s, workspace, st)) return rc;
  return dtype == CSN_BF16 ? forward<true>(o.p[0], o.ld[0], o.p[1], o.ld[1], o.p[2], o.ld[2], y, pre, R, C, F, st)
                           : forward<false>(o.p[0], o.ld[0], o.p[1], o.ld[1], o.p[2], o.ld[2], y, pre, R, C, F, st);
}

extern "C" int csn_silu_gated_linear_bwd(const void* x, int64_t ldx, const void* w_gate, int64_t ld_gate,
                                         const void* w_up, int64_t ld_up, const void* dy, int64_t ld_dy, const float* pre, void* dx,
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
  if (!even(dy) || !even(x) || !even(w_gate) || !even(w_up) || !al16b(pre) || !al16b(dx) || !al16b(dw_gate) || !al16b(dw_up))
    return set_error(CSN_ERR_INVALID, "csn_silu_gated_linear_bwd: missing or misaligned pointer");
  Operands o(x, ldx, w_gate, ld_gate, w_up, ld_up, R, C, F);
  const Scratch s(R, C, F, o.copies, true);
  if (!workspace || !al16b(workspace) || workspace_bytes < s.total)
    return set_error(CSN_ERR_INVALID, "csn_silu_gated_linear_bwd: workspace smaller than csn_silu_gated_linear_workspace_bytes");
  KernelTimer kt("silu_gated_linear_bwd", st);
  if (int rc = o.copy(R, C, F, s, workspace, st)) return rc;
  return dtype == CSN_BF16 ? backward<true>(o.p[0], o.ld[0], o.p[1], o.ld[1], o.p[2], o.ld[2], dy, ld_dy, pre, dx, dw_gate, dw_up, R, C,
                                            F, s, workspace, st)
                           : backward<false>(o.p[0], o.ld[0], o.p[1], o.ld[1], o.p[2], o.ld[2], dy, ld_dy, pre, dx, dw_gate, dw_up, R,
                                             C, F, s, workspace, st);
}

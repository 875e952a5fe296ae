// csn_linear_attention_tc.cu -- the passes of linear attention (csn_linear_attention.cuh) over 16-bit rows on the tensor cores.
//
// Blocks of 128 steps; with l = exp(log_decay), rows i, j of a block of n, X the state that enters (forward):
//   P_ij = l^(i-j) (a_i . b_j) for j <= i,  out = so (diag(l^(i+1)) A X + P V),  X <- l^n X + (diag(l^(n-1-j)) B)^T V
// and mirrored where time runs down.  A CTA runs through the blocks of one segment of one head:
//   warps 0 to 7 turn A B^T into P, in its place in tensor memory, fade A X, which P V is then added to, and write out, half a
//   row to a thread;
//   warps 8 to 15 fade B, half a row to a thread, and keep the state in registers, half of the entries along b at one place of v;
//   warp 16 loads the tiles of a, b (two stages) and v (one) by TMA;
//   warp 17 issues the four products: A B^T early, A X when the state is there, (l^.. B)^T V, P V.
// Shared memory has no room for a copy of each operand, so they follow one another in place: B, then the first part of the
// faded B; A, then its last part.
//
// Roundings.  P and the state as an operand of A X are rounded to the tensors' type: out itself is, and these two add as
// much again.  The state is not: it stays float32 in registers, and the faded B that enters it is split into parts that
// hold 22 bits or more: three of bfloat16, two of float16.  float16 ends at 65504 and loses bits below 2^-14, so rows of P,
// places of v of the state, and the faded B of a block are first scaled by a power of two that brings the
// largest entry into [2^14, 2^15), and what comes of them is scaled back in float32.
//
// What bounds it: a block's chain, 3.6 to 3.9 us for 128 x 128 states in bf16: A X, the second half of the faded B, its products,
// the state's update and its rounding follow one another, while scores, P and out of the blocks beside run next to them.  Of
// its cycles the shared memory moves data in about two thirds (352 KB of operands for the products of a block, of which the three
// parts of the faded B take 192, and 130 KB that threads write and read), the schedulers issue in 40 %, the tensor
// pipe is active in 32 %, HBM at 0.6 of its rate.  B8 T4096 H16 D128 bf16 forward 135 us (4.0 TB/s), float16 165, D64 93; the three
// passes of its gradients 380 us.  One CTA an SM: 230 KB of shared memory and all of tensor memory.
// Slower, forward: one warpgroup for each half of the work 413 us; P through shared memory 166; the faded B after A X instead of
// half a block ahead 148; rows of out through shared memory 153, since the tiles behind them came late; spilled registers 10 %
// for 160 bytes a thread.  What a sequence's unit derives from ballots or per-lane loads costs the same (the registers of every
// warp), which is why Unit searches with uniform values.
#include <algorithm>
#include <cstdint>

#include "csn_linear_attention.cuh"
#include "csn_tc.cuh"

namespace csn {
namespace {

using namespace tc;
using namespace la;

constexpr int STEPS = 128;      // of a block
constexpr int BOX = 128 * 128;  // bytes of 128 rows x 64 places
constexpr int LOADS = 16, PRODUCTS = 17, THREADS = 20 * 32;
// Registers of a thread of warps 0 to 7, 8 to 15 and the rest: 256 x 72 + 256 x 152 + 128 x 24 = 60416 of the 640 x 96 = 61440
// that a CTA is launched with.
constexpr int FEW = 24, SOME = 72, MANY = 152;
constexpr int MAX_PASSES = 3;

__host__ __device__ constexpr int tile_a(int nk) { return nk * BOX; }
constexpr int smem_bytes(int nk, int nv, bool bf16) { return 4 * tile_a(nk) + nv * BOX + 2 * BOX + (bf16 ? tile_a(nk) : 0) + 1024; }

struct Job {
  CUtensorMap a, b, v;
  Pass pass;
};
struct Jobs {
  Job job[MAX_PASSES];
};

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  return BF16 ? pack<__nv_bfloat16>(a, b) : pack<__half>(a, b);
}
template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
  if (BF16) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  return __half22float2(*reinterpret_cast<__half2*>(&v));
}

// the larger of `top` and |a|, unless that is not finite
__device__ __forceinline__ float finite_max(float top, float a) {
  a = fabsf(a);
  return fmaxf(top, a < __int_as_float(0x7f800000) ? a : 0.0f);
}
// the power of two that brings `top` into [2^14, 2^15), as far as float32 has it and its inverse, and that inverse
__device__ __forceinline__ float scale_up(float top, float& down) {
  const uint32_t e = top == 0.0f ? 141u : max(__float_as_uint(top) >> 23, 15u);
  down = __uint_as_float((e - 14) << 23);
  return __uint_as_float((268 - e) << 23);
}

// 32 bytes in one access, p on a multiple of them
__device__ __forceinline__ void store8(void* p, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
               "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

// 16 bytes: chunk c (8 places) of row r of a tile of boxes of `rows` rows
__device__ __forceinline__ char* chunk_at(char* tile, int rows, int r, int c) {
  return tile + (c / 8) * rows * 128 + r * 128 + ((c % 8) ^ (r & 7)) * 16;
}
__device__ __forceinline__ void arrive_warp(uint64_t* b) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(b);
}

template <bool BF16, int NK, int NV, bool OUT>
__global__ void __launch_bounds__(THREADS, 1) blocks_tc_kernel(const __grid_constant__ Jobs jobs, const Batch B, int count) {
  constexpr int TA = tile_a(NK), PARTS = BF16 ? 3 : 2;
  extern __shared__ char raw[];
  __shared__ uint64_t full_ab[2], full_v, scores, met, keys[2], updated, probs, summed, state, out_read[2], drained;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile uint32_t gave_up;
  __shared__ __align__(16) float place_scale[2][128];
  __shared__ float power[STEPS + 1];
  __shared__ float tops[2][128], place_top[2][128], warp_top[2][8];
  __shared__ __align__(16) float near[32], fan[64];  // powers of the distances to a side of 32 steps, and to its diagonal
  char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  char* const tv = smem + 4 * TA;       // stage s: a at smem + 2 s TA, b behind it
  char* const sp = tv + NV * BOX;       // the state as an operand
  char* const third = sp + 2 * BOX;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  const Job& J = jobs.job[blockIdx.x % count];
  const Pass& P = J.pass;
  const int h = (int)(blockIdx.x / count % B.H);
  const Unit U(B, blockIdx.x / count / B.H, !OUT, P.back);
  const bool back = P.back, cut = U.len > B.seg;
  if (U.s < 0 || (!OUT && U.ends(back))) return;
  const int steps = U.to - U.from, blocks = (steps + STEPS - 1) / STEPS;

  // steps of block n: first .. first + have - 1 of the sequence
  auto block = [&](int n, int& have) {
    const int b = back ? blocks - 1 - n : n;
    have = min(STEPS, steps - b * STEPS);
    return U.from + b * STEPS;
  };
  auto load_ab = [&](int n) {
    int have;
    const int row = (B.cu ? (int)U.row0 : 0) + block(n, have), w = B.cu ? 0 : (int)U.s;
    char* a = smem + (n & 1) * 2 * TA;
    if (elect_one()) {
      mbar_expect(&full_ab[n & 1], (OUT ? 2 : 1) * TA);
#pragma unroll
      for (int i = 0; i < NK; ++i) {
        if (OUT) tma_load(a + i * BOX, &J.a, i * 64, h / P.a.shared, row, w, &full_ab[n & 1]);
        tma_load(a + TA + i * BOX, &J.b, i * 64, h / P.b.shared, row, w, &full_ab[n & 1]);
      }
    }
    __syncwarp();
  };
  auto load_v = [&](int n) {
    int have;
    const int row = (B.cu ? (int)U.row0 : 0) + block(n, have), w = B.cu ? 0 : (int)U.s;
    if (elect_one()) {
      mbar_expect(&full_v, NV * BOX);
#pragma unroll
      for (int i = 0; i < NV; ++i) tma_load(tv + i * BOX, &J.v, i * 64, h / P.v.shared, row, w, &full_v);
    }
    __syncwarp();
  };
  if (warp == LOADS) {  // the first tiles are on their way while the rest is set up
    if (elect_one()) {
      mbar_init(&full_ab[0], 1), mbar_init(&full_ab[1], 1), mbar_init(&full_v, 1), mbar_init(&scores, 1), mbar_init(&met, 1);
      mbar_init(&updated, 1), mbar_init(&probs, 8), mbar_init(&summed, 1);
      mbar_init(&state, 8), mbar_init(&out_read[0], 8), mbar_init(&out_read[1], 8), mbar_init(&drained, 1);
      mbar_init(&keys[0], 8), mbar_init(&keys[1], 8);
      mbar_init_fence();
      gave_up = 0;
    }
    __syncwarp();
    if (blocks > 0) load_ab(0), load_v(0);
    if (blocks > 1) load_ab(1);
  }
  if (warp == PRODUCTS) tmem_alloc<512>(&tmem_slot);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t t_scores = tmem_slot, t_update = t_scores + 128, t_out = t_update + 64 * NK;  // two of out
  if (warp < 16) {  // while the first tiles are on their way
    const unsigned t = threadIdx.x;
    if (t <= STEPS) power[t] = fade(B.log_decay[h], t);
    else if (t - 256 < 32u) near[t - 256] = fade(B.log_decay[h], back ? t - 256 : 287 - t);
    else if (t - 320 < 63u) fan[t - 320] = fade(B.log_decay[h], abs((int)t - 351));
    asm volatile("bar.sync 3, 512;" ::: "memory");
  }
  if (warp >= 16) fewer_registers<FEW>();
  if (warp == LOADS) {  // ------------------------------------------------------------ loads
    int ab = min(blocks, 2), vv = min(blocks, 1);  // blocks loaded
    bool ok = true;
    for (int n = 0; n + 1 < blocks && ok; ++n) {
      if (!(ok = __all_sync(0xffffffffu, mbar_wait(OUT ? &summed : &updated, n & 1, &gave_up)))) break;
      load_v(n + 1), ++vv;
      if (n + 2 < blocks) load_ab(n + 2), ++ab;
    }
    // copies in flight end before the shared memory does: where a wait gave up, and otherwise these have long been awaited
    for (int n = max(ab - 2, 0); n < ab; ++n)
      for (uint32_t i = 0; i < POLLS && !mbar_try(&full_ab[n & 1], (n >> 1) & 1); ++i) {}
    for (uint32_t i = 0; vv > 0 && i < POLLS && !mbar_try(&full_v, (vv - 1) & 1); ++i) {}
  } else if (warp == PRODUCTS) {  // -------------------------------------------------- products
    constexpr uint32_t I_SCORES = instruction(BF16, false, false, 128, 128), I_INTER = instruction(BF16, false, false, 128, 64 * NV);
    constexpr uint32_t I_INTRA = instruction(BF16, false, true, 128, 64 * NV), I_UPDATE = instruction(BF16, true, true, 128, 64 * NK);
    const uint64_t d_v = operand(smem_addr(tv), BOX), d_sp = operand(smem_addr(sp), BOX), d_third = operand(smem_addr(third), BOX);
    bool ok = true;
    auto wait = [&](uint64_t* b, int n) {
      ok = ok && __all_sync(0xffffffffu, mbar_wait(b, n & 1, &gave_up));
      return ok;
    };
    // A B^T of block n, while the state is still on its way
    auto issue_scores = [&](int n) {
      if (!wait(&full_ab[n & 1], n >> 1)) return;
      fence_after();
      const uint64_t d_a = operand(smem_addr(smem + (n & 1) * 2 * TA), BOX);
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < 4 * NK; ++k) {
          const uint64_t at = d_a + (k / 4) * (BOX >> 4) + (k % 4) * 2;
          mma(t_scores, at, at + (TA >> 4), I_SCORES, k > 0);
        }
        mma_commit(&scores);
      }
      __syncwarp();
    };
    if (OUT && blocks > 0) issue_scores(0);
    for (int n = 0; n < blocks && ok; ++n) {
      const uint64_t d_a = operand(smem_addr(smem + (n & 1) * 2 * TA), BOX), d_b = d_a + (TA >> 4);
      if (OUT) {
        if (!wait(&state, n) || (n > 1 && !wait(&out_read[n & 1], (n >> 1) - 1))) break;
        fence_after();
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < 4 * NK; ++k)
            mma(t_out + (n & 1) * 64 * NV, d_a + (k / 4) * (BOX >> 4) + (k % 4) * 2, d_sp + (k / 4) * (NV * BOX / 2 >> 4) + (k % 4) * 2, I_INTER, k > 0);
          mma_commit(&met);
        }
        __syncwarp();
      } else if (!wait(&full_ab[n & 1], n >> 1)) {
        break;
      }
      if (!wait(&full_v, n)) break;
      for (int q = 0; q < 2 && wait(&keys[q], n); ++q) {  // 64 rows of the faded B at a time
        fence_after();
        if (elect_one()) {
#pragma unroll
          for (int p = 0; p < PARTS; ++p) {
            const uint64_t d = (p == 0 ? d_b : p == 2 || !BF16 ? d_a : d_third) + q * (8192 >> 4);
#pragma unroll
            for (int k = 0; k < 4; ++k) mma(t_update, d_v + q * (8192 >> 4) + k * (2048 >> 4), d + k * (2048 >> 4), I_UPDATE, q > 0 || p > 0 || k > 0);
          }
          if (q == 1) mma_commit(&updated);
        }
        __syncwarp();
      }
      if (!ok) break;
      if (!OUT) continue;
      if (!wait(&probs, n)) break;
      fence_after();
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          mma_tmem(t_out + (n & 1) * 64 * NV, t_scores + k / 4 * 64 + k % 4 * 8, d_v + k * (2048 >> 4), I_INTRA, true);
        mma_commit(&summed);
      }
      __syncwarp();
      // P lies where the next scores go
      if (n + 1 < blocks && wait(&summed, n)) issue_scores(n + 1);
    }
    if (!ok) {
      if (elect_one()) mma_commit(&drained);
      __syncwarp();
      for (uint32_t i = 0; i < POLLS && !mbar_try(&drained, 0); ++i) {}
    }
  } else if (warp < 8) {  // ------------------------------------------------- P, and out
    fewer_registers<SOME>();
    if (OUT) {
      const int quarter = warp % 4, side = warp / 4, i = quarter * 32 + lane;  // row of the block
      const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
      const float both = P.so * P.sb;
      // rows whose pieces of 16 places (8, of float32) are sectors of 32 bytes, which store8 wants on such a border
      const bool sectors = (reinterpret_cast<uintptr_t>(P.out) & 31) == 0, eights = P.V % 8 == 0, whole_sectors = P.V % 16 == 0 && sectors;
      // 32 products of this thread's row, c of four, faded and times `up`; `have`: places of the block
      auto products = [&](int c, int have, float up, float2 (&v)[16]) {
        tmem_load16(t_scores + lanes + c * 32, reinterpret_cast<float*>(v));
        tmem_load16(t_scores + lanes + c * 32 + 16, reinterpret_cast<float*>(v + 8));
        const int apart = 32 * (back ? c - quarter : quarter - c);
        if (apart == 0) {
          const float* p = fan + 31 + lane;
          const uint32_t in = back ? (c * 32 + 32 > have ? have > c * 32 ? (1u << (have - c * 32)) - 1 : 0u : ~0u) & ~0u << lane : (2u << lane) - 1;
          tmem_load_wait();
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float2 w = mul2(v[e], mul2(make_float2(p[-2 * e], p[-2 * e - 1]), twice(up)));
            v[e] = make_float2(in & 1u << 2 * e ? w.x : 0.0f, in & 2u << 2 * e ? w.y : 0.0f);
          }
        } else {
          const float2 edge = twice(power[apart - (back ? lane : 31 - lane)] * up);
          tmem_load_wait();
#pragma unroll
          for (int e = 0; e < 16; e += 2) {
            const float4 f = *reinterpret_cast<const float4*>(&near[2 * e]);
            v[e] = mul2(v[e], mul2(edge, make_float2(f.x, f.y))), v[e + 1] = mul2(v[e + 1], mul2(edge, make_float2(f.z, f.w)));
          }
          if (back && c * 32 + 32 > have) {
#pragma unroll
            for (int e = 0; e < 16; ++e) v[e] = make_float2(c * 32 + 2 * e < have ? v[e].x : 0.0f, c * 32 + 2 * e + 1 < have ? v[e].y : 0.0f);
          }
        }
      };
      for (int n = 0; n < blocks; ++n) {
        int have;
        const int first = block(n, have);
        bool ok = mbar_wait(&scores, n & 1, &gave_up);
        __syncwarp();
        fence_after();
        float down = 1.0f, up = both;
        if (!BF16) {
          // a row with an infinity is one in any case, and out has no use for what 2^60 leaves below 1
          float top = 0.0f;
#pragma unroll 1
          for (int c = 2 * side; c < 2 * side + 2; ++c) {
            if (back ? c < quarter : c > quarter) continue;
            float2 v[16];
            products(c, have, both, v);
#pragma unroll
            for (int e = 0; e < 16; ++e) top = fmaxf(top, fmaxf(fabsf(v[e].x), fabsf(v[e].y)));
          }
          tops[side][i] = top;
          asm volatile("bar.sync 1, 256;" ::: "memory");
          up = scale_up(fmaxf(fmaxf(tops[0][i], tops[1][i]), 0x1p-46f), down) * both;
        }
#pragma unroll 1
        for (int c = 2 * side; c < 2 * side + 2; ++c) {
          uint32_t w[16] = {};
          if (back ? c >= quarter : c <= quarter) {
            float2 v[16];
            products(c, have, up, v);
#pragma unroll
            for (int e = 0; e < 16; ++e) w[e] = pack2<BF16>(v[e].x, v[e].y);
          }
          tmem_store16(t_scores + lanes + side * 64 + (c & 1) * 16, w);  // over scores that this warp has read
        }
        // A X, faded, is what P V is added to
        const float inter = P.so * power[i < have ? (back ? have - 1 - i : i + 1) : 0] * (BF16 ? 1.0f : 1.0f / down);
        const uint32_t t_mine = t_out + (n & 1) * 64 * NV + side * 32 * NV + lanes;
        ok = mbar_wait(&met, n & 1, &gave_up) && ok;
        __syncwarp();
        fence_after();
#pragma unroll 1
        for (int c = 0; c < 32 * NV; c += 16) {
          float2 a[8];
          tmem_load16(t_mine + c, reinterpret_cast<float*>(a));
          tmem_load_wait();
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            if (!BF16) a[e] = mul2(a[e], *reinterpret_cast<const float2*>(&place_scale[n & 1][side * 32 * NV + c + 2 * e]));
            a[e] = mul2(a[e], twice(inter));
          }
          tmem_store16(t_mine + c, reinterpret_cast<const uint32_t*>(a));
        }
        tmem_store_wait();
        fence_before();
        arrive_warp(&probs);

        ok = mbar_wait(&summed, n & 1, &gave_up) && ok;
        __syncwarp();
        fence_after();
        const bool there = i < have;
        const int64_t at = ((U.row0 + first + i) * B.H + h) * (int64_t)P.V;
#pragma unroll 1
        for (int k = 0; k < 2 * NV; ++k) {  // 16 places at a time
          const int c = (side * 2 * NV + k) * 16;
          float2 v[8];
          tmem_load16(t_mine + k * 16, reinterpret_cast<float*>(v));
          tmem_load_wait();
          if (k == 2 * NV - 1) {
            fence_before();
            arrive_warp(&out_read[n & 1]);
          }
          if (!BF16) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = mul2(v[e], twice(down));
          }
          if (!ok) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = twice(__int_as_float(0x7fffffff));
          }
          if (!there || c >= P.V) continue;
          // a row to a thread, whole sectors at a time
          uint32_t w[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) w[e] = pack2<BF16>(v[e].x, v[e].y);
          if (P.wide && eights && sectors) {
            float* to = static_cast<float*>(P.out) + at + c;
            store8(to, reinterpret_cast<uint32_t*>(v));
            if (c + 8 < P.V) store8(to + 8, reinterpret_cast<uint32_t*>(v + 4));
          } else if (P.wide) {
            float* to = static_cast<float*>(P.out) + at + c;
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (c + e < P.V) to[e] = e % 2 ? v[e / 2].y : v[e / 2].x;
          } else if (whole_sectors) {
            store8(static_cast<uint16_t*>(P.out) + at + c, w);
          } else if (eights) {
            uint16_t* to = static_cast<uint16_t*>(P.out) + at + c;
            *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
            if (c + 8 < P.V) *reinterpret_cast<uint4*>(to + 8) = make_uint4(w[4], w[5], w[6], w[7]);
          } else {
            uint16_t* to = static_cast<uint16_t*>(P.out) + at + c;
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (c + e < P.V) to[e] = (uint16_t)(w[e / 2] >> (e % 2 * 16));
          }
        }
      }
    }
  } else if (warp < 16) {  // --------------------------------- the faded B, and the state
    more_registers<MANY>();
    const int r = threadIdx.x & 127, side = (warp - 8) / 4;  // row of the block; place of v
    const int k0 = side * 32 * NK;                           // entries k0 .. along b
    const uint32_t lanes = (uint32_t)(warp % 4 * 32) << 16;
    const bool mine = r < P.V && r < 64 * NV;
    const int64_t size = (int64_t)P.K * P.V;
    float x[32 * NK];
#pragma unroll
    for (int k = 0; k < 32 * NK; ++k) x[k] = 0.0f;
    const float* const enters = cut ? P.made : P.state;
    if (OUT && enters && mine) {
      const float* p = enters + ((cut ? U.unit : U.s) * B.H + h) * size + k0 * P.sr + r * P.sc;
#pragma unroll
      for (int k = 0; k < 32 * NK; ++k)
        if (k0 + k < P.K) x[k] = p[k * P.sr];
    }
    bool ok = true;
    auto put_state = [&](int n) {  // as an operand of block n: row = place of v
      float up = 1.0f;
      if (!BF16) {
        float top = 0.0f, down;
#pragma unroll
        for (int k = 0; k < 32 * NK; ++k) top = fmaxf(top, fabsf(x[k]));
        place_top[side][r] = top;
        asm volatile("bar.sync 2, 256;" ::: "memory");
        up = scale_up(fmaxf(place_top[0][r], place_top[1][r]), down);
        place_scale[n & 1][r] = down;
      }
      if (r < 64 * NV) {
#pragma unroll
        for (int c = 0; c < 4 * NK; ++c) {
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = pack2<BF16>(x[c * 8 + 2 * e] * up, x[c * 8 + 2 * e + 1] * up);
          *reinterpret_cast<uint4*>(chunk_at(sp, 64 * NV, r, side * 4 * NK + c)) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
      fence_async();
      fence_before();
      arrive_warp(&state);
    };
    if (OUT && blocks > 0) put_state(0);
    // The faded B of a block is made 64 rows at a time, 2 NK chunks of a row to a thread, the first 64 while the products of
    // the block before run.
    const int row = (warp & 1) * 32 + lane, c0 = (warp - 8) / 2 * 2 * NK;
    float down = 1.0f, next_down = 1.0f, up = P.sb;
    uint32_t early[PARTS][8 * NK];
    // the parts of chunk c of row `at` of B, whose factor is f; nothing of rows that are not the sequence's, whatever they hold
    auto split = [&](const char* at, bool in, float2 f, uint32_t* w0, uint32_t* w1, uint32_t* w2) {
      const uint4 x4 = in ? *reinterpret_cast<const uint4*>(at) : make_uint4(0, 0, 0, 0);
      const uint32_t x[4] = {x4.x, x4.y, x4.z, x4.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float2 v = mul2(unpack2<BF16>(x[e]), f);
        if (BF16) {  // the upper halves of what is left, cut off: each part takes 7 bits at least, and the last is rounded to 8 more
          const uint32_t ux = __float_as_uint(v.x), uy = __float_as_uint(v.y);
          w0[e] = __byte_perm(ux, uy, 0x7632);
          v = fma2(make_float2(__uint_as_float(ux & 0xffff0000u), __uint_as_float(uy & 0xffff0000u)), twice(-1.0f), v);
          const uint32_t sx = __float_as_uint(v.x), sy = __float_as_uint(v.y);
          w1[e] = __byte_perm(sx, sy, 0x7632);
          v = fma2(make_float2(__uint_as_float(sx & 0xffff0000u), __uint_as_float(sy & 0xffff0000u)), twice(-1.0f), v);
          w2[e] = pack2<BF16>(v.x, v.y);
        } else {
          w0[e] = pack2<BF16>(v.x, v.y);
          v = fma2(unpack2<BF16>(w0[e]), twice(-1.0f), v);
          w1[e] = pack2<BF16>(v.x, v.y);
        }
      }
    };
    auto factor = [&](int i, int have) { return twice(i < have ? power[back ? i + 1 : have - 1 - i] * up : 0.0f); };
    auto begin = [&](int n) {  // the first 64 rows of block n
      int have;
      block(n, have);
      const char* const tb = smem + (n & 1) * 2 * TA + TA;
      ok = mbar_wait(&full_ab[n & 1], (n >> 1) & 1, &gave_up) && ok;
      __syncwarp();
      if (!BF16) {
        float top = 0.0f;
        up = P.sb;
        if (r < have) {
          const float f = factor(r, have).x;
#pragma unroll
          for (int c = 0; c < 4 * NK; ++c) {
            const uint4 q = *reinterpret_cast<const uint4*>(chunk_at(const_cast<char*>(tb), 128, r, side * 4 * NK + c));
            const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 v = unpack2<BF16>(w[e]);
              top = finite_max(finite_max(top, v.x * f), v.y * f);
            }
          }
        }
        const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
        if (lane == 0) warp_top[n & 1][warp - 8] = __uint_as_float(bits);
        asm volatile("bar.sync 2, 256;" ::: "memory");
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, warp_top[n & 1][i]);
        up *= scale_up(top, next_down);
      }
      const float2 f = factor(row, have);
#pragma unroll
      for (int c = 0; c < 2 * NK; ++c)
        split(chunk_at(const_cast<char*>(tb), 128, row, c0 + c), row < have, f, &early[0][4 * c], &early[1][4 * c], &early[PARTS - 1][4 * c]);
    };
    auto put = [&](char* tile, int i, int c, const uint32_t* w) {
      *reinterpret_cast<uint4*>(chunk_at(tile, 128, i, c0 + c)) = make_uint4(w[0], w[1], w[2], w[3]);
    };
    if (blocks > 0) begin(0);
    for (int n = 0; n < blocks; ++n) {
      int have;
      block(n, have);
      char* const ta = smem + (n & 1) * 2 * TA;
      char* const tb = ta + TA;
      down = next_down;
      if (OUT) ok = mbar_wait(&scores, n & 1, &gave_up) && ok;  // B has been read
      __syncwarp();
#pragma unroll
      for (int c = 0; c < 2 * NK; ++c) {
        put(tb, row, c, &early[0][4 * c]);
        if (BF16) put(third, row, c, &early[1][4 * c]);
      }
      if (B.cu && have < STEPS) {  // rows of the next sequence in v
        ok = mbar_wait(&full_v, n & 1, &gave_up) && ok;
#pragma unroll
        for (int c = 0; c < 4 * NV; ++c)
          if (r >= have) *reinterpret_cast<uint4*>(chunk_at(tv, 128, r, side * 4 * NV + c)) = make_uint4(0, 0, 0, 0);
      }
      const float2 f = factor(row + 64, have);
      uint32_t rest[8 * NK];
#pragma unroll
      for (int c = 0; c < 2 * NK; ++c) {
        uint32_t w0[4], w1[4];
        split(chunk_at(tb, 128, row + 64, c0 + c), row + 64 < have, f, w0, BF16 ? w1 : &rest[4 * c], &rest[4 * c]);
        put(tb, row + 64, c, w0);
        if (BF16) put(third, row + 64, c, w1);
        if (c == NK - 1) {
          if (OUT) ok = mbar_wait(&met, n & 1, &gave_up) && ok;  // A has been read, and the state
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 2 * NK; ++i) put(ta, row, i, &early[PARTS - 1][4 * i]);
          fence_async();
          fence_before();
          arrive_warp(&keys[0]);
        }
      }
#pragma unroll
      for (int c = 0; c < 2 * NK; ++c) put(ta, row + 64, c, &rest[4 * c]);
      fence_async();
      fence_before();
      arrive_warp(&keys[1]);
      if (n + 1 < blocks) begin(n + 1);

      const float whole = power[have];
      ok = mbar_wait(&updated, n & 1, &gave_up) && ok;
      __syncwarp();
      fence_after();
#pragma unroll
      for (int c = 0; c < 32 * NK; c += 16) {
        float u[16];
        tmem_load16(t_update + lanes + k0 + c, u);
        tmem_load_wait();
#pragma unroll
        for (int e = 0; e < 16; ++e) x[c + e] = fmaf(whole, x[c + e], BF16 ? u[e] : u[e] * down);
      }
      fence_before();
      if (OUT && n + 1 < blocks) put_state(n + 1);
    }
    float* to = OUT ? (P.last && U.ends(back) ? P.last + (U.s * B.H + h) * size : nullptr) : P.made + (U.unit * B.H + h) * size;
    if (to && mine) {
#pragma unroll
      for (int k = 0; k < 32 * NK; ++k)
        if (k0 + k < P.K) to[(k0 + k) * P.sr + r * P.sc] = ok ? x[k] : __int_as_float(0x7fffffff);
    }
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == PRODUCTS) tmem_free<512>(tmem_slot);
}

template <bool BF16, int NK, int NV, bool OUT>
cudaError_t launch(const Jobs& jobs, const Batch& B, int count, cudaStream_t st) {
  constexpr int smem = smem_bytes(NK, NV, BF16);
  if (cudaError_t e = allow_smem<blocks_tc_kernel<BF16, NK, NV, OUT>>(smem)) return e;
  blocks_tc_kernel<BF16, NK, NV, OUT><<<(unsigned)(unit_grid(B, !OUT) * B.H * count), THREADS, smem, st>>>(jobs, B, count);
  return cudaSuccess;
}
template <bool BF16, int NK, int NV>
cudaError_t launch(const Jobs& jobs, const Batch& B, int count, bool first, cudaStream_t st) {
  return first ? launch<BF16, NK, NV, false>(jobs, B, count, st) : launch<BF16, NK, NV, true>(jobs, B, count, st);
}
template <bool BF16>
cudaError_t launch(const Jobs& jobs, const Batch& B, int nk, int nv, int count, bool first, cudaStream_t st) {
  if (nk == 1 && nv == 1) return launch<BF16, 1, 1>(jobs, B, count, first, st);
  if (nk == 1) return launch<BF16, 1, 2>(jobs, B, count, first, st);
  if (nv == 1) return launch<BF16, 2, 1>(jobs, B, count, first, st);
  return launch<BF16, 2, 2>(jobs, B, count, first, st);
}

bool map_stream(CUtensorMap* map, const Batch& B, const Stream& x, int D, bool bf16) {
  const int64_t sizes[4] = {D, B.H / x.shared, B.T, B.cu ? 1 : B.S}, strides[3] = {x.head, x.row, x.seq};
  return make_map4(map, x.p, sizes, strides, STEPS, bf16);
}

}  // namespace

namespace la {

int tensor_passes(const Batch& B, const Pass* passes, int count, bool first, bool bf16, cudaStream_t st) {
  // passes whose tiles have one shape run side by side in one launch
  bool done[MAX_PASSES] = {};
  for (int i = 0; i < count; ++i) {
    if (done[i]) continue;
    const int nk = passes[i].K > 64 ? 2 : 1, nv = passes[i].V > 64 ? 2 : 1;
    Jobs jobs;
    int n = 0;
    for (int j = i; j < count; ++j) {
      const Pass& p = passes[j];
      if (done[j] || (p.K > 64 ? 2 : 1) != nk || (p.V > 64 ? 2 : 1) != nv) continue;
      done[j] = true;
      Job& job = jobs.job[n++];
      job.pass = p;
      if (!map_stream(&job.a, B, p.a, p.K, bf16) || !map_stream(&job.b, B, p.b, p.K, bf16) || !map_stream(&job.v, B, p.v, p.V, bf16))
        return set_error(CSN_ERR_CUDA, "csn_linear_attention: tensor map");
    }
    for (int j = n; j < MAX_PASSES; ++j) jobs.job[j] = jobs.job[0];
    KernelTimer kt(first ? "linear_attention_first" : "linear_attention", st);
    const cudaError_t e = bf16 ? launch<true>(jobs, B, nk, nv, n, first, st) : launch<false>(jobs, B, nk, nv, n, first, st);
    if (e != cudaSuccess) return set_cuda_error(e, "csn_linear_attention: shared memory");
  }
  return CSN_OK;
}

}  // namespace la
}  // namespace csn

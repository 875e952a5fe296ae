// csn_tc.cuh -- asynchronous and tensor-core building blocks for sm_100a: mbarriers, TMA tile loads, tensor memory and tcgen05.mma,
// as inline PTX, and the tensor maps on the host.
//
// Every wait is bounded.  A wait that runs out sets the CTA's `gave_up` word; every other wait of the CTA then ends
// too, the CTA drains what it has in flight, frees its tensor memory and returns, and its epilogue writes NaN in
// place of results.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace csn {
namespace tc {

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

// One lane of a converged warp, for the instructions that one thread issues.  The warp stays together around them, so
// that what they take (descriptors, addresses) is uniform and needs no moving: a loop of one lane alone bounded
// every tile (R2048 C4096 F8192 forward 196 us against 174).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

__device__ __forceinline__ void mbar_init(uint64_t* b, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(b)), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_init_fence() {
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}
__device__ __forceinline__ void mbar_expect(uint64_t* b, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_addr(b)), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint64_t* b, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_addr(b)), "r"(parity)
      : "memory");
  return ok != 0;
}

// address in CTA `rank` of the cluster
__device__ __forceinline__ uint32_t peer_addr(const void* p, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_addr(p)), "r"(rank));
  return a;
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Waits for the phase `parity` of b to end.  A wait can last as long as a tile: a k block takes 0.4 us of the tensor cores, or
// 0.7 where nothing of it is in L2 and every SM reads, and the largest tile that is accepted has 65536, 24 to 49 ms.  A
// poll takes tens of nanoseconds at least, so the limit is a second and more.  (It is a constant: as an argument of the
// kernel it cost few_rows_kernel up to 6 %.)
constexpr uint32_t POLLS = 1u << 26;
__device__ __forceinline__ bool mbar_wait(uint64_t* b, uint32_t parity, volatile uint32_t* gave_up) {
  for (uint32_t i = 0; i < POLLS; ++i) {
    if (mbar_try(b, parity)) return true;
    if ((i & 1023) == 1023 && *gave_up) return false;
  }
  *gave_up = 1;
  return false;
}

// ------------------------------------------------------------------------- TMA
// the box of `map` at (x, y) to shared memory, counted on b
__device__ __forceinline__ void tma_load(void* dst, const CUtensorMap* map, int x, int y, uint64_t* b) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          smem_addr(dst)),
      "l"(map), "r"(x), "r"(y), "r"(smem_addr(b))
      : "memory");
}

// the same into this CTA's shared memory, counted on a barrier of either CTA of a pair
__device__ __forceinline__ void tma_load_pair(void* dst, const CUtensorMap* map, int x, int y, uint32_t barrier) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], "
      "[%4];" ::"r"(smem_addr(dst)),
      "l"(map), "r"(x), "r"(y), "r"(barrier)
      : "memory");
}

// ---------------------------------------------------------------- tensor memory
// the _pair forms: both CTAs of a pair call them
template <int COLS>
__device__ __forceinline__ void tmem_alloc_pair(uint32_t* slot) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(slot)), "n"(COLS)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
}
template <int COLS>
__device__ __forceinline__ void tmem_free_pair(uint32_t base) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "n"(COLS));
}
template <int COLS>
__device__ __forceinline__ void tmem_alloc(uint32_t* slot) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(slot)), "n"(COLS)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
template <int COLS>
__device__ __forceinline__ void tmem_free(uint32_t base) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "n"(COLS));
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// 16 columns of this warp's 32 lanes: thread = lane, register = column
__device__ __forceinline__ void tmem_load16(uint32_t addr, float* v) {
  uint32_t r[16];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
                 "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(addr));
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_load_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// -------------------------------------------------------------------------- MMA
// Shared-memory operand of 16-bit elements in 128-byte swizzled rows (what a TMA box of 64 elements a row leaves).
//   K-major: a row is 64 neighbouring k of one m (n); 8 rows make a 1024-byte group (SBO), a k step of 16 is 32 bytes.
//   MN-major: a row is 64 neighbouring m of one k; 8 rows of k make a 1024-byte group (SBO), the next 64 m are `lbo`
//   bytes on, a k step of 16 is 2048 bytes.
__device__ __forceinline__ uint64_t operand(uint32_t addr, uint32_t lbo) {
  return (uint64_t)((addr & 0x3ffff) >> 4) | (uint64_t)((lbo & 0x3ffff) >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 |
         (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

// kind::f16 instruction: float32 accumulators, both operands bf16 or both fp16, each K-major or MN-major, M x N
__host__ __device__ constexpr uint32_t instruction(bool bf16, bool a_mn, bool b_mn, int m, int n) {
  return 1u << 4 | (bf16 ? 1u : 0u) << 7 | (bf16 ? 1u : 0u) << 10 | (a_mn ? 1u : 0u) << 15 | (b_mn ? 1u : 0u) << 16 |
         (uint32_t)(n >> 3) << 17 | (uint32_t)(m >> 4) << 24;
}

__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
      : "memory");
}
// b counts one arrival when every MMA issued so far by this thread is done
__device__ __forceinline__ void mma_commit(uint64_t* b) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(b))
               : "memory");
}

// A pair's product: each CTA holds half of A's m rows and half of B's n rows at the same places of its shared memory,
// and gets its m rows of the result.  One thread of CTA 0 issues it for both.
__device__ __forceinline__ void mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
      : "memory");
}
// the barrier at b's place in both CTAs counts one arrival when every pair product issued so far is done
__device__ __forceinline__ void mma_commit_pair(uint64_t* b) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                   smem_addr(b)),
               "h"((uint16_t)3)
               : "memory");
}

// ------------------------------------------------------------------------- host
// Tensor map of a row-major 16-bit matrix [rows, cols] with `ld` elements a row (ld % 8 == 0, p 16-byte aligned),
// read in boxes of 64 columns x box_rows rows with 128-byte swizzle; what lies outside reads as 0.
bool make_map(CUtensorMap* map, const void* p, int64_t rows, int64_t cols, int64_t ld, int box_rows, bool bf16);
int sm_count();

}  // namespace tc
}  // namespace csn

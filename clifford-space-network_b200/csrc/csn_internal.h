// csn_internal.h -- error reporting shared by the library's translation units.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "../../include/csn_b200.h"

namespace csn {

// Record `msg` as this thread's last error and return `code`.
int set_error(int code, const char* msg);
int set_cuda_error(cudaError_t e, const char* where);
// cudaGetLastError() after a batch of launches.
int check_launch(const char* where);

}  // namespace csn

namespace csn {

// Allows KERNEL `bytes` of dynamic shared memory, once on each device (a call of the runtime costs as much as a launch).
template <auto KERNEL>
cudaError_t allow_smem(int bytes) {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (done.load() & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(reinterpret_cast<const void*>(KERNEL), cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.fetch_or(bit);
  return e;
}

// Optional per-kernel timing (off by default).  When enabled with
// csn_timing_enable(1), every library launch wrapped in a KernelTimer records a pair
// of CUDA events on its own stream; csn_timing_read() sums the elapsed times.
bool timing_on();
void timing_push(const char* name, cudaEvent_t start, cudaEvent_t stop);

struct KernelTimer {
  const char* name;
  cudaStream_t st;
  cudaEvent_t e0 = nullptr, e1 = nullptr;
  KernelTimer(const char* n, cudaStream_t s) : name(n), st(s) {
    if (timing_on() && cudaEventCreate(&e0) == cudaSuccess && cudaEventCreate(&e1) == cudaSuccess)
      cudaEventRecord(e0, st);
    else
      e0 = e1 = nullptr;
  }
  ~KernelTimer() {
    if (e0) {
      cudaEventRecord(e1, st);
      timing_push(name, e0, e1);
    }
  }
};

}  // namespace csn

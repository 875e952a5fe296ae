// csn_tc.cu -- host side of the tensor-core kernels: tensor maps through the driver's encoder.
#include "csn_tc.cuh"

#include <atomic>

namespace csn {
namespace tc {
namespace {
using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                            const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                            CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

Encode encoder() {
  static std::atomic<Encode> found{nullptr};
  Encode e = found.load();
  if (!e) {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult how;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &how) != cudaSuccess ||
        how != cudaDriverEntryPointSuccess)
      return nullptr;
    e = reinterpret_cast<Encode>(fn);
    found.store(e);
  }
  return e;
}
}  // namespace

bool make_map4(CUtensorMap* map, const void* p, const int64_t* sizes, const int64_t* strides, int box, bool bf16) {
  Encode e = encoder();
  int dev = 0;
  if (!e || cudaGetDevice(&dev) != cudaSuccess || cudaSetDevice(dev) != cudaSuccess) return false;
  cuuint64_t dims[4], steps[3];
  for (int i = 0; i < 4; ++i) dims[i] = (cuuint64_t)sizes[i];
  for (int i = 0; i < 3; ++i) steps[i] = sizes[i + 1] > 1 ? (cuuint64_t)strides[i] * 2 : 16;
  const cuuint32_t boxes[4] = {64, 1, (cuuint32_t)box, 1}, step[4] = {1, 1, 1, 1};
  return e(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(p), dims, steps,
           boxes, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool make_map(CUtensorMap* map, const void* p, int64_t rows, int64_t cols, int64_t ld, int box_rows, bool bf16) {
  Encode e = encoder();
  int dev = 0;
  // the encoder needs a context on this thread, and a thread that has launched nothing yet has none
  if (!e || cudaGetDevice(&dev) != cudaSuccess || cudaSetDevice(dev) != cudaSuccess) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld * 2};
  const cuuint32_t box[2] = {64, (cuuint32_t)box_rows}, step[2] = {1, 1};
  return e(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(p), dims,
           strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int sm_count() {
  static std::atomic<int> cached[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  int n = cached[dev].load();
  if (!n) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
    cached[dev].store(n);
  }
  return n;
}

}  // namespace tc
}  // namespace csn

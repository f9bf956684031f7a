// Host side of the 8-bit product (fp8_core.cuh): tensor maps, choice of the tile, launch.
#include <cuda.h>
#include <cuda_runtime.h>
#include <string.h>

#include <atomic>

#include "../../core/core.h"
#include "fp8_core.cuh"
#include "gemm_host.h"
#include "mccl_ops.h"

using namespace mccl;
using namespace mccl::fp8;

namespace {

// Bytes [outer][rows][cols] (outer 0: a matrix), rows `ld` apart; box = 128 columns x boxRows.  Elements outside read as zero.
mcclResult_t mapOf(CUtensorMap* map, const void* base, uint64_t outer, uint64_t rows, uint64_t cols, uint64_t ld, uint32_t boxRows) {
  static gemm::EncodeTiledFn fn = gemm::encodeTiled();
  if (fn == nullptr) MCCLFAIL(mcclSystemError);
  const cuuint64_t dims[3] = {cols, rows, outer};
  const cuuint64_t strides[2] = {ld, rows * ld};
  const cuuint32_t box[3] = {kBlock, boxRows, 1}, elemStrides[3] = {1, 1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, outer ? 3 : 2, const_cast<void*>(base), dims, strides, box, elemStrides,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    MCCL_WARN("cuTensorMapEncodeTiled failed with %d (base %p, %llu x %llu x %llu bytes, row pitch %llu)", (int)r, base, (unsigned long long)outer,
              (unsigned long long)rows, (unsigned long long)cols, (unsigned long long)ld);
    return mcclInvalidArgument;
  }
  return mcclSuccess;
}

template <int BN>
mcclResult_t launchAs(const Args& a, int dev, int grid, cudaStream_t s) {
  auto* kernel = fp8Kernel<BN>;
  static std::atomic<uint64_t> prepared{0};                // a bit per device: the attribute stays with the function
  if (!(prepared.load(std::memory_order_relaxed) >> (dev & 63) & 1)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<BN>::TOTAL) != cudaSuccess) { cudaGetLastError(); return mcclSystemError; }
    prepared.fetch_or(1ull << (dev & 63));
  }
  kernel<<<grid, kThreads, Smem<BN>::TOTAL, s>>>(a);
  return cudaGetLastError() == cudaSuccess ? mcclSuccess : mcclSystemError;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace

extern "C" {

mcclResult_t mcclFp8Gemm(const void* x, int64_t ldx, const void* xScale, int64_t ldxScale, const void* w, const void* wScale, int64_t ldwScale, void* y,
                         const void* ends, int ends64, int groups, int64_t rows, int N, int K, mcclStream_t stream) {
  const int kb = (K + kBlock - 1) / kBlock;
  if (groups <= 0 || groups > grouped::kMaxGroups || (ends == nullptr && groups != 1) || rows < 0 || rows > INT32_MAX - 256 || N <= 0 || K <= 0 ||
      N > INT32_MAX - 256 || K > INT32_MAX - 256 || N % 8 || K % 16) return mcclInvalidArgument;
  if (rows == 0) return mcclSuccess;
  if (!x || !xScale || !w || !wScale || !y || !aligned16(x) || !aligned16(w) || !aligned16(y) || ldx < K || ldx % 16 || ldxScale < kb || ldxScale % 4 ||
      ldwScale < kb || ldwScale % 4 || ((reinterpret_cast<uintptr_t>(xScale) | reinterpret_cast<uintptr_t>(wScale)) & 3u)) return mcclInvalidArgument;
  int dev = 0;
  cudaGetDevice(&dev);
  cudaSetDevice(dev);                                      // binds the context to this thread, for the driver's encoder
  const int64_t rowTiles = ends == nullptr ? (rows + BM - 1) / BM : rows / BM + (rows < groups ? rows : groups);
  const int sms = gemm::gemmSmCount(), bn = N > 128 && rowTiles * ((N + 255) / 256) >= sms ? 256 : 128;
  const int64_t tiles = rowTiles * ((N + bn - 1) / bn);
  if (tiles > INT32_MAX) return mcclInvalidArgument;
  Args a;
  memset(&a, 0, sizeof(a));
  MCCLCHECK(mapOf(&a.mapA, x, 0, rows, K, ldx, BM));
  MCCLCHECK(mapOf(&a.mapB, w, groups, N, K, K, bn));
  a.sx = static_cast<const uint8_t*>(xScale);
  a.sw = static_cast<const uint8_t*>(wScale);
  a.ldsx = ldxScale; a.ldsw = ldwScale;
  a.ends = ends; a.ends64 = ends64; a.groups = groups;
  a.rows = (int)rows; a.N = N; a.K = K;
  a.out = static_cast<__nv_bfloat16*>(y);
  a.errFlag = gemm::gemmErrFlag(dev);
  if (a.errFlag == nullptr) return mcclSystemError;
  a.budgetNs = 2000000000ull;
  const int grid = (int)(tiles < sms ? tiles : sms);
  return bn == 256 ? launchAs<256>(a, dev, grid, reinterpret_cast<cudaStream_t>(stream)) : launchAs<128>(a, dev, grid, reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"

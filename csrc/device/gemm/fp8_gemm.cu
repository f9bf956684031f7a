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

template <int BN>
mcclResult_t launchAs(const Args& a, int dev, int grid, bool behind, cudaStream_t s) {
  auto* kernel = fp8Kernel<BN>;
  static std::atomic<uint64_t> prepared{0};                // a bit per device: the attribute stays with the function
  if (!(prepared.load(std::memory_order_relaxed) >> (dev & 63) & 1)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<BN>::TOTAL) != cudaSuccess) { cudaGetLastError(); return mcclSystemError; }
    prepared.fetch_or(1ull << (dev & 63));
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Smem<BN>::TOTAL;
  cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = behind ? 1 : 0;
  if (cudaLaunchKernelEx(&cfg, kernel, a) != cudaSuccess) { cudaGetLastError(); return mcclSystemError; }
  return mcclSuccess;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// x: e4m3 with its scales; `behind`: made by the kernel launched last on the stream, which lets this one start before that has ended.
mcclResult_t product(const void* x, int64_t ldx, const void* xScale, int64_t ldxScale, const void* w, int64_t ldw, const void* wScale, int64_t ldwScale, void* y,
                     const void* ends, int ends64, int groups, int64_t rows, int N, int K, bool behind, mcclStream_t stream) {
  const int kb = (K + kBlock - 1) / kBlock;
  if (groups <= 0 || groups > grouped::kMaxGroups || (ends == nullptr && groups != 1) || rows < 0 || rows > INT32_MAX - 256 || N <= 0 || K <= 0 ||
      N > INT32_MAX - 256 || K > INT32_MAX - 256 || N % 8 || K % 16) return mcclInvalidArgument;
  if (rows == 0) return mcclSuccess;
  if (!x || !xScale || !w || !wScale || !y || !aligned16(x) || !aligned16(w) || !aligned16(y) || ldx < K || ldx % 16 || ldw < K || ldw % 16 || ldxScale < kb || ldxScale % 4 ||
      ldwScale < kb || ldwScale % 4 || ((reinterpret_cast<uintptr_t>(xScale) | reinterpret_cast<uintptr_t>(wScale)) & 3u)) return mcclInvalidArgument;
  int dev = 0;
  cudaGetDevice(&dev);
  cudaSetDevice(dev);                                      // binds the context to this thread, for the driver's encoder
  if (gemm::thinWanted(rows, ends != nullptr, groups, N, K))
    return gemm::thinGemm(gemm::ThinCall{x, w, ldx, ldw, true, xScale, wScale, ldxScale, ldwScale, y, ends, ends64, groups, rows, N, K, behind}, dev, stream);
  const int64_t rowTiles = ends == nullptr ? (rows + BM - 1) / BM : rows / BM + (rows < groups ? rows : groups);
  const int sms = gemm::gemmSmCount();
  const int bn = gemm::pickColumns(ends == nullptr ? (double)rowTiles : (double)(rows / BM) + 0.5 * (double)(rows < groups ? rows : groups), N, sms);
  const int64_t tiles = rowTiles * ((N + bn - 1) / bn);
  if (tiles > INT32_MAX) return mcclInvalidArgument;
  Args a;
  memset(&a, 0, sizeof(a));
  MCCLCHECK(gemm::rowsMap(&a.mapA, x, 1, 0, rows, K, ldx, BM));
  MCCLCHECK(gemm::rowsMap(&a.mapB, w, 1, groups, N, K, ldw, bn));
  MCCLCHECK(gemm::outputMap(&a.mapC, y, 0, rows, N, 32));
  a.sx = static_cast<const uint8_t*>(xScale);
  a.sw = static_cast<const uint8_t*>(wScale);
  a.ldsx = ldxScale; a.ldsw = ldwScale;
  a.ends = ends; a.ends64 = ends64; a.groups = groups;
  a.rows = (int)rows; a.N = N; a.K = K;
  a.out = static_cast<__nv_bfloat16*>(y);
  MCCLCHECK(gemm::errorWord(dev, &a.errFlag));
  a.budgetNs = gemm::waitNs();
  a.blockNs = gemm::blockNs();
  const int grid = (int)(tiles < sms ? tiles : sms);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return bn == 256 ? launchAs<256>(a, dev, grid, behind, s) : launchAs<128>(a, dev, grid, behind, s);
}

}  // namespace

extern "C" {

mcclResult_t mcclFp8Gemm(const void* x, int64_t ldx, const void* xScale, int64_t ldxScale, const void* w, int64_t ldw, const void* wScale, int64_t ldwScale, void* y,
                         const void* ends, int ends64, int groups, int64_t rows, int N, int K, mcclStream_t stream) {
  return product(x, ldx, xScale, ldxScale, w, ldw, wScale, ldwScale, y, ends, ends64, groups, rows, N, K, false, stream);
}

mcclResult_t mcclFp8GemmBf16Rows(const void* x, int64_t ldx, void* q, int64_t ldq, void* qScale, int64_t ldqScale, const void* w, int64_t ldw, const void* wScale, int64_t ldwScale,
                                 void* y, const void* ends, int ends64, int groups, int64_t rows, int N, int K, mcclStream_t stream) {
  MCCLCHECK(mcclFp8QuantizeRows(x, ldx, q, ldq, qScale, ldqScale, rows, K, stream));
  return product(q, ldq, qScale, ldqScale, w, ldw, wScale, ldwScale, y, ends, ends64, groups, rows, N, K, rows > 0, stream);
}

}  // extern "C"

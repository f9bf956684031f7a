// Host side of the products by pairs of SMs (pair_core.cuh): when they are used, launch.
#include <cuda.h>
#include <cuda_runtime.h>
#include <string.h>

#include <algorithm>
#include <atomic>

#include "../../core/core.h"
#include "gemm_host.h"
#include "pair_core.cuh"

using namespace mccl;
using namespace mccl::pair;

namespace {

template <int MODE>
mcclResult_t launchAs(const Args& a, int dev, int pairs, bool beside, cudaStream_t s) {
  auto* kernel = pairKernel<MODE>;
  static std::atomic<uint64_t> prepared{0};                // a bit per device: the attribute stays with the function
  if (!(prepared.load(std::memory_order_relaxed) >> (dev & 63) & 1)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES) != cudaSuccess) { cudaGetLastError(); return mcclSystemError; }
    prepared.fetch_or(1ull << (dev & 63));
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * pairs);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = SMEM_BYTES;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = beside ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, kernel, a) != cudaSuccess) { cudaGetLastError(); return mcclSystemError; }
  return mcclSuccess;
}

int64_t rowTilesAtMost(int mode, int64_t rows, int groups, int N) {
  return mode == WEIGHT ? (int64_t)groups * ((N + kRows - 1) / kRows) : rows / kRows + std::min<int64_t>(rows, groups);
}

}  // namespace

// 1024 rows a group on the average, and a tile for every pair (both measured beside pairKernel).
bool mccl::gemm::pairWanted(int mode, int64_t rows, int groups, int N, int K) {
  const int width = mode == FORWARD ? N : K;
  return rows >= 1024 * (int64_t)groups && rowTilesAtMost(mode, rows, groups, N) * ((width + BN - 1) / BN) >= gemmSmCount() / 2;
}

mcclResult_t mccl::gemm::pairGemm(const PairCall& c, int device, void* stream) {
  const int pairs = gemmSmCount() / 2, width = c.mode == FORWARD ? c.N : c.K;
  const int64_t tiles = rowTilesAtMost(c.mode, c.rows, c.groups, c.N) * ((width + BN - 1) / BN);
  if (tiles > INT32_MAX) return mcclInvalidArgument;
  Args a;
  memset(&a, 0, sizeof(a));
  if (c.mode == WEIGHT) {
    MCCLCHECK(rowsMap(&a.mapA, c.a, 2, 0, c.rows, c.N, c.lda, 64));
    MCCLCHECK(rowsMap(&a.mapB, c.b, 2, 0, c.rows, c.K, c.ldb, 64));
  } else {
    MCCLCHECK(rowsMap(&a.mapA, c.a, 2, 0, c.rows, c.mode == DATA ? c.N : c.K, c.lda, BM));
    MCCLCHECK(rowsMap(&a.mapB, c.b, 2, c.groups, c.N, c.K, c.K, c.mode == DATA ? 64 : HALF));
  }
  MCCLCHECK(outputMap(&a.mapC, c.out, c.mode == WEIGHT ? c.groups : 0, c.mode == WEIGHT ? c.N : c.rows, width, 32));
  a.ends = c.ends; a.ends64 = c.ends64; a.groups = c.groups;
  a.rows = (int)c.rows;
  a.contracted = c.mode == DATA ? c.N : c.K;
  a.tileRows = c.N; a.width = width;
  a.out = static_cast<__nv_bfloat16*>(c.out);
  MCCLCHECK(errorWord(device, &a.errFlag));
  a.budgetNs = gemm::waitNs();
  a.blockNs = gemm::blockNs();
  const int grid = (int)std::min<int64_t>(tiles, pairs);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return c.mode == FORWARD ? launchAs<FORWARD>(a, device, grid, false, s) : c.mode == DATA ? launchAs<DATA>(a, device, grid, false, s) : launchAs<WEIGHT>(a, device, grid, c.beside, s);
}

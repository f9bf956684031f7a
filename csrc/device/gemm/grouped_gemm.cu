// Host side of the products of ragged groups of rows (grouped_core.cuh): tensor maps, choice of the tile, launch.
#include <cuda.h>
#include <cuda_runtime.h>
#include <string.h>

#include <atomic>
#include <cmath>

#include "../../core/core.h"
#include "gemm_host.h"
#include "grouped_core.cuh"
#include "mccl_ops.h"

using namespace mccl;
using namespace mccl::grouped;

int mccl::gemm::pickColumns(double rowTiles, int width, int sms) {
  if (width <= 128) return 128;
  auto waves = [&](int bn) {
    const double w = rowTiles * ((width + bn - 1) / bn) / sms;
    return w > 8 ? w : std::ceil(w);
  };
  return waves(128) * 0.8 < waves(256) ? 128 : 256;
}

namespace {

mcclResult_t encode(CUtensorMap* map, const void* base, int elementBytes, uint64_t outer, uint64_t rows, uint64_t cols, uint64_t ld, uint32_t boxCols,
                    uint32_t boxRows, CUtensorMapSwizzle swizzle) {
  static gemm::EncodeTiledFn fn = gemm::encodeTiled();
  if (fn == nullptr) MCCLFAIL(mcclSystemError);
  const cuuint64_t dims[3] = {cols, rows, outer};
  const cuuint64_t strides[2] = {ld * elementBytes, rows * ld * elementBytes};
  const cuuint32_t box[3] = {boxCols, boxRows, 1}, elemStrides[3] = {1, 1, 1};
  const CUresult r = fn(map, elementBytes == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8, outer ? 3 : 2, const_cast<void*>(base), dims,
                        strides, box, elemStrides, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    MCCL_WARN("cuTensorMapEncodeTiled failed with %d (base %p, %llu x %llu x %llu, row pitch %llu)", (int)r, base, (unsigned long long)outer,
              (unsigned long long)rows, (unsigned long long)cols, (unsigned long long)ld);
    return mcclInvalidArgument;
  }
  return mcclSuccess;
}

}  // namespace

mcclResult_t mccl::gemm::rowsMap(CUtensorMap* map, const void* base, int elementBytes, uint64_t outer, uint64_t rows, uint64_t cols, uint64_t ld,
                                 uint32_t boxRows) {
  return encode(map, base, elementBytes, outer, rows, cols, ld, 128 / elementBytes, boxRows, CU_TENSOR_MAP_SWIZZLE_128B);
}
mcclResult_t mccl::gemm::outputMap(CUtensorMap* map, void* base, uint64_t outer, uint64_t rows, uint64_t cols, int boxCols) {
  return encode(map, base, 2, outer, rows, cols, cols, boxCols, 32, boxCols == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
}

namespace {

// The current device, its context bound to this thread: the driver's encoder needs it, and a thread of the autograd engine that has
// launched nothing yet has none.
int boundDevice() {
  int dev = 0;
  cudaGetDevice(&dev);
  cudaSetDevice(dev);
  return dev;
}

template <int BN, int MODE, bool WHOLE>
mcclResult_t launchAs(const Args& a, int dev, int grid, bool beside, cudaStream_t s) {
  auto* kernel = groupedKernel<BN, MODE, WHOLE>;
  static std::atomic<uint64_t> prepared{0};                // a bit per device: the attribute stays with the function
  if (!(prepared.load(std::memory_order_relaxed) >> (dev & 63) & 1)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (Smem<BN, WHOLE>::TOTAL)) != cudaSuccess) { cudaGetLastError(); return mcclSystemError; }
    prepared.fetch_or(1ull << (dev & 63));
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = (Smem<BN, WHOLE>::TOTAL);
  cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = beside ? 1 : 0;
  if (cudaLaunchKernelEx(&cfg, kernel, a) != cudaSuccess) { cudaGetLastError(); return mcclSystemError; }
  return mcclSuccess;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

struct Shape { const void* ends; int ends64, E; int64_t T; int N, K; };

bool valid(const Shape& s) {
  return s.ends != nullptr && s.E > 0 && s.E <= kMaxGroups && s.T >= 0 && s.T <= INT32_MAX - 256 && s.N > 0 && s.K > 0 && s.N <= INT32_MAX - 256 && s.K <= INT32_MAX - 256 &&
         s.N % 8 == 0 && s.K % 8 == 0;
}
bool validRows(const void* p, int64_t ld, int cols) { return p != nullptr && aligned16(p) && ld >= cols && ld % 8 == 0; }

template <int MODE, bool WHOLE = false>
mcclResult_t run(Args& a, const Shape& s, int dev, int64_t rowTiles, cudaStream_t stream, int bn, bool beside = false) {
  MCCLCHECK(gemm::errorWord(dev, &a.errFlag));
  a.budgetNs = gemm::waitNs();
  a.blockNs = gemm::blockNs();
  a.ends = s.ends; a.ends64 = s.ends64; a.groups = s.E; a.rows = (int)s.T;
  const int64_t tiles = rowTiles * ((a.width + bn - 1) / bn);
  if (tiles > INT32_MAX) return mcclInvalidArgument;
  const int sms = gemm::gemmSmCount(), grid = (int)(tiles < sms ? tiles : sms);
  return bn == 256 ? launchAs<256, MODE, WHOLE>(a, dev, grid, beside, stream) : launchAs<128, MODE, WHOLE>(a, dev, grid, beside, stream);
}

// Row tiles of all groups: at most one beside the full ones for each group.
int64_t rowTilesAtMost(const Shape& s) { return s.T / BM + (s.T < s.E ? s.T : s.E); }
// and half of one on the average.
double rowTilesExpected(const Shape& s) { return (double)(s.T / BM) + 0.5 * (double)(s.T < s.E ? s.T : s.E); }

// dw; `beside`: may run beside the product launched last on the stream.
mcclResult_t weightGradient(const void* dy, int64_t lddy, const void* x, int64_t ldx, void* dw, const void* ends, int ends64, int groups,
                            int64_t rows, int N, int K, bool beside, mcclStream_t stream) {
  const Shape s{ends, ends64, groups, rows, N, K};
  if (!valid(s) || dw == nullptr || !aligned16(dw)) return mcclInvalidArgument;
  if (rows == 0)
    return cudaMemsetAsync(dw, 0, (size_t)groups * N * K * 2, reinterpret_cast<cudaStream_t>(stream)) == cudaSuccess ? mcclSuccess : mcclSystemError;
  if (!validRows(dy, lddy, N) || !validRows(x, ldx, K)) return mcclInvalidArgument;
  const int dev = boundDevice();
  if (gemm::pairWanted(WEIGHT, rows, groups, N, K))
    return gemm::pairGemm(gemm::PairCall{WEIGHT, dy, x, lddy, ldx, dw, ends, ends64, groups, rows, N, K, beside}, dev, stream);
  Args a;
  memset(&a, 0, sizeof(a));
  const int64_t rt = (int64_t)groups * ((N + BM - 1) / BM);
  const int bn = gemm::pickColumns((double)rt, K, gemm::gemmSmCount());
  MCCLCHECK(gemm::rowsMap(&a.mapA, dy, 2, 0, rows, N, lddy, 64));
  MCCLCHECK(gemm::rowsMap(&a.mapB, x, 2, 0, rows, K, ldx, 64));
  a.tileRows = N; a.width = K;
  a.out = static_cast<__nv_bfloat16*>(dw);
  const bool whole = rows <= 64 * (int64_t)groups;         // one block of rows an expert on the average
  MCCLCHECK(gemm::outputMap(&a.mapC, dw, groups, N, K, whole ? 64 : 32));
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return whole ? run<WEIGHT, true>(a, s, dev, rt, st, bn, beside) : run<WEIGHT>(a, s, dev, rt, st, bn, beside);
}

}  // namespace

extern "C" {

int mcclGroupedGemmMaxGroups(void) { return kMaxGroups; }

mcclResult_t mcclGroupedGemm(const void* x, int64_t ldx, const void* w, void* y, const void* ends, int ends64, int groups, int64_t rows, int N, int K,
                             mcclStream_t stream) {
  const Shape s{ends, ends64, groups, rows, N, K};
  if (!valid(s)) return mcclInvalidArgument;
  if (rows == 0) return mcclSuccess;
  if (!validRows(x, ldx, K) || w == nullptr || y == nullptr || !aligned16(w) || !aligned16(y)) return mcclInvalidArgument;
  const int dev = boundDevice();
  if (gemm::thinWanted(rows, true, groups, N, 2ll * K)) {
    gemm::ThinCall c{};
    c.x = x; c.w = w; c.ldx = ldx; c.ldw = K; c.out = y; c.ends = ends; c.ends64 = ends64; c.groups = groups; c.rows = rows; c.N = N; c.K = K;
    return gemm::thinGemm(c, dev, stream);
  }
  if (gemm::pairWanted(FORWARD, rows, groups, N, K))
    return gemm::pairGemm(gemm::PairCall{FORWARD, x, w, ldx, K, y, ends, ends64, groups, rows, N, K, false}, dev, stream);
  Args a;
  memset(&a, 0, sizeof(a));
  const int64_t rt = rowTilesAtMost(s);
  const int bn = gemm::pickColumns(rowTilesExpected(s), N, gemm::gemmSmCount());
  MCCLCHECK(gemm::rowsMap(&a.mapA, x, 2, 0, rows, K, ldx, BM));
  MCCLCHECK(gemm::rowsMap(&a.mapB, w, 2, groups, N, K, K, bn));
  a.contracted = K; a.width = N;
  a.out = static_cast<__nv_bfloat16*>(y);
  MCCLCHECK(gemm::outputMap(&a.mapC, y, 0, rows, N, 32));
  return run<FORWARD>(a, s, dev, rt, reinterpret_cast<cudaStream_t>(stream), bn);
}

mcclResult_t mcclGroupedGemmBackwardData(const void* dy, int64_t lddy, const void* w, void* dx, const void* ends, int ends64, int groups, int64_t rows,
                                         int N, int K, mcclStream_t stream) {
  const Shape s{ends, ends64, groups, rows, N, K};
  if (!valid(s)) return mcclInvalidArgument;
  if (rows == 0) return mcclSuccess;
  if (!validRows(dy, lddy, N) || w == nullptr || dx == nullptr || !aligned16(w) || !aligned16(dx)) return mcclInvalidArgument;
  const int dev = boundDevice();
  if (gemm::pairWanted(DATA, rows, groups, N, K))
    return gemm::pairGemm(gemm::PairCall{DATA, dy, w, lddy, K, dx, ends, ends64, groups, rows, N, K, false}, dev, stream);
  Args a;
  memset(&a, 0, sizeof(a));
  const int64_t rt = rowTilesAtMost(s);
  const int bn = gemm::pickColumns(rowTilesExpected(s), K, gemm::gemmSmCount());
  MCCLCHECK(gemm::rowsMap(&a.mapA, dy, 2, 0, rows, N, lddy, BM));
  MCCLCHECK(gemm::rowsMap(&a.mapB, w, 2, groups, N, K, K, 64));
  a.contracted = N; a.width = K;
  a.out = static_cast<__nv_bfloat16*>(dx);
  MCCLCHECK(gemm::outputMap(&a.mapC, dx, 0, rows, K, 32));
  return run<DATA>(a, s, dev, rt, reinterpret_cast<cudaStream_t>(stream), bn);
}

mcclResult_t mcclGroupedGemmBackwardWeight(const void* dy, int64_t lddy, const void* x, int64_t ldx, void* dw, const void* ends, int ends64, int groups,
                                           int64_t rows, int N, int K, mcclStream_t stream) {
  return weightGradient(dy, lddy, x, ldx, dw, ends, ends64, groups, rows, N, K, false, stream);
}

mcclResult_t mcclGroupedGemmBackward(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* w, void* dx, void* dw, const void* ends, int ends64,
                                     int groups, int64_t rows, int N, int K, mcclStream_t stream) {
  MCCLCHECK(mcclGroupedGemmBackwardData(dy, lddy, w, dx, ends, ends64, groups, rows, N, K, stream));
  return weightGradient(dy, lddy, x, ldx, dw, ends, ends64, groups, rows, N, K, rows > 0, stream);
}

}  // extern "C"

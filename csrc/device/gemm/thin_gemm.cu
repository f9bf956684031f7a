// Host side of the products with few rows (thin_core.cuh): choice of the tile and of the CTAs that share one, launch.
#include <cuda.h>
#include <cuda_runtime.h>
#include <string.h>

#include <algorithm>
#include <atomic>

#include "../../core/core.h"
#include "gemm_host.h"
#include "thin_core.cuh"

using namespace mccl;
using namespace mccl::thin;

namespace {

template <int BT, bool FP8>
mcclResult_t launchAs(Args& a, const gemm::ThinCall& c, int dev, int tiles, int shares, int slices, cudaStream_t s) {
  auto* kernel = thinKernel<BT, FP8>;
  static std::atomic<uint64_t> prepared{0};                // a bit per device: the attribute stays with the function
  if (!(prepared.load(std::memory_order_relaxed) >> (dev & 63) & 1)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<BT>::TOTAL) != cudaSuccess) { cudaGetLastError(); return mcclSystemError; }
    prepared.fetch_or(1ull << (dev & 63));
  }
  MCCLCHECK(gemm::rowsMap(&a.mapX, c.x, FP8 ? 1 : 2, 0, c.rows, c.K, c.ldx, BT));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * slices), (unsigned)c.groups, (unsigned)shares);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Smem<BT>::TOTAL;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = slices; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = c.behind ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, kernel, a) != cudaSuccess) { cudaGetLastError(); return mcclSystemError; }
  return mcclSuccess;
}

template <bool FP8>
mcclResult_t launch(int bt, Args& a, const gemm::ThinCall& c, int dev, int tiles, int shares, int slices, cudaStream_t s) {
  switch (bt) {
    case 16: return launchAs<16, FP8>(a, c, dev, tiles, shares, slices, s);
    case 32: return launchAs<32, FP8>(a, c, dev, tiles, shares, slices, s);
    default: return launchAs<64, FP8>(a, c, dev, tiles, shares, slices, s);
  }
}

// CTAs that run at a time.  Two fit an SM, but clusters do not fill the last of them: 128 rows of 8192 by 3584 columns with 280 CTAs in clusters of
// five 19 us, with 224 in clusters of four 13 us.
int64_t placesFor(int64_t sms) { return 2 * sms * 7 / 8; }

int64_t expertsWithRows(int64_t rows, int groups) { return std::min<int64_t>(rows, groups); }

}  // namespace

// Where a tile's contraction can be shared by two CTAs or more (8 bits, 100 rows of 8192 by 11008 columns, which cannot: 32 us here, 21 us in tiles of
// 128 rows), and for up to 32 rows whose weights' rows are not short (one row of 4096 by 22016 columns 14.5 us here, 26 us there; of 1024 by
// 50304 columns 14.4 and 12.9 us).  With groups, whose rows the host does not know: where the tiles of 128 rows x 128 columns are no more than
// the SMs (64 rows for 32 experts of 2048 x 5504, which are more: 106 us here, 103 us there), and the CTAs that find no rows are few (two rows, 64
// experts of 2048 x 1024 in 8 bits: 10.6 us here, 9.0 us there).
bool mccl::gemm::thinWanted(int64_t rows, bool ragged, int groups, int N, int64_t kBytes) {
  const int64_t nTiles = (N + BM - 1) / BM, sms = gemmSmCount();
  if (ragged) return (rows / BM + expertsWithRows(rows, groups)) * nTiles <= sms && groups * nTiles <= 2 * sms;
  if (rows <= 32) return nTiles <= sms || kBytes >= 2048;
  return 2 * nTiles * ((rows + 63) / 64) <= placesFor(sms);
}

mcclResult_t mccl::gemm::thinGemm(const ThinCall& c, int device, void* stream) {
  const bool ragged = c.ends != nullptr;
  const int sms = gemmSmCount(), nTiles = (c.N + BM - 1) / BM;
  // Rows of a tile: those of a group where they are known, twice the mean where not.
  const int64_t experts = ragged ? expertsWithRows(c.rows, c.groups) : 1, rows = ragged ? 2 * ((c.rows + experts - 1) / experts) : c.rows;
  const int bt = rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
  const int64_t shares = (rows + bt - 1) / bt;             // an expert with more rows than expected walks them in turns
  const int perUnit = c.fp8 ? 512 : 64, units = (c.K + perUnit - 1) / perUnit;
  const int64_t places = placesFor(sms), tiles = (int64_t)nTiles * c.groups * shares;       // those of experts without rows start, too
  const int slices = (int)std::max<int64_t>(1, std::min<int64_t>({8, places / tiles, units}));
  Args a;
  memset(&a, 0, sizeof(a));
  MCCLCHECK(rowsMap(&a.mapW, c.w, c.fp8 ? 1 : 2, c.groups, c.N, c.K, c.ldw, BM));
  a.sx = static_cast<const uint8_t*>(c.sx);
  a.sw = static_cast<const uint8_t*>(c.sw);
  a.ldsx = c.ldsx; a.ldsw = c.ldsw;
  a.ends = c.ends; a.ends64 = c.ends64; a.groups = c.groups;
  a.rows = (int)c.rows; a.N = c.N; a.K = c.K; a.slices = slices;
  a.out = static_cast<__nv_bfloat16*>(c.out);
  MCCLCHECK(errorWord(device, &a.errFlag));
  a.budgetNs = gemm::waitNs();
  a.blockNs = gemm::blockNs();
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return c.fp8 ? launch<true>(bt, a, c, device, nTiles, (int)shares, slices, s) : launch<false>(bt, a, c, device, nTiles, (int)shares, slices, s);
}

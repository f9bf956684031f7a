// Host-side helpers the GEMM launchers share (defined in tp_gemm.cu).
#pragma once

#include <cuda.h>
#include <stdint.h>

#include "mccl.h"

namespace mccl {
namespace gemm {

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
// cuTensorMapEncodeTiled of the driver; null where it cannot be had.
EncodeTiledFn encodeTiled();
// The device-visible word in which a GEMM kernel records that it gave up (mcclTpGemmLastError).  mcclInternalError where one has done so and
// nobody has read it: what it left unwritten is not built upon.
mcclResult_t errorWord(int device, int** word);
// How long a wait of a kernel may take: two seconds, and 20 us for each block of contractions it covers, which take 0.1 to 0.4 us each
// (mcclDbgGemmWaitNs).
uint64_t waitNs();
uint64_t blockNs();
// Multiprocessors of the current device.
int gemmSmCount();

// y [rows, N] = x w^T for few rows (thin_core.cuh): bf16, or e4m3 with scales; ends null: one group.  `behind`: launched right behind the
// kernel that makes x and its scales, which lets it start early.
struct ThinCall {
  const void *x, *w;
  int64_t ldx, ldw;                     // elements
  bool fp8;
  const void *sx, *sw;
  int64_t ldsx, ldsw;
  void* out;
  const void* ends;
  int ends64, groups;
  int64_t rows;
  int N, K;
  bool behind;
};
// Whether this many rows are better served by the thin form.  kBytes: of a row of the weights.
bool thinWanted(int64_t rows, bool ragged, int groups, int N, int64_t kBytes);
mcclResult_t thinGemm(const ThinCall& c, int device, void* stream);
// The products of groups by pairs of SMs (pair_core.cuh).  mode: 0 y = x w^T, 1 dx = dy w, 2 dw = dy^T x.
struct PairCall {
  int mode;
  const void *a, *b;                    // x or dy; w, or x for mode 2
  int64_t lda, ldb;                     // elements a row; ldb for mode 2
  void* out;
  const void* ends;
  int ends64, groups;
  int64_t rows;
  int N, K;
  bool beside;                          // may run beside the product launched last on the stream
};
// Whether groups of this many rows are better served by pairs.
bool pairWanted(int mode, int64_t rows, int groups, int N, int K);
mcclResult_t pairGemm(const PairCall& c, int device, void* stream);
// Columns of a tile of 128 rows, 128 or 256, by the waves that so many row tiles of `width` columns make.  A wave of tiles of 128 columns takes 0.8 of one
// of 256 (8 bits, contraction of 8192: 21 and 26 us), so the narrow tile is for where SMs would stand idle.
int pickColumns(double rowTiles, int width, int sms);
// Tensor map of [outer][rows][cols] (outer 0: a matrix) of 2-byte (bf16) or 1-byte elements, rows `ld` elements apart: boxes of 128 bytes x
// boxRows, 128-byte swizzle, zeros outside.
mcclResult_t rowsMap(CUtensorMap* map, const void* base, int elementBytes, uint64_t outer, uint64_t rows, uint64_t cols, uint64_t ld, uint32_t boxRows);
// Of the output, contiguous bf16 [outer][rows][cols] (outer 0: a matrix): boxes of 32 or 64 columns x 32 rows, swizzled over their width.
mcclResult_t outputMap(CUtensorMap* map, void* base, uint64_t outer, uint64_t rows, uint64_t cols, int boxCols);

}  // namespace gemm
}  // namespace mccl

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
// The device-visible word in which a GEMM kernel records that it gave up (mcclTpGemmLastError); null where it cannot be had.
int* gemmErrFlag(int device);
// Multiprocessors of the current device.
int gemmSmCount();

}  // namespace gemm
}  // namespace mccl

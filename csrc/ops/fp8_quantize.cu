// bf16 -> 8-bit floating point (e4m3) with a power-of-two scale (e8m0) for each block of 128 of a row, or of 128 rows x 128.
//   scale = 2^e with the smallest e for which the block's largest magnitude is at most 448 2^e (a block of zeros: 1),
//   q = the nearest e4m3 number to x / scale, the even one of two.
// The exponent comes from the bits of the largest magnitude: 448 = 1.75 x 2^8, so it is that of the magnitude less eight, or less seven
// where its mantissa is above 1.75.  x / scale is exact.  Numbers that are not finite take no part in the scale and become NaN.
// Bound by memory: two bytes read, one written for each value.  No counterpart in the reference.
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "mccl.h"
#include "mccl_ops.h"

namespace {

constexpr int kBlock = 128, kThreads = 256;

// Magnitudes of eight bf16 numbers as one 16-bit maximum; numbers that are not finite count as zero.
__device__ __forceinline__ uint32_t largest(const uint4& q) {
  auto two = [](uint32_t w) {
    w &= 0x7fff7fffu;
    const uint32_t big = __vcmpgtu2(w, 0x7f7f7f7fu);       // all ones where not finite
    return w & ~big;
  };
  const uint32_t m = __vmaxu2(__vmaxu2(two(q.x), two(q.y)), __vmaxu2(two(q.z), two(q.w)));
  return max(m & 0xffffu, m >> 16);
}
// The scale's byte (its exponent plus 127) for a largest magnitude of these bf16 bits.
__device__ __forceinline__ uint32_t scaleByte(uint32_t a) {
  if (a == 0) return 127;
  const int e = (int)(a >> 7) - ((a & 0x7f) <= 0x60 ? 8 : 7);
  return (uint32_t)max(e, 0);
}
__device__ __forceinline__ uint32_t four(uint32_t lo, uint32_t hi, float inv) {
  float f[4] = {__uint_as_float(lo << 16), __uint_as_float(lo & 0xffff0000u), __uint_as_float(hi << 16), __uint_as_float(hi & 0xffff0000u)};
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = __fmaf_rn(f[i], 0.f, f[i] * inv);          // Inf x 0: NaN, where the conversion would give 448
  const uint32_t a = __nv_cvt_float2_to_fp8x2(make_float2(f[0], f[1]), __NV_SATFINITE, __NV_E4M3);
  const uint32_t b = __nv_cvt_float2_to_fp8x2(make_float2(f[2], f[3]), __NV_SATFINITE, __NV_E4M3);
  return a | b << 16;
}
__device__ __forceinline__ uint2 quantize(const uint4& q, uint32_t byte) {
  const float inv = __uint_as_float((254u - byte) << 23);  // byte <= 247
  return make_uint2(four(q.x, q.y, inv), four(q.z, q.w, inv));
}

// Eight threads a block of 128, sixteen values each, four blocks a thread.  8192 x 8192: with sixteen threads a block and one block in
// flight a thread 55 us, with four 47 us, with eight threads a block 37 us (5.4 TB/s).
// I: the type the blocks of all rows are counted in (a 64-bit division costs as much as the rest).
constexpr int kPieces = 4, kPerBlock = 8;
template <class I>
__global__ void __launch_bounds__(kThreads) quantizeRowsKernel(const __nv_bfloat16* x, int64_t ldx, uint8_t* q, int64_t ldq, uint8_t* scale, int64_t lds, int64_t rows,
                                                               int K, int blocks) {
  // Launched with programmatic stream serialization, which hides its launch behind the end of what runs before; everything here comes after
  // that.  Then a product behind this may start, which itself waits for this grid's end where it reads what it makes.  (One row of 4096 by
  // 11008 columns, quantised and multiplied, call after call: 14.9 -> 13.3 us.)
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const I total = (I)rows * (I)blocks, b0 = (I)blockIdx.x * (kThreads / kPerBlock * kPieces) + (threadIdx.x / kPerBlock);
  const int in = (threadIdx.x % kPerBlock) * 16;
  uint4 v[kPieces][2];
  int64_t row[kPieces];
  int blk[kPieces];
#pragma unroll
  for (int u = 0; u < kPieces; ++u) {
    const I b = b0 + (I)(u * (kThreads / kPerBlock)), r = b < total ? b / (I)blocks : 0;
    row[u] = (int64_t)r;
    blk[u] = b < total ? (int)(b - r * (I)blocks) : -1;
    const int col = blk[u] * kBlock + in;                  // K is a multiple of 16: all sixteen or none
    const uint4* from = reinterpret_cast<const uint4*>(x + row[u] * ldx + col);
    const bool live = blk[u] >= 0 && col < K;
    v[u][0] = live ? from[0] : make_uint4(0, 0, 0, 0);
    v[u][1] = live ? from[1] : make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int u = 0; u < kPieces; ++u) {
    uint32_t a = max(largest(v[u][0]), largest(v[u][1]));
#pragma unroll
    for (int o = kPerBlock / 2; o > 0; o >>= 1) a = max(a, __shfl_xor_sync(0xffffffffu, a, o));
    const uint32_t byte = scaleByte(a);
    const int col = blk[u] * kBlock + in;
    if (blk[u] >= 0 && col < K) {
      const uint2 lo = quantize(v[u][0], byte), hi = quantize(v[u][1], byte);
      *reinterpret_cast<uint4*>(q + row[u] * ldq + col) = make_uint4(lo.x, lo.y, hi.x, hi.y);
    }
    if (blk[u] >= 0 && in == 0) scale[row[u] * lds + blk[u]] = (uint8_t)byte;
  }
}

// One CTA a block of 128 x 128, all of them along the grid's first dimension: each thread eight rows' pieces of eight values.  8192 x 8192 41 us,
// 4.9 TB/s; 3584 x 8192 20.5 us.
__global__ void __launch_bounds__(kThreads) quantizeTilesKernel(const __nv_bfloat16* x, uint8_t* q, int64_t ldq, uint8_t* scale, int64_t lds, int rows, int K,
                                                                int rowBlocks, int colBlocks) {
  __shared__ uint32_t warpMax[kThreads / 32];
  const uint32_t across = blockIdx.x / (uint32_t)colBlocks;
  const int cb = (int)(blockIdx.x - across * (uint32_t)colBlocks), rb = (int)(across % (uint32_t)rowBlocks);
  const int64_t outer = across / (uint32_t)rowBlocks;
  const int col = cb * kBlock + (threadIdx.x & 15) * 8;
  x += outer * rows * K;
  q += outer * rows * ldq;
  uint4 v[8];
  uint32_t a = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = rb * kBlock + i * 16 + (threadIdx.x >> 4);
    v[i] = r < rows && col < K ? *reinterpret_cast<const uint4*>(x + (int64_t)r * K + col) : make_uint4(0, 0, 0, 0);
    a = max(a, largest(v[i]));
  }
  a = __reduce_max_sync(0xffffffffu, a);
  if ((threadIdx.x & 31) == 0) warpMax[threadIdx.x >> 5] = a;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) a = max(a, warpMax[w]);
  const uint32_t byte = scaleByte(a);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = rb * kBlock + i * 16 + (threadIdx.x >> 4);
    if (r < rows && col < K) *reinterpret_cast<uint2*>(q + r * ldq + col) = quantize(v[i], byte);
  }
  if (threadIdx.x == 0) scale[(outer * rowBlocks + rb) * lds + cb] = (uint8_t)byte;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
mcclResult_t launchedOk() { return cudaGetLastError() == cudaSuccess ? mcclSuccess : mcclSystemError; }

}  // namespace

extern "C" {

mcclResult_t mcclFp8QuantizeRows(const void* x, int64_t ldx, void* q, int64_t ldq, void* scale, int64_t ldScale, int64_t rows, int K, mcclStream_t stream) {
  const int blocks = (K + kBlock - 1) / kBlock;
  if (rows < 0 || K <= 0 || K > INT32_MAX - 256 || K % 16 || ldx < K || ldx % 8 || ldq < K || ldq % 16 || ldScale < blocks) return mcclInvalidArgument;
  if (rows == 0) return mcclSuccess;
  if (!x || !q || !scale || !aligned16(x) || !aligned16(q) || rows * blocks > (int64_t)INT32_MAX * 16) return mcclInvalidArgument;
  const int64_t per = kThreads / kPerBlock * kPieces, ctas = (rows * blocks + per - 1) / per;
  auto* kernel = rows * blocks < (1ll << 31) - per ? quantizeRowsKernel<uint32_t> : quantizeRowsKernel<int64_t>;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = reinterpret_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, kernel, static_cast<const __nv_bfloat16*>(x), ldx, static_cast<uint8_t*>(q), ldq, static_cast<uint8_t*>(scale), ldScale, rows, K, blocks);
  return launchedOk();
}

mcclResult_t mcclFp8QuantizeTiles(const void* x, void* q, int64_t ldq, void* scale, int64_t ldScale, int64_t outer, int rows, int K, mcclStream_t stream) {
  if (outer < 0 || rows <= 0 || K <= 0 || K > INT32_MAX - 256 || rows > INT32_MAX - 256 || K % 16 || ldq < K || ldq % 16 || ldScale < (K + kBlock - 1) / kBlock)
    return mcclInvalidArgument;
  if (outer == 0) return mcclSuccess;
  const int rowBlocks = (rows + kBlock - 1) / kBlock, colBlocks = (K + kBlock - 1) / kBlock;
  if (!x || !q || !scale || !aligned16(x) || !aligned16(q)) return mcclInvalidArgument;
  // a grid ends at 2^31 - 1 blocks: matrices in turn
  const int64_t each = (int64_t)rowBlocks * colBlocks, per = INT32_MAX / each;
  if (per == 0) return mcclInvalidArgument;
  for (int64_t o = 0; o < outer; o += per) {
    const int64_t n = outer - o < per ? outer - o : per;
    quantizeTilesKernel<<<dim3((unsigned)(n * each)), kThreads, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
        static_cast<const __nv_bfloat16*>(x) + o * rows * K, static_cast<uint8_t*>(q) + o * rows * ldq, ldq,
        static_cast<uint8_t*>(scale) + o * rowBlocks * ldScale, ldScale, rows, K, rowBlocks, colBlocks);
  }
  return launchedOk();
}

}  // extern "C"

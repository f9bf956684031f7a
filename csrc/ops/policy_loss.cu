// Clipped policy loss with a KL term over the logits of a language-model head, for tuning by rewards.
//   lp   = z[a] - logsumexp(z)                       the token's log-probability now
//   r    = exp(lp - old)                             against the policy that sampled it
//   l    = -min(r A, clamp(r, 1 - lo, 1 + hi) A) + beta (exp(ref - lp) - (ref - lp) - 1)
//   loss = sum of w l, divided by the sum of w where the mean is wanted
//   d loss / d z[j] = c ([j = a] - p[j]),  c = w (d l / d lp) / sum of w,  d l / d lp = (-r A where r A is the smaller, else 0) + beta (1 - exp(ref - lp))
// Forward: a CTA per row (a cluster of up to eight where there are few rows), one pass with a running maximum and sum of exponentials
// (online_softmax.cuh); then one cluster works out all rows' terms and adds them up, in 64 bits: lp is a small difference, and the
// terms have both signs.  Backward: reads the logits again and writes the gradient, a
// row of weight zero, or one that the clamp holds without a KL term, is written as zeros without being read.
// No counterpart in the reference (it has no model code).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "mccl.h"
#include "mccl_ops.h"
#include "online_softmax.cuh"

namespace {

using namespace mccl;

constexpr int kThreads = 256;                  // as in the cross-entropy: several small CTAs an SM, so that the ends of rows lie beside other rows' loads
constexpr int kUnroll = 4;                     // 16-byte pieces in flight per thread in long rows

template <class T> constexpr int kVec = 16 / (int)sizeof(T);

__device__ __forceinline__ float toFloat(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float toFloat(__half x) { return __half2float(x); }
__device__ __forceinline__ float toFloat(float x) { return x; }
template <class T> __device__ __forceinline__ T fromFloat(float x);
template <> __device__ __forceinline__ __nv_bfloat16 fromFloat<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half fromFloat<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ float fromFloat<float>(float x) { return x; }

template <class T>
__device__ __forceinline__ void unpack(const uint4& q, float (&f)[kVec<T>]) {
  const T* e = reinterpret_cast<const T*>(&q);
#pragma unroll
  for (int k = 0; k < kVec<T>; ++k) f[k] = toFloat(e[k]);
}
template <>
__device__ __forceinline__ void unpack<__nv_bfloat16>(const uint4& q, float (&f)[8]) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) { f[2 * k] = __uint_as_float(w[k] << 16); f[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u); }
}
template <class T>
__device__ __forceinline__ uint4 pack(const float (&f)[kVec<T>]) {
  uint4 q;
  T* e = reinterpret_cast<T*>(&q);
#pragma unroll
  for (int k = 0; k < kVec<T>; ++k) e[k] = fromFloat<T>(f[k]);
  return q;
}

// What the loss of a row is made of besides its logits.  `stats` holds three numbers a row for the backward pass: the maximum, one
// over the sum of exponentials, and w dl/dlp.
struct RowInputs {
  const int64_t* tokens;
  const float *old, *ref, *advantages;         // ref: nullable
  const void* weights;                         // nullable: all ones
  int boolWeights;                             // one byte a row, not a float
  double lo, hi, beta;
  __device__ __forceinline__ float weight(int64_t row) const {
    if (weights == nullptr) return 1.f;
    return boolWeights ? (static_cast<const uint8_t*>(weights)[row] ? 1.f : 0.f) : static_cast<const float*>(weights)[row];
  }
};

__device__ __forceinline__ void clusterMeet() { asm volatile("barrier.cluster.arrive.release;\n barrier.cluster.wait.acquire;" ::: "memory"); }
__device__ __forceinline__ uint32_t atRank(const void* here, int rank) {
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(here)), "r"(rank));
  return at;
}

// stats[row], stats[rows + row] = maximum and sum of exp(x - maximum).  gridDim.y CTAs share a row, as one cluster: each leaves its pair in
// its shared memory, and the first adds them up rank by rank.
// Instructions bound it beside memory: 8192 x 50257 bf16 with the rows' terms 147 us, 5.6 TB/s; 170 us where the distance of a thread's pieces is
// no constant, hence SHARED (whether there are several CTAs).
template <class T, int U, bool SHARED>
__global__ void __launch_bounds__(kThreads, 6) policyForwardKernel(const T* logits, int64_t rows, int64_t ld, int vocab, float* stats) {
  __shared__ MaxSum warpAcc[kThreads / 32];
  __shared__ __align__(8) MaxSum mine;
  const int64_t row = blockIdx.x;
  const int share = SHARED ? (int)blockIdx.y : 0, stride = SHARED ? (int)gridDim.y * kThreads : kThreads;
  const T* x = logits + row * ld;
  MaxSum acc{kLowest, 0.f};
  const Span sp = spanOf(x, vocab);
  const uint4* v = reinterpret_cast<const uint4*>(x + sp.head);
  for (int i = share * kThreads + threadIdx.x; i < sp.vecs; i += U * stride) {
    uint4 q[U];
#pragma unroll
    for (int u = 0; u < U; ++u) if (i + u * stride < sp.vecs) q[u] = v[i + u * stride];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u * stride >= sp.vecs) continue;
      float f[kVec<T>];
      unpack<T>(q[u], f);
      pushAll(acc, f);
    }
  }
  const int tail = sp.head + sp.vecs * kVec<T>;
  if (share == 0 && (int)threadIdx.x < sp.head) push(acc, toFloat(x[threadIdx.x]));
  if (share == 0 && tail + (int)threadIdx.x < vocab) push(acc, toFloat(x[tail + threadIdx.x]));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    MaxSum other{__shfl_xor_sync(0xffffffffu, acc.m, o), __shfl_xor_sync(0xffffffffu, acc.s, o)};
    acc = combine(acc, other);
  }
  if ((threadIdx.x & 31) == 0) warpAcc[threadIdx.x >> 5] = acc;
  __syncthreads();
  MaxSum t{kLowest, 0.f};
  if (threadIdx.x == 0) {
    t = warpAcc[0];
    for (int w = 1; w < kThreads / 32; ++w) t = combine(t, warpAcc[w]);
  }
  if (SHARED) {
    if (threadIdx.x == 0) mine = t;
    clusterMeet();
    if (threadIdx.x == 0 && share == 0)
      for (int p = 1; p < (int)gridDim.y; ++p) {
        MaxSum r;
        asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(r.m), "=f"(r.s) : "r"(atRank(&mine, p)) : "memory");
        t = combine(t, r);
      }
    clusterMeet();                             // no CTA leaves before its pair has been read
  }
  if (threadIdx.x != 0 || share != 0) return;
  stats[row] = t.m;
  stats[rows + row] = t.s;
}

__device__ __forceinline__ double warpSum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// One cluster over all rows: log-probabilities, terms and slopes, and their sums in a fixed order.  stats[rows + row] becomes one over the sum,
// stats[2 rows + row] = w dl/dlp; *loss = sum of w l [/ sum of w], *inverse = one over what it was divided by.  A batch whose weights add
// up to zero has loss zero and no gradient.
constexpr int kRowThreads = 512;
template <class T>
__global__ void __launch_bounds__(kRowThreads) policyRowsKernel(const T* logits, int64_t rows, int64_t ld, int vocab, RowInputs in, int mean, float* logp,
                                                                float* stats, float* loss, float* inverse) {
  __shared__ double partial[2][kRowThreads / 32], mine[2];
  double sumL = 0., sumW = 0.;
  for (int64_t row = (int64_t)blockIdx.x * kRowThreads + threadIdx.x; row < rows; row += (int64_t)gridDim.x * kRowThreads) {
    const int64_t tok = in.tokens[row];
    const float w = in.weight(row), m = stats[row], nan = __int_as_float(0x7fffffff);
    const float s = m == INFINITY ? nan : stats[rows + row];       // inf - inf in the exponent
    const bool valid = tok >= 0 && tok < vocab;
    // A token that is no column: of no weight, or the loss and the row's gradient are NaN.
    const double lp = valid ? (double)toFloat(logits[row * ld + tok]) - (double)m - log((double)s) : w == 0.f ? 0. : (double)nan;
    logp[row] = (float)lp;
    double l = 0., slope = 0.;
    if (w != 0.f) {
      const double a = in.advantages[row], r = exp(lp - (double)in.old[row]);
      const double plain = r * a, held = fmin(fmax(r, 1. - in.lo), 1. + in.hi) * a;
      l = plain > held ? -held : -plain;
      slope = plain > held ? 0. : -plain;      // of equals, and of NaN, the unclamped one
      if (in.ref != nullptr) {
        const double d = (double)in.ref[row] - lp, e = exp(d);
        l += in.beta * (e - d - 1.);
        slope += in.beta * (1. - e);
      }
      l *= w;
      slope *= w;
    }
    sumL += l;
    sumW += w;
    stats[rows + row] = 1.f / s;
    stats[2 * rows + row] = (float)slope;
  }
  sumL = warpSum(sumL);
  sumW = warpSum(sumW);
  if ((threadIdx.x & 31) == 0) { partial[0][threadIdx.x >> 5] = sumL; partial[1][threadIdx.x >> 5] = sumW; }
  __syncthreads();
  if (threadIdx.x < 32) {
    const bool has = threadIdx.x < kRowThreads / 32;
    sumL = warpSum(has ? partial[0][threadIdx.x] : 0.);
    sumW = warpSum(has ? partial[1][threadIdx.x] : 0.);
    if (threadIdx.x == 0) { mine[0] = sumL; mine[1] = sumW; }
  }
  if (gridDim.x > 1) {
    clusterMeet();
    if (threadIdx.x == 0 && blockIdx.x == 0)
      for (int p = 1; p < (int)gridDim.x; ++p) {
        double l, w;
        asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(l) : "r"(atRank(&mine[0], p)) : "memory");
        asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(w) : "r"(atRank(&mine[1], p)) : "memory");
        sumL += l;
        sumW += w;
      }
    clusterMeet();                             // no CTA leaves before its sums have been read
  }
  if (threadIdx.x != 0 || blockIdx.x != 0) return;
  const bool none = mean && sumW == 0.;
  const double over = none ? 0. : mean ? 1. / sumW : 1.;
  *loss = none ? 0.f : (float)(sumL * over);   // weights that add up to infinity: NaN
  *inverse = (float)over;
}

// exp for a gradient in T: one with the type's precision.
template <class T> __device__ __forceinline__ float gradExp(float x) { return __expf(x); }
template <> __device__ __forceinline__ float gradExp<float>(float x) { return expf(x); }

// Bound by memory: 8192 x 50257 bf16, every row read, 258 us, 6.4 TB/s; with a tenth of the rows of weight zero 248 us, 6.3 TB/s.  blockIdx.y: which slice of the row.  SAME: a row's 16-byte boundaries lie at the same elements in the logits and in the gradient.
template <class T, int U, bool SAME>
__global__ void __launch_bounds__(kThreads) policyBackwardKernel(const T* logits, int64_t rows, int64_t ld, T* grad, int64_t gradLd, int vocab, int width,
                                                                 const int64_t* tokens, const float* stats, const float* gradOut,
                                                                 const float* inverse) {
  const int64_t row = (int64_t)gridDim.x - 1 - blockIdx.x;     // the last rows, which the forward pass left in L2, first
  const T* x = logits + row * ld;
  T* g = grad + row * gradLd;
  const float slope = stats[2 * rows + row];
  const float c = slope * (*inverse) * (*gradOut);
  const bool zero = slope == 0.f || c == 0.f;
  const float m = stats[row], is = -c * stats[rows + row];
  const int64_t tok = tokens[row];
  auto one = [&](int j, float xj) -> float {
    if (j >= vocab || zero) return 0.f;
    const float p = gradExp<T>(xj - m) * is;
    return j == tok ? p + c : p;
  };
  const Span sp = spanOf(g, width);
  uint4* out = reinterpret_cast<uint4*>(g + sp.head);
  const int stride = (int)gridDim.y * kThreads;
  for (int i = (int)blockIdx.y * kThreads + threadIdx.x; i < sp.vecs; i += U * stride) {
    uint4 q[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u * stride >= sp.vecs || zero) continue;
      if (SAME) {
        q[u] = reinterpret_cast<const uint4*>(x + sp.head)[i + u * stride];
      } else {
        T* e = reinterpret_cast<T*>(&q[u]);
#pragma unroll
        for (int k = 0; k < kVec<T>; ++k) e[k] = x[sp.head + (i + u * stride) * kVec<T> + k];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u * stride >= sp.vecs) continue;
      if (zero) { out[i + u * stride] = make_uint4(0, 0, 0, 0); continue; }
      const int j0 = sp.head + (i + u * stride) * kVec<T>;
      float f[kVec<T>];
      unpack<T>(q[u], f);
      if (j0 + kVec<T> <= vocab && (tok < j0 || tok >= j0 + kVec<T>)) {
#pragma unroll
        for (int k = 0; k < kVec<T>; ++k) f[k] = gradExp<T>(f[k] - m) * is;
      } else {
#pragma unroll
        for (int k = 0; k < kVec<T>; ++k) f[k] = one(j0 + k, f[k]);
      }
      out[i + u * stride] = pack<T>(f);
    }
  }
  if (blockIdx.y == 0) {
    const int tail = sp.head + sp.vecs * kVec<T>, h = threadIdx.x, t = tail + (int)threadIdx.x;
    if (h < sp.head) g[h] = fromFloat<T>(one(h, zero ? 0.f : toFloat(x[h])));
    if (t < width) g[t] = fromFloat<T>(one(t, zero ? 0.f : toFloat(x[t])));
  }
}

// Rows that the threads walk in two turns or fewer take the form with one piece in flight.
template <class T> bool shortRow(int n) { return n <= 2 * kVec<T> * kThreads; }

// CTAs per row: few rows are shared by up to eight, as long as there are no more than six an SM and each keeps two turns of its loads
// (one row of 131072 bf16 logits, whole forward pass: 8 us; one CTA needs 23 us to read it).
template <class T>
int rowSplit(int64_t rows, int n) {
  int r = 1;
  while (r < 8 && rows * r * 2 <= 148 * 6 && n / (r * 2) >= 2 * kVec<T> * kThreads) r *= 2;
  return r;
}

template <class T>
void forward(const void* logits, int64_t rows, int64_t ld, int vocab, const RowInputs& in, int mean, float* logp, float* stats, float* loss, float* inverse,
             cudaStream_t s) {
  const T* z = static_cast<const T*>(logits);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  cfg.attrs = &attr;
  cfg.stream = s;
  if (rows > 0) {
    const int shares = rowSplit<T>(rows, vocab);
    cfg.gridDim = dim3((unsigned)rows, (unsigned)shares);
    cfg.blockDim = dim3(kThreads);
    attr.val.clusterDim.x = 1; attr.val.clusterDim.y = shares; attr.val.clusterDim.z = 1;
    cfg.numAttrs = shares > 1 ? 1 : 0;
    auto* kernel = shares > 1 ? policyForwardKernel<T, kUnroll, true> : shortRow<T>(vocab) ? policyForwardKernel<T, 1, false> : policyForwardKernel<T, kUnroll, false>;
    cudaLaunchKernelEx(&cfg, kernel, z, rows, ld, vocab, stats);
  }
  const int ctas = rows <= kRowThreads ? 1 : rows >= 8 * kRowThreads ? 8 : (int)((rows + kRowThreads - 1) / kRowThreads);
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(kRowThreads);
  attr.val.clusterDim.x = ctas; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
  cfg.numAttrs = ctas > 1 ? 1 : 0;
  cudaLaunchKernelEx(&cfg, policyRowsKernel<T>, z, rows, ld, vocab, in, mean, logp, stats, loss, inverse);
}

template <class T, bool SAME>
void backwardAs(const void* logits, int64_t rows, int64_t ld, void* grad, int64_t gradLd, int vocab, int width, const int64_t* tokens, const float* stats,
                const float* gradOut, const float* inverse, cudaStream_t s) {
  auto* kernel = shortRow<T>(width) ? policyBackwardKernel<T, 1, SAME> : policyBackwardKernel<T, kUnroll, SAME>;
  kernel<<<dim3((unsigned)rows, (unsigned)rowSplit<T>(rows, width)), kThreads, 0, s>>>(static_cast<const T*>(logits), rows, ld, static_cast<T*>(grad), gradLd,
                                                                                       vocab, width, tokens, stats, gradOut, inverse);
}

template <class T>
void backward(const void* logits, int64_t rows, int64_t ld, void* grad, int64_t gradLd, int vocab, int width, const int64_t* tokens, const float* stats,
              const float* gradOut, const float* inverse, cudaStream_t s) {
  const bool same = ((reinterpret_cast<uintptr_t>(logits) ^ reinterpret_cast<uintptr_t>(grad)) & 15u) == 0 && ((ld - gradLd) * (int64_t)sizeof(T)) % 16 == 0;
  (same ? backwardAs<T, true> : backwardAs<T, false>)(logits, rows, ld, grad, gradLd, vocab, width, tokens, stats, gradOut, inverse, s);
}

mcclResult_t launchedOk() { return cudaGetLastError() == cudaSuccess ? mcclSuccess : mcclSystemError; }
bool shaped(int64_t rows, int64_t ld, int vocab, int width) { return rows >= 0 && rows <= INT32_MAX && vocab > 0 && width >= vocab && ld >= width; }

}  // namespace

extern "C" {

mcclResult_t mcclPolicyLossForward(const void* logits, mcclDataType_t dt, int64_t rows, int64_t ld, int vocab, const int64_t* tokens, const float* oldLogp,
                                   const float* refLogp, const float* advantages, const void* weights, int boolWeights, double clipLow, double clipHigh,
                                   double klCoef, int mean, float* logp, float* stats, float* loss, float* inverse, mcclStream_t stream) {
  if (!shaped(rows, ld, vocab, vocab) || !loss || !inverse) return mcclInvalidArgument;
  if (rows > 0 && (!logits || !tokens || !oldLogp || !advantages || !logp || !stats)) return mcclInvalidArgument;
  const RowInputs in{tokens, oldLogp, refLogp, advantages, weights, boolWeights, clipLow, clipHigh, klCoef};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (dt != mcclBfloat16 && dt != mcclFloat16 && dt != mcclFloat32) return mcclInvalidArgument;
  auto* fn = dt == mcclBfloat16 ? forward<__nv_bfloat16> : dt == mcclFloat16 ? forward<__half> : forward<float>;
  fn(logits, rows, ld, vocab, in, mean, logp, stats, loss, inverse, s);
  return launchedOk();
}

mcclResult_t mcclPolicyLossBackward(const void* logits, mcclDataType_t dt, int64_t rows, int64_t ld, void* grad, int64_t gradLd, int vocab, int width,
                                    const int64_t* tokens, const float* stats, const float* gradOut, const float* inverse, mcclStream_t stream) {
  if (!shaped(rows, ld, vocab, width) || gradLd < width) return mcclInvalidArgument;
  if (dt != mcclBfloat16 && dt != mcclFloat16 && dt != mcclFloat32) return mcclInvalidArgument;
  if (rows == 0) return mcclSuccess;
  if (!logits || !grad || !tokens || !stats || !gradOut || !inverse) return mcclInvalidArgument;
  auto* fn = dt == mcclBfloat16 ? backward<__nv_bfloat16> : dt == mcclFloat16 ? backward<__half> : backward<float>;
  fn(logits, rows, ld, grad, gradLd, vocab, width, tokens, stats, gradOut, inverse, reinterpret_cast<cudaStream_t>(stream));
  return launchedOk();
}

}  // extern "C"

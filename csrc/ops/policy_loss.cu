// Clipped policy loss with a KL term over the logits of a language-model head, for tuning by rewards.
//   lp   = z[a] - logsumexp(z)                       the token's log-probability now
//   r    = exp(lp - old)                             against the policy that sampled it
//   l    = -min(r A, clamp(r, 1 - lo, 1 + hi) A) + beta (exp(ref - lp) - (ref - lp) - 1)
//   loss = sum of w l, divided by the sum of w where the mean is wanted
//   d loss / d z[j] = c ([j = a] - p[j]),  c = w (d l / d lp) / sum of w,  d l / d lp = (-r A where r A is the smaller, else 0) + beta (1 - exp(ref - lp))
// Forward: one CTA per row, one pass with a running maximum and sum of exponentials (online_softmax.cuh); what the row's scalar
// terms need is worked out once, in 64 bits: lp is a difference of numbers ten times its rounding apart from the reference's.  The
// rows' terms have both signs, so their sum is kept in 64 bits too.  Backward: reads the logits again and writes the gradient, a
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

template <class T, int U>
__global__ void __launch_bounds__(kThreads, 6) policyForwardKernel(const T* logits, int64_t rows, int64_t ld, int vocab, RowInputs in, float* logp,
                                                                   double* term, float* stats) {
  __shared__ MaxSum warpAcc[kThreads / 32];
  const int64_t row = blockIdx.x;
  const T* x = logits + row * ld;
  MaxSum acc{kLowest, 0.f};
  const Span sp = spanOf(x, vocab);
  const uint4* v = reinterpret_cast<const uint4*>(x + sp.head);
  for (int i = threadIdx.x; i < sp.vecs; i += U * kThreads) {
    uint4 q[U];
#pragma unroll
    for (int u = 0; u < U; ++u) if (i + u * kThreads < sp.vecs) q[u] = v[i + u * kThreads];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u * kThreads >= sp.vecs) continue;
      float f[kVec<T>];
      unpack<T>(q[u], f);
      pushAll(acc, f);
    }
  }
  const int tail = sp.head + sp.vecs * kVec<T>;
  if ((int)threadIdx.x < sp.head) push(acc, toFloat(x[threadIdx.x]));
  if (tail + (int)threadIdx.x < vocab) push(acc, toFloat(x[tail + threadIdx.x]));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    MaxSum other{__shfl_xor_sync(0xffffffffu, acc.m, o), __shfl_xor_sync(0xffffffffu, acc.s, o)};
    acc = combine(acc, other);
  }
  if ((threadIdx.x & 31) == 0) warpAcc[threadIdx.x >> 5] = acc;
  __syncthreads();
  if (threadIdx.x != 0) return;
  MaxSum t = warpAcc[0];
  for (int w = 1; w < kThreads / 32; ++w) t = combine(t, warpAcc[w]);
  const float nan = __int_as_float(0x7fffffff);
  if (t.m == INFINITY) t.s = nan;              // inf - inf in the exponent
  const int64_t tok = in.tokens[row];
  const float w = in.weight(row);
  const bool valid = tok >= 0 && tok < vocab;
  // A token that is no column: of no weight, or the loss and the row's gradient are NaN.
  const double lp = valid ? (double)toFloat(x[tok]) - (double)t.m - log((double)t.s) : w == 0.f ? 0. : (double)nan;
  logp[row] = (float)lp;
  double l = 0., slope = 0.;
  if (w != 0.f) {
    const double a = in.advantages[row], r = exp(lp - (double)in.old[row]);
    const double plain = r * a, held = fmin(fmax(r, 1. - in.lo), 1. + in.hi) * a;
    l = plain > held ? -held : -plain;
    slope = plain > held ? 0. : -plain;        // of equals, and of NaN, the unclamped one
    if (in.ref != nullptr) {
      const double d = (double)in.ref[row] - lp, e = exp(d);
      l += in.beta * (e - d - 1.);
      slope += in.beta * (1. - e);
    }
    l *= w;
    slope *= w;
  }
  term[row] = l;
  stats[row] = t.m;
  stats[rows + row] = 1.f / t.s;
  stats[2 * rows + row] = (float)slope;
}

// *loss = sum of the terms [/ sum of the weights], *inverse = one over what it was divided by, in a fixed order.  A batch whose
// weights add up to zero has loss zero and no gradient.
__global__ void __launch_bounds__(1024) policyReduceKernel(const double* term, int64_t rows, RowInputs in, int mean, float* loss, float* inverse) {
  __shared__ double accT[32], accW[32];
  double t = 0., w = 0.;
  for (int64_t i = threadIdx.x; i < rows; i += 4 * 1024) {
    double x[4];
    float y[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const bool in_ = i + u * 1024 < rows;
      x[u] = in_ ? term[i + u * 1024] : 0.;
      y[u] = in_ && mean ? in.weight(i + u * 1024) : 0.f;
    }
    t += (x[0] + x[1]) + (x[2] + x[3]);
    w += ((double)y[0] + y[1]) + ((double)y[2] + y[3]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) { t += __shfl_xor_sync(0xffffffffu, t, o); w += __shfl_xor_sync(0xffffffffu, w, o); }
  if ((threadIdx.x & 31) == 0) { accT[threadIdx.x >> 5] = t; accW[threadIdx.x >> 5] = w; }
  __syncthreads();
  if (threadIdx.x >= 32) return;
  t = accT[threadIdx.x];
  w = accW[threadIdx.x];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) { t += __shfl_xor_sync(0xffffffffu, t, o); w += __shfl_xor_sync(0xffffffffu, w, o); }
  if (threadIdx.x != 0) return;
  const double over = !mean ? 1. : w == 0. ? 0. : 1. / w;
  *loss = over == 0. ? 0.f : (float)(t * over);
  *inverse = (float)over;
}

// exp for a gradient in T: one with the type's precision.
template <class T> __device__ __forceinline__ float gradExp(float x) { return __expf(x); }
template <> __device__ __forceinline__ float gradExp<float>(float x) { return expf(x); }

// blockIdx.y: which slice of the row.  SAME: a row's 16-byte boundaries lie at the same elements in the logits and in the gradient.
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

// CTAs per row in the backward pass: few rows are shared by up to eight, as long as there are no more than six an SM and each keeps
// two turns of its loads.
template <class T>
int rowSplit(int64_t rows, int n) {
  int r = 1;
  while (r < 8 && rows * r * 2 <= 148 * 6 && n / (r * 2) >= 2 * kVec<T> * kThreads) r *= 2;
  return r;
}

template <class T>
void forward(const void* logits, int64_t rows, int64_t ld, int vocab, const RowInputs& in, float* logp, double* term, float* stats, cudaStream_t s) {
  auto* kernel = shortRow<T>(vocab) ? policyForwardKernel<T, 1> : policyForwardKernel<T, kUnroll>;
  kernel<<<(unsigned)rows, kThreads, 0, s>>>(static_cast<const T*>(logits), rows, ld, vocab, in, logp, term, stats);
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
                                   double klCoef, int mean, float* logp, double* term, float* stats, float* loss, float* inverse, mcclStream_t stream) {
  if (!shaped(rows, ld, vocab, vocab) || !loss || !inverse) return mcclInvalidArgument;
  if (rows > 0 && (!logits || !tokens || !oldLogp || !advantages || !logp || !term || !stats)) return mcclInvalidArgument;
  const RowInputs in{tokens, oldLogp, refLogp, advantages, weights, boolWeights, clipLow, clipHigh, klCoef};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (dt != mcclBfloat16 && dt != mcclFloat16 && dt != mcclFloat32) return mcclInvalidArgument;
  if (rows > 0) {
    auto* fn = dt == mcclBfloat16 ? forward<__nv_bfloat16> : dt == mcclFloat16 ? forward<__half> : forward<float>;
    fn(logits, rows, ld, vocab, in, logp, term, stats, s);
  }
  policyReduceKernel<<<1, 1024, 0, s>>>(term, rows, in, mean, loss, inverse);
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

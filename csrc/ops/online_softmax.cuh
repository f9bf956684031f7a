// A running maximum and sum of exponentials over a row of logits: one pass over the data.
#pragma once

#include <stdint.h>

#include "f32x2.cuh"

namespace mccl {

struct MaxSum { float m, s; };                 // running maximum and sum of exp(x - m)
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLowest = -3.402823466e38f;    // a maximum of nothing: not above any finite number, and minus itself zero
__device__ __forceinline__ MaxSum combine(MaxSum a, MaxSum b) {
  const float m = fmaxf(a.m, b.m);
  return MaxSum{m, a.s * __expf(a.m - m) + b.s * __expf(b.m - m)};
}
// Values enter one after another: s = s exp(m - x) + 1 where x is a new maximum and s + exp(x - m) where not.  The maximum
// is subtracted before anything is scaled: exp(x - m) as 2^(x log2e - m log2e) would save an instruction, but it rounds
// m log2e (an error of |m| 2^-24 in every exponent) and overflows for logits near the type's lowest value, which masks are made
// of.
__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ void add(MaxSum& a, bool up, float e) { a.s = up ? __fmaf_rn(a.s, e, 1.f) : __fadd_rn(a.s, e); }
__device__ __forceinline__ void push(MaxSum& a, float x) {
  add(a, x > a.m, ex2(-fabsf((x - a.m) * kLog2e)));
  a.m = fmaxf(a.m, x);
}
// N of them.  Instructions bound the pass here, at eight values of nine slots each a turn (cross-entropy of 8192 x 50257: 201 us):
// the maxima first, then differences and products two at a time, then the sums, predicated: 148 us, 5.6 TB/s.  (With a
// branch for a new maximum, which some lane of a warp takes nearly always: 254 us.)
template <int N>
__device__ __forceinline__ void pushAll(MaxSum& a, const float (&f)[N]) {
  float m[N + 1], e[N];
  m[0] = a.m;
#pragma unroll
  for (int k = 0; k < N; ++k) m[k + 1] = fmaxf(m[k], f[k]);
#pragma unroll
  for (int k = 0; k < N; k += 2) {
    float d0, d1;
    split((f2(f[k], f[k + 1]) + f2(-m[k], -m[k + 1])) * f2(kLog2e), &d0, &d1);
    e[k] = ex2(-fabsf(d0));
    e[k + 1] = ex2(-fabsf(d1));
  }
#pragma unroll
  for (int k = 0; k < N; ++k) add(a, f[k] > m[k], e[k]);
  a.m = m[N];
}

// The part of a row between its first and last 16-byte boundary: [head, head + (16 / sizeof(T)) * vecs) of n elements.
struct Span { int head, vecs; };
template <class T>
__device__ __forceinline__ Span spanOf(const T* x, int n) {
  constexpr int kVec = 16 / (int)sizeof(T);
  int head = (int)((16u - (uint32_t)(reinterpret_cast<uintptr_t>(x) & 15u)) & 15u) / (int)sizeof(T);
  if (head > n) head = n;
  return Span{head, (n - head) / kVec};
}

}  // namespace mccl

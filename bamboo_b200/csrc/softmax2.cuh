// Softmax in base 2.  With k = scale * log2(e) the kernels sum 2^(k x - r) for an INTEGER reference r: partial sums with different references
// meet exactly (powers of two).  soft_add keeps r >= max(k x); where r is the maximum of a part of the logits only, the caller bounds
// the sum that may come of it.  A row is kept as the pair (r, s): softmax_j = 2^(k x_j - r) / s, log
// softmax_j = (k x_j - r - log2 s) ln 2, the latter once per row in 64 bits.  k comes in two parts (K2): rounded to 32 bits it would
// be another temperature, 1.3e-8 off, which moves every log-probability of a sequence to the same side (measured on four
// sequences of 1024 tokens: the sum of log-ratios 2.7e-5 off, in two parts 2e-6, which is the rounding of the log-probabilities).
// What is left is ex2.approx: over arguments in (-1, 0] its results are 2.2e-8 too small in the mean, which puts up to 3e-8 on
// every log-probability (a softmax in 32 bits over logits divided by the temperature: 2e-8 to 2e-7).
#pragma once
#include "common.cuh"
#include <math.h>

// k = hi + lo, hi with 16 significant bits (x hi is exact for a bf16 x), lo > 0 (so that -inf stays -inf)
struct K2 { float hi, lo; };
inline K2 split_k(double scale) {
  const double k = scale * 1.4426950408889634;
  int e;
  const double m = frexp(k, &e);                       // [0.5, 1)
  double hi = ldexp(floor(m * 65536.0), e - 16);
  if (hi == k) hi = ldexp(floor(m * 65536.0) - 1.0, e - 16);
  return {(float)hi, (float)(k - hi)};
}

namespace bb {

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// k x - r
__device__ __forceinline__ float expo(float x, K2 k, float r) { return fmaf(x, k.lo, fmaf(x, k.hi, -r)); }
__device__ __forceinline__ float2 expo2(float2 x, K2 k, float r) {
  return fma2(x, make_float2(k.lo, k.lo), fma2(x, make_float2(k.hi, k.hi), make_float2(-r, -r)));
}

// Partial sums (r, s), r an integer or -inf (nothing yet)
__device__ __forceinline__ void soft_merge(float& r, float& s, float r2, float s2) {
  const float rn = fmaxf(r, r2);
  // (equal references add as they are: -inf - -inf would be NaN)
  s = (r == rn ? s : s * ex2(r - rn)) + (r2 == rn ? s2 : s2 * ex2(r2 - rn));
  r = rn;
}
// N (even, or 1) logits added to (r, s).  The reference is an integer only as far as a float's integers go: at 2^20 the rounding of k x
// to the reference's grid costs the exponent 2^-20, at 2^31 all of it (a mask of -1e10 would be 2^0 or 2^300, by chance).  So it is not taken from below
// `lowest`: logits down there add nothing to what stands above, and rows without any other are the caller's to look at again.
constexpr float SOFT_FAR = 0x1p20f;
template <int N> __device__ __forceinline__ void soft_add(float& r, float& s, const float* f, K2 k, float lowest) {
  float top = f[0];
#pragma unroll
  for (int i = 1; i < N; ++i) top = fmaxf(top, f[i]);
  const float rn = fmaxf(ceilf(expo(top, k, 0.f)), lowest);
  if (rn > r) { s *= ex2(r - rn); r = rn; }            // (nothing yet: 0 * 2^-inf)
  if constexpr (N == 1) {
    s += ex2(expo(f[0], k, r));
  } else {
    float2 sum = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const float2 t = expo2(make_float2(f[i], f[i + 1]), k, r);
      sum = add2(sum, make_float2(ex2(t.x), ex2(t.y)));
    }
    s += sum.x + sum.y;
  }
}

// k d for a difference of logits, which may be -inf
__device__ __forceinline__ float expo_gap(float d, K2 k) { return fmaf(d, k.lo, d * k.hi); }

// log softmax of logit x in 64 bits; a row without any finite logit (s = 0) has no distribution: -inf; s < 0: a row kept as its largest logit and
// the sum over differences from it
__device__ __forceinline__ double row_logp(float x, K2 k, float r, float s) {
  const double k2 = (double)k.hi + (double)k.lo;
  if (s == 0.f) return -INFINITY;
  if (s < 0.f) return ((double)x - (double)r) * k2 * 0.69314718055994531 - log((double)-s);
  return ((double)x * k2 - ((double)r + log2((double)s))) * 0.69314718055994531;
}

}  // namespace bb

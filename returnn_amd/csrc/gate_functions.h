// The gates' non-linearities.
#pragma once

#include <hip/hip_runtime.h>

namespace rtn {

// 1 / (1 + e^-x) (returnn/native_op.py:1102-1104) in float32, in 15 instructions; with expf and a division there are 32, a chain that a
// thread goes through three times per pair and step while nothing else runs on its SIMD.
//  * e^-x = 2^t (1 + r), t = -x log2 e as rounded, r = -x - t ln 2 what the rounding left out.
//  * 1 / d by a Newton step from the hardware's reciprocal; `lo` is what d = 1 + e lost by rounding.  The reciprocal is that of d / 4: the hardware
//    gives zero for what is below the normal numbers, as 1 / d is from x = -87.34 on.
// Error against 64 bits, 2-norm, of 2^20 arguments evenly spread over +-0.1, +-1, +-3, +-8 and +-20, with expf and a division / here: 4.4e-8 / 3.0e-8,
// 4.0e-8 / 2.9e-8, 3.8e-8 / 2.4e-8, 3.8e-8 / 1.9e-8, 3.5e-8 / 1.8e-8.  Largest in ulp: 2.1 / 1.2, 2.0 / 1.3, 2.1 / 2.1, 2.1 / 2.4,
// 2.5 / 3.1: where the result is small it is e^x, whose error is the hardware's and a rounding.
__device__ __forceinline__ float exp_f32(float w) {
  const float t = w * 1.44269504088896f;
  const float e = __builtin_amdgcn_exp2f(t);
  const float r = __builtin_fmaf(t, 1.904654299957767e-09f, __builtin_fmaf(t, -0.693147182464599609375f, w));  // ln 2 in two parts
  return __builtin_fmaf(e, r, e);
}
// what goes through exp_f32 (minimum keeps a NaN; at infinity r would be one)
__device__ __forceinline__ float sigmoid_exponent(float x) { return -__builtin_elementwise_minimum(x, 100.f); }
// 1 / d of a d of at least 1, about
__device__ __forceinline__ float reciprocal_f32(float d) { return 0.25f * __builtin_amdgcn_rcpf(0.25f * d); }
// sigmoid of x from e = exp_f32 of that, d = 1 + e and q = reciprocal_f32(d)
__device__ __forceinline__ float sigmoid_of(float x, float e, float d, float q) {
  const float lo = e - (d - 1.f);
  const float s = __builtin_fmaf(__builtin_fmaf(-lo, q, __builtin_fmaf(-d, q, 1.f)), q, q);
  return x < -88.72283f ? 0.f : s;  // (where e^-x is no float32 any more, down to minus infinity)
}
__device__ __forceinline__ float sigmoid_f32(float x) {
  const float e = exp_f32(sigmoid_exponent(x)), d = 1.f + e;
  return sigmoid_of(x, e, d, reciprocal_f32(d));
}

// tanh in float32 without a branch: both sides of |x| = 0.75, 23 instructions that the compiler puts between those of other gates.  (tanhf branches
// at 0.625: 16 and 28 instructions, both of them as soon as one lane is on the other side.)
//  * near: x + x u P(u), u = x^2, P of degree 5 by least squares of the relative error, reweighted to its maximum: 0.03 ulp.
//  * far: 1 - 2 / (1 + e^2|x|), what is subtracted is below 0.37, and so are its errors.
// Error against 64 bits, 2-norm and largest in ulp, of arguments evenly spread over +-0.1, +-1, +-3 and +-20, tanhf / here: 2.56e-8 / 2.54e-8, 3.43e-8 /
// 3.18e-8, 2.13e-8 / 2.10e-8, 1.24e-8 / 1.23e-8; 0.55 / 0.52, 1.38 / 1.31, 1.38 / 1.28, 1.30 / 1.23.  us per call, with tanhf / this, of arguments that
// nearly all were near: T = 32, 4 rows of n = 64 19.0 / 18.2; T = 300, 32 rows of n = 1024 1077 / 1071; T = 200, 3 rows of n = 2048 1235 / 1222.
__device__ __forceinline__ float tanh_exponent(float x) {
  const float a = __builtin_elementwise_minimum(__builtin_fabsf(x), 20.f);
  return a + a;
}
// tanh of x from q = 1 / (1 + exp_f32 of that)
__device__ __forceinline__ float tanh_of(float x, float q) {
  const float u = x * x;
  float p = __builtin_fmaf(u, 0.001736935111694038f, -0.007657254114747047f);
  p = __builtin_fmaf(u, p, 0.021452033892273903f);
  p = __builtin_fmaf(u, p, -0.053892724215984344f);
  p = __builtin_fmaf(u, p, 0.1333269476890564f);
  p = __builtin_fmaf(u, p, -0.33333316445350647f);
  const float near = __builtin_fmaf(u, x * p, x);
  const float far = __builtin_fmaf(q, -2.f, 1.f);
  return __builtin_copysignf(__builtin_fabsf(x) < 0.75f ? near : far, x);  // (of -0 as well, where the sum of `near` is +0)
}
__device__ __forceinline__ float tanh_f32(float x) { return tanh_of(x, __builtin_amdgcn_rcpf(1.f + exp_f32(tanh_exponent(x)))); }

// Gate non-linearities.  float32 runs keep to 32 bits (1e-5 relative is the bar there).  bfloat16 runs round every result to 8 bits of
// mantissa anyway, so they use the hardware exp2 and reciprocal (about 1 ulp of float32 each):
// sigmoid(x) = 1 / (1 + 2^(-x log2 e)), tanh(x) = 2 sigmoid(2x) - 1.  The latter's error is 2e-7 absolute: of an |x| below 1e-4 more than the rounding.
template <typename AT>
struct Act;

template <>
struct Act<float> {
  static __device__ __forceinline__ float sigmoid(float x) { return sigmoid_f32(x); }
  static __device__ __forceinline__ float tanh(float x) { return tanh_f32(x); }
};

template <>
struct Act<__bf16> {
  static __device__ __forceinline__ float sigmoid(float x) {
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * x));
  }
  static __device__ __forceinline__ float tanh(float x) {
    // (2 r - 1 as one fused multiply-add: 2 r is exact, so this is bit for bit r + r - 1)
    return __builtin_fmaf(2.f, __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-2.8853900817779268f * x)), -1.f);
  }
};

}  // namespace rtn

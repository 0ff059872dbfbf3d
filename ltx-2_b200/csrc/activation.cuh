// Activation functions and their derivatives on packed fp32 pairs (sm_100a).
//
// Both activations are z * sigmoid(u):  GELU-tanh with u = 2 sqrt(2/pi) (z + 0.044715 z^3),
// SiLU with u = z.  With e = 2^(-u log2 e) and s = 1 / (1 + e):
//   act(z) = z s,   act'(z) = s + z s (1 - s) u'(z).
// The exponential and the reciprocal are the approximate instructions (a few 2^-23 relative).
#pragma once

#include "ptx.cuh"

namespace ltxfp8 {

enum ActKind : int { kActNone = 0, kActGeluTanh = 1, kActSilu = 2 };

constexpr float kNegLog2e = -1.4426950408889634f;

// e = 2^(-u(z) log2 e); infinite where the sigmoid vanishes.
template <int kAct>
__device__ __forceinline__ float2 act_exp(const float2 z) {
  float2 a;
  if constexpr (kAct == kActGeluTanh) {
    const float c1 = kGeluC1, c3 = kGeluC3;
    a = __fmul2_rn(__ffma2_rn(__fmul2_rn(z, z), make_float2(c3, c3), make_float2(c1, c1)), z);
  } else {
    const float c = kNegLog2e;
    a = __fmul2_rn(z, make_float2(c, c));
  }
  return make_float2(ex2_approx(a.x), ex2_approx(a.y));
}

template <int kAct>
__device__ __forceinline__ float2 act_apply(const float2 z) {
  if constexpr (kAct == kActNone) {
    return z;
  } else {
    const float2 d = __fadd2_rn(act_exp<kAct>(z), make_float2(1.0f, 1.0f));
    return __fmul2_rn(z, make_float2(rcp_approx(d.x), rcp_approx(d.y)));
  }
}

// With q = z u'(z): act' = s + s (q - q s).  q - q s is one fused step, so 1 - s loses nothing
// where s is small; where s is near 1 the term is an absolute error of 2^-24 q in a value near 1.
// GELU's q is a cubic: |z| has to stay below 10^12 (act_grad_scale), or an infinite q meets 1 - s = 0
// or s = 0.  Where e vanishes, s has to be 1 exactly: the approximate reciprocal of 1.0 is 1.0, which
// test_act_extremes_gpu.py holds to (an ulp less would be 2^-24 q).  Forming q from at most z = 16, which
// would not need that, costs an instruction a value: 6143 x 16384 106.5 -> 110.5 us.
template <int kAct>
__device__ __forceinline__ float2 act_grad(const float2 z) {
  const float2 d = __fadd2_rn(act_exp<kAct>(z), make_float2(1.0f, 1.0f));
  const float2 s = make_float2(rcp_approx(d.x), rcp_approx(d.y));
  float2 q = z;
  if constexpr (kAct == kActGeluTanh) {
    constexpr float kU1 = 2.0f * 0.7978845608028654f, kU3 = 3.0f * 0.044715f * kU1;
    const float u1 = kU1, u3 = kU3;
    q = __fmul2_rn(z, __ffma2_rn(__fmul2_rn(z, z), make_float2(u3, u3), make_float2(u1, u1)));
  }
  const float2 v = __ffma2_rn(make_float2(-s.x, -s.y), q, q);
  return __ffma2_rn(s, v, s);
}

// The scale of a group of e4m3 codes that act_grad is taken of, at most 2^16 (|z| < 2^25): the
// smallest code but zero, 2^-9, is 128 there, where the derivative of either activation has become 0
// or 1 to fp32, so a larger scale changes nothing.  Infinity and NaN stay.
__device__ __forceinline__ float act_grad_scale(float s) { return isfinite(s) ? fminf(s, 65536.0f) : s; }

}  // namespace ltxfp8

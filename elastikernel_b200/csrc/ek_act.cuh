// Gate functions of the gated feed-forward block and their slopes, in fp32.
//
//   silu       f = z s(z),            f' = s + z s (1 - s)
//   gelu       f = z Phi(z),          f' = Phi + z phi(z)
//   gelu_tanh  f = z s(2u(z)),        f' = s + z s (1 - s) 2u'(z)
//              u = sqrt(2/pi) (z + 0.044715 z^3);  (1 + tanh u) / 2 = s(2u)
//
// s is the logistic function, Phi and phi the normal distribution and density.
// Phi is taken as erfc(-z / sqrt 2) / 2, which keeps its relative precision for
// negative z where 1 + erf cancels. u's argument is held within +-30, where s
// has long reached 0 or 1, so that z^3 cannot overflow into inf * 0, by comparisons
// that a NaN passes: a minimum or maximum would take the bound for it.
#pragma once
#include "ek_ptx.cuh"

namespace ek {

enum GateFn : int { kGateSilu = 0, kGateGelu = 1, kGateGeluTanh = 2 };

__device__ __forceinline__ float logistic_f(float z) { return __fdividef(1.0f, 1.0f + __expf(-z)); }

// s(2u(z)) and, with slope, z s (1 - s) 2u'(z)
__device__ __forceinline__ float gelu_tanh_s(float z, float& tail) {
  constexpr float k2 = 1.5957691216057308f, c = 0.044715f;  // 2 sqrt(2 / pi)
  const float zc = z < -30.0f ? -30.0f : z > 30.0f ? 30.0f : z, z2 = zc * zc;
  const float s = logistic_f(k2 * zc * (1.0f + c * z2));
  tail = zc * s * (1.0f - s) * k2 * (1.0f + 3.0f * c * z2);
  return s;
}

template <int kFn>
__device__ __forceinline__ float gate_f(float z) {
  if constexpr (kFn == kGateSilu) return z * logistic_f(z);
  if constexpr (kFn == kGateGelu) return z * (0.5f * erfcf(z * -0.70710678118654752f));
  float tail;
  return z * gelu_tanh_s(z, tail);
}

// f(z) and f'(z)
template <int kFn>
__device__ __forceinline__ void gate_f_df(float z, float& f, float& df) {
  if constexpr (kFn == kGateSilu) {
    const float s = logistic_f(z);
    f = z * s;
    df = s + f * (1.0f - s);
  } else if constexpr (kFn == kGateGelu) {
    const float cdf = 0.5f * erfcf(z * -0.70710678118654752f);
    f = z * cdf;
    df = cdf + z * (0.39894228040143268f * __expf(-0.5f * z * z));
  } else {
    float tail;
    const float s = gelu_tanh_s(z, tail);
    f = z * s;
    df = s + tail;
  }
}

// The gate function of a launch is a run-time choice: one uniform branch around
// a loop over registers, so the three forms share a kernel.
template <class Body>
__device__ __forceinline__ void with_gate(int fn, Body&& body) {
  if (fn == kGateSilu)
    body(std::integral_constant<int, kGateSilu>{});
  else if (fn == kGateGelu)
    body(std::integral_constant<int, kGateGelu>{});
  else
    body(std::integral_constant<int, kGateGeluTanh>{});
}

}  // namespace ek

// The gates of a gated linear layer: act(a) and act'(a) in float32.
//
//   silu       a s(a)                        s the logistic function
//   gelu       a Phi(a)                      Phi the normal distribution's
//   gelu_tanh  a s(2 c (a + k a^3))          c = sqrt(2 / pi), k = 0.044715: a / 2 (1 + tanh(c (a + k a^3)))
//   relu       max(a, 0)
//   sigmoid    s(a)
//
// s(v) = 1 / (1 + e^-v) and 1 - s(v) = 1 / (1 + e^v) are formed each by itself, and Phi from
// the complementary error function, so that small values keep their digits.
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

#include "lmp_hip_transformer.h"

namespace lmp_hip {
namespace {

// The larger of s(v) and s(-v) is 1 / (1 + e^-|v|), the smaller e^-|v| times that.  The
// reciprocal, of a number from 1 to 2, is the hardware's with one step of Newton's: within a unit.
__device__ __forceinline__ void logistic(float v, float& s, float& rest) {
  const float e = expf(-fabsf(v)), d = 1.0f + e, r = __builtin_amdgcn_rcpf(d);
  const float big = __builtin_fmaf(__builtin_fmaf(-d, r, 1.0f), r, r), small = e * big;
  s = v < 0 ? small : big;
  rest = v < 0 ? big : small;
}

template <int GATE>
__device__ __forceinline__ void gate_at(float a, float& act, float& slope) {
  constexpr float kTwoC = 1.5957691216057308f, kCube = 0.044715f;
  float s, rest;
  if constexpr (GATE == LMP_GATE_SILU) {
    logistic(a, s, rest);
    act = a * s;
    slope = s + act * rest;
  } else if constexpr (GATE == LMP_GATE_GELU) {
    s = 0.5f * erfcf(a * -0.70710678118654752f);
    act = a * s;
    slope = s + a * expf(a * a * -0.5f) * 0.39894228040143268f;
  } else if constexpr (GATE == LMP_GATE_GELU_TANH) {
    logistic(a * kTwoC * (1.0f + kCube * a * a), s, rest);
    act = a * s;
    // Past 64 act or rest is 0 (e^-19000): bounded, so that a * a stays finite beside it.
    const float b = fminf(fabsf(a), 64.0f);
    slope = s + act * rest * (kTwoC * (1.0f + 3.0f * kCube * b * b));
  } else if constexpr (GATE == LMP_GATE_RELU) {
    act = a < 0.0f ? 0.0f : a;
    slope = a > 0.0f ? 1.0f : 0.0f;
  } else {
    logistic(a, s, rest);
    act = s;
    slope = s * rest;
  }
}

// Calls f with the gate as a constant.
template <class F>
__host__ __device__ __forceinline__ auto with_gate(int gate, F&& f) {
  switch (gate) {
    case LMP_GATE_SILU: return f(std::integral_constant<int, LMP_GATE_SILU>{});
    case LMP_GATE_GELU: return f(std::integral_constant<int, LMP_GATE_GELU>{});
    case LMP_GATE_GELU_TANH: return f(std::integral_constant<int, LMP_GATE_GELU_TANH>{});
    case LMP_GATE_RELU: return f(std::integral_constant<int, LMP_GATE_RELU>{});
    default: return f(std::integral_constant<int, LMP_GATE_SIGMOID>{});
  }
}

}  // namespace
}  // namespace lmp_hip

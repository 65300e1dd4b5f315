// activation.cuh -- the activations of the gated projections and their derivatives, in f32.
#pragma once
#include <cuda_runtime.h>

#include "gicc/ops.hpp"

namespace gicc {
namespace act {

// x / (1 + e^-t).  A t far below zero makes the exponential infinite and the quotient 0.
__device__ __forceinline__ float logistic(float t) { return __fdividef(1.0f, 1.0f + __expf(-t)); }

// sqrt(2/pi), and 0.044715 of the tanh form of GELU
constexpr float kGeluK = 0.7978845608028654f;
constexpr float kGeluC = 0.044715f;

__device__ __forceinline__ float value(float g, int kind) {
  if (kind == ops::ACT_SILU) return g * logistic(g);
  if (kind == ops::ACT_GELU) return 0.5f * g * (1.0f + erff(g * 0.7071067811865476f));
  // 0.5 (1 + tanh z) = logistic(2 z)
  return g * logistic(2.0f * kGeluK * g * (1.0f + kGeluC * g * g));
}

// act(g), and its derivative in *d
__device__ __forceinline__ float value_grad(float g, int kind, float* d) {
  if (kind == ops::ACT_SILU) {
    const float s = logistic(g);
    *d = s * (1.0f + g * (1.0f - s));
    return g * s;
  }
  if (kind == ops::ACT_GELU) {
    const float phi = 0.5f * (1.0f + erff(g * 0.7071067811865476f));
    *d = phi + g * 0.3989422804014327f * __expf(-0.5f * g * g);
    return g * phi;
  }
  const float s = logistic(2.0f * kGeluK * g * (1.0f + kGeluC * g * g));
  *d = s + g * 2.0f * s * (1.0f - s) * kGeluK * (1.0f + 3.0f * kGeluC * g * g);
  return g * s;
}

}  // namespace act
}  // namespace gicc

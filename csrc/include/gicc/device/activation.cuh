// activation.cuh -- the activations of the gated projections and their derivatives, in f32.
#pragma once
#include <cuda_runtime.h>

#include "gicc/ops.hpp"

namespace gicc {
namespace act {

// 1 / (1 + e^-t).  0 where t is below -87.3: __fdividef gives 0 for a divisor beyond 2^126.  (By the
// exponential of -|t| it would go on, but 8192 x 1024 -> 8192 took 227 to 243 us instead of 216 with it,
// for values of silu below 1.1e-36.)
__device__ __forceinline__ float logistic(float t) { return __fdividef(1.0f, 1.0f + __expf(-t)); }

// Phi(g) = (1 + erf(g / sqrt 2)) / 2, and e^(-g^2/2) in *e.  The sum with erf cancels where g is far
// below zero (relative error 4 % at -5), so the tail is computed itself, in the form of Hastings'
// approximations (Abramowitz and Stegun 7.1.26): Phi(-|g|) = e^(-g^2/2) w P(w), w = 1 / (1 + 0.3 |g|).  P is
// our own minimax fit of degree 7 (relative error 2^-21 in f32 arithmetic, |g| <= 13.5, beyond which f32 has no
// such value).  8192 x 1024 -> 8192, beside the sum with erff in the same run: this form 265 us against
// 264, CUDA's erfcf 432 against 298.
__device__ __forceinline__ float normal_cdf(float g, float* e) {
  *e = __expf(-0.5f * g * g);
  const float w = __fdividef(1.0f, fmaf(0.3f, fabsf(g), 1.0f));
  float p = 0.03593176f;
  p = fmaf(p, w, -0.15827608f);
  p = fmaf(p, w, 0.20820672f);
  p = fmaf(p, w, -0.05539394f);
  p = fmaf(p, w, 0.12946925f);
  p = fmaf(p, w, 0.09963748f);
  p = fmaf(p, w, 0.12079836f);
  p = fmaf(p, w, 0.11962639f);
  const float tail = p * w * *e;
  return g < 0.0f ? tail : 1.0f - tail;
}

// sqrt(2/pi), and 0.044715 of the tanh form of GELU
constexpr float kGeluK = 0.7978845608028654f;
constexpr float kGeluC = 0.044715f;

__device__ __forceinline__ float value(float g, int kind) {
  if (kind == ops::ACT_SILU) return g * logistic(g);
  if (kind == ops::ACT_GELU) {
    float e;
    return g * normal_cdf(g, &e);
  }
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
    float e;
    const float phi = normal_cdf(g, &e);
    *d = phi + g * 0.3989422804014327f * e;
    return g * phi;
  }
  const float s = logistic(2.0f * kGeluK * g * (1.0f + kGeluC * g * g));
  // s (1 - s) first, and g^2 bounded: it is 0 long before they overflow
  *d = s + 2.0f * s * (1.0f - s) * g * kGeluK * (1.0f + 3.0f * kGeluC * fminf(g * g, 1e30f));
  return g * s;
}

}  // namespace act
}  // namespace gicc

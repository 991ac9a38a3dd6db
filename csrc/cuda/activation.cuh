// The activations of the linear operator and their derivatives, in 32 bits.
#pragma once
#include "layers.cuh"

namespace hipress {

__device__ __forceinline__ float exp2_fast(float x) {   // within 2^-22 of it
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Phi(p) and the density phi(p) of the normal distribution.  erfc(z) for z >= 0 by Abramowitz
// and Stegun's formula 7.1.26, within 1.5e-7: far below half a unit of the 16-bit results, and
// two special-function instructions an element where erff() takes a dozen more.
__device__ __forceinline__ void normal_cdf(float p, float& cdf, float& pdf) {
  const float z = fabsf(p) * 0.7071067811865476f;
  const float t = rcp_fast(fmaf(0.3275911f, z, 1.f)), e = exp2_fast(p * p * -0.7213475204444817f);
  float q = fmaf(t, 1.061405429f, -1.453152027f);
  q = fmaf(t, q, 1.421413741f);
  q = fmaf(t, q, -0.284496736f);
  q = fmaf(t, q, 0.254829592f);
  q *= 0.5f * t * e;
  cdf = p > 0.f ? 1.f - q : q;
  pdf = 0.3989422804014327f * e;
}

// the tanh form is p times the logistic function of 2 u
constexpr float kTanhC = 0.7978845608028654f, kTanhA = 0.044715f, kLog2e = 1.4426950408889634f;
__device__ __forceinline__ float tanh_gate(float p) {
  const float u = kTanhC * fmaf(kTanhA * p * p, p, p);
  return rcp_fast(1.f + exp2_fast(-2.f * kLog2e * u));
}

template <int ACT>
__device__ __forceinline__ float activate(float p) {
  if (ACT == HP_ACT_RELU) return p > 0.f ? p : (p != p ? p : 0.f);
  if (ACT == HP_ACT_GELU) {
    float c, d;
    normal_cdf(p, c, d);
    return p * c;
  }
  if (ACT == HP_ACT_GELU_TANH) return p * tanh_gate(p);
  return p;
}

template <int ACT>
__device__ __forceinline__ float slope(float p) {
  if (ACT == HP_ACT_RELU) return p > 0.f ? 1.f : 0.f;
  if (ACT == HP_ACT_GELU) {
    float c, d;
    normal_cdf(p, c, d);
    return fmaf(p, d, c);
  }
  if (ACT == HP_ACT_GELU_TANH) {
    const float g = tanh_gate(p), du = 2.f * kTanhC * fmaf(3.f * kTanhA, p * p, 1.f);
    return fmaf(p * g * (1.f - g), du, g);
  }
  return 1.f;
}

}  // namespace hipress

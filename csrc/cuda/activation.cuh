// The activations of the linear operator and their derivatives, in 32 bits.
#pragma once
#include "layers.cuh"

namespace hipress {

// Phi(p) and the density phi(p) of the normal distribution
__device__ __forceinline__ void normal_cdf(float p, float& cdf, float& pdf) {
  pdf = 0.3989422804014327f * expf(-0.5f * p * p);
  cdf = 0.5f * erfcf(-0.7071067811865476f * p);
}

template <int ACT>
__device__ __forceinline__ float activate(float p) {
  if (ACT == HP_ACT_RELU) return p > 0.f ? p : (p != p ? p : 0.f);
  if (ACT == HP_ACT_GELU) {
    float c, d;
    normal_cdf(p, c, d);
    return p * c;
  }
  if (ACT == HP_ACT_GELU_TANH) {
    const float u = 0.7978845608028654f * fmaf(0.044715f * p * p, p, p);
    return 0.5f * p * (1.f + tanhf(u));
  }
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
    const float t = tanhf(0.7978845608028654f * fmaf(0.044715f * p * p, p, p));
    return fmaf(0.5f * p * (1.f - t * t), 0.7978845608028654f * fmaf(3.f * 0.044715f, p * p, 1.f), 0.5f * (1.f + t));
  }
  return 1.f;
}

}  // namespace hipress

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

// The normal distribution's tail Q(|p|), and e = exp(-p p / 2).  Q is e t times a polynomial in
// t = 1 / (1 + a |p|) of degree 5, a and the coefficients chosen for the least largest relative error
// of Q exp(p p / 2) over 0..14 (a linear program for each a): 4.2e-6 in 32 bits, 2^-17.9.  Relative,
// since GELU of a negative p is p times the tail itself; e's exponent of up to 122 in 32 bits adds
// 2^-16.6 at -13.  Half a unit of fp16 is 2^-12 of a value at least.  Two special-function
// instructions an element where erff() takes a dozen more.
__device__ __forceinline__ float normal_tail(float p, float& e) {
  const float t = rcp_fast(fmaf(0.3081703f, fabsf(p), 1.f));
  e = exp2_fast(p * p * -0.7213475204444817f);
  float q = fmaf(t, -0.0753871202f, 0.189065352f);
  q = fmaf(t, q, 0.00776021322f);
  q = fmaf(t, q, 0.136384055f);
  q = fmaf(t, q, 0.118987784f);
  q = fmaf(t, q, 0.12318778f);
  return q * t * e;
}

// the tanh form is p times the logistic function of 2 u
constexpr float kTanhC = 0.7978845608028654f, kTanhA = 0.044715f, kLog2e = 1.4426950408889634f;
__device__ __forceinline__ float tanh_gate(float p) {
  const float u = kTanhC * fmaf(kTanhA * p * p, p, p);
  return rcp_fast(1.f + exp2_fast(-2.f * kLog2e * u));
}

template <int ACT>
__device__ __forceinline__ float activate(float p) {
  if (ACT == HP_ACT_RELU) return p < 0.f ? 0.f : p;   // NaN stays
  if (ACT == HP_ACT_GELU) {   // p Phi(p) = max(p, 0) - |p| Q(|p|), whose second term is none at infinity
    float e;
    const float q = normal_tail(p, e);
    return fmaf(-fminf(fabsf(p), 64.f), q, fmaxf(p, 0.f));
  }
  if (ACT == HP_ACT_GELU_TANH) return p * tanh_gate(p);
  return p;
}

// p comes back from 16 bits, where a large one may have become an infinity.  Beyond 64 either form is
// zero or one to the last bit, and every factor below is finite.
template <int ACT>
__device__ __forceinline__ float slope(float p) {
  if (ACT == HP_ACT_RELU) return p > 0.f ? 1.f : 0.f;
  if (ACT == HP_ACT_GELU) {
    float e;
    const float q = normal_tail(p, e), near = fminf(fmaxf(p, -64.f), 64.f);   // e is no number where p is none
    return fmaf(near * 0.3989422804014327f, e, p > 0.f ? 1.f - q : q);
  }
  if (ACT == HP_ACT_GELU_TANH) {
    const float g = tanh_gate(p), near = fminf(fmaxf(p, -64.f), 64.f);        // nor is g
    const float du = 2.f * kTanhC * fmaf(3.f * kTanhA, near * near, 1.f);
    return fmaf(near * g * (1.f - g), du, g);
  }
  return 1.f;
}

}  // namespace hipress

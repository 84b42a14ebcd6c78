// Activations of a gated block and their derivatives, and the approximate exponential that
// epilogues use.
#pragma once

#include <cuda_runtime.h>

#include "ffn.h"

namespace mb {

namespace {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 1 / (1 + exp(-x)).  FAST: approximate exponential, a few 2^-22 of it for the |x| below 16 that
// bfloat16 results show; the approximate reciprocal is off by one unit in the last place.
template <bool FAST>
__device__ __forceinline__ float sigmoid(float x) {
  return rcp_approx(1.f + (FAST ? exp2_approx(-kLog2e * x) : expf(-x)));
}

// The normal distribution function and its density.  FAST: formula 7.1.26 of Abramowitz and
// Stegun, "Handbook of Mathematical Functions" (1964), off by less than 1.5e-7 / 2, in its form
// for the tail, whose exponential is the density's.  Of the tail itself that is 0.16% at -5, where x p is
// -1.4e-6, and 1% at -8, where it is -5e-15.
template <bool FAST>
__device__ __forceinline__ void normal(float x, float& p, float& density) {
  constexpr float kRoot2Pi = 0.3989422804014327f;  // 1 / sqrt(2 pi)
  if constexpr (FAST) {
    const float z = fabsf(x) * 0.70710678f;
    const float t = rcp_approx(fmaf(0.3275911f, z, 1.f));
    const float e = exp2_approx(-0.5f * kLog2e * x * x);
    float q = fmaf(1.061405429f, t, -1.453152027f);
    q = fmaf(q, t, 1.421413741f);
    q = fmaf(q, t, -0.284496736f);
    q = fmaf(q, t, 0.254829592f);
    const float tail = 0.5f * q * t * e;
    p = x < 0.f ? tail : 1.f - tail;
    density = kRoot2Pi * e;
  } else {
    p = 0.5f * erfcf(-0.70710678f * x);
    density = kRoot2Pi * expf(-0.5f * x * x);
  }
}

constexpr float kTanhScale = 0.7978845608028654f, kTanhCubic = 0.044715f;  // sqrt(2 / pi)

// act(x); 0.5 (1 + tanh(u)) is sigmoid(2 u).
template <int ACT, bool FAST>
__device__ __forceinline__ float activation(float x) {
  if constexpr (ACT == kSilu) return x * sigmoid<FAST>(x);
  if constexpr (ACT == kGelu) {
    float p, d;
    normal<FAST>(x, p, d);
    return x * p;
  }
  return x * sigmoid<FAST>(2.f * kTanhScale * fmaf(kTanhCubic * x * x, x, x));
}

// act(x) and its derivative.
template <int ACT, bool FAST>
__device__ __forceinline__ float activation_slope(float x, float& slope) {
  if constexpr (ACT == kSilu) {
    const float p = sigmoid<FAST>(x), y = x * p;
    slope = fmaf(y, 1.f - p, p);
    return y;
  }
  if constexpr (ACT == kGelu) {
    float p, d;
    normal<FAST>(x, p, d);
    slope = fmaf(x, d, p);
    return x * p;
  }
  // beyond 30 the sigmoid is 0 or 1, and its derivative's square must not overflow
  const float t = fminf(fmaxf(x, -30.f), 30.f), t2 = kTanhCubic * t * t;
  const float p = sigmoid<FAST>(2.f * kTanhScale * fmaf(t2, t, t)), y = x * p;
  slope = fmaf(y * (1.f - p), 2.f * kTanhScale * fmaf(3.f, t2, 1.f), p);
  return y;
}

// v = act(v) * w
template <bool FAST, int N>
__device__ __forceinline__ void activate(int act, float (&v)[N], const float (&w)[N]) {
  if (act == kSilu) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = activation<kSilu, FAST>(v[i]) * w[i];
  } else if (act == kGelu) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = activation<kGelu, FAST>(v[i]) * w[i];
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = activation<kGeluTanh, FAST>(v[i]) * w[i];
  }
}

// From gate x, factor y and the gradient of act(x) y: the gradients of both.
template <bool FAST>
__device__ __forceinline__ void gate_grad(int act, float x, float y, float dh, float& dx, float& dy) {
  float slope, h;
  if (act == kSilu)
    h = activation_slope<kSilu, FAST>(x, slope);
  else if (act == kGelu)
    h = activation_slope<kGelu, FAST>(x, slope);
  else
    h = activation_slope<kGeluTanh, FAST>(x, slope);
  dx = dh * y * slope;
  dy = dh * h;
}

// Four of them, for bfloat16.
template <int ACT>
__device__ __forceinline__ void gate_grads(const float (&x)[4], const float (&y)[4], const float (&dh)[4],
                                           float (&dx)[4], float (&dy)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float slope;
    const float h = activation_slope<ACT, true>(x[i], slope);
    dx[i] = dh[i] * y[i] * slope;
    dy[i] = dh[i] * h;
  }
}
__device__ __forceinline__ void gate_grad4(int act, const float (&x)[4], const float (&y)[4], const float (&dh)[4],
                                           float (&dx)[4], float (&dy)[4]) {
  if (act == kSilu)
    gate_grads<kSilu>(x, y, dh, dx, dy);
  else if (act == kGelu)
    gate_grads<kGelu>(x, y, dh, dx, dy);
  else
    gate_grads<kGeluTanh>(x, y, dh, dx, dy);
}

}  // namespace

}  // namespace mb

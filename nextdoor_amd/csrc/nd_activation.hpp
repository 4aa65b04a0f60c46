// Activations of a model's layers and their derivatives, in 32 bits.
#pragma once

#include <hip/hip_runtime.h>

#include "../../include/nextdoor_amd.h"
#include "nd_matrix.hpp"

namespace nd {

// 1 / (1 + exp(-x))
__device__ __forceinline__ float logistic(float x) { return __builtin_amdgcn_rcpf(1.f + exp2_fast(x * -1.4426950408889634f)); }

// The normal distribution's integral up to x, P(x), as logistic(x p(x^2)): p is a polynomial fitted to log(P(x) / P(-x)) / x over 0 ..
// 5.5, where P is off by 3e-8 at most (8e-8 with the roundings); beyond, p only grows, and P(-x) is below 2e-8.  -log2(e) is in
// the coefficients.
__device__ __forceinline__ float normal_integral(float x) {
  const float t = x * x;
  float s = -0x1.5c37c2p-28f;
  s = __builtin_fmaf(s, t, 0x1.99c602p-22f);
  s = __builtin_fmaf(s, t, -0x1.7fdb6cp-17f);
  s = __builtin_fmaf(s, t, 0x1.4ea9d4p-13f);
  s = __builtin_fmaf(s, t, 0x1.8a7896p-14f);
  s = __builtin_fmaf(s, t, -0x1.ad6798p-4f);
  s = __builtin_fmaf(s, t, -0x1.26aeccp+1f);
  return __builtin_amdgcn_rcpf(1.f + exp2_fast(x * s));
}
__device__ __forceinline__ float normal_density(float x) { return 0.39894228040143268f * exp2_fast(x * x * -0.72134752044448170f); }

constexpr float kTanhInside = 0.79788456080286536f, kTanhCube = 0.044715f;  // gelu(tanh): x (1 + tanh(inside (x + cube x^3))) / 2

// a(x) of N values.  (One branch for all: the kernels of a type and a shape do not come once for each activation.)
template <int N>
__device__ __forceinline__ void activate(int activation, float (&x)[N]) {
  if (activation == ND_RELU) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = x[i] < 0.f ? 0.f : x[i];  // (NaN stays)
  } else if (activation == ND_GELU) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] *= normal_integral(x[i]);
  } else if (activation == ND_GELU_TANH) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] *= logistic(2.f * kTanhInside * x[i] * __builtin_fmaf(kTanhCube * x[i], x[i], 1.f));
  } else if (activation == ND_SILU) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] *= logistic(x[i]);
  }
}

// x becomes a(x), slope a'(x), which is 0 or 1 where a is flat to 32 bits: x may be infinite there, as what a 16-bit float does not hold.
template <int N>
__device__ __forceinline__ void activate_with_slope(int activation, float (&x)[N], float (&slope)[N]) {
  if (activation == ND_RELU) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      slope[i] = x[i] > 0.f ? 1.f : 0.f;
      x[i] = x[i] < 0.f ? 0.f : x[i];  // (NaN stays)
    }
  } else if (activation == ND_GELU) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float integral = normal_integral(x[i]), density = normal_density(x[i]);
      slope[i] = density == 0.f ? integral : __builtin_fmaf(x[i], density, integral);
      x[i] *= integral;
    }
  } else if (activation == ND_GELU_TANH) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float square = kTanhCube * x[i] * x[i], s = logistic(2.f * kTanhInside * x[i] * (1.f + square));
      const float flat = s * (1.f - s);
      slope[i] = flat == 0.f ? s : __builtin_fmaf(2.f * kTanhInside * x[i] * flat, __builtin_fmaf(3.f, square, 1.f), s);
      x[i] *= s;
    }
  } else if (activation == ND_SILU) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float s = logistic(x[i]), flat = s * (1.f - s);
      slope[i] = flat == 0.f ? s : __builtin_fmaf(x[i], flat, s);
      x[i] *= s;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) slope[i] = 1.f;
  }
}

}  // namespace nd

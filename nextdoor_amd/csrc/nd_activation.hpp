// Activations of a model's layers and their derivatives, in 32 bits.
#pragma once

#include <hip/hip_runtime.h>

#include "../../include/nextdoor_amd.h"
#include "nd_matrix.hpp"

namespace nd {

// 1 / (1 + exp(-x))
__device__ __forceinline__ float logistic(float x) { return __builtin_amdgcn_rcpf(1.f + exp2_fast(x * -1.4426950408889634f)); }

// The normal distribution at x: its integral up to x, and its density.  The integral is a polynomial in 1 / (1 + p |x|) times the
// density (Abramowitz and Stegun 7.1.26, off by at most 1.5e-7 of erf): one exponential serves both.
__device__ __forceinline__ void normal_distribution(float x, float& integral, float& density) {
  const float u = fabsf(x) * 0.70710678118654752f, e = exp2_fast(x * x * -0.72134752044448170f);
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3275911f, u, 1.f));
  float s = 1.061405429f;
  s = __builtin_fmaf(s, t, -1.453152027f);
  s = __builtin_fmaf(s, t, 1.421413741f);
  s = __builtin_fmaf(s, t, -0.284496736f);
  s = __builtin_fmaf(s, t, 0.254829592f);
  const float tail = 0.5f * s * t * e;
  integral = x < 0.f ? tail : 1.f - tail;
  density = 0.39894228040143268f * e;
}

constexpr float kTanhInside = 0.79788456080286536f, kTanhCube = 0.044715f;  // gelu(tanh): x (1 + tanh(inside (x + cube x^3))) / 2

// a(x) of N values.  (One branch for all: the kernels of a type and a shape do not come once for each activation.)
template <int N>
__device__ __forceinline__ void activate(int activation, float (&x)[N]) {
  if (activation == ND_RELU) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = x[i] > 0.f ? x[i] : x[i] != x[i] ? x[i] : 0.f;
  } else if (activation == ND_GELU) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float integral, density;
      normal_distribution(x[i], integral, density);
      x[i] *= integral;
    }
  } else if (activation == ND_GELU_TANH) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] *= logistic(2.f * kTanhInside * x[i] * __builtin_fmaf(kTanhCube * x[i], x[i], 1.f));
  } else if (activation == ND_SILU) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] *= logistic(x[i]);
  }
}

// x becomes a(x), slope a'(x).
template <int N>
__device__ __forceinline__ void activate_with_slope(int activation, float (&x)[N], float (&slope)[N]) {
  if (activation == ND_RELU) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      slope[i] = x[i] > 0.f ? 1.f : 0.f;
      x[i] = x[i] > 0.f ? x[i] : x[i] != x[i] ? x[i] : 0.f;
    }
  } else if (activation == ND_GELU) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float integral, density;
      normal_distribution(x[i], integral, density);
      slope[i] = __builtin_fmaf(x[i], density, integral);
      x[i] *= integral;
    }
  } else if (activation == ND_GELU_TANH) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float square = kTanhCube * x[i] * x[i], s = logistic(2.f * kTanhInside * x[i] * (1.f + square));
      slope[i] = __builtin_fmaf(2.f * kTanhInside * x[i] * s * (1.f - s), __builtin_fmaf(3.f, square, 1.f), s);
      x[i] *= s;
    }
  } else if (activation == ND_SILU) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float s = logistic(x[i]);
      slope[i] = s * __builtin_fmaf(x[i], 1.f - s, 1.f);
      x[i] *= s;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) slope[i] = 1.f;
  }
}

}  // namespace nd

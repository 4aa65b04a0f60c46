// Dropout from the sampling engine's random stream (C entry: nd_dropout).
//
//   u_o = draw 0 of slot o at `step` in the grouped form of nd_philox.hpp (four slots to a block)
//   y_o = [u_o >= p] x_o / (1 - p) (+ residual_o)
//
// The mask is a function of (seed, step, slot): the backward pass computes it again and nothing is
// stored.  An element that is dropped counts as 0 whatever it holds, NaN and infinities included.
//
// Bound by memory: ten rounds of Philox for four elements hide behind the loads (65537 x 1021 in 16 bits: 268 MB in 50 us, 5.3
// TB/s with what the last cache still holds, as fast as a copy; 8192 x 1024 with a residual, and its gradient: 9 us each).
#include "../../include/nextdoor_amd.h"

#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "nd_errors.hpp"
#include "nd_matrix.hpp"
#include "nd_philox.hpp"

namespace nd {
namespace {

constexpr int kDropoutThreads = 256;
constexpr int kDropoutSlots = 8;  // of one lane: two Philox blocks, and 16 bytes of a 16-bit type

struct DropoutParams {
  const void* x;
  const void* residual;
  void* y;
  int64_t n;
  uint64_t seed;
  uint32_t step;
  uint32_t first_kept;  // kept: word >> 8 at least this (p * 2^24, rounded up: the same as u >= p)
  float scale;
};

template <class T>
struct alignas(sizeof(T) * kDropoutSlots <= 16 ? 16 : 32) DropoutRun {
  T v[kDropoutSlots];
};

// VECTOR: every array is aligned to 16 bytes, whole runs of eight move as vectors.
template <class T, bool RESIDUAL, bool VECTOR>
__global__ __launch_bounds__(kDropoutThreads) void dropout_kernel(DropoutParams p) {
  const int64_t base = (((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * kDropoutThreads + threadIdx.x) * kDropoutSlots;
  if (base >= p.n) return;
  const T* x = (const T*)p.x + base;
  const T* r = (const T*)p.residual + base;
  T* y = (T*)p.y + base;
  const int64_t left = p.n - base;
  DropoutRun<T> in, add;
  if (VECTOR && left >= kDropoutSlots) {
    in = *(const DropoutRun<T>*)x;
    if (RESIDUAL) add = *(const DropoutRun<T>*)r;
  } else {
#pragma unroll
    for (int i = 0; i < kDropoutSlots; ++i) {
      in.v[i] = i < left ? x[i] : T(0.f);
      if (RESIDUAL) add.v[i] = i < left ? r[i] : T(0.f);
    }
  }
  DropoutRun<T> out;
#pragma unroll
  for (int b = 0; b < kDropoutSlots / 4; ++b) {
    const PhiloxBlock words = grouped_first_block_scalar_seed(p.seed, (uint64_t)(base >> 2) + b, p.step);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float value = (words.w[i] >> 8) >= p.first_kept ? (float)in.v[4 * b + i] * p.scale : 0.f;
      if (RESIDUAL) value += (float)add.v[4 * b + i];
      out.v[4 * b + i] = (T)value;
    }
  }
  if (VECTOR && left >= kDropoutSlots) {
    *(DropoutRun<T>*)y = out;
  } else {
#pragma unroll
    for (int i = 0; i < kDropoutSlots; ++i)
      if (i < left) y[i] = out.v[i];
  }
}

template <class T>
hipError_t launch_dropout(const DropoutParams& p, hipStream_t stream) {
  const int64_t lanes = (p.n + kDropoutSlots - 1) / kDropoutSlots;
  const int64_t blocks = (lanes + kDropoutThreads - 1) / kDropoutThreads, most = 1 << 22;  // (a row of a grid has fewer than 2^32 threads)
  const dim3 grid((uint32_t)std::min(blocks, most), (uint32_t)((blocks + most - 1) / most));
  const bool vector = (((uintptr_t)p.x | (uintptr_t)p.y | (uintptr_t)p.residual) & 15) == 0;
  if (p.residual) {
    if (vector) dropout_kernel<T, true, true><<<grid, kDropoutThreads, 0, stream>>>(p);
    else dropout_kernel<T, true, false><<<grid, kDropoutThreads, 0, stream>>>(p);
  } else {
    if (vector) dropout_kernel<T, false, true><<<grid, kDropoutThreads, 0, stream>>>(p);
    else dropout_kernel<T, false, false><<<grid, kDropoutThreads, 0, stream>>>(p);
  }
  return hipGetLastError();
}

}  // namespace
}  // namespace nd

extern "C" int nd_dropout(const void* d_x, const void* d_residual, void* d_y, int64_t n, int dtype, double p,
                          uint64_t seed, uint32_t step, void* stream) {
  return nd::guarded([&]() -> int {
    if (n < 0 || (n > 0 && (!d_x || !d_y))) return nd::fail("bad argument");
    if (!(p >= 0.0 && p <= 1.0)) return nd::fail("dropout: p is a probability, " + std::to_string(p) + " given");
    if (step >> 31) return nd::fail("dropout: step numbers are below 2^31");
    if (n > (int64_t)1 << 40) return nd::fail("dropout: at most 2^40 elements");
    if (n == 0) return 0;
    nd::DropoutParams q;
    q.x = d_x;
    q.residual = d_residual;
    q.y = d_y;
    q.n = n;
    q.seed = seed;
    q.step = step;
    q.first_kept = (uint32_t)ceil((double)(float)p * 16777216.0);
    q.scale = p < 1.0 ? (float)(1.0 / (1.0 - p)) : 0.f;
    hipError_t e;
    if (dtype == ND_F32) e = nd::launch_dropout<float>(q, (hipStream_t)stream);
    else if (dtype == ND_F16) e = nd::launch_dropout<_Float16>(q, (hipStream_t)stream);
    else if (dtype == ND_BF16) e = nd::launch_dropout<__bf16>(q, (hipStream_t)stream);
    else return nd::fail("dropout: unknown type " + std::to_string(dtype));
    if (e != hipSuccess) return nd::fail(std::string("dropout: ") + hipGetErrorString(e));
    return 0;
  });
}

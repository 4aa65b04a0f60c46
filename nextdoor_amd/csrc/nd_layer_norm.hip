// Layer norm and its gradients (C entries: nd_layer_norm_*).
//
//   mean_i, rstd_i = 1 / sqrt(variance_i + eps) of row i;  n = (x - mean_i) rstd_i;  out = n w + b
//   e = dout w;  dx = rstd_i (e - mean(e) - n mean(e n));  dw = sum over the rows of dout n,  db = that of dout
//
// Bound by memory: a row is read once and stays in registers for its two sums, the deviations' squares being taken once the
// mean is known.  LANES lanes have a row, each VALUES of its places; a workgroup has a number of rows at a time and asks for the next
// ones before it sums those it has.  w and b, and in the backward pass the sums for dw and db, stay in registers over all rows of a
// workgroup; another kernel adds the workgroups' sums.  Forward and backward, in 16 bits 8192 x 1024: 11 and 16 us (3.1 TB/s, of which
// the start of workgroups and the last rows' sums are a third), 16384 x 4096: 59 and 88 (4.6 TB/s, as fast as a copy); in 32 bits
// 20011 x 1021, places one by one: 34 and 42 (4.8 and 5.8, some of it from the last cache); the sums' kernel 4 to 5.
#include "../../include/nextdoor_amd.h"

#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "nd_column_sums.hpp"
#include "nd_errors.hpp"
#include "nd_matrix.hpp"

namespace nd {
namespace {

struct NormParams {
  const char* x;
  const char* dout;
  int64_t x_bytes, dout_bytes;  // of a row
  const void *weight, *bias;
  void* out;  // backward: dx, or null
  float *mean, *rstd;
  float* sums;  // [workgroup][2][dim], or null
  void *dweight, *dbias;  // where there is one workgroup: written here, each unless it is null
  int64_t rows;
  int32_t dim;
  int32_t weight_32;
  float eps;
};

// VALUES places of a row: VECTOR: runs of eight, each 16 bytes aligned (32 bits: twice that), LANES runs apart; else single ones.
template <class T, int LANES, int VALUES, bool VECTOR>
struct Places {
  static constexpr int kRun = VECTOR ? 8 : 1;
  T v[VALUES];
  __device__ __forceinline__ static int column(int i, int lane) { return (i / kRun * LANES + lane) * kRun + i % kRun; }
  __device__ __forceinline__ void load(const char* row, int dim, int lane) {
    if constexpr (VECTOR) {
#pragma unroll
      for (int i = 0; i < VALUES; i += 8) {
        const int c = column(i, lane);
        u32x4 w[sizeof(T) / 2];
#pragma unroll
        for (unsigned j = 0; j < sizeof(T) / 2; ++j) w[j] = c < dim ? ((const u32x4*)(row + (int64_t)c * sizeof(T)))[j] : u32x4{0, 0, 0, 0};
        __builtin_memcpy(&v[i], w, sizeof(w));
      }
    } else {
#pragma unroll
      for (int i = 0; i < VALUES; ++i) {
        const int c = column(i, lane);
        v[i] = c < dim ? ((const T*)row)[c] : T(0.f);
      }
    }
  }
  __device__ __forceinline__ static void store(char* row, int dim, int lane, const float (&x)[VALUES]) {
    if constexpr (VECTOR) {
#pragma unroll
      for (int i = 0; i < VALUES; i += 8) {
        const int c = column(i, lane);
        T out[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) out[j] = (T)x[i + j];
        u32x4 w[sizeof(T) / 2];
        __builtin_memcpy(w, out, sizeof(w));
        if (c < dim) {
#pragma unroll
          for (unsigned j = 0; j < sizeof(T) / 2; ++j) ((u32x4*)(row + (int64_t)c * sizeof(T)))[j] = w[j];
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < VALUES; ++i) {
        const int c = column(i, lane);
        if (c < dim) ((T*)row)[c] = (T)x[i];
      }
    }
  }
  // Weights: of this type or in 32 bits; a null array is `otherwise` everywhere.
  __device__ __forceinline__ static void load_weights(const void* w, bool in_32, float otherwise, int dim, int lane, float (&x)[VALUES]) {
    if (!w) {
#pragma unroll
      for (int i = 0; i < VALUES; ++i) x[i] = otherwise;
    } else if (in_32) {
      Places<float, LANES, VALUES, VECTOR> all;
      all.load((const char*)w, dim, lane);
#pragma unroll
      for (int i = 0; i < VALUES; ++i) x[i] = all.v[i];
    } else {
      Places all;
      all.load((const char*)w, dim, lane);
#pragma unroll
      for (int i = 0; i < VALUES; ++i) x[i] = (float)all.v[i];
    }
  }
};

// The sums of two values over the LANES lanes of a row; `turn` counts the calls (every wave of the workgroup makes them all).
template <int LANES, int THREADS>
__device__ __forceinline__ float2 row_sums(float2 v, float2 (*scratch)[THREADS / 64], int turn) {
#pragma unroll
  for (int d = (LANES < 64 ? LANES : 64) / 2; d > 0; d >>= 1) {
    v.x += __shfl_xor(v.x, d);
    v.y += __shfl_xor(v.y, d);
  }
  if constexpr (LANES > 64) {
    constexpr int kWaves = LANES / 64;
    const int wave = threadIdx.x >> 6, first = wave / kWaves * kWaves;
    if ((threadIdx.x & 63) == 0) scratch[turn & 1][wave] = v;
    __syncthreads();  // (two arrays in turn: this one is written again only after the barrier of the next call)
    v = make_float2(0.f, 0.f);
#pragma unroll 4
    for (int w = 0; w < kWaves; ++w) {
      v.x += scratch[turn & 1][first + w].x;
      v.y += scratch[turn & 1][first + w].y;
    }
  }
  return v;
}

template <class T, int LANES, int VALUES, int THREADS, int AHEAD, bool VECTOR>
__global__ __launch_bounds__(THREADS) void norm_forward_kernel(NormParams p) {
  using Row = Places<T, LANES, VALUES, VECTOR>;
  constexpr int kGroups = THREADS / LANES;
  __shared__ float2 scratch[2][THREADS / 64];
  const int lane = threadIdx.x % LANES;
  const int64_t stride = (int64_t)gridDim.x * kGroups;
  Row next[AHEAD];
  int64_t row = (int64_t)blockIdx.x * kGroups + threadIdx.x / LANES;
#pragma unroll
  for (int a = 0; a < AHEAD; ++a)
    if (row + a * stride < p.rows) next[a].load(p.x + (row + a * stride) * p.x_bytes, p.dim, lane);
  float w[VALUES], b[VALUES];
  Row::load_weights(p.weight, p.weight_32, 1.f, p.dim, lane, w);
  Row::load_weights(p.bias, p.weight_32, 0.f, p.dim, lane, b);
  int turn = 0;
  for (int64_t base = (int64_t)blockIdx.x * kGroups; base < p.rows; base += AHEAD * stride) {
#pragma unroll
    for (int a = 0; a < AHEAD; ++a, row += stride) {
      const bool there = row < p.rows;
      float x[VALUES], sum = 0.f;
#pragma unroll
      for (int i = 0; i < VALUES; ++i) {
        x[i] = there ? (float)next[a].v[i] : 0.f;
        sum += x[i];
      }
      if (row + AHEAD * stride < p.rows) next[a].load(p.x + (row + AHEAD * stride) * p.x_bytes, p.dim, lane);
      const float mean = row_sums<LANES, THREADS>(make_float2(sum, 0.f), scratch, turn++).x / p.dim;
      sum = 0.f;
#pragma unroll
      for (int i = 0; i < VALUES; ++i) {
        x[i] = Row::column(i, lane) < p.dim ? x[i] - mean : 0.f;
        sum = __builtin_fmaf(x[i], x[i], sum);
      }
      const float variance = row_sums<LANES, THREADS>(make_float2(sum, 0.f), scratch, turn++).x / p.dim;
      const float rstd = 1.f / sqrtf(variance + p.eps);
#pragma unroll
      for (int i = 0; i < VALUES; ++i) x[i] = __builtin_fmaf(x[i] * rstd, w[i], b[i]);
      if (there) {
        Row::store((char*)p.out + row * p.dim * (int64_t)sizeof(T), p.dim, lane, x);
        if (lane == 0) {
          p.mean[row] = mean;
          p.rstd[row] = rstd;
        }
      }
    }
  }
}

template <class T, int LANES, int VALUES, int THREADS, int AHEAD, bool VECTOR>
__global__ __launch_bounds__(THREADS) void norm_backward_kernel(NormParams p) {
  using Row = Places<T, LANES, VALUES, VECTOR>;
  constexpr int kGroups = THREADS / LANES;
  __shared__ float2 scratch[2][THREADS / 64];
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
  const int64_t stride = (int64_t)gridDim.x * kGroups;
  Row next[AHEAD], next_dout[AHEAD];
  float next_mean[AHEAD], next_rstd[AHEAD];
  auto ask = [&](int a, int64_t row) {
    if (row >= p.rows) return;
    next[a].load(p.x + row * p.x_bytes, p.dim, lane);
    next_dout[a].load(p.dout + row * p.dout_bytes, p.dim, lane);
    next_mean[a] = p.mean[row];
    next_rstd[a] = p.rstd[row];
  };
  int64_t row = (int64_t)blockIdx.x * kGroups + group;
#pragma unroll
  for (int a = 0; a < AHEAD; ++a) ask(a, row + a * stride);
  constexpr bool kKeepWeights = VALUES <= 8;  // (the longest rows read them again each time, from the caches)
  float w[VALUES], dw[VALUES], db[VALUES];
  if (kKeepWeights) Row::load_weights(p.weight, p.weight_32, 1.f, p.dim, lane, w);
#pragma unroll
  for (int i = 0; i < VALUES; ++i) dw[i] = db[i] = 0.f;
  int turn = 0;
  for (int64_t base = (int64_t)blockIdx.x * kGroups; base < p.rows; base += AHEAD * stride) {
#pragma unroll
    for (int a = 0; a < AHEAD; ++a, row += stride) {
      const bool there = row < p.rows;
      const float mean = next_mean[a], rstd = next_rstd[a];
      if (!kKeepWeights) Row::load_weights(p.weight, p.weight_32, 1.f, p.dim, lane, w);
      float n[VALUES], e[VALUES];
      float2 sum = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < VALUES; ++i) {
        const bool inside = there && Row::column(i, lane) < p.dim;
        const float d = inside ? (float)next_dout[a].v[i] : 0.f;
        n[i] = inside ? ((float)next[a].v[i] - mean) * rstd : 0.f;
        dw[i] = __builtin_fmaf(d, n[i], dw[i]);
        db[i] += d;
        e[i] = d * w[i];
        sum.x += e[i];
        sum.y = __builtin_fmaf(e[i], n[i], sum.y);
      }
      ask(a, row + AHEAD * stride);
      if (p.out) {
        sum = row_sums<LANES, THREADS>(sum, scratch, turn++);
        const float mean_e = sum.x / p.dim, mean_en = sum.y / p.dim;
#pragma unroll
        for (int i = 0; i < VALUES; ++i) e[i] = (e[i] - __builtin_fmaf(n[i], mean_en, mean_e)) * rstd;
        if (there) Row::store((char*)p.out + row * p.dim * (int64_t)sizeof(T), p.dim, lane, e);
      }
    }
  }
  if (!p.sums && !p.dweight && !p.dbias) return;
  // The groups' sums: half of them leave theirs in LDS, the other half adds them, until one is left.
  __shared__ float part[kGroups > 1 ? kGroups / 2 : 1][2][kGroups > 1 ? LANES * VALUES : 1];
#pragma unroll
  for (int half = kGroups / 2; half > 0; half >>= 1) {
    __syncthreads();
    if (group >= half && group < 2 * half) {
#pragma unroll
      for (int i = 0; i < VALUES; ++i) {
        part[group - half][0][i * LANES + lane] = dw[i];
        part[group - half][1][i * LANES + lane] = db[i];
      }
    }
    __syncthreads();
    if (group < half) {
#pragma unroll
      for (int i = 0; i < VALUES; ++i) {
        dw[i] += part[group][0][i * LANES + lane];
        db[i] += part[group][1][i * LANES + lane];
      }
    }
  }
  if (group > 0) return;
  auto put = [&](void* to, int c, float v) {
    if (!to) return;
    if (p.weight_32) ((float*)to)[c] = v;
    else ((T*)to)[c] = (T)v;
  };
#pragma unroll
  for (int i = 0; i < VALUES; ++i) {
    const int c = Row::column(i, lane);
    if (c >= p.dim) continue;
    if (p.sums) {
      float* sums = p.sums + (int64_t)blockIdx.x * 2 * p.dim;
      sums[c] = dw[i];
      sums[p.dim + c] = db[i];
    } else {
      put(p.dweight, c, dw[i]);
      put(p.dbias, c, db[i]);
    }
  }
}

// Rows by size: eight places to a lane, sixteen for the longest, and as many lanes as that takes; `rows` of a workgroup at a time in
// the backward pass, which has one workgroup of 1024 lanes to a compute unit, so that few sums are left to add.  The forward pass
// has workgroups of 256 or what a row takes.
struct NormShape {
  int most, lanes, rows;
};
constexpr NormShape kNormShapes[] = {{64, 8, 128}, {128, 16, 64}, {256, 32, 32}, {512, 64, 16}, {1024, 128, 8}, {2048, 256, 4}, {4096, 512, 2}, {8192, 1024, 1}, {16384, 1024, 1}};
constexpr int kForwardLanes = 1 << 19, kBackwardBlocks = 256;
constexpr int kAlone = 6;  // times at most that one workgroup takes the next rows: less than another launch, which adds up sums, costs
int shape_of(int32_t dim) {
  int i = 0;
  while (dim > kNormShapes[i].most) ++i;
  return i;
}
int64_t backward_blocks(int64_t rows, int32_t dim) {
  const int at_once = kNormShapes[shape_of(dim)].rows;
  if (rows <= kAlone * at_once) return 1;
  return std::max<int64_t>(1, std::min<int64_t>(kBackwardBlocks, (rows + at_once - 1) / at_once));
}

template <class T, int LANES, int VALUES>
void launch_norm_of(const NormParams& p, bool backward, bool vector, hipStream_t stream) {
  if (backward) {
    const uint32_t blocks = (uint32_t)backward_blocks(p.rows, p.dim);
    if (vector) norm_backward_kernel<T, LANES, VALUES, 1024, VALUES == 8 && sizeof(T) == 2 ? 2 : 1, true><<<blocks, 1024, 0, stream>>>(p);
    else norm_backward_kernel<T, LANES, VALUES, 1024, 1, false><<<blocks, 1024, 0, stream>>>(p);
  } else {
    constexpr int kThreads = LANES < 256 ? 256 : LANES, kGroups = kThreads / LANES;
    const uint32_t blocks = (uint32_t)std::min<int64_t>((p.rows + kGroups - 1) / kGroups, kForwardLanes / kThreads);
    if (vector) norm_forward_kernel<T, LANES, VALUES, kThreads, 1, true><<<blocks, kThreads, 0, stream>>>(p);
    else norm_forward_kernel<T, LANES, VALUES, kThreads, 1, false><<<blocks, kThreads, 0, stream>>>(p);
  }
}
template <class T>
void launch_norm(const NormParams& p, bool backward, hipStream_t stream) {
  const uintptr_t at = (uintptr_t)p.x | (uintptr_t)p.out | (uintptr_t)p.weight | (uintptr_t)p.bias | (uintptr_t)p.x_bytes |
                       (backward ? (uintptr_t)p.dout | (uintptr_t)p.dout_bytes : 0);
  const bool vector = p.dim % 8 == 0 && (at & 15) == 0;
  switch (shape_of(p.dim)) {
    case 0: return launch_norm_of<T, 8, 8>(p, backward, vector, stream);
    case 1: return launch_norm_of<T, 16, 8>(p, backward, vector, stream);
    case 2: return launch_norm_of<T, 32, 8>(p, backward, vector, stream);
    case 3: return launch_norm_of<T, 64, 8>(p, backward, vector, stream);
    case 4: return launch_norm_of<T, 128, 8>(p, backward, vector, stream);
    case 5: return launch_norm_of<T, 256, 8>(p, backward, vector, stream);
    case 6: return launch_norm_of<T, 512, 8>(p, backward, vector, stream);
    case 7: return launch_norm_of<T, 1024, 8>(p, backward, vector, stream);
    default: return launch_norm_of<T, 1024, 16>(p, backward, vector, stream);
  }
}

int64_t norm_workspace(const nd_layer_norm* a) {
  const int64_t blocks = backward_blocks(a->rows, a->dim);
  return (a->dweight || a->dbias) && blocks > 1 ? blocks * 2 * a->dim * 4 : 0;
}

std::string refuse(const nd_layer_norm* a) {
  if (!a) return "null argument";
  if (a->dtype != ND_F32 && a->dtype != ND_F16 && a->dtype != ND_BF16) return "unknown type " + std::to_string(a->dtype);
  if (a->weight_dtype != a->dtype && a->weight_dtype != ND_F32) return "weights have the type of x or 32 bits";
  if (a->rows < 0 || a->rows > (int64_t)1 << 40) return "between 0 and 2^40 rows, " + std::to_string(a->rows) + " given";
  if (a->dim < 1 || a->dim > ND_LAYER_NORM_MAX_DIM)
    return "rows of 1 to " + std::to_string(ND_LAYER_NORM_MAX_DIM) + " values, " + std::to_string(a->dim) + " given";
  if (!(a->eps >= 0.f && a->eps < INFINITY)) return "eps is a number of at least 0";
  if (a->x_row < 0 || a->dout_row < 0 || a->x_row >> 40 || a->dout_row >> 40) return "rows lie 0 to 2^40 elements apart";
  return "";
}

int run_norm(const nd_layer_norm* a, bool backward, void* stream) {
  std::string why = refuse(a);
  if (!why.empty()) return fail("layer norm: " + why);
  const bool some = a->rows > 0;
  const int size = a->dtype == ND_F32 ? 4 : 2, weight_size = a->weight_dtype == ND_F32 ? 4 : 2;
  struct {
    const void* at;
    bool needed;
    int size;
  } const arrays[] = {{a->x, some, size},
                      {a->weight, false, weight_size},
                      {a->bias, false, weight_size},
                      {a->mean, some, 4},
                      {a->rstd, some, 4},
                      {backward ? a->dout : a->out, some, size},
                      {backward ? a->dx : nullptr, false, size},
                      {backward ? a->dweight : nullptr, false, weight_size},
                      {backward ? a->dbias : nullptr, false, weight_size}};
  for (const auto& x : arrays) {
    if (x.needed && !x.at) return fail("layer norm: null array");
    if ((uintptr_t)x.at % x.size) return fail("layer norm: arrays are aligned as their elements are");
  }
  const bool weights = backward && (a->dweight || a->dbias);
  const int64_t room = backward ? norm_workspace(a) : 0;
  if (room > 0 && (a->workspace_bytes < room || !a->workspace || ((uintptr_t)a->workspace & 15)))
    return fail("layer norm: the workspace has " + std::to_string(a->workspace ? a->workspace_bytes : 0) + " bytes, " + std::to_string(room) +
                " needed, aligned to 16");
  if (!weights && (!some || (backward && !a->dx))) return 0;
  NormParams p = {};
  p.x = (const char*)a->x;
  p.x_bytes = a->x_row * size;
  p.dout = (const char*)a->dout;
  p.dout_bytes = a->dout_row * size;
  p.weight = a->weight;
  p.bias = a->bias;
  p.out = backward ? a->dx : a->out;
  p.mean = a->mean;
  p.rstd = a->rstd;
  p.sums = room > 0 ? (float*)a->workspace : nullptr;
  p.dweight = backward ? a->dweight : nullptr;
  p.dbias = backward ? a->dbias : nullptr;
  p.rows = a->rows;
  p.dim = a->dim;
  p.weight_32 = a->weight_dtype == ND_F32;
  p.eps = a->eps;
  if (a->dtype == ND_F32) launch_norm<float>(p, backward, (hipStream_t)stream);
  else if (a->dtype == ND_F16) launch_norm<_Float16>(p, backward, (hipStream_t)stream);
  else launch_norm<__bf16>(p, backward, (hipStream_t)stream);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && p.sums) {
    const int64_t blocks = backward_blocks(a->rows, a->dim), columns = 2 * a->dim;
    const hipStream_t s = (hipStream_t)stream;
    if (a->weight_dtype == ND_F32) e = column_join<float>(p.sums, blocks, columns, nullptr, a->dweight, a->dim, a->dbias, s);
    else if (a->weight_dtype == ND_F16) e = column_join<_Float16>(p.sums, blocks, columns, nullptr, a->dweight, a->dim, a->dbias, s);
    else e = column_join<__bf16>(p.sums, blocks, columns, nullptr, a->dweight, a->dim, a->dbias, s);
  }
  if (e != hipSuccess) return fail(std::string("layer norm: ") + hipGetErrorString(e));
  return 0;
}

}  // namespace
}  // namespace nd

extern "C" {

int64_t nd_layer_norm_workspace(const nd_layer_norm* a) {
  if (!nd::refuse(a).empty()) return -1;
  return nd::norm_workspace(a);
}
int nd_layer_norm_forward(const nd_layer_norm* a, void* stream) {
  return nd::guarded([&]() -> int { return nd::run_norm(a, false, stream); });
}
int nd_layer_norm_backward(const nd_layer_norm* a, void* stream) {
  return nd::guarded([&]() -> int { return nd::run_norm(a, true, stream); });
}

}  // extern "C"

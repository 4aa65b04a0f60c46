// Layer norm and its gradients (C entries: nd_layer_norm_*).
//
//   mean_i, rstd_i = 1 / sqrt(variance_i + eps) of row i;  n = (x - mean_i) rstd_i;  out = n w + b
//   e = dout w;  dx = rstd_i (e - mean(e) - n mean(e n));  dw = sum over the rows of dout n,  db = that of dout
//
// Bound by memory: a row is read once and stays in registers for its two sums, the deviations' squares being taken once the
// mean is known.  LANES lanes have a row, each VALUES of its places; a workgroup has a number of rows at a time and asks for the next
// ones before it sums those it has.  w and b, and in the backward pass the sums for dw and db, stay in registers over all rows of a
// workgroup; another kernel adds the workgroups' sums.  Forward and backward, in 16 bits 8192 x 1024: 10 and 16 us (3.2 TB/s, of which
// the start of workgroups and the last rows' sums are a third), 16384 x 4096: 48 and 87 (5.6 and 4.6 TB/s); in 32 bits 20011 x 1021: 32
// and 42 (5.1 and 5.8, some of it from the last cache); the sums' kernel 4 to 5.  Rows of fewer than 64 values leave lanes without places:
// 128 MiB of rows of 32, 16 and 8 16-bit values 4.1, 2.5 and 1.4 TB/s forward, 4.4, 2.8 and 1.6 backward.
#include "../../include/nextdoor_amd.h"

#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

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

// How a row's places are shared out among lanes.  kWhole: runs of 16 bytes, one after another, of which rows are multiples; kOver: the
// same, but the last run ends where the row ends and begins among the places of the one before, which are not counted twice (and are
// written twice, the same); kSingle: one by one, rows shorter than a run.  Loads need no alignment but the elements'.  (Place by place
// 20011 x 1021 in 16 bits took 21.6 and 32.9 us for 16.5 and 30.9, 8000 x 4001 32.5 and 49 for 24 and 45.)
enum class Runs { kWhole, kOver, kSingle };

// VALUES places of a row with a lane, in runs that lie LANES runs apart.
template <class T, int LANES, int VALUES, Runs RUNS, int RUN = RUNS == Runs::kSingle ? 1 : 16 / sizeof(T)>
struct Places {
  static constexpr int kRun = RUN;
  using Word = std::conditional_t<RUNS == Runs::kSingle, T, uint32_t>;  // (pairs of 16-bit values stay as they are until they are used)
  struct __attribute__((packed, aligned(sizeof(T)))) Run {
    Word w[kRun * sizeof(T) / sizeof(Word)];
  };
  T v[VALUES];
  // The first place of the run that place i belongs to, and where that run is read.
  __device__ __forceinline__ static int first(int i, int lane) { return (i / kRun * LANES + lane) * kRun; }
  __device__ __forceinline__ static int at(int i, int lane, int dim) { return min(first(i, lane), dim - kRun); }
  __device__ __forceinline__ static int column(int i, int lane, int dim) { return at(i, lane, dim) + i % kRun; }
  __device__ __forceinline__ static bool there(int i, int lane, int dim) { return first(i, lane) < dim; }
  // (past the row's end a run is at the end, and all of its places belong to others)
  __device__ __forceinline__ static bool counts(int i, int lane, int dim) {
    return RUNS == Runs::kOver ? column(i, lane, dim) >= first(i, lane) : there(i, lane, dim);
  }
  __device__ __forceinline__ void load(const char* row, int dim, int lane) {
#pragma unroll
    for (int i = 0; i < VALUES; i += kRun) {
      const Run r = *(const Run*)(row + (uint32_t)at(i, lane, dim) * sizeof(T));
      __builtin_memcpy(&v[i], &r, sizeof(r));
    }
  }
  __device__ __forceinline__ static void store(char* row, int dim, int lane, const float (&x)[VALUES]) {
#pragma unroll
    for (int i = 0; i < VALUES; i += kRun) {
      T out[kRun];
#pragma unroll
      for (int j = 0; j < kRun; ++j) out[j] = (T)x[i + j];
      Run r;
      __builtin_memcpy(&r, out, sizeof(r));
      if (there(i, lane, dim)) *(Run*)(row + (uint32_t)at(i, lane, dim) * sizeof(T)) = r;
    }
  }
  // Weights: of this type or in 32 bits; a null array is `otherwise` everywhere.
  __device__ __forceinline__ static void load_weights(const void* w, bool in_32, float otherwise, int dim, int lane, float (&x)[VALUES]) {
    if (!w) {
#pragma unroll
      for (int i = 0; i < VALUES; ++i) x[i] = otherwise;
    } else if (in_32) {
      Places<float, LANES, VALUES, RUNS, RUN> all;
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
    // (four at a time, those in pairs, so that the chain of roundings is not as long as the waves are many; in pairs of all sixteen the longest
    // rows' gradients spilled registers)
    constexpr int kAtOnce = kWaves < 4 ? kWaves : 4;
    v = make_float2(0.f, 0.f);
#pragma unroll 1
    for (int w = 0; w < kWaves; w += kAtOnce) {
      float2 s[kAtOnce];
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) s[i] = scratch[turn & 1][first + w + i];
#pragma unroll
      for (int d = kAtOnce / 2; d > 0; d >>= 1)
#pragma unroll
        for (int i = 0; i < d; ++i) {
          s[i].x += s[i + d].x;
          s[i].y += s[i + d].y;
        }
      v.x += s[0].x;
      v.y += s[0].y;
    }
  }
  return v;
}

// Which row of those that a workgroup has at a time; the same for a whole wave, and so are its addresses, where a row has 64 lanes.
template <int LANES>
__device__ __forceinline__ int group_of() {
  return LANES < 64 ? threadIdx.x / LANES : uniform(threadIdx.x / LANES);
}

template <class T, int LANES, int VALUES, int THREADS, int AHEAD, Runs RUNS>
__global__ __launch_bounds__(THREADS) void norm_forward_kernel(NormParams p) {
  using Row = Places<T, LANES, VALUES, RUNS>;
  constexpr int kGroups = THREADS / LANES;
  __shared__ float2 scratch[2][THREADS / 64];
  const int lane = threadIdx.x % LANES, group = group_of<LANES>();
  const int64_t stride = (int64_t)gridDim.x * kGroups;
  Row next[AHEAD];
  int64_t row = (int64_t)blockIdx.x * kGroups + group;
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
        sum += Row::counts(i, lane, p.dim) ? x[i] : 0.f;
      }
      if (row + AHEAD * stride < p.rows) next[a].load(p.x + (row + AHEAD * stride) * p.x_bytes, p.dim, lane);
      const float mean = row_sums<LANES, THREADS>(make_float2(sum, 0.f), scratch, turn++).x / p.dim;
      sum = 0.f;
#pragma unroll
      for (int i = 0; i < VALUES; ++i) {
        x[i] -= mean;
        sum = __builtin_fmaf(x[i], Row::counts(i, lane, p.dim) ? x[i] : 0.f, sum);
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

template <class T, int LANES, int VALUES, int THREADS, int AHEAD, Runs RUNS>
__global__ __launch_bounds__(THREADS) void norm_backward_kernel(NormParams p) {
  using Row = Places<T, LANES, VALUES, RUNS>;
  constexpr int kGroups = THREADS / LANES;
  __shared__ float2 scratch[2][THREADS / 64];
  const int lane = threadIdx.x % LANES, group = group_of<LANES>();
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
        const float d = there ? (float)next_dout[a].v[i] : 0.f;
        n[i] = there ? ((float)next[a].v[i] - mean) * rstd : 0.f;
        dw[i] = __builtin_fmaf(d, n[i], dw[i]);
        db[i] += d;
        e[i] = d * w[i];
        const float counted = Row::counts(i, lane, p.dim) ? e[i] : 0.f;
        sum.x += counted;
        sum.y = __builtin_fmaf(counted, n[i], sum.y);
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
    if (!Row::counts(i, lane, p.dim)) continue;
    const int c = Row::column(i, lane, p.dim);
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

// Rows by size: eight places to a lane, sixteen for the longest, and as many lanes as that takes, 8 at least (with 16
// lanes for up to 128 places and 64 for up to 512 alone, 92000 x 256 in 16 bits took 26.5 and 39 us for 17 and 31, 300000 x 64 24 and 34
// for 14.6 and 29); `rows` of a workgroup at a time in the backward pass, which has one workgroup of 1024 lanes to a compute unit, so that few sums are left to add.  The forward pass
// has workgroups of 256 or what a row takes.
struct NormShape {
  int most, lanes, rows;
};
constexpr NormShape kNormShapes[] = {{64, 8, 128}, {128, 16, 64}, {256, 32, 32}, {512, 64, 16}, {1024, 128, 8}, {2048, 256, 4}, {4096, 512, 2}, {8192, 1024, 1}, {16384, 1024, 1}};
constexpr int kForwardLanes = 1 << 19, kBackwardBlocks = 256;
// Times at most that one workgroup takes the next rows: less than another launch, which adds up sums, costs where a program makes each call
// (48 x 1024 13.1 us for 15.7, 4 x 16384 18 for 21.5; in a graph 12.9 for 8.7 and 18 for 21.3).
constexpr int kAlone = 6;
int shape_of(int32_t dim) {
  int i = 0;
  while (dim > kNormShapes[i].most) ++i;
  return i;
}
int64_t backward_blocks(int64_t rows, int32_t dim, bool weights) {  // (for dx alone there is no such launch: 48 x 1024 5.0 us for 11.2, 6 x 16384 4.4 for 16)
  const int at_once = kNormShapes[shape_of(dim)].rows;
  if (weights && rows <= kAlone * at_once) return 1;
  return std::max<int64_t>(1, std::min<int64_t>(kBackwardBlocks, (rows + at_once - 1) / at_once));
}

template <class T, int LANES, int VALUES, Runs RUNS>
void launch_backward(const NormParams& p, hipStream_t stream) {
  const uint32_t blocks = (uint32_t)backward_blocks(p.rows, p.dim, p.sums || p.dweight || p.dbias);
  norm_backward_kernel<T, LANES, VALUES, 1024, VALUES == 8 && sizeof(T) == 2 ? 2 : 1, RUNS><<<blocks, 1024, 0, stream>>>(p);
}
template <class T, int LANES, int VALUES, Runs RUNS>
void launch_forward(const NormParams& p, hipStream_t stream) {
  constexpr int kThreads = LANES < 256 ? 256 : LANES, kGroups = kThreads / LANES;
  const uint32_t blocks = (uint32_t)std::min<int64_t>((p.rows + kGroups - 1) / kGroups, kForwardLanes / kThreads);
  norm_forward_kernel<T, LANES, VALUES, kThreads, 1, RUNS><<<blocks, kThreads, 0, stream>>>(p);
}
// FORWARD: lanes to a row in the forward pass: half as many for 513 to 8192 places of 16 bits, sixteen to each, as less waits for others
// then (20011 x 1024: 15.6 us for 17.3, 5000 x 8000: 28 for 34; in 32 bits equal or slower).
template <class T, int LANES, int VALUES, int FORWARD = LANES>
void launch_norm_of(const NormParams& p, bool backward, hipStream_t stream) {
  constexpr int kForwardValues = VALUES * LANES / FORWARD;
  if (p.dim % (16 / sizeof(T)) == 0) {
    if (backward) launch_backward<T, LANES, VALUES, Runs::kWhole>(p, stream);
    else launch_forward<T, FORWARD, kForwardValues, Runs::kWhole>(p, stream);
  } else {
    if (backward) launch_backward<T, LANES, VALUES, Runs::kOver>(p, stream);
    else launch_forward<T, FORWARD, kForwardValues, Runs::kOver>(p, stream);
  }
}
template <class T>
void launch_norm(const NormParams& p, bool backward, hipStream_t stream) {
  if (p.dim < (int)(16 / sizeof(T))) {
    if (backward) launch_backward<T, 8, 1, Runs::kSingle>(p, stream);
    else launch_forward<T, 8, 1, Runs::kSingle>(p, stream);
    return;
  }
  constexpr bool k16 = sizeof(T) == 2;
  switch (shape_of(p.dim)) {
    case 0: return launch_norm_of<T, 8, 8>(p, backward, stream);
    case 1: return launch_norm_of<T, 16, 8>(p, backward, stream);
    case 2: return launch_norm_of<T, 32, 8>(p, backward, stream);
    case 3: return launch_norm_of<T, 64, 8>(p, backward, stream);
    case 4: return launch_norm_of<T, 128, 8, k16 ? 64 : 128>(p, backward, stream);
    case 5: return launch_norm_of<T, 256, 8, k16 ? 128 : 256>(p, backward, stream);
    case 6: return launch_norm_of<T, 512, 8, k16 ? 256 : 512>(p, backward, stream);
    case 7: return launch_norm_of<T, 1024, 8, k16 ? 512 : 1024>(p, backward, stream);
    default: return launch_norm_of<T, 1024, 16>(p, backward, stream);
  }
}

int64_t norm_workspace(const nd_layer_norm* a) {
  if (!a->dweight && !a->dbias) return 0;
  const int64_t blocks = backward_blocks(a->rows, a->dim, true);
  return blocks > 1 ? blocks * 2 * a->dim * 4 : 0;
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
    const int64_t blocks = backward_blocks(a->rows, a->dim, true), columns = 2 * a->dim;
    const hipStream_t s = (hipStream_t)stream;
    if (a->weight_dtype == ND_F32) e = column_join<float>(p.sums, blocks, columns, a->dweight, a->dim, a->dbias, s);
    else if (a->weight_dtype == ND_F16) e = column_join<_Float16>(p.sums, blocks, columns, a->dweight, a->dim, a->dbias, s);
    else e = column_join<__bf16>(p.sums, blocks, columns, a->dweight, a->dim, a->dbias, s);
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

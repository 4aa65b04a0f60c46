// Softmax cross entropy of rows against a large vocabulary (C entries: nd_vocabulary_loss_*).
//
//   z_iv = h_i . w_v,  lse_i = log sum_v exp z_iv,  loss_i = lse_i - z_{i, t_i}
//   g_iv = dloss_i (exp(z_iv - lse_i) - [v = t_i]),  dh = g w,  dw = g^T h
// A row whose target is no class (the engine's "no vertex" is |V|) has loss 0 and no gradient.
//
// The logits are never kept.  Forward: a workgroup makes a tile of Z^T = W H^T and keeps one maximum and one sum of a row
// for it; a second kernel joins them.  Backward: for one piece of the vocabulary after another the tiles are made again,
// turned into g (16 bits, in a workspace of one piece) and multiplied by w and by h.
#include "../../include/nextdoor_amd.h"

#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "nd_errors.hpp"
#include "nd_matrix.hpp"

namespace nd {
namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kTile = 128;             // rows and columns of a workgroup's product: four waves of 64 x 64
constexpr int kDepth = 64;             // places of the sum per round
constexpr float kGradientOne = 32768.f;  // what |g| = max |dloss| is held as (below the largest 16-bit float)

struct LossParams {
  const void *hidden, *weight;
  const int32_t* target;
  const float* dloss;
  float *loss, *lse;
  void *dhidden, *dweight;
  int32_t rows, classes, dim;
  // workspace
  float2* partials;   // forward: (maximum, sum) of a row over 64 classes, in powers of two; [part][row]
  u32x4* gradient;    // backward: g of one piece of the vocabulary, see gradient_place
  float* dhidden_sum; // [rows][dim], if there is more than one piece
  float* largest;     // max |dloss|
  void* hidden_known; // hidden, the rows without a target zero
  int32_t row_blocks; // of 32 rows, a multiple of 4
  int32_t class0, class_end;  // the piece
};

// g of 32 rows x 32 classes is kept as it leaves the product that made it, ready to be an operand (PAIRED order over the
// classes): slice s has classes 16 s .. + 15, half h of it (row r, classes 16 s + 4 h .. + 3 and 16 s + 8 + 4 h .. + 3) in
// 16 bytes.  The rows are permuted so that reads by columns meet different banks.
__device__ __forceinline__ int gradient_place(int r, int s, int h) { return s * 64 + h * 32 + (r ^ ((h | 2 * s) << 2)); }
constexpr int kGradientBlock = 128;  // 16-byte chunks of 32 rows x 32 classes

// ---- operands of a round of 64 places, 128 rows ----------------------------------------------------

// A matrix whose rows are the operand's rows: [row][place].
struct ByRows {
  const char* base;
  int64_t row_bytes;
  int row0, row_end, places;
  static constexpr int kChunks = kTile * kDepth / 8;
  __device__ __forceinline__ void load(u32x4* tile, int place0) const {
#pragma unroll
    for (int i = 0; i < kChunks / 256; ++i) {
      const int at = threadIdx.x + 256 * i, r = at / 8, c = at % 8;
      u32x4 v = {0, 0, 0, 0};
      if (row0 + r < row_end && place0 + c * 8 < places)
        v = *(const u32x4*)(base + (int64_t)(row0 + r) * row_bytes + (int64_t)(place0 + c * 8) * 2);
      tile[tile_place<8>(r, c)] = v;
    }
  }
  template <bool PAIRED>
  __device__ __forceinline__ static u32x4 operand(const u32x4* tile, int row, int s, int lane) {
    static_assert(!PAIRED, "read by rows only in the plain order");
    return read_operand_by_rows<8>(tile, row, s, lane);
  }
};

// A matrix whose rows are the places: [place][row].
struct ByColumns {
  const char* base;
  int64_t row_bytes;
  int row0, row_end, places;
  static constexpr int kChunks = kTile * kDepth / 8;
  __device__ __forceinline__ void load(u32x4* tile, int place0) const {
#pragma unroll
    for (int i = 0; i < kChunks / 256; ++i) {
      const int at = threadIdx.x + 256 * i, r = at / 16, c = at % 16;
      u32x4 v = {0, 0, 0, 0};
      if (place0 + r < places && row0 + c * 8 < row_end)
        v = *(const u32x4*)(base + (int64_t)(place0 + r) * row_bytes + (int64_t)(row0 + c * 8) * 2);
      tile[tile_place<16>(r, c)] = v;
    }
  }
  template <bool PAIRED>
  __device__ __forceinline__ static u32x4 operand(const u32x4* tile, int row, int s, int lane) {
    return read_operand_by_columns<16, PAIRED>(tile, 16 * s, row, lane);
  }
};

// g with the rows of the loss as rows, places = classes of the piece.
struct GradientByRows {
  const u32x4* base;
  int row_blocks, row0;
  static constexpr int kChunks = kTile * kDepth / 8;
  __device__ __forceinline__ void load(u32x4* tile, int place0) const {
#pragma unroll
    for (int i = 0; i < kChunks / 256; ++i) {
      const int at = threadIdx.x + 256 * i, vb = at / (4 * kGradientBlock);
      tile[at] = base[((int64_t)(place0 / 32 + vb) * row_blocks + row0 / 32) * kGradientBlock + at % (4 * kGradientBlock)];
    }
  }
  template <bool PAIRED>
  __device__ __forceinline__ static u32x4 operand(const u32x4* tile, int row, int s, int lane) {
    static_assert(PAIRED, "kept in the paired order");
    return tile[((s >> 1) * 4 + row / 32) * kGradientBlock + gradient_place(lane & 31, s & 1, lane >> 5)];
  }
};

// g with the classes of the piece as rows, places = rows of the loss.
struct GradientByColumns {
  const u32x4* base;
  int row_blocks, row0;
  static constexpr int kChunks = kTile * kDepth / 8;
  __device__ __forceinline__ void load(u32x4* tile, int place0) const {
#pragma unroll
    for (int i = 0; i < kChunks / 256; ++i) {
      const int at = threadIdx.x + 256 * i, vb = at / (2 * kGradientBlock);
      tile[at] = base[((int64_t)(row0 / 32 + vb) * row_blocks + place0 / 32) * kGradientBlock + at % (2 * kGradientBlock)];
    }
  }
  template <bool PAIRED>
  __device__ __forceinline__ static u32x4 operand(const u32x4* tile, int row, int s, int lane) {
    static_assert(!PAIRED, "read in the plain order");
    const int h = lane >> 5, at = (lane & 15) >> 2, slice = (lane >> 4) & 1, hh = lane & 1, upper = (lane >> 1) & 1;
    const u32x4* block = tile + ((row / 32) * 2 + (s >> 1)) * kGradientBlock;
    const int r = 16 * (s & 1) + 8 * h + at;
    const u32x2 a = read_columns((const char*)(block + gradient_place(r, slice, hh)) + upper * 8);
    const u32x2 b = read_columns((const char*)(block + gradient_place(r + 4, slice, hh)) + upper * 8);
    u32x4 out;
    out[0] = a[0];
    out[1] = a[1];
    out[2] = b[0];
    out[3] = b[1];
    return out;
  }
};

// acc += A B^T over all places; a wave has rows 64 * (wave / 2) of A and 64 * (wave % 2) of B.
template <class T, bool PAIRED, class A, class B>
__device__ __forceinline__ void multiply(f32x16 (&acc)[2][2], const A& a, const B& b, int places, u32x4* tile_a, u32x4* tile_b) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int k = 0; k < places; k += kDepth) {
    __syncthreads();
    a.load(tile_a, k);
    b.load(tile_b, k);
    __syncthreads();
#pragma unroll
    for (int s = 0; s < kDepth / 16; ++s) {
      u32x4 fa[2], fb[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        fa[i] = A::template operand<PAIRED>(tile_a, 64 * (wave >> 1) + 32 * i, s, lane);
        fb[i] = B::template operand<PAIRED>(tile_b, 64 * (wave & 1) + 32 * i, s, lane);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = product_32x32x16<T>(fa[i], fb[j], acc[i][j]);
    }
  }
}

// ---- Z^T = W H^T ----------------------------------------------------------------------------------
// Rows of the result are classes and lie in a lane's registers, its column is the lane's row of the loss: the softmax over
// classes is mostly a lane's own.  BACKWARD: g instead of the maxima and sums.
template <class T, bool BACKWARD>
__global__ __launch_bounds__(256) void logits_kernel(LossParams p) {
  __shared__ u32x4 tile_a[ByRows::kChunks], tile_b[ByRows::kChunks];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
  const int class0 = p.class0 + blockIdx.x * kTile, row0 = blockIdx.y * kTile;
  const int64_t row_bytes = (int64_t)p.dim * 2;
  f32x16 z[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) z[i][j] = f32x16{};
  multiply<T, false>(z, ByRows{(const char*)p.weight, row_bytes, class0, p.class_end, p.dim},
                     ByRows{(const char*)p.hidden, row_bytes, row0, p.rows, p.dim}, p.dim, tile_a, tile_b);
  const int wave_class0 = class0 + 64 * (wave >> 1);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int row = row0 + 64 * (wave & 1) + 32 * j + (lane & 31);
    if (!BACKWARD) {
      float m = -INFINITY;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int n = 0; n < 16; ++n) {
          const int c = wave_class0 + 32 * i + 8 * (n / 4) + 4 * h + n % 4;
          z[i][j][n] = c < p.class_end ? z[i][j][n] : -INFINITY;
          m = fmaxf(m, z[i][j][n]);
        }
      const float m2 = pair_max(m) * kLog2e, base = m2 == -INFINITY ? 0.f : m2;
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int n = 0; n < 16; ++n) sum += exp2_fast(__builtin_fmaf(z[i][j][n], kLog2e, -base));
      sum = pair_sum(sum);
      if (h == 0 && row < p.rows) p.partials[((int64_t)blockIdx.x * 2 + (wave >> 1)) * p.rows + row] = make_float2(m2, sum);
    } else {
      const bool there = row < p.rows;
      const int target = there ? p.target[row] : -1;
      const bool has = target >= 0 && target < p.classes;
      const float largest = *p.largest;
      const float each = has && largest > 0.f ? p.dloss[row] / largest * kGradientOne : 0.f;
      const float lse2 = there ? p.lse[row] * kLog2e : 0.f;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        f32x16 g;
#pragma unroll
        for (int n = 0; n < 16; ++n) {
          const int c = wave_class0 + 32 * i + 8 * (n / 4) + 4 * h + n % 4;
          float v = exp2_fast(__builtin_fmaf(z[i][j][n], kLog2e, -lse2));
          if (c == target) v -= 1.f;
          g[n] = has && c < p.class_end ? v * each : 0.f;
        }
        const int64_t block = (int64_t)((wave_class0 - p.class0) / 32 + i) * p.row_blocks + (row - (lane & 31)) / 32;
#pragma unroll
        for (int s = 0; s < 2; ++s)
          p.gradient[block * kGradientBlock + gradient_place(lane & 31, s, h)] = pack_operand<T>(g, s);
      }
    }
  }
}

// Joins the maxima and sums of 64 rows; loss = lse - z of the target, its logit from the vectors themselves.
template <class T>
__global__ __launch_bounds__(256) void join_kernel(LossParams p, int parts) {
  __shared__ float2 partial[4][64];
  __shared__ float lses[64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int row0 = blockIdx.x * 64, row = row0 + lane;
  float m = -INFINITY, sum = 0.f;
  if (row < p.rows)
    for (int i = wave; i < parts; i += 4) {
      const float2 one = p.partials[(int64_t)i * p.rows + row];
      const float top = fmaxf(m, one.x), base = top == -INFINITY ? 0.f : top;
      sum = sum * exp2_fast(m - base) + one.y * exp2_fast(one.x - base);
      m = top;
    }
  partial[wave][lane] = make_float2(m, sum);
  __syncthreads();
  if (wave == 0) {
    for (int i = 1; i < 4; ++i) {
      const float2 one = partial[i][lane];
      const float top = fmaxf(m, one.x), base = top == -INFINITY ? 0.f : top;
      sum = sum * exp2_fast(m - base) + one.y * exp2_fast(one.x - base);
      m = top;
    }
    lses[lane] = (m + log2f(sum)) * kLn2;
    if (row < p.rows) p.lse[row] = lses[lane];
  }
  __syncthreads();
  for (int i = wave; i < 64 && row0 + i < p.rows; i += 4) {
    const int target = p.target[row0 + i];
    const bool has = target >= 0 && target < p.classes;
    float z = 0.f;
    if (has) {
      const u32x4* a = (const u32x4*)((const char*)p.hidden + (int64_t)(row0 + i) * p.dim * 2);
      const u32x4* b = (const u32x4*)((const char*)p.weight + (int64_t)target * p.dim * 2);
      for (int c = lane; c < p.dim / 8; c += 64) {
        const u32x4 x = a[c], y = b[c];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          z = __builtin_fmaf(unpack_low<T>(x[n]), unpack_low<T>(y[n]), z);
          z = __builtin_fmaf(unpack_high<T>(x[n]), unpack_high<T>(y[n]), z);
        }
      }
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) z += __shfl_xor(z, d);
    if (lane == 0) p.loss[row0 + i] = has ? lses[i] - z : 0.f;
  }
}

// max |dloss|: g is held relative to it, so that 16-bit floats hold the gradient of a mean over any number of rows.
__global__ __launch_bounds__(1024) void largest_kernel(LossParams p) {
  __shared__ float tops[16];
  float m = 0.f;
  for (int i = threadIdx.x; i < p.rows; i += 1024) if (p.target[i] >= 0 && p.target[i] < p.classes) m = fmaxf(m, fabsf(p.dloss[i]));
#pragma unroll
  for (int d = 1; d < 64; d *= 2) m = fmaxf(m, __shfl_xor(m, d));
  if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = m;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 16; ++i) m = fmaxf(m, tops[i]);
    *p.largest = m;
  }
}

// A row without a target sends nothing to dw, whatever it holds: 0 x NaN would be NaN.
__global__ __launch_bounds__(256) void known_rows_kernel(LossParams p) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int chunks = p.dim / 8;
  if (i >= (int64_t)p.rows * chunks) return;
  const int target = p.target[i / chunks];
  u32x4 v = {0, 0, 0, 0};
  if (target >= 0 && target < p.classes) v = ((const u32x4*)p.hidden)[i];
  ((u32x4*)p.hidden_known)[i] = v;
}

// dh of the piece: a row of the result is a row of the loss, its column (the lane's) a column of the vectors.
template <class T>
__global__ __launch_bounds__(256) void dhidden_kernel(LossParams p) {
  __shared__ u32x4 tile_a[GradientByRows::kChunks], tile_b[ByColumns::kChunks];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
  const int column0 = blockIdx.x * kTile, row0 = blockIdx.y * kTile, classes = p.class_end - p.class0;
  f32x16 acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) acc[i][j] = f32x16{};
  multiply<T, true>(acc, GradientByRows{p.gradient, p.row_blocks, row0},
                    ByColumns{(const char*)p.weight + (int64_t)p.class0 * p.dim * 2, (int64_t)p.dim * 2, column0, p.dim, classes},
                    classes, tile_a, tile_b);
  const float factor = *p.largest / kGradientOne;
  const bool first = p.class0 == 0, last = p.class_end == p.classes;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int column = column0 + 64 * (wave & 1) + 32 * j + (lane & 31);
#pragma unroll
      for (int n = 0; n < 16; ++n) {
        const int row = row0 + 64 * (wave >> 1) + 32 * i + 8 * (n / 4) + 4 * h + n % 4;
        if (row >= p.rows || column >= p.dim) continue;
        const int64_t at = (int64_t)row * p.dim + column;
        const float sum = acc[i][j][n] * factor + (first ? 0.f : p.dhidden_sum[at]);
        if (last) ((T*)p.dhidden)[at] = (T)sum;
        else p.dhidden_sum[at] = sum;
      }
    }
}

// dw of the piece's classes, whole at once.
template <class T>
__global__ __launch_bounds__(256) void dweight_kernel(LossParams p) {
  __shared__ u32x4 tile_a[GradientByColumns::kChunks], tile_b[ByColumns::kChunks];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
  const int column0 = blockIdx.x * kTile, class0 = blockIdx.y * kTile;  // in the piece
  f32x16 acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) acc[i][j] = f32x16{};
  multiply<T, false>(acc, GradientByColumns{p.gradient, p.row_blocks, class0},
                     ByColumns{(const char*)p.hidden_known, (int64_t)p.dim * 2, column0, p.dim, p.rows}, p.rows, tile_a, tile_b);
  const float factor = *p.largest / kGradientOne;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int column = column0 + 64 * (wave & 1) + 32 * j + (lane & 31);
#pragma unroll
      for (int n = 0; n < 16; ++n) {
        const int c = p.class0 + class0 + 64 * (wave >> 1) + 32 * i + 8 * (n / 4) + 4 * h + n % 4;
        if (c < p.class_end && column < p.dim) ((T*)p.dweight)[(int64_t)c * p.dim + column] = (T)(acc[i][j][n] * factor);
      }
    }
}

// ---- host -----------------------------------------------------------------------------------------

int64_t round_up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// Classes of a piece: g of all rows stays within 256 MiB (the last-level cache), but at least 2048 classes.
int64_t piece_classes(int64_t rows, int64_t classes) {
  const int64_t fit = ((int64_t)256 << 20) / (2 * round_up(std::max<int64_t>(rows, 1), kTile)) / kTile * kTile;
  return std::min(round_up(classes, kTile), std::max<int64_t>(fit, 2048));
}

struct LossWorkspace {
  int64_t partials, gradient, dhidden_sum, largest, hidden_known, bytes;
};
LossWorkspace workspace_of(int64_t rows, int64_t classes, int64_t dim, bool backward) {
  LossWorkspace w = {};
  auto take = [&](int64_t bytes) {
    const int64_t at = w.bytes;
    w.bytes += round_up(bytes, 256);
    return at;
  };
  if (!backward) {
    w.partials = take(round_up(classes, kTile) / 64 * rows * (int64_t)sizeof(float2));
  } else {
    const int64_t piece = piece_classes(rows, classes);
    w.largest = take(sizeof(float));
    w.hidden_known = take(rows * dim * 2);
    w.gradient = take(round_up(rows, kTile) * piece * 2);
    if (piece < classes) w.dhidden_sum = take(rows * dim * (int64_t)sizeof(float));
  }
  return w;
}

template <class T>
void launch_forward(LossParams p, hipStream_t stream) {
  const dim3 grid((p.classes + kTile - 1) / kTile, (p.rows + kTile - 1) / kTile);
  logits_kernel<T, false><<<grid, 256, 0, stream>>>(p);
  join_kernel<T><<<(p.rows + 63) / 64, 256, 0, stream>>>(p, (int)grid.x * 2);
}

template <class T>
void launch_backward(LossParams p, hipStream_t stream) {
  largest_kernel<<<1, 1024, 0, stream>>>(p);
  if (p.rows > 0)
    known_rows_kernel<<<(uint32_t)(((int64_t)p.rows * (p.dim / 8) + 255) / 256), 256, 0, stream>>>(p);
  const int64_t piece = piece_classes(p.rows, p.classes);
  const uint32_t row_tiles = (p.rows + kTile - 1) / kTile, column_tiles = (p.dim + kTile - 1) / kTile;
  for (int64_t at = 0; at < p.classes; at += piece) {
    p.class0 = (int32_t)at;
    p.class_end = (int32_t)std::min<int64_t>(at + piece, p.classes);
    const uint32_t class_tiles = (p.class_end - p.class0 + kTile - 1) / kTile;
    if (p.rows > 0) {
      logits_kernel<T, true><<<dim3(class_tiles, row_tiles), 256, 0, stream>>>(p);
      dhidden_kernel<T><<<dim3(column_tiles, row_tiles), 256, 0, stream>>>(p);
    }
    dweight_kernel<T><<<dim3(column_tiles, class_tiles), 256, 0, stream>>>(p);
  }
}

int run_loss(const nd_vocabulary_loss* a, bool backward, void* stream) {
  if (!a) return fail("vocabulary loss: null argument");
  if (a->dtype != ND_F16 && a->dtype != ND_BF16) return fail("vocabulary loss: 16-bit types only (ND_F16, ND_BF16)");
  if (a->rows < 0 || a->rows > ND_VOCABULARY_MAX_ROWS)
    return fail("vocabulary loss: between 0 and " + std::to_string(ND_VOCABULARY_MAX_ROWS) + " rows, " + std::to_string(a->rows) + " given");
  if (a->classes < 1 || a->classes > ND_VOCABULARY_MAX_CLASSES)
    return fail("vocabulary loss: between 1 and " + std::to_string(ND_VOCABULARY_MAX_CLASSES) + " classes, " +
                std::to_string(a->classes) + " given");
  if (a->dim < 8 || a->dim > ND_VOCABULARY_MAX_DIM || a->dim % 8 != 0)
    return fail("vocabulary loss: the vectors' size is a multiple of 8 up to " + std::to_string(ND_VOCABULARY_MAX_DIM) + ", " +
                std::to_string(a->dim) + " given");
  if (a->rows == 0 && !backward) return 0;
  const LossWorkspace w = workspace_of(a->rows, a->classes, a->dim, backward);
  if (a->workspace_bytes < w.bytes)
    return fail("vocabulary loss: the workspace has " + std::to_string(a->workspace_bytes) + " bytes, " + std::to_string(w.bytes) + " needed");
  const void* in[] = {a->weight, a->workspace, a->dweight, a->hidden, a->dhidden};
  const bool needed[] = {true, true, backward, a->rows > 0, backward && a->rows > 0};
  for (int i = 0; i < 5; ++i)
    if (needed[i] && (!in[i] || ((uintptr_t)in[i] & 15))) return fail("vocabulary loss: null array, or one not aligned to 16 bytes");
  if (a->rows > 0 && (!a->target || !a->lse || (backward ? !a->dloss : !a->loss))) return fail("vocabulary loss: null array");
  LossParams p = {};
  p.hidden = a->hidden;
  p.weight = a->weight;
  p.target = a->target;
  p.dloss = a->dloss;
  p.loss = a->loss;
  p.lse = a->lse;
  p.dhidden = a->dhidden;
  p.dweight = a->dweight;
  p.rows = (int32_t)a->rows;
  p.classes = (int32_t)a->classes;
  p.dim = a->dim;
  char* work = (char*)a->workspace;
  p.partials = (float2*)(work + w.partials);
  p.gradient = (u32x4*)(work + w.gradient);
  p.dhidden_sum = (float*)(work + w.dhidden_sum);
  p.largest = (float*)(work + w.largest);
  p.hidden_known = work + w.hidden_known;
  p.row_blocks = (int32_t)(round_up(a->rows, kTile) / 32);
  p.class_end = p.classes;
  if (backward) {
    if (a->dtype == ND_BF16) launch_backward<__bf16>(p, (hipStream_t)stream);
    else launch_backward<_Float16>(p, (hipStream_t)stream);
  } else {
    if (a->dtype == ND_BF16) launch_forward<__bf16>(p, (hipStream_t)stream);
    else launch_forward<_Float16>(p, (hipStream_t)stream);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(std::string("vocabulary loss: ") + hipGetErrorString(e));
  return 0;
}

}  // namespace
}  // namespace nd

extern "C" {

int64_t nd_vocabulary_loss_workspace(int64_t rows, int64_t classes, int32_t dim, int backward) {
  if (rows < 0 || rows > ND_VOCABULARY_MAX_ROWS || classes < 1 || classes > ND_VOCABULARY_MAX_CLASSES || dim < 1 ||
      dim > ND_VOCABULARY_MAX_DIM)
    return -1;
  return nd::workspace_of(rows, classes, dim, backward != 0).bytes;
}

int nd_vocabulary_loss_forward(const nd_vocabulary_loss* a, void* stream) {
  return nd::guarded([&]() -> int { return nd::run_loss(a, false, stream); });
}

int nd_vocabulary_loss_backward(const nd_vocabulary_loss* a, void* stream) {
  return nd::guarded([&]() -> int { return nd::run_loss(a, true, stream); });
}

}  // extern "C"

// Softmax cross entropy of rows against a large vocabulary (C entries: nd_vocabulary_loss_*).
//
//   z_iv = h_i . w_v,  lse_i = log sum_v exp z_iv,  loss_i = lse_i - z_{i, t_i}
//   g_iv = dloss_i (exp(z_iv - lse_i) - [v = t_i]),  dh = g w,  dw = g^T h
// A row whose target is no class (the engine's "no vertex" is |V|) has loss 0 and no gradient.
//
// The logits are never kept.  Forward: a workgroup makes a tile of Z^T = W H^T and keeps one maximum and one sum of a row
// for it; a second kernel joins them.  Backward, vectors of up to 224: dh and dw each make the logits once more and turn them
// into g in registers, where it is the operand of their second product.  Longer vectors: the logits are made once more for one
// piece of the vocabulary after another, and g (16 bits, in a workspace of one piece) is multiplied by w and by h.
#include "../../include/nextdoor_amd.h"

#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "nd_errors.hpp"
#include "nd_matrix.hpp"
#include "nd_row_tiles.hpp"

namespace nd {
namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// What g is held times: in 16-bit floats such that max |dloss| becomes this (below their largest); bfloat16 has the exponents of
// 32 bits, and a constant keeps the smallest weights of a mean over millions of rows among the normal numbers.
constexpr float kGradientOne = 32768.f, kGradientScale = 4294967296.f;
constexpr float kLeastLargest = 0x1p-100f;  // max |dloss| that this is done for: one over it is still finite, and less is 0 in 16 bits
constexpr int kClassPad = 256;           // a piece of the vocabulary is filled up to a multiple of it

struct LossParams {
  const void *hidden, *weight;
  const int32_t* target;
  const float* dloss;
  float *loss, *lse;
  void *dhidden, *dweight;
  int32_t rows, classes, dim;
  // workspace
  float2* partials;    // forward: (maximum, sum) of a row over one wave's classes, in powers of two; [part][row]
  u32x4* gradient;     // backward: g of one piece of the vocabulary, see gradient_place
  float* dhidden_sums; // [split][rows][dim]
  float* dweight_sums; // [split][classes of the piece][dim]
  float* scale;        // what g is held times, and one over it
  void* hidden_known;  // hidden, filled up to padded_rows; rows without a target are zero; twice, if g_rows says so
  // of a row: g = +-exp2(z log2(e) + shift) - [class = target] each; no target: each 0, shift -inf, target -1
  float *row_each, *row_shift;
  int32_t* row_target;
  int32_t padded_rows;
  // longer vectors: rows that g is kept for.  Few rows: twice padded_rows, g rounded and what the rounding left, for dw
  int32_t g_rows;
  int32_t class0, class_end;  // the piece
  int32_t dhidden_split, dweight_split;
};

// g of 32 rows x 32 classes is kept as it leaves the product that made it, ready to be an operand (PAIRED order over the
// classes): slice s has classes 16 s .. + 15, half h of it (row r, classes 16 s + 4 h .. + 3 and 16 s + 8 + 4 h .. + 3) in
// 16 bytes.  The rows are permuted so that reads by columns meet different banks.
__device__ __forceinline__ int gradient_place(int r, int s, int h) { return s * 64 + h * 32 + (r ^ ((h | 2 * s) << 2)); }
// The gradient of a row is -each at its target and small elsewhere: that one rounding of g would show in every column of dh.
// So g is formed with `each` rounded to 16 bits, where the target's is exact but for its own weight, and the rows of dh, in 32
// bits, are multiplied by each / (each rounded); dw takes g in two parts, rounded and rest.  Longer vectors do so where rows are
// few; over many such roundings are as good as any.
template <class T>
__device__ __forceinline__ float row_ratio(float each) {
  const float rounded = unpack_low<T>(pack_pair<T>(each, 0.f)), ratio = each / rounded;
  return rounded != 0.f && fabsf(ratio - 1.f) < 0.01f ? ratio : 1.f;
}
constexpr int kGradientBlock = 128;  // 16-byte chunks of 32 rows x 32 classes
constexpr int kGradientBlockBytes = kGradientBlock * 16;

// ---- the shape of a workgroup's product -------------------------------------------------------------
// kWavesM x kWavesN waves, each with kM x kN results of 32 x 32, kDepth places of the sum per round.
template <int WAVES_M, int WAVES_N, int M, int N, int DEPTH>
struct Shape {
  static constexpr int kWavesM = WAVES_M, kWavesN = WAVES_N, kM = M, kN = N, kDepth = DEPTH;
  static constexpr int kThreads = 64 * WAVES_M * WAVES_N;
  static constexpr int kTileM = 32 * WAVES_M * M, kTileN = 32 * WAVES_N * N;
  static constexpr int kWavesPerSimd = DEPTH > 64 ? 1 : 2;  // (at least; what LDS has room for)
};

// ---- operands: ROWS rows, DEPTH places of the sum a round, brought to LDS by THREADS threads --------------
// issue() asks for the tile of a round, operand() reads 32 rows x 16 places of it.  What lies past the last place is 0 in
// one of the two operands and some value of the same array in the other; what lies past the last row is some row.

// A matrix whose rows are the operand's rows: [row][place].
template <int ROWS, int DEPTH, int THREADS>
struct ByRows {
  static constexpr int kRowChunks = DEPTH / 8, kChunks = ROWS * kRowChunks, kTurns = kChunks / THREADS;
  static_assert(kChunks % THREADS == 0, "");
  const char* base;
  uint32_t offset[kTurns];
  int places, chunk;
  __device__ __forceinline__ ByRows(const void* matrix, int64_t row_bytes, int row0, int row_end, int places_)
      : base((const char*)matrix + row0 * row_bytes), places(places_) {
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
      const int at = threadIdx.x + THREADS * i, r = at / kRowChunks, c = (at % kRowChunks) ^ tile_swizzle<kRowChunks>(r);
      offset[i] = (uint32_t)(min(r, row_end - 1 - row0) * row_bytes + c * 16);
      chunk = c;  // (the same in every turn: THREADS / kRowChunks is a multiple of 16 rows)
    }
  }
  __device__ __forceinline__ void issue(u32x4* tile, uint32_t wave_lds, int place0) const {
    const char* at = base + (int64_t)place0 * 2;
    if (place0 + DEPTH <= places) {
#pragma unroll
      for (int i = 0; i < kTurns; ++i) load_to_lds(at, offset[i], wave_lds + THREADS * 16 * i);
    } else {
      const bool there = place0 + chunk * 8 < places;
#pragma unroll
      for (int i = 0; i < kTurns; ++i) {
        if (there) load_to_lds(at, offset[i], wave_lds + THREADS * 16 * i);
        else tile[threadIdx.x + THREADS * i] = u32x4{0, 0, 0, 0};
      }
    }
  }
  template <bool PAIRED>
  __device__ __forceinline__ static u32x4 operand(const u32x4* tile, int row, int s, int lane) {
    static_assert(!PAIRED, "read by rows only in the plain order");
    return read_operand_by_rows<kRowChunks>(tile, row, s, lane);
  }
};

// A matrix whose rows are the places: [place][row].
template <int ROWS, int DEPTH, int THREADS>
struct ByColumns {
  static constexpr int kRowChunks = ROWS / 8, kChunks = DEPTH * kRowChunks, kTurns = kChunks / THREADS;
  static_assert(kChunks % THREADS == 0, "");
  const char* base;
  int64_t row_bytes;
  uint32_t offset[kTurns];
  int places;
  __device__ __forceinline__ ByColumns(const void* matrix, int64_t row_bytes_, int row0, int row_end, int places_)
      : base((const char*)matrix + (int64_t)row0 * 2), row_bytes(row_bytes_), places(places_) {
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
      const int at = threadIdx.x + THREADS * i, r = at / kRowChunks, c = (at % kRowChunks) ^ tile_swizzle<kRowChunks>(r);
      offset[i] = (uint32_t)(r * row_bytes) + (row0 + c * 8 < row_end ? c * 16 : 0);
    }
  }
  __device__ __forceinline__ void issue(u32x4*, uint32_t wave_lds, int place0) const {
    const char* at = base + place0 * row_bytes;
    if (place0 + DEPTH <= places) {
#pragma unroll
      for (int i = 0; i < kTurns; ++i) load_to_lds(at, offset[i], wave_lds + THREADS * 16 * i);
    } else {  // rows past the last place: the last one (the other operand is 0 there)
#pragma unroll
      for (int i = 0; i < kTurns; ++i) {
        const int r = (threadIdx.x + THREADS * i) / kRowChunks, past = max(place0 + r - (places - 1), 0);
        load_to_lds(at, offset[i] - (uint32_t)(past * row_bytes), wave_lds + THREADS * 16 * i);
      }
    }
  }
  template <bool PAIRED>
  __device__ __forceinline__ static u32x4 operand(const u32x4* tile, int row, int s, int lane) {
    return read_operand_by_columns<kRowChunks, PAIRED>(tile, 16 * s, row, lane);
  }
};

// g with the rows of the loss as rows, places = classes of the piece.
template <int ROWS, int DEPTH, int THREADS>
struct GradientByRows {
  static constexpr int kChunks = ROWS * DEPTH / 8, kTurns = kChunks / THREADS, kBlocks = ROWS / 32;
  static_assert(kChunks % THREADS == 0, "");
  const char* base;
  int64_t step;
  uint32_t offset[kTurns];
  __device__ __forceinline__ GradientByRows(const u32x4* gradient, int padded_rows, int row0)
      : base((const char*)gradient + (int64_t)(row0 / 32) * kGradientBlockBytes), step((int64_t)(padded_rows / 32) * kGradientBlockBytes) {
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
      const int at = threadIdx.x + THREADS * i;
      offset[i] = (uint32_t)(at / (kBlocks * kGradientBlock) * step) + at % (kBlocks * kGradientBlock) * 16;
    }
  }
  __device__ __forceinline__ void issue(u32x4*, uint32_t wave_lds, int place0) const {
    const char* at = base + place0 / 32 * step;
#pragma unroll
    for (int i = 0; i < kTurns; ++i) load_to_lds(at, offset[i], wave_lds + THREADS * 16 * i);
  }
  template <bool PAIRED>
  __device__ __forceinline__ static u32x4 operand(const u32x4* tile, int row, int s, int lane) {
    static_assert(PAIRED, "kept in the paired order");
    return tile[((s >> 1) * kBlocks + row / 32) * kGradientBlock + gradient_place(lane & 31, s & 1, lane >> 5)];
  }
};

// g with the classes of the piece as rows, places = rows of the loss.
template <int ROWS, int DEPTH, int THREADS>
struct GradientByColumns {
  static constexpr int kChunks = ROWS * DEPTH / 8, kTurns = kChunks / THREADS, kBlocks = DEPTH / 32;
  static_assert(kChunks % THREADS == 0, "");
  const char* base;
  uint32_t offset[kTurns];
  __device__ __forceinline__ GradientByColumns(const u32x4* gradient, int padded_rows, int class0) {
    const int64_t step = (int64_t)(padded_rows / 32) * kGradientBlockBytes;
    base = (const char*)gradient + class0 / 32 * step;
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
      const int at = threadIdx.x + THREADS * i;
      offset[i] = (uint32_t)(at / (kBlocks * kGradientBlock) * step) + at % (kBlocks * kGradientBlock) * 16;
    }
  }
  __device__ __forceinline__ void issue(u32x4*, uint32_t wave_lds, int place0) const {
    const char* at = base + (int64_t)(place0 / 32) * kGradientBlockBytes;
#pragma unroll
    for (int i = 0; i < kTurns; ++i) load_to_lds(at, offset[i], wave_lds + THREADS * 16 * i);
  }
  template <bool PAIRED>
  __device__ __forceinline__ static u32x4 operand(const u32x4* tile, int row, int s, int lane) {
    static_assert(!PAIRED, "read in the plain order");
    const int h = lane >> 5, at = (lane & 15) >> 2, slice = (lane >> 4) & 1, hh = lane & 1, upper = (lane >> 1) & 1;
    const u32x4* block = tile + ((row / 32) * kBlocks + (s >> 1)) * kGradientBlock;
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

// acc += A B^T over the places place0 .. place_end - 1: while the matrix cores work on one tile the next is on its way to
// the other half of LDS.  One barrier a round: at it, this round's tile has arrived for all and the last one's is free.
// tiles: twice a round's tiles of LDS, which the caller may use again after a barrier.
//
// 256 x 256 x 64, eight waves of 4 x 2 results: an operand read from LDS serves two or four products.  The three products of 4096
// rows x 131072 classes x 1024 run at 1.03 to 1.16 PFLOP/s, matrix cores busy 56 to 60 % at the 1.8 GHz that the GPU keeps up under
// them; more stages, operands fetched one slice ahead and another wave priority all gave the same.
template <class A, class B>
constexpr int kTileChunks = 2 * (A::kChunks + B::kChunks);
template <class T, class S, bool PAIRED, class A, class B>
__device__ __forceinline__ void multiply(f32x16 (&acc)[S::kM][S::kN], const A& a, const B& b, int place0, int place_end, u32x4* tiles) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m0 = wave / S::kWavesN * 32 * S::kM, n0 = wave % S::kWavesN * 32 * S::kN;
#pragma unroll
  for (int i = 0; i < S::kM; ++i)
#pragma unroll
    for (int j = 0; j < S::kN; ++j) acc[i][j] = f32x16{};
  const uint32_t lds = lds_address(tiles) + wave * 1024;
  constexpr int kHalf = A::kChunks + B::kChunks;
  int half = 0;
  auto issue = [&](int into, int place) {
    a.issue(tiles + into * kHalf, lds + into * kHalf * 16, place);
    b.issue(tiles + into * kHalf + A::kChunks, lds + (into * kHalf + A::kChunks) * 16, place);
  };
  if (place0 < place_end) issue(0, place0);
  for (int place = place0; place < place_end; place += S::kDepth) {
    wait_for_loads_and_others();
    if (place + S::kDepth < place_end) issue(half ^ 1, place + S::kDepth);
    const u32x4 *tile_a = tiles + half * kHalf, *tile_b = tile_a + A::kChunks;
#pragma unroll
    for (int s = 0; s < S::kDepth / 16; ++s) {
      u32x4 fa[S::kM], fb[S::kN];
#pragma unroll
      for (int j = 0; j < S::kN; ++j) fb[j] = B::template operand<PAIRED>(tile_b, n0 + 32 * j, s, lane);
#pragma unroll
      for (int i = 0; i < S::kM; ++i) fa[i] = A::template operand<PAIRED>(tile_a, m0 + 32 * i, s, lane);
#pragma unroll
      for (int i = 0; i < S::kM; ++i)
#pragma unroll
        for (int j = 0; j < S::kN; ++j) acc[i][j] = product_32x32x16<T>(fa[i], fb[j], acc[i][j]);
    }
    half ^= 1;
  }
}

// ---- Z^T = W H^T ----------------------------------------------------------------------------------
// Rows of the result are classes and lie in a lane's registers, its column is the lane's row of the loss: the softmax over
// classes is mostly a lane's own.  BACKWARD: g instead of the maxima and sums.  4096 rows x 131072 classes x 1024: 1.01 to 1.07
// ms; a quarter of the classes with g, 268 MB written: 286 us, 0.96 PFLOP/s.  1021 x 100003 x 520: 140 us, 0.76 PFLOP/s: 1564 tiles
// are 6.1 to a compute unit, and the last 8 of 520 places take a round of 64.
template <class T, class S, bool BACKWARD>
__global__ __launch_bounds__(S::kThreads, S::kWavesPerSimd) void logits_kernel(LossParams p, int row_tiles) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
  const uint32_t block = block_by_die();
  const int class_tile = uniform(block / row_tiles), class0 = p.class0 + class_tile * S::kTileM;
  const int row0 = uniform(block % row_tiles) * S::kTileN;
  const int64_t row_bytes = (int64_t)p.dim * 2;
  using Classes = ByRows<S::kTileM, S::kDepth, S::kThreads>;
  using Rows = ByRows<S::kTileN, S::kDepth, S::kThreads>;
  __shared__ u32x4 tiles[kTileChunks<Classes, Rows>];
  f32x16 z[S::kM][S::kN];
  // (a tile of nothing but the piece's filling has no class to read: it reads the last one, and g is 0)
  multiply<T, S, false>(z, Classes(p.weight, row_bytes, min(class0, p.class_end - 1), p.class_end, p.dim),
                        Rows(BACKWARD ? p.hidden_known : p.hidden, row_bytes, row0, BACKWARD ? p.padded_rows : p.rows, p.dim), 0, p.dim, tiles);
  const int wave_class0 = class0 + wave / S::kWavesN * 32 * S::kM;
  const int wave_row0 = row0 + wave % S::kWavesN * 32 * S::kN;
  const bool whole = wave_class0 + 32 * S::kM <= p.class_end;
#pragma unroll
  for (int j = 0; j < S::kN; ++j) {
    const int row = wave_row0 + 32 * j + (lane & 31);
    if (!BACKWARD) {
      float m = -INFINITY;
      if (!whole) {
#pragma unroll
        for (int i = 0; i < S::kM; ++i)
#pragma unroll
          for (int n = 0; n < 16; ++n)
            if (wave_class0 + 32 * i + 8 * (n / 4) + 4 * h + n % 4 >= p.class_end) z[i][j][n] = -INFINITY;
      }
#pragma unroll
      for (int i = 0; i < S::kM; ++i)
#pragma unroll
        for (int n = 0; n < 16; ++n) m = fmaxf(m, z[i][j][n]);
      const float m2 = pair_max(m) * kLog2e, base = m2 == -INFINITY ? 0.f : m2;
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < S::kM; ++i)
#pragma unroll
        for (int n = 0; n < 16; ++n) sum += exp2_fast(__builtin_fmaf(z[i][j][n], kLog2e, -base));
      sum = pair_sum(sum);
      if (h == 0 && row < p.rows)
        p.partials[((int64_t)class_tile * S::kWavesM + wave / S::kWavesN) * p.rows + row] = make_float2(m2, sum);
    } else {
      const int target = p.row_target[row];
      const bool in_parts = p.g_rows > p.padded_rows;
      const float exact = p.row_each[row], ratio = in_parts ? row_ratio<T>(exact) : 1.f, each = exact / ratio;
      const float shift = p.row_shift[row] - log2f(ratio);
      const uint32_t negative = each < 0.f ? 0x80000000u : 0u;
      const bool targets_here = __builtin_amdgcn_ballot_w64(target >= wave_class0 && target < wave_class0 + 32 * S::kM) != 0;
      const bool negatives = __builtin_amdgcn_ballot_w64(negative) != 0;
#pragma unroll
      for (int i = 0; i < S::kM; ++i) {
        f32x16 g;
#pragma unroll
        for (int n = 0; n < 16; ++n) g[n] = exp2_fast(__builtin_fmaf(z[i][j][n], kLog2e, shift));
        if (negatives) {
#pragma unroll
          for (int n = 0; n < 16; ++n) g[n] = __uint_as_float(__float_as_uint(g[n]) ^ negative);
        }
        if (targets_here || !whole) {
          const int c0 = wave_class0 + 32 * i + 4 * h;
#pragma unroll
          for (int n = 0; n < 16; ++n) {
            const int c = c0 + 8 * (n / 4) + n % 4;
            if (c == target) g[n] -= each;
            if (c >= p.class_end) g[n] = 0.f;
          }
        }
        const int64_t at = (int64_t)((wave_class0 - p.class0) / 32 + i) * (p.g_rows / 32) + (row - (lane & 31)) / 32;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const u32x4 gf = pack_operand<T>(g, s);
          p.gradient[at * kGradientBlock + gradient_place(lane & 31, s, h)] = gf;
          if (in_parts) {
            // (dh has `each` rounded, so has this: what is left over of both, of g with `each` itself)
            u32x4 rest;
#pragma unroll
            for (int n = 0; n < 4; ++n)
              rest[n] = pack_pair<T>(g[8 * s + 2 * n] * ratio - unpack_low<T>(gf[n]), g[8 * s + 2 * n + 1] * ratio - unpack_high<T>(gf[n]));
            p.gradient[(at + p.padded_rows / 32) * kGradientBlock + gradient_place(lane & 31, s, h)] = rest;
          }
        }
      }
    }
  }
}

constexpr int kRound = 64;  // classes in a round of the kernel for short vectors

// Rounds of a share of n: whole ones, spread evenly.
__device__ __forceinline__ void rounds_of(int rounds, int i, int n, int& begin, int& end) {
  begin = uniform((int)((int64_t)rounds * i / n));
  end = uniform((int)((int64_t)rounds * (i + 1) / n));
}

// The same for vectors of up to 256: a workgroup has 256 rows, a wave 64 of them (two columns of Z^T a lane) in registers, and
// goes over its share of the classes with a running maximum and sum.  Each read of the classes serves two products.  8192 rows x
// 56944 classes: 132 us at 128 (0.90 PFLOP/s, matrix cores busy 47 %, the exponentials between the products the rest), 235 at 256.
template <class T, int NB>
__global__ __launch_bounds__(256, 2) void logits_short_kernel(LossParams p, int row_tiles, int splits) {
  constexpr int kChunks = HeadTile<NB>::kChunks, kSize = kRound * kChunks;
  __shared__ u32x4 tiles[2][kSize];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), h = lane >> 5;
  const uint32_t block = block_by_die();
  const int split = uniform(block / row_tiles), row0 = uniform(block % row_tiles) * 256 + wave * 64;
  int begin, end;
  rounds_of((p.classes + kRound - 1) / kRound, split, splits, begin, end);
  const int64_t row_bytes = (int64_t)p.dim * 2;
  const TileLoader<NB, kRound> w(p.weight, row_bytes, 0, 0, p.dim);
  const uint32_t lds = lds_address(&tiles[0][0]) + wave * 1024;
  if (begin < end) w.issue(lds, row_bytes, begin * kRound, p.classes);
  u32x4 hf[2][2 * NB];
  float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int row = row0 + 32 * j + (lane & 31);
    load_rows<NB>(hf[j], (const char*)p.hidden + row * row_bytes, row < p.rows, p.dim, h);
  }
  int half = 0;
  for (int i = begin; i < end; ++i, half ^= 1) {
    wait_for_loads_and_others();
    if (i + 1 < end) w.issue(lds + (half ^ 1) * kSize * 16, row_bytes, (i + 1) * kRound, p.classes);
    if (row0 >= p.rows) continue;
    const u32x4* tile = tiles[half];
    f32x16 z[2][kRound / 32];
#pragma unroll
    for (int t = 0; t < kRound / 32; ++t) {
      z[0][t] = z[1][t] = f32x16{};
#pragma unroll
      for (int s = 0; s < 2 * NB; ++s) {
        const u32x4 wf = read_operand_by_rows<kChunks>(tile, 32 * t, s, lane);
        z[0][t] = product_32x32x16<T>(wf, hf[0][s], z[0][t]);
        z[1][t] = product_32x32x16<T>(wf, hf[1][s], z[1][t]);
      }
    }
    if ((i + 1) * kRound > p.classes) {
#pragma unroll
      for (int t = 0; t < kRound / 32; ++t)
#pragma unroll
        for (int n = 0; n < 16; ++n)
          if (i * kRound + 32 * t + 8 * (n / 4) + 4 * h + n % 4 >= p.classes) z[0][t][n] = z[1][t][n] = -INFINITY;
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float m = z[j][0][0];
#pragma unroll
      for (int t = 0; t < kRound / 32; ++t)
#pragma unroll
        for (int n = 0; n < 16; ++n) m = fmaxf(m, z[j][t][n]);
      m = pair_max(m) * kLog2e;
      // the sums are taken relative to a maximum that may be up to 2^8 too small, and are rarely scaled again
      if (__builtin_amdgcn_ballot_w64(m > top[j] + 8.f)) {
        const float higher = fmaxf(m, top[j]);
        sum[j] *= higher == -INFINITY ? 0.f : exp2_fast(top[j] - higher);
        top[j] = higher;
      }
      // (a round's weights among themselves first: a share may have a hundred thousand classes, and that many equal weights
      // added to one sum would all be rounded alike)
      const float base = top[j] == -INFINITY ? 0.f : top[j];
      float part = 0.f;
#pragma unroll
      for (int t = 0; t < kRound / 32; ++t)
#pragma unroll
        for (int n = 0; n < 16; ++n) part += exp2_fast(__builtin_fmaf(z[j][t][n], kLog2e, -base));
      sum[j] += part;
    }
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int row = row0 + 32 * j + (lane & 31);
    const float all = pair_sum(sum[j]);
    if (h == 0 && row < p.rows) p.partials[(int64_t)split * p.rows + row] = make_float2(top[j], all);
  }
}

// Joins two (maximum, sum) pairs, in powers of two.
__device__ __forceinline__ void join(float2& a, float2 b) {
  const float top = fmaxf(a.x, b.x), base = top == -INFINITY ? 0.f : top;
  a.y = a.y * exp2_fast(a.x - base) + b.y * exp2_fast(b.x - base);
  a.x = top;
}

// Joins the maxima and sums of 8 rows; loss = lse - z of the target, its logit from the vectors themselves.  A row's parts
// are shared out among 128 lanes: there may be very many (a row of a vocabulary of millions) and few rows.  4096 rows of 1024
// parts: 16 us, 50 MB (3.1 TB/s).
template <class T>
__global__ __launch_bounds__(1024) void join_kernel(LossParams p, int parts) {
  __shared__ float2 partial[16][8];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int row0 = blockIdx.x * 8, mine = row0 + (lane & 7);
  float2 all = make_float2(-INFINITY, 0.f);
  if (mine < p.rows) {
    const float2* from = p.partials + mine;
    int i = threadIdx.x >> 3;
    for (; i + 3 * 128 < parts; i += 4 * 128) {
      float2 four[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) four[j] = from[(int64_t)(i + 128 * j) * p.rows];
#pragma unroll
      for (int j = 0; j < 4; ++j) join(all, four[j]);
    }
    for (; i < parts; i += 128) join(all, from[(int64_t)i * p.rows]);
  }
#pragma unroll
  for (int d = 8; d < 64; d *= 2) join(all, make_float2(__shfl_xor(all.x, d), __shfl_xor(all.y, d)));
  if (lane < 8) partial[wave][lane] = all;
  __syncthreads();
  const int row = row0 + wave;
  if (wave >= 8 || row >= p.rows) return;
  all = partial[0][wave];
  for (int i = 1; i < 16; ++i) join(all, partial[i][wave]);
  const float lse = (all.x + log2f(all.y)) * kLn2;
  const int target = p.target[row];
  const bool has = target >= 0 && target < p.classes;
  float z = 0.f;
  if (has) {
    const u32x4* a = (const u32x4*)((const char*)p.hidden + (int64_t)row * p.dim * 2);
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
  if (lane == 0) {
    p.lse[row] = lse;
    p.loss[row] = has ? lse - z : 0.f;
  }
}

// g in 16-bit floats is held relative to max |dloss|, so that they hold the gradient of a mean over any number of rows.  What is
// not finite does not count: the other rows' dh are as they would be without it.  One workgroup, no atomics: 4 bytes a row are little next to the products that follow.
__global__ __launch_bounds__(1024) void largest_kernel(LossParams p) {
  __shared__ float tops[16];
  float m = 0.f;
  for (int i = threadIdx.x; i < p.rows; i += 1024)
    if (p.target[i] >= 0 && p.target[i] < p.classes && fabsf(p.dloss[i]) < INFINITY) m = fmaxf(m, fabsf(p.dloss[i]));
#pragma unroll
  for (int d = 1; d < 64; d *= 2) m = fmaxf(m, __shfl_xor(m, d));
  if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = m;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 16; ++i) m = fmaxf(m, tops[i]);
    m = fmaxf(m, kLeastLargest);  // (also where there is none)
    p.scale[0] = kGradientOne / m;
    p.scale[1] = m / kGradientOne;
  }
}

// Before the backward products: hidden, filled up with rows of zeros and with zeros for the rows without a target (such a
// row sends nothing to dw, whatever it holds: 0 x NaN would be NaN), and what g takes of each row.  (4096 x 1024: 6 us.)
template <class T, bool SCALED>
__global__ __launch_bounds__(256) void prepare_kernel(LossParams p) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int chunks = p.dim / 8;
  if (i >= (int64_t)p.padded_rows * chunks) return;
  const int row = (int)(i / chunks), target = row < p.rows ? p.target[row] : -1;
  const bool has = target >= 0 && target < p.classes;
  u32x4 v = {0, 0, 0, 0};
  if (has) v = ((const u32x4*)p.hidden)[i];
  ((u32x4*)p.hidden_known)[i] = v;
  const float each = has ? p.dloss[row] * (SCALED ? p.scale[0] : kGradientScale) : 0.f;
  if (p.g_rows > p.padded_rows) ((u32x4*)p.hidden_known)[i + (int64_t)p.padded_rows * chunks] = v;
  if (i % chunks == 0) {
    p.row_each[row] = each;
    p.row_shift[row] = has ? log2f(fabsf(each)) - p.lse[row] * kLog2e : -INFINITY;
    p.row_target[row] = has ? target : -1;
  }
  if (!SCALED && i == 0) p.scale[1] = 1.f / kGradientScale;
}

// ---- backward, vectors of up to 224 --------------------------------------------------------------------
template <int NB>
struct ShortTiles {
  // Rows of the other side in a round.  Vectors above 160 leave registers for one product of 32 x 32 at a time only (192: 792 us
  // with 34 registers spilled, 712; 8192 rows x 56944 classes).
  static constexpr int kRound = NB > 5 ? 32 : 64;
  static constexpr int kSize = 64 * HeadTile<NB>::kChunks;  // (results leave through both halves: 32 rows of each of four waves)
  u32x4 tiles[2][kSize];
  float shifts[2][64], eaches[2][64];
  int32_t targets[2][64];
};

// dh: one workgroup has 128 rows, a wave 32 of them (lane's row is a column of Z^T = W H^T) in registers, and goes over its
// share of the classes; G^T is the second operand of dH^T = W^T G^T as it leaves the exponentials.
template <class T, int NB>
__device__ __forceinline__ void dhidden_short(const LossParams& p, uint32_t block, int row_tiles, bool alone, ShortTiles<NB>& lds_tiles) {
  constexpr int kRound = ShortTiles<NB>::kRound, kChunks = HeadTile<NB>::kChunks, kSize = ShortTiles<NB>::kSize;
  auto& tiles = lds_tiles.tiles;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), h = lane >> 5;
  const int split = uniform(block / row_tiles), row0 = uniform(block % row_tiles) * 128 + wave * 32, row = row0 + (lane & 31);
  const bool work = row0 < p.padded_rows;  // (wave-uniform: padded_rows is a multiple of 32)
  int begin, end;
  rounds_of((p.classes + kRound - 1) / kRound, split, p.dhidden_split, begin, end);
  const int64_t row_bytes = (int64_t)p.dim * 2;
  const TileLoader<NB, kRound> w(p.weight, row_bytes, 0, 0, p.dim);
  const uint32_t lds = lds_address(&tiles[0][0]) + wave * 1024;
  if (begin < end) w.issue(lds, row_bytes, begin * kRound, p.classes);
  u32x4 hf[2 * NB];
  load_rows<NB>(hf, (const char*)p.hidden_known + row * row_bytes, work, p.dim, h);
  const int target = work ? p.row_target[row] : -1;
  const float exact = work ? p.row_each[row] : 0.f, ratio = row_ratio<T>(exact), each = exact / ratio;
  const float shift = work ? p.row_shift[row] - log2f(ratio) : -INFINITY;
  const uint32_t negative = each < 0.f ? 0x80000000u : 0u;
  const bool negatives = __builtin_amdgcn_ballot_w64(negative) != 0;
  f32x16 acc[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) acc[b] = f32x16{};
  int half = 0;
  for (int i = begin; i < end; ++i, half ^= 1) {
    wait_for_loads_and_others();
    if (i + 1 < end) w.issue(lds + (half ^ 1) * kSize * 16, row_bytes, (i + 1) * kRound, p.classes);
    if (!work) continue;
    const int class0 = i * kRound;
    const u32x4* tile = tiles[half];
    const bool edge = class0 + kRound > p.classes ||
                      __builtin_amdgcn_ballot_w64(target >= class0 && target < class0 + kRound) != 0;
#pragma unroll
    for (int t = 0; t < kRound / 32; ++t) {
      f32x16 g = {};
#pragma unroll
      for (int s = 0; s < 2 * NB; ++s) g = product_32x32x16<T>(read_operand_by_rows<kChunks>(tile, 32 * t, s, lane), hf[s], g);
#pragma unroll
      for (int n = 0; n < 16; ++n) g[n] = exp2_fast(__builtin_fmaf(g[n], kLog2e, shift));
      // (branches inside the round: with a body of its own for rounds without an edge the compiler runs out of registers,
      // 276 us where this takes 232)
      if (negatives) {
#pragma unroll
        for (int n = 0; n < 16; ++n) g[n] = __uint_as_float(__float_as_uint(g[n]) ^ negative);
      }
      if (edge) {
        const int c0 = class0 + 32 * t + 4 * h;
#pragma unroll
        for (int n = 0; n < 16; ++n) {
          const int c = c0 + 8 * (n / 4) + n % 4;
          if (c == target) g[n] -= each;
          if (c >= p.classes) g[n] = 0.f;
        }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const u32x4 gf = pack_operand<T>(g, j);
#pragma unroll
        for (int b = 0; b < NB; ++b)
          acc[b] = product_32x32x16<T>(read_operand_by_columns<kChunks, true>(tile, 32 * t + 16 * j, 32 * b, lane), gf, acc[b]);
      }
    }
  }
  __syncthreads();
  if (row0 >= p.rows) return;
  const float factor = p.scale[1] * ratio;
  if (alone)
    store_rows<T, NB>((T*)p.dhidden + (int64_t)row0 * p.dim, p.dim, p.rows - row0, acc, factor, p.dim,
                      &tiles[0][0] + wave * 32 * kChunks);
  else if (row < p.rows)
    store_sums<NB>(p.dhidden_sums + ((int64_t)split * p.rows + row) * p.dim, acc, factor, p.dim, h);
}

// dw: one workgroup has 128 classes, a wave 32 of them (lane's class is a column of Z = H W^T), and goes over its share of the
// rows, whose shifts are read from LDS.  In rounds in which a target is one of the classes g is multiplied in two parts,
// rounded and rest (see row_ratio: here a row is no lane's own, and the rows of h have their logits to make).
template <class T, int NB>
__device__ __forceinline__ void dweight_short(const LossParams& p, uint32_t block, int class_tiles, ShortTiles<NB>& lds_tiles) {
  constexpr int kRound = ShortTiles<NB>::kRound, kChunks = HeadTile<NB>::kChunks, kSize = ShortTiles<NB>::kSize;
  auto& tiles = lds_tiles.tiles;
  auto& shifts = lds_tiles.shifts;
  auto& eaches = lds_tiles.eaches;
  auto& targets = lds_tiles.targets;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), h = lane >> 5;
  const int split = uniform(block / class_tiles), class0 = uniform(block % class_tiles) * 128 + wave * 32, mine = class0 + (lane & 31);
  int begin, end;
  rounds_of(p.padded_rows / kRound, split, p.dweight_split, begin, end);
  const int64_t row_bytes = (int64_t)p.dim * 2;
  const TileLoader<NB, kRound> rows(p.hidden_known, row_bytes, 0, 0, p.dim);
  const uint32_t lds = lds_address(&tiles[0][0]) + wave * 1024;
  auto issue = [&](int half, int i) {
    rows.issue(lds + half * kSize * 16, row_bytes, i * kRound, p.padded_rows);
#pragma unroll
    for (int j = 0; j < kRound; j += 64) {
      if (wave == 0) load_words_to_lds((const char*)(p.row_shift + i * kRound + j), min(lane, kRound - 1) * 4, lds_address(shifts[half] + j));
      if (wave == 1) load_words_to_lds((const char*)(p.row_target + i * kRound + j), min(lane, kRound - 1) * 4, lds_address(targets[half] + j));
      if (wave == 2) load_words_to_lds((const char*)(p.row_each + i * kRound + j), min(lane, kRound - 1) * 4, lds_address(eaches[half] + j));
    }
  };
  if (begin < end) issue(0, begin);
  const bool work = class0 < p.classes;
  u32x4 wf[2 * NB];
  load_rows<NB>(wf, (const char*)p.weight + mine * row_bytes, mine < p.classes, p.dim, h);
  f32x16 acc[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) acc[b] = f32x16{};
  int half = 0;
  for (int i = begin; i < end; ++i, half ^= 1) {
    wait_for_loads_and_others();
    if (i + 1 < end) issue(half ^ 1, i + 1);
    if (!work) continue;
    const u32x4* tile = tiles[half];
    // a row of the round whose target is a class of the wave, or whose gradient is negative
    bool odd = false;
#pragma unroll
    for (int j = 0; j < kRound; j += 64)
      odd = odd || (targets[half][j + lane] >= class0 && targets[half][j + lane] < class0 + 32) || eaches[half][j + lane] < 0.f;
    const bool edge = __builtin_amdgcn_ballot_w64(odd) != 0;
#pragma unroll
    for (int t = 0; t < kRound / 32; ++t) {
      f32x16 g = {};
#pragma unroll
      for (int s = 0; s < 2 * NB; ++s) g = product_32x32x16<T>(read_operand_by_rows<kChunks>(tile, 32 * t, s, lane), wf[s], g);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x4 shift = *(const f32x4*)&shifts[half][32 * t + 8 * q + 4 * h];
#pragma unroll
        for (int n = 0; n < 4; ++n) g[4 * q + n] = exp2_fast(__builtin_fmaf(g[4 * q + n], kLog2e, shift[n]));
      }
      if (edge) {
#pragma unroll
        for (int n = 0; n < 16; ++n) {
          const int at = 32 * t + 8 * (n / 4) + 4 * h + n % 4;
          const float each = eaches[half][at];
          if (each < 0.f) g[n] = -g[n];
          if (targets[half][at] == mine) g[n] -= each;
        }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const u32x4 gf = pack_operand<T>(g, j);
#pragma unroll
        for (int b = 0; b < NB; ++b)
          acc[b] = product_32x32x16<T>(read_operand_by_columns<kChunks, true>(tile, 32 * t + 16 * j, 32 * b, lane), gf, acc[b]);
        if (edge) {
          u32x4 rest;
#pragma unroll
          for (int n = 0; n < 4; ++n)
            rest[n] = pack_pair<T>(g[8 * j + 2 * n] - unpack_low<T>(gf[n]), g[8 * j + 2 * n + 1] - unpack_high<T>(gf[n]));
#pragma unroll
          for (int b = 0; b < NB; ++b)
            acc[b] = product_32x32x16<T>(read_operand_by_columns<kChunks, true>(tile, 32 * t + 16 * j, 32 * b, lane), rest, acc[b]);
        }
      }
    }
  }
  __syncthreads();
  if (!work) return;
  const float factor = p.scale[1];
  if (p.dweight_split == 1)
    store_rows<T, NB>((T*)p.dweight + (int64_t)class0 * p.dim, p.dim, p.classes - class0, acc, factor, p.dim,
                      &tiles[0][0] + wave * 32 * kChunks);
  else if (mine < p.classes)
    store_sums<NB>(p.dweight_sums + ((int64_t)split * p.classes + mine) * p.dim, acc, factor, p.dim, h);
}

// Both in one launch: the first `dhidden_blocks` workgroups and the rest (neither waits for the other's last ones).  Four
// products of rows x classes x size: 8192 x 56944 x 128: 497 us, 0.96 PFLOP/s, matrix cores busy 53 %.
template <class T, int NB>
__global__ __launch_bounds__(256, 2) void gradients_short_kernel(LossParams p, int dhidden_blocks, int row_tiles, bool alone, int class_tiles) {
  __shared__ ShortTiles<NB> tiles;
  if ((int)blockIdx.x < dhidden_blocks) dhidden_short<T, NB>(p, block_by_die(blockIdx.x, dhidden_blocks), row_tiles, alone, tiles);
  else dweight_short<T, NB>(p, block_by_die(blockIdx.x - dhidden_blocks, gridDim.x - dhidden_blocks), class_tiles, tiles);
}

// ---- backward, longer vectors ------------------------------------------------------------------------------
// What a workgroup of the two products below leaves.  Result rows are columns of the vectors and lie in a lane's
// registers, four next to each other at a time; the result's column is the lane's row of the output.
// A sum of its own among several, in 32 bits:
template <class S>
__device__ __forceinline__ void store_tile_sums(const f32x16 (&acc)[S::kM][S::kN], float factor, float* sums, bool add, int row0, int row_end,
                                           int column0, int columns) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
#pragma unroll
  for (int j = 0; j < S::kN; ++j) {
    const int row = row0 + 32 * (wave % S::kWavesN * S::kN + j) + (lane & 31);
    if (row >= row_end) continue;
#pragma unroll
    for (int i = 0; i < S::kM; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int column = column0 + 32 * (wave / S::kWavesN * S::kM + i) + 8 * g + 4 * h;
        if (column >= columns) continue;
        f32x4* at = (f32x4*)(sums + (int64_t)row * columns + column);
        f32x4 v;
#pragma unroll
        for (int n = 0; n < 4; ++n) v[n] = acc[i][j][4 * g + n] * factor;
        *at = add ? v + *at : v;
      }
  }
}
// The result itself: rounded, turned through the wave's own part of LDS and stored 16 bytes a lane, whole rows of
// 32 * kM columns side by side (stored from the registers as they are, 64 bytes side by side, this took twice as long).
template <class T, class S>
__device__ __forceinline__ void store_result(const f32x16 (&acc)[S::kM][S::kN], float factor, T* out, int row0, int row_end, int column0,
                                             int columns, u32x4* tiles) {
  constexpr int kRowChunks = 4 * S::kM;  // of a row in the wave's part
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
  u32x4* part = tiles + wave * 32 * kRowChunks;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < S::kN; ++j) {
    const int r = lane & 31, first = row0 + 32 * (wave % S::kWavesN * S::kN + j);
#pragma unroll
    for (int i = 0; i < S::kM; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        u32x2 v;
        v[0] = pack_pair<T>(acc[i][j][4 * g] * factor, acc[i][j][4 * g + 1] * factor);
        v[1] = pack_pair<T>(acc[i][j][4 * g + 2] * factor, acc[i][j][4 * g + 3] * factor);
        ((u32x2*)(part + r * kRowChunks + ((4 * i + g) ^ (r & (kRowChunks - 1)))))[h] = v;
      }
    // (one wave's LDS operations are done in order: no barrier between its own writes and reads)
#pragma unroll
    for (int n = 0; n < kRowChunks / 2; ++n) {
      const int at = lane + 64 * n, rr = at / kRowChunks, c = at % kRowChunks;
      const u32x4 v = part[rr * kRowChunks + (c ^ (rr & (kRowChunks - 1)))];
      const int row = first + rr, column = column0 + 32 * (wave / S::kWavesN * S::kM) + 8 * c;
      if (row < row_end && column < columns) *(u32x4*)(out + (int64_t)row * columns + column) = v;
    }
  }
}

// The share `i` of `n` in a sum over `places`, in whole rounds.
__device__ __forceinline__ void share_of(int places, int depth, int i, int n, int& begin, int& end) {
  const int rounds = (places + depth - 1) / depth, each = (rounds + n - 1) / n;
  begin = uniform(min(i * each * depth, places));
  end = uniform(min(begin + each * depth, places));
}

// dh of the piece (4096 rows x 32768 classes x 1024: 237 us, 1.16 PFLOP/s).
template <class T, class S>
__global__ __launch_bounds__(S::kThreads, 2) void dhidden_kernel(LossParams p, int row_tiles, int column_tiles, bool alone) {
  using Columns = ByColumns<S::kTileM, S::kDepth, S::kThreads>;
  using Rows = GradientByRows<S::kTileN, S::kDepth, S::kThreads>;
  __shared__ u32x4 tiles[kTileChunks<Columns, Rows>];
  const uint32_t block = block_by_die();
  const int of = row_tiles * column_tiles, split = uniform(block / of), tile = uniform(block % of);
  const int row0 = uniform(tile / column_tiles) * S::kTileN, column0 = uniform(tile % column_tiles) * S::kTileM;
  const int classes = p.class_end - p.class0;
  int begin, end;
  share_of(classes, S::kDepth, split, p.dhidden_split, begin, end);
  f32x16 acc[S::kM][S::kN];
  multiply<T, S, true>(acc, Columns((const char*)p.weight + (int64_t)p.class0 * p.dim * 2, (int64_t)p.dim * 2, column0, p.dim, classes),
                       Rows(p.gradient, p.g_rows, row0), begin, end, tiles);
  // the lane's rows are columns of the result
  const int wave = threadIdx.x >> 6, mine = row0 + 32 * (wave % S::kWavesN * S::kN) + (threadIdx.x & 31);
#pragma unroll
  for (int j = 0; j < S::kN; ++j) {
    const float ratio = p.g_rows > p.padded_rows && mine + 32 * j < p.rows ? row_ratio<T>(p.row_each[mine + 32 * j]) : 1.f;
#pragma unroll
    for (int i = 0; i < S::kM; ++i)
#pragma unroll
      for (int n = 0; n < 16; ++n) acc[i][j][n] *= ratio;
  }
  const float factor = p.scale[1];
  if (alone) store_result<T, S>(acc, factor, (T*)p.dhidden, row0, p.rows, column0, p.dim, tiles);
  else store_tile_sums<S>(acc, factor, p.dhidden_sums + (int64_t)split * p.rows * p.dim, p.class0 > 0, row0, p.rows, column0, p.dim);
}

// dw of the piece's classes (the same sizes: 245 us, 1.12 PFLOP/s).
template <class T, class S>
__global__ __launch_bounds__(S::kThreads, 2) void dweight_kernel(LossParams p, int class_tiles, int column_tiles) {
  using Columns = ByColumns<S::kTileM, S::kDepth, S::kThreads>;
  using Classes = GradientByColumns<S::kTileN, S::kDepth, S::kThreads>;
  __shared__ u32x4 tiles[kTileChunks<Columns, Classes>];
  const uint32_t block = block_by_die();
  const int of = class_tiles * column_tiles, split = uniform(block / of), tile = uniform(block % of);
  const int class0 = uniform(tile / column_tiles) * S::kTileN, column0 = uniform(tile % column_tiles) * S::kTileM;
  const int classes = p.class_end - p.class0;
  int begin, end;
  share_of(p.g_rows, S::kDepth, split, p.dweight_split, begin, end);
  f32x16 acc[S::kM][S::kN];
  multiply<T, S, false>(acc, Columns(p.hidden_known, (int64_t)p.dim * 2, column0, p.dim, p.g_rows),
                        Classes(p.gradient, p.g_rows, class0), begin, end, tiles);
  const float factor = p.scale[1];
  if (p.dweight_split == 1)
    store_result<T, S>(acc, factor, (T*)p.dweight + (int64_t)p.class0 * p.dim, class0, classes, column0, p.dim, tiles);
  else store_tile_sums<S>(acc, factor, p.dweight_sums + (int64_t)split * classes * p.dim, false, class0, classes, column0, p.dim);
}

// out = the sum of `split` arrays of n values, n a multiple of 8, four values a lane.  SHARES lanes share out the arrays: one
// where there are few (18726 x 256 values, 3 arrays: 27 us with sixteen lanes, most of them idle), sixteen where there are
// many and the result is small.
template <class T, int SHARES>
__global__ __launch_bounds__(256) void add_sums_kernel(const float* sums, T* out, int64_t n, int split) {
  constexpr int kLanes = 256 / SHARES;
  __shared__ f32x4 partial[SHARES][kLanes + 1];
  const int at = threadIdx.x % kLanes, share = threadIdx.x / kLanes;
  const int64_t i = ((int64_t)blockIdx.x * kLanes + at) * 4;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  if (i < n) {
    const float* from = sums + i;
    int s = share;
    for (; s + 3 * SHARES < split; s += 4 * SHARES) {
      f32x4 four[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) four[j] = *(const f32x4*)(from + (s + j * SHARES) * n);
#pragma unroll
      for (int j = 0; j < 4; ++j) v += four[j];
    }
    for (; s < split; s += SHARES) v += *(const f32x4*)(from + s * n);
  }
  if constexpr (SHARES > 1) {
    partial[share][at] = v;
    __syncthreads();
    if (share != 0) return;
    for (int s = 1; s < min(split, SHARES); ++s) v += partial[s][at];
  }
  if (i >= n) return;
  u32x2 o;
  o[0] = pack_pair<T>(v[0], v[1]);
  o[1] = pack_pair<T>(v[2], v[3]);
  *(u32x2*)(out + i) = o;
}

// ---- host -----------------------------------------------------------------------------------------

int64_t round_up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

constexpr int kFewRows = 128;  // up to here tiles of 64 rows of the loss, beyond it tiles of 256
constexpr int64_t kWorkgroups = 256;  // what fills the GPU, one to a compute unit
// More rows, but tiles of 256 x 256 for less than half of the compute units: smaller ones throughout (both directions in us: 24
// tiles, 268 rows x 2864 x 784, 118 -> 75; 114 tiles, 266 x 14352 x 696, 122 -> 109; 192 tiles, 2000 x 6000 x 1024, 185 -> 213, so not
// there).
bool few_tiles(int64_t rows, int64_t classes) { return rows > kFewRows && ((rows + 255) / 256) * ((classes + 255) / 256) <= kWorkgroups / 2; }
// Vectors whose g stays in registers, and whose rows do in the forward pass.  8192 rows x 56944 classes, dh and dw in us so and
// over a g in memory (933 MB): 495 and 757 at 128, 600 and 835 at 160, 712 and 864 at 192, 801 and 968 at 224; at 256 the sums
// leave too few registers (1576 and 935).  Forward, and by tiles: 185 and 264 at 136, 235 and 324 at 256.
constexpr int64_t kShortVector = 224, kShortForward = 256;
constexpr int64_t kPieceBytes = (int64_t)256 << 20;  // of what is kept for one piece of the work
constexpr int64_t kMostElements = ((int64_t)1 << 34) - 1024;  // of a matrix: one launch has fewer than 2^32 threads, of four each
constexpr int64_t kMostWorkgroups = 0xffffff;                 // of 256 threads, for the same reason

// How the work is cut; the workspace's parts as offsets.
struct LossPlan {
  int64_t forward_rows, padded_rows, g_rows, piece, column_tiles, logits_split, dhidden_split, dweight_split;
  bool alone;  // the only sum of dh
  int64_t partials, gradient, dhidden_sums, dweight_sums, scale, row_each, row_shift, row_target, hidden_known, bytes;
};

LossPlan plan_of(int64_t rows, int64_t classes, int64_t dim, bool backward) {
  LossPlan w = {};
  auto take = [&](int64_t bytes) {
    const int64_t at = w.bytes;
    w.bytes += round_up(bytes, 256);
    return at;
  };
  auto split = [](int64_t workgroups, int64_t tiles, int64_t rounds, int64_t least) {  // at least so many rounds to a share
    return std::max<int64_t>(1, std::min(workgroups / std::max<int64_t>(tiles, 1), rounds / least));
  };
  const bool is_short = dim <= (backward ? kShortVector : kShortForward);
  if (!backward) {
    w.logits_split = is_short ? split(4 * kWorkgroups, (rows + 255) / 256, (classes + kRound - 1) / kRound, 1) : 1;
    // Longer vectors leave a pair for each row and 64 classes, a sixteenth of the logits: rows are taken as many at a time as
    // have 256 MiB of them, at least a tile.
    const int64_t row_bytes = (is_short ? w.logits_split : round_up(classes, kClassPad) / 64) * (int64_t)sizeof(float2);
    w.forward_rows = is_short ? rows : std::min(rows, std::max<int64_t>(kPieceBytes / row_bytes / 256, 1) * 256);
    w.partials = take(w.forward_rows * row_bytes);
    return w;
  }
  const bool small = few_tiles(rows, classes);
  const int64_t tile_rows = rows <= kFewRows || small ? 64 : 256;
  w.padded_rows = round_up(std::max<int64_t>(rows, 1), is_short ? kRound : tile_rows);
  w.g_rows = !is_short && rows <= kFewRows ? 2 * w.padded_rows : w.padded_rows;
  if (is_short) {
    w.dhidden_split = split(2 * kWorkgroups, (w.padded_rows + 127) / 128, (classes + kRound - 1) / kRound, 1);
    w.dweight_split = split(2 * kWorkgroups, (classes + 127) / 128, w.padded_rows / kRound, 4);
    w.alone = w.dhidden_split == 1;
    w.piece = classes;
  } else {
    w.column_tiles = (dim + 255) / 256;
    // g of a piece: 256 MiB (4096 rows x 131072 classes x 1024: 4.23 ms with pieces of 128 to 512 MiB, 4.14 with one of 1024,
    // 5.1 of 64), up to four times that where it would leave compute units without a tile of dw.  Each piece reads and writes the
    // sums of dh, 8 bytes for 6 operations a class: 300 / classes of its time.  So no fewer classes than eight times the vectors,
    // or than 4 GiB hold; and no fewer than 1024, which are more than that for over two million rows (131072 rows x 40000 x 4096: 118 ms
    // with 4 GiB, 121 with 8; 2097152 x 10000 x 264: 81 ms with 4, 74 with 9; 4194240 rows of it: 163 with 8, 150 with 18)
    const int64_t fit = kPieceBytes / (2 * w.g_rows), fill = std::min(kWorkgroups / w.column_tiles * kClassPad, 4 * fit);
    const int64_t sums = std::min(8 * dim, std::max<int64_t>(16 * fit, 1024));
    w.piece = std::min(round_up(classes, kClassPad), round_up(std::max({fit, fill, sums}), kClassPad));
    w.dhidden_split = split(kWorkgroups, w.padded_rows / tile_rows * w.column_tiles, w.piece / 64, 4);
    w.dweight_split = split(kWorkgroups, w.piece / (small ? 64 : kClassPad) * w.column_tiles, w.g_rows / 64, 4);
    w.alone = w.dhidden_split == 1 && w.piece >= classes;
    w.gradient = take(w.g_rows * w.piece * 2);
  }
  w.scale = take(2 * sizeof(float));
  w.row_each = take(w.padded_rows * 4);
  w.row_shift = take(w.padded_rows * 4);
  w.row_target = take(w.padded_rows * 4);
  w.hidden_known = take(w.g_rows * dim * 2);
  if (!w.alone) w.dhidden_sums = take(w.dhidden_split * rows * dim * (int64_t)sizeof(float));
  if (w.dweight_split > 1) w.dweight_sums = take(w.dweight_split * std::min(w.piece, classes) * dim * (int64_t)sizeof(float));
  return w;
}

template <class T, class S, bool BACKWARD>
int launch_logits(const LossParams& p, int64_t covered_rows, int64_t covered_classes, hipStream_t stream) {
  const int64_t row_tiles = (covered_rows + S::kTileN - 1) / S::kTileN, class_tiles = (covered_classes + S::kTileM - 1) / S::kTileM;
  logits_kernel<T, S, BACKWARD><<<(uint32_t)(row_tiles * class_tiles), S::kThreads, 0, stream>>>(p, (int)row_tiles);
  return (int)class_tiles * S::kWavesM;
}
// Shapes (classes x rows): few rows leave the products bound by the reading of the class vectors; few tiles, by the rounds of a
// lone workgroup, of which these have a quarter of the work and half as many (268 rows x 2864 x 784: 41 -> 27 us forward, 74 -> 48 backward).
template <class T, bool BACKWARD>
int launch_logits(const LossParams& p, int64_t covered_rows, int64_t covered_classes, hipStream_t stream) {
  if (few_tiles(p.rows, p.classes)) return launch_logits<T, Shape<2, 2, 2, 1, 128>, BACKWARD>(p, covered_rows, covered_classes, stream);
  if (p.rows <= kFewRows) return launch_logits<T, Shape<4, 1, 2, 2, 64>, BACKWARD>(p, covered_rows, covered_classes, stream);
  return launch_logits<T, Shape<2, 4, 4, 2, 64>, BACKWARD>(p, covered_rows, covered_classes, stream);
}

template <class T, int NB>
int launch_logits_short(const LossParams& p, int splits, hipStream_t stream) {
  const int row_tiles = (p.rows + 255) / 256;
  logits_short_kernel<T, NB><<<(uint32_t)(row_tiles * splits), 256, 0, stream>>>(p, row_tiles, splits);
  return splits;
}

template <class T>
void launch_forward(const LossParams& p, const LossPlan& w, hipStream_t stream) {
  int parts;
  if (p.dim > kShortForward) {
    const int64_t rows = p.rows;
    for (int64_t at = 0; at < rows; at += w.forward_rows) {
      LossParams q = p;
      q.rows = (int32_t)std::min(w.forward_rows, rows - at);
      q.hidden = (const char*)p.hidden + at * p.dim * 2;
      q.target += at;
      q.loss += at;
      q.lse += at;
      parts = launch_logits<T, false>(q, q.rows, q.classes, stream);
      join_kernel<T><<<(q.rows + 7) / 8, 1024, 0, stream>>>(q, parts);
    }
    return;
  }
  if (p.dim > 224) parts = launch_logits_short<T, 8>(p, (int)w.logits_split, stream);
  else if (p.dim > 192) parts = launch_logits_short<T, 7>(p, (int)w.logits_split, stream);
  else if (p.dim > 160) parts = launch_logits_short<T, 6>(p, (int)w.logits_split, stream);
  else if (p.dim > 128) parts = launch_logits_short<T, 5>(p, (int)w.logits_split, stream);
  else if (p.dim > 96) parts = launch_logits_short<T, 4>(p, (int)w.logits_split, stream);
  else if (p.dim > 64) parts = launch_logits_short<T, 3>(p, (int)w.logits_split, stream);
  else if (p.dim > 32) parts = launch_logits_short<T, 2>(p, (int)w.logits_split, stream);
  else parts = launch_logits_short<T, 1>(p, (int)w.logits_split, stream);
  join_kernel<T><<<(p.rows + 7) / 8, 1024, 0, stream>>>(p, parts);
}

template <class T, class S>
void launch_dhidden(const LossParams& p, const LossPlan& w, hipStream_t stream) {
  const int row_tiles = p.padded_rows / S::kTileN;
  dhidden_kernel<T, S><<<(uint32_t)(row_tiles * w.column_tiles * w.dhidden_split), S::kThreads, 0, stream>>>(p, row_tiles, (int)w.column_tiles, w.alone);
}
template <class T, class S>
void launch_dweight(const LossParams& p, const LossPlan& w, hipStream_t stream) {
  const int class_tiles = (p.class_end - p.class0 + S::kTileN - 1) / S::kTileN;
  dweight_kernel<T, S><<<(uint32_t)(class_tiles * w.column_tiles * w.dweight_split), S::kThreads, 0, stream>>>(p, class_tiles, (int)w.column_tiles);
}

template <class T>
void launch_add_sums(const float* sums, void* out, int64_t n, int64_t split, hipStream_t stream) {
  if (split <= 16) add_sums_kernel<T, 1><<<(uint32_t)((n / 4 + 255) / 256), 256, 0, stream>>>(sums, (T*)out, n, (int)split);
  else add_sums_kernel<T, 16><<<(uint32_t)((n / 4 + 15) / 16), 256, 0, stream>>>(sums, (T*)out, n, (int)split);
}

template <class T, int NB>
void launch_short(const LossParams& p, const LossPlan& w, hipStream_t stream) {
  const int row_tiles = (p.padded_rows + 127) / 128, class_tiles = (p.classes + 127) / 128;
  const int64_t dhidden_blocks = row_tiles * w.dhidden_split, dweight_blocks = class_tiles * w.dweight_split;
  auto launch = [&](int64_t blocks, int64_t of_dhidden) {
    gradients_short_kernel<T, NB><<<(uint32_t)blocks, 256, 0, stream>>>(p, (int)of_dhidden, row_tiles, w.alone, class_tiles);
  };
  if (dhidden_blocks + dweight_blocks <= kMostWorkgroups) {
    launch(dhidden_blocks + dweight_blocks, dhidden_blocks);
  } else {  // (over two billion classes)
    launch(dhidden_blocks, dhidden_blocks);
    launch(dweight_blocks, 0);
  }
}

template <class T>
void launch_backward(LossParams p, const LossPlan& w, hipStream_t stream) {
  if (p.rows == 0) {  // no sum at all
    const int64_t n = (int64_t)p.classes * p.dim;
    launch_add_sums<T>(nullptr, p.dweight, n, 0, stream);
    return;
  }
  const uint32_t prepare_blocks = (uint32_t)((w.padded_rows * (p.dim / 8) + 255) / 256);
  if (std::is_same<T, _Float16>::value) {
    largest_kernel<<<1, 1024, 0, stream>>>(p);
    prepare_kernel<T, true><<<prepare_blocks, 256, 0, stream>>>(p);
  } else {
    prepare_kernel<T, false><<<prepare_blocks, 256, 0, stream>>>(p);
  }
  auto add_dweight = [&](int64_t class0, int64_t classes) {
    const int64_t n = classes * p.dim;
    if (w.dweight_split > 1)
      launch_add_sums<T>(p.dweight_sums, (T*)p.dweight + class0 * p.dim, n, p.dweight_split, stream);
  };
  if (p.dim <= kShortVector) {
    switch ((p.dim + 31) / 32) {
      case 1: launch_short<T, 1>(p, w, stream); break;
      case 2: launch_short<T, 2>(p, w, stream); break;
      case 3: launch_short<T, 3>(p, w, stream); break;
      case 4: launch_short<T, 4>(p, w, stream); break;
      case 5: launch_short<T, 5>(p, w, stream); break;
      case 6: launch_short<T, 6>(p, w, stream); break;
      default: launch_short<T, 7>(p, w, stream); break;
    }
    add_dweight(0, p.classes);
  } else
  for (int64_t at = 0; at < p.classes; at += w.piece) {
    p.class0 = (int32_t)at;
    p.class_end = (int32_t)std::min<int64_t>(at + w.piece, p.classes);
    const int64_t classes = p.class_end - p.class0;
    launch_logits<T, true>(p, p.padded_rows, round_up(classes, kClassPad), stream);
    const bool small = few_tiles(p.rows, p.classes), few = p.rows <= kFewRows || small;
    // shapes of the two products: columns of the vectors x rows of the output
    if (few) launch_dhidden<T, Shape<4, 2, 2, 1, 64>>(p, w, stream);
    else launch_dhidden<T, Shape<2, 4, 4, 2, 64>>(p, w, stream);
    if (small) launch_dweight<T, Shape<4, 2, 2, 1, 64>>(p, w, stream);
    else launch_dweight<T, Shape<2, 4, 4, 2, 64>>(p, w, stream);
    add_dweight(at, classes);
  }
  if (!w.alone) {
    const int64_t n = (int64_t)p.rows * p.dim;
    launch_add_sums<T>(p.dhidden_sums, p.dhidden, n, p.dhidden_split, stream);
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
  if (a->rows * a->dim > kMostElements || a->classes * a->dim > kMostElements)
    return fail("vocabulary loss: at most " + std::to_string(kMostElements) + " elements to a matrix");
  if (a->rows == 0 && !backward) return 0;
  const LossPlan w = plan_of(a->rows, a->classes, a->dim, backward);
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
  p.dhidden_sums = (float*)(work + w.dhidden_sums);
  p.dweight_sums = (float*)(work + w.dweight_sums);
  p.scale = (float*)(work + w.scale);
  p.row_each = (float*)(work + w.row_each);
  p.row_shift = (float*)(work + w.row_shift);
  p.row_target = (int32_t*)(work + w.row_target);
  p.hidden_known = work + w.hidden_known;
  p.g_rows = (int32_t)w.g_rows;
  p.padded_rows = (int32_t)w.padded_rows;
  p.dhidden_split = (int32_t)w.dhidden_split;
  p.dweight_split = (int32_t)w.dweight_split;
  p.class_end = p.classes;
  if (backward) {
    if (a->dtype == ND_BF16) launch_backward<__bf16>(p, w, (hipStream_t)stream);
    else launch_backward<_Float16>(p, w, (hipStream_t)stream);
  } else {
    if (a->dtype == ND_BF16) launch_forward<__bf16>(p, w, (hipStream_t)stream);
    else launch_forward<_Float16>(p, w, (hipStream_t)stream);
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
  return nd::plan_of(rows, classes, dim, backward != 0).bytes;
}

int nd_vocabulary_loss_forward(const nd_vocabulary_loss* a, void* stream) {
  return nd::guarded([&]() -> int { return nd::run_loss(a, false, stream); });
}

int nd_vocabulary_loss_backward(const nd_vocabulary_loss* a, void* stream) {
  return nd::guarded([&]() -> int { return nd::run_loss(a, true, stream); });
}

}  // extern "C"

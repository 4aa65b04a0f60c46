// Causal attention over packed sequences with grouped heads (C entries: nd_packed_*).
//
// Token i of sequence [first_i, last_i) attends to the keys first_i .. i:
//   s_ij = scale q_i . k_j,  lse_i = log sum_j exp s_ij,  p_ij = exp(s_ij - lse_i),  o_i = sum_j p_ij v_j
//   delta_i = do_i . o_i,    ds_ij = p_ij (do_i . v_j - delta_i)
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum ds_ij q_i,  dv_j = sum p_ij do_i  (over i and the group's heads)
// A token of no sequence (the rest of a buffer that is longer than its sequences) has o = 0, lse = -inf, no gradient.
//
// Tiles are cut from the packed tokens, not from the sequences: a row's mask is the interval [first_i, i], so a tile
// may hold many short sequences and part of a long one, and no tile is padded for a short one.
#include "../../include/nextdoor_amd.h"

#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>
#include <vector>

#include "nd_errors.hpp"
#include "nd_matrix.hpp"
#include "nd_row_tiles.hpp"

namespace nd {
namespace {

constexpr int kPlanThreads = 256;
constexpr int kOrderThreads = 1024;
constexpr int kRows = 128;    // rows of a workgroup: four waves of 32
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// A row's sums are kept relative to a maximum that is taken anew only when it has grown by this much (in powers of two):
// weights stay below 2^8, which costs 32-bit sums and 16-bit floats nothing, and the sums are rarely scaled again.
constexpr float kTopSlack = 8.f;
constexpr int kExactDeltaRounds = 4;
constexpr int kTopParts = 256;  // workgroups that look for the largest output gradient and value

struct PackedPlan {
  const int32_t* first;  // of the sequence a token belongs to; tokens from `covered` on belong to none
  const int32_t* last;   // one past it
  const int32_t* query_order;  // tiles of kRows tokens, those with most keys first
  const int32_t* key_order;    // those with most queries first
  // No sequence is longer than a tile: tile i is the whole sequences in tokens short_starts[i] .. short_starts[i + 1] - 1
  // (short_tiles of them; 0: there are longer sequences).
  const int32_t* short_starts;
  int32_t tokens, covered, tiles, short_tiles;
};

struct AttentionParams {
  PackedPlan plan;
  const void *q, *k, *v, *out, *dout;
  void *out_w, *dq, *dk, *dv;
  float *lse, *lse2, *delta;  // [heads][tokens]; the backward kernels': lse in powers of two less what p is held times, delta times k (whole sequences to a tile: as it is)
  // what the chunks of a tile whose work is cut leave: [chunk][token][head][dim] of out or dq, [chunk][head][token] of
  // maxima and sums, [chunk][token][kv_head][dim] of dk and dv
  float *row_sums, *dk_sums, *dv_sums;
  float2* row_tops;
  uint32_t* gradient_tops;  // 16-bit floats, backward: [kTopParts], see attention_top_kernel
  int64_t q_token, q_head, k_token, k_head, v_token, v_head, dout_token, dout_head;  // in bytes
  int32_t heads, kv_heads, group, dim;
  int32_t chunk, max_chunks;          // rounds that a workgroup of the query kernels takes, chunks of a tile at most
  int32_t key_chunk, max_key_chunks;  // of the key kernel
  int32_t head_split;                 // shares of a group's heads in the key kernel
  float scale, scale_log2;  // scale_log2 > 0
  uint32_t flip;          // sign bits of a pair: q is taken negative for a negative scale
};

// Where each token's sequence begins and ends: a binary search a token, bound by its latency (5 us for 1024 sequences).
__global__ __launch_bounds__(kPlanThreads) void packed_plan_kernel(const int32_t* starts, int32_t sequences,
                                                                   int32_t tokens, int32_t* first, int32_t* last) {
  const int64_t t = (int64_t)blockIdx.x * kPlanThreads + threadIdx.x;
  if (t >= tokens) return;
  // the last sequence that starts at or before t (empty ones start where the next does)
  int32_t lo = 0, hi = sequences;
  while (hi - lo > 1) {
    const int32_t mid = lo + (hi - lo) / 2;  // (there may be more than 2^30 of them, most of them empty)
    if (starts[mid] <= t) lo = mid;
    else hi = mid;
  }
  const bool in = sequences > 0 && t < starts[sequences];
  // (the bounds are those of a checked array; whatever a caller has on the device, no token outside is ever read)
  first[t] = in ? min(max(starts[lo], 0), (int32_t)t) : (int32_t)t;
  last[t] = in ? max(min(starts[lo + 1], tokens), (int32_t)t + 1) : (int32_t)t;
}

// Tiles by falling work, so that the last workgroups to start are short ones: a counting sort.  Workgroup 0: the keys a tile of
// queries reads; workgroup 1: the queries a tile of keys is read by.  (The order of equal ones is left open: it decides when
// a tile runs and nothing else.)  One launch a batch, 3.5 us for 23 sequences of up to 1999.
__global__ __launch_bounds__(kOrderThreads) void packed_order_kernel(const int32_t* first, const int32_t* last, int32_t tokens,
                                                                     int32_t covered, int32_t tiles, int32_t* query_order,
                                                                     int32_t* key_order) {
  __shared__ int32_t count[kOrderThreads];
  const bool keys = blockIdx.x == 1;
  int shift = 0;
  while ((tokens / kColumns >> shift) >= kOrderThreads - 2) ++shift;
  auto bucket = [&](int64_t tile) {
    const int64_t t0 = tile * kRows;
    if (t0 >= covered) return kOrderThreads - 1;
    const int32_t t1 = (int32_t)min(t0 + kRows, (int64_t)covered);
    const int32_t work = keys ? last[t1 - 1] - (int32_t)t0 : t1 - first[t0];
    return kOrderThreads - 2 - min(work / kColumns >> shift, kOrderThreads - 2);
  };
  count[threadIdx.x] = 0;
  __syncthreads();
  for (int64_t i = threadIdx.x; i < tiles; i += kOrderThreads) atomicAdd(&count[bucket(i)], 1);
  __syncthreads();
  for (int d = 1; d < kOrderThreads; d *= 2) {
    const int v = threadIdx.x >= d ? count[threadIdx.x - d] : 0;
    __syncthreads();
    count[threadIdx.x] += v;
    __syncthreads();
  }
  // count: one past the last place of a bucket
  for (int64_t i = threadIdx.x; i < tiles; i += kOrderThreads)
    (keys ? key_order : query_order)[atomicSub(&count[bucket(i)], 1) - 1] = (int32_t)i;
}

// A tile's rounds are cut into chunks of about `chunk` where that shortens what the GPU would wait for at the end: a long
// row among short ones, or few rows.  Chunks leave sums in 32 bits that another kernel joins.
__host__ __device__ __forceinline__ int64_t chunks_of(int64_t rounds, int64_t chunk, int64_t most) {
  const int64_t n = rounds <= 2 * chunk ? 1 : (rounds + chunk - 1) / chunk;
  return n < most ? n : most;
}

// What a workgroup has: heads side by side (their tiles share keys), and, where they fill the eight dies evenly, a die's
// heads next to each other; then the tiles by falling work; then the chunks, the first ones last.  A chunk that a tile does
// not have ends at once, but workgroups go to the parts of a die in turn: the empty ones stay together, or half of the GPU
// would get nothing else (chunks next to each other: 264 us where this takes 177).
__device__ __forceinline__ void chunk_tile_and_head(int max_chunks, int heads, int& chunk, int& rank, int& head) {
  const uint32_t each = gridDim.x / max_chunks, block = blockIdx.x % each;
  chunk = max_chunks - 1 - uniform(blockIdx.x / each);
  rank = uniform(block / heads);
  head = uniform(block % heads);
  if (heads % 8 == 0) head = (head % 8) * (heads / 8) + head / 8;
}

// ---- values that are not finite ---------------------------------------------------------------------
// A key that a row does not see has weight 0 in the matrix products, and 0 x NaN is NaN: an infinity or NaN of one sequence, or
// of a later token, would reach every row whose tile holds it.  A wave whose sums have turned out not finite (one instruction
// for each at its end) takes them again here, pair by pair, leaving out the pairs that the mask leaves out; what a row
// does see comes out as it should, finite or not.  Lane: a row and half of its columns, 16 s + 8 h .. + 7; 32-bit arithmetic on
// the vector units, so that a wave takes some 0.5 us for each key.
template <int NB>
__device__ __forceinline__ bool all_finite(const f32x16 (&acc)[NB]) {
  float zero = 0.f;
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int i = 0; i < 16; ++i) zero = __builtin_fmaf(acc[b][i], 0.f, zero);
  return zero == 0.f;
}
// Rows are read again for every pair: few registers, and none that the sums above would have to leave.
template <class T>
__device__ __forceinline__ float dot_rows(const char* a, const char* b, int dim, int h) {
  float sum = 0.f;
#pragma unroll 1
  for (int c = 16 * h; c < 2 * dim; c += 32) {
    const u32x4 x = *(const u32x4*)(a + c), y = *(const u32x4*)(b + c);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      sum = __builtin_fmaf(unpack_low<T>(x[j]), unpack_low<T>(y[j]), sum);
      sum = __builtin_fmaf(unpack_high<T>(x[j]), unpack_high<T>(y[j]), sum);
    }
  }
  return pair_sum(sum);
}
template <int NB>
struct HalfRow {
  float v[16 * NB];
};
// acc = acc shrink + weight row
template <class T, int NB>
__device__ __forceinline__ void add_row(HalfRow<NB>& acc, float shrink, float weight, const char* row, int dim, int h) {
#pragma unroll
  for (int s = 0; s < 2 * NB; ++s) {
    if (16 * s + 8 * h >= dim) continue;
    const u32x4 v = *(const u32x4*)(row + 32 * s + 16 * h);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      acc.v[8 * s + 2 * j] = __builtin_fmaf(weight, unpack_low<T>(v[j]), acc.v[8 * s + 2 * j] * shrink);
      acc.v[8 * s + 2 * j + 1] = __builtin_fmaf(weight, unpack_high<T>(v[j]), acc.v[8 * s + 2 * j + 1] * shrink);
    }
  }
}
// A lane's half of a result row: `row` as the final values, or, if it is null, `sums` in 32 bits.
template <class T, int NB>
__device__ __forceinline__ void store_half(T* row, float* sums, const HalfRow<NB>& acc, float factor, int dim, int h) {
#pragma unroll
  for (int s = 0; s < 2 * NB; ++s) {
    const int column = 16 * s + 8 * h;
    if (column >= dim) continue;
    if (row) {
      u32x4 v;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = pack_pair<T>(acc.v[8 * s + 2 * j] * factor, acc.v[8 * s + 2 * j + 1] * factor);
      *(u32x4*)(row + column) = v;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) sums[column + j] = acc.v[8 * s + j] * factor;
    }
  }
}

// (there: first <= row.  The rows of lanes that are not there are read all the same: a row that is.)
template <class T, int NB>
__device__ __forceinline__ void forward_carefully(const AttentionParams& p, int head, int kv_head, int row, int first, int begin, int stop,
                                                  int row_end, int chunk, int chunks) {
  const int h = (threadIdx.x & 63) >> 5;
  const bool there = first <= row;
  const float scale = p.flip ? -p.scale_log2 : p.scale_log2;
  const char* q = (const char*)p.q + (int64_t)(there ? row : begin) * p.q_token + (int64_t)head * p.q_head;
  HalfRow<NB> acc = {};
  float top = -INFINITY, sum = 0.f;
#pragma unroll 1
  for (int key = begin; key < stop; ++key) {
    const bool sees = there && key >= first && key <= row;
    if (__builtin_amdgcn_ballot_w64(sees) == 0) continue;
    const float s = dot_rows<T>(q, (const char*)p.k + (int64_t)key * p.k_token + (int64_t)kv_head * p.k_head, p.dim, h) * scale;
    if (!sees) continue;
    const float higher = fmaxf(top, s), base = higher == -INFINITY ? 0.f : higher;
    const float shrink = exp2_fast(top - base), weight = exp2_fast(s - base);
    top = higher;
    sum = sum * shrink + weight;
    add_row<T, NB>(acc, shrink, weight, (const char*)p.v + (int64_t)key * p.v_token + (int64_t)kv_head * p.v_head, p.dim, h);
  }
  if (row >= row_end) return;
  const int64_t at = (int64_t)head * p.plan.tokens + row;
  if (chunks > 1) {
    if (h == 0) p.row_tops[(int64_t)chunk * p.heads * p.plan.tokens + at] = make_float2(top, sum);
    store_half<T, NB>(nullptr, p.row_sums + (((int64_t)chunk * p.plan.tokens + row) * p.heads + head) * p.dim, acc, 1.f, p.dim, h);
    return;
  }
  if (h == 0) p.lse[at] = (top + log2f(sum)) * kLn2;
  store_half<T, NB>((T*)p.out_w + ((int64_t)row * p.heads + head) * p.dim, nullptr, acc, there ? 1.f / sum : 0.f, p.dim, h);
}

// ---- what 16-bit floats hold ------------------------------------------------------------------------------
// The backward pass rounds p and ds to 16 bits as operands.  The smallest 16-bit floats are steps of 2^-24, and p of a row of
// thousands of keys and the ds of a mean's gradient are near that or below, while dq and dk are not (8000 keys, output gradients of 1e-3:
// dq and dk off by 0.003 without this and by 0.00046 with it, of which 0.0004 are the result's own rounding); above 65504 they would
// be infinite.  So the kernels hold 2^15 p, and k 2^15 ds with a power of two k, at least 1 / (4 B) and below 1 / (2 B), B = dim
// max |do| max |v| >= |dp|: |k 2^15 ds| <= 2^15.  2^15 goes into the exponent that makes p, k into the subtraction of delta, which is
// kept times k: not one instruction more.  The maxima are those of the batch, from a launch before, or, where a workgroup has whole
// sequences in LDS, its own.  bfloat16 has the exponents of 32 bits: both are 1.
template <class T>
struct Held {
  static constexpr float kShift = 0.f, kWeight = 1.f;
};
template <>
struct Held<_Float16> {
  static constexpr float kShift = 15.f, kWeight = 32768.f;
};
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t max_of_halves(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
__device__ __forceinline__ uint32_t top_of(u32x4 v) {
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t low = v[j] & 0x7fff, high = v[j] >> 16 & 0x7fff;
    top = max(top, max(low < 0x7c00 ? low : 0, high < 0x7c00 ? high : 0));
  }
  return top;
}
template <int CONTROL>
__device__ __forceinline__ uint32_t turned(uint32_t v) { return __builtin_amdgcn_update_dpp(0, v, CONTROL, 0xf, 0xf, true); }
__device__ __forceinline__ uint32_t top_of_wave(uint32_t top) {
  // sixteen lanes by turning them by 1, 2, 4 and 8, then the four sixteens
  top = max_of_halves(top, turned<0x121>(top));
  top = max_of_halves(top, turned<0x122>(top));
  top = max_of_halves(top, turned<0x124>(top));
  top = max_of_halves(top, turned<0x128>(top));
  const auto rows = __builtin_amdgcn_permlane16_swap(top, top, false, false);
  top = max_of_halves(rows[0], rows[1]);
  const auto halves = __builtin_amdgcn_permlane32_swap(top, top, false, false);
  return max_of_halves(halves[0], halves[1]);
}
// The largest |x| of a part of the tokens, as 16-bit floats: low half of dout, high half of v.  What is not finite does not count: its rows are
// taken carefully.  A launch and its latency where there is little to read (8.3 thousand tokens, 6 heads of 80 and 3: 12 MB in 4.6 us).
__device__ __forceinline__ uint32_t top_of(const char* x, int64_t token_bytes, int64_t head_bytes, uint32_t heads, uint32_t chunks, int64_t begin,
                                           int64_t end) {
  const uint32_t n = (uint32_t)(end - begin) * heads * chunks;  // (a launch holds 2^31 rows of up to 16 chunks at most, a part a 256th)
  uint32_t top = 0;
#pragma unroll 4
  for (uint32_t i = threadIdx.x; i < n; i += 1024) {
    const uint32_t c = i % chunks, row = i / chunks;
    top = max(top, top_of(*(const u32x4*)(x + (begin + row / heads) * token_bytes + row % heads * head_bytes + c * 16)));
  }
  return top;
}
__global__ __launch_bounds__(1024) void attention_top_kernel(AttentionParams p) {
  __shared__ uint32_t tops[16];
  const int64_t begin = (int64_t)p.plan.covered * blockIdx.x / kTopParts, end = (int64_t)p.plan.covered * (blockIdx.x + 1) / kTopParts;
  uint32_t top = top_of((const char*)p.dout, p.dout_token, p.dout_head, p.heads, p.dim / 8, begin, end) |
                 top_of((const char*)p.v, p.v_token, p.v_head, p.kv_heads, p.dim / 8, begin, end) << 16;
  top = top_of_wave(top);
  if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int i = 1; i < 16; ++i) top = max_of_halves(top, tops[i]);
  p.gradient_tops[blockIdx.x] = top;
}
// k for a pair of them.
__device__ __forceinline__ float scale_of_tops(uint32_t top, int dim) {
  const float most = unpack_low<_Float16>(top) * unpack_high<_Float16>(top) * (float)dim;  // B, between 2^-46 and 2^39, or 0
  return __uint_as_float((uint32_t)uniform(most > 0.f ? 252 - (__float_as_uint(most) >> 23) : 127) << 23);  // (its exponent e: 2^(-2 - e))
}
// 1 / k, of a power of two.
__device__ __forceinline__ float one_over(float k) { return __uint_as_float(0x7f000000 - __float_as_uint(k)); }
// k of the whole batch, by every wave for itself.
template <class T>
__device__ __forceinline__ float gradient_scale(const AttentionParams& p) {
  if constexpr (!std::is_same<T, _Float16>::value) return 1.f;
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < kTopParts; i += 64) top = max_of_halves(top, p.gradient_tops[i + (threadIdx.x & 63)]);
  return scale_of_tops(top_of_wave(top), p.dim);
}

// ---- rows with one key ----------------------------------------------------------------------------------
// The first token of a sequence has itself as its only key: its weight is 1 and ds = p (dp - delta) = 0 whatever it holds.  Weights
// made again from lse are 1 +- some 2^-24 |s|, which would leave noise where nothing belongs (and an optimizer that normalises makes
// full steps of it).  The kernels for long sequences take its lse as infinite, which makes the weight 0 and with it ds (NaN, where the
// row is not finite), and put the weight of the pair back to 1 for dv.  The kernel for short ones has a factor of each row in LDS
// anyway, which is 0 for it: p (0 dp - 0); its dv has the weight as it is, 1 once rounded to 16 bits (up to logits of a thousand).
// (There the weight of the pair by comparisons took 440 us where this takes 436 at heads of 128, and 424 with neither.)
__device__ __forceinline__ float one_key_lse2(float lse) { return INFINITY + (lse - lse); }
// A result's 32 x 32 weights, rows = queries, where the lane's key is query `at` + 4 h of them and its own query's only key (at = -32: it is not).
template <class T>
__device__ __forceinline__ void one_key_weight(f32x16& weights, int at) {
  asm volatile("" : "+v"(at));  // (else the sixteen comparisons are kept over the whole loop: 21 to 82 scalar registers spilled)
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (8 * (i / 4) + i % 4 == at && weights[i] == weights[i]) weights[i] = Held<T>::kWeight;
}
// For the same reason: delta = sum p dp, and the weights' own sum, by which the errors that they share go out of it, so that a row's ds add up
// to 0.  (Logits so large that 32 bits hold no weight have no sum to go by.)
template <class T>
__device__ __forceinline__ float delta_of(float sum, float weights) {
  constexpr float kOne = Held<T>::kWeight;
  return weights > 0.5f * kOne && weights < 2.f * kOne ? sum / weights : sum * (1.f / kOne);
}

template <class T, int NB>
__device__ __forceinline__ void dq_carefully(const AttentionParams& p, int head, int kv_head, int row, int first, int begin, int stop,
                                             int row_end, float delta, int chunk, int chunks) {
  const int h = (threadIdx.x & 63) >> 5;
  const bool there = first <= row;
  const float scale = p.flip ? -p.scale_log2 : p.scale_log2;
  const float lse2 = there ? p.lse[(int64_t)head * p.plan.tokens + row] * kLog2e : 0.f;
  const char* q = (const char*)p.q + (int64_t)(there ? row : begin) * p.q_token + (int64_t)head * p.q_head;
  const char* d = (const char*)p.dout + (int64_t)(there ? row : begin) * p.dout_token + (int64_t)head * p.dout_head;
  HalfRow<NB> acc = {};
#pragma unroll 1
  for (int key = begin; key < stop; ++key) {
    const bool sees = there && key >= first && key <= row;
    if (__builtin_amdgcn_ballot_w64(sees) == 0) continue;
    const char* k = (const char*)p.k + (int64_t)key * p.k_token + (int64_t)kv_head * p.k_head;
    const float dp = dot_rows<T>(d, (const char*)p.v + (int64_t)key * p.v_token + (int64_t)kv_head * p.v_head, p.dim, h);
    const float ds = first == row ? (dp - dp) + (lse2 - lse2)  // (see one_key_lse2)
                                  : exp2_fast(__builtin_fmaf(dot_rows<T>(q, k, p.dim, h), scale, -lse2)) * (dp - delta);
    if (sees) add_row<T, NB>(acc, 1.f, ds, k, p.dim, h);
  }
  if (row >= row_end) return;
  const int64_t at = (int64_t)row * p.heads + head;
  store_half<T, NB>(chunks > 1 ? nullptr : (T*)p.dq + at * p.dim,
                    chunks > 1 ? p.row_sums + ((int64_t)chunk * p.plan.tokens * p.heads + at) * p.dim : nullptr, acc, p.scale, p.dim, h);
}

// Rounds begin .. stop - 1 of `round` queries each, as the dk, dv kernel counts them; part: of the sums, or -1.
template <class T, int NB>
__device__ __forceinline__ void dk_dv_carefully(const AttentionParams& p, int kv_head, int head0, int key, int last, int tile0, int end,
                                                int round, int head_rounds, int begin, int stop, int key_end, int part, float k_scale) {
  const int h = (threadIdx.x & 63) >> 5;
  const bool there = last > key;
  const float scale = p.flip ? -p.scale_log2 : p.scale_log2;
  const char* k = (const char*)p.k + (int64_t)(there ? key : tile0) * p.k_token + (int64_t)kv_head * p.k_head;
  const char* v = (const char*)p.v + (int64_t)(there ? key : tile0) * p.v_token + (int64_t)kv_head * p.v_head;
  const bool begins = there && p.plan.first[key] == key;  // (query `key` has this key only: see one_key_lse2)
#pragma unroll 1
  for (int which = 0; which < 2; ++which) {  // dv, dk
    HalfRow<NB> acc = {};
#pragma unroll 1
    for (int n = begin; n < stop; ++n) {
      const int head = head0 + n / head_rounds, m0 = tile0 + n % head_rounds * round;
#pragma unroll 1
      for (int query = m0; query < min(m0 + round, end); ++query) {
        const bool sees = there && query >= key && query < last;
        if (__builtin_amdgcn_ballot_w64(sees) == 0) continue;
        const int64_t at = (int64_t)head * p.plan.tokens + query;
        const char* q = (const char*)p.q + (int64_t)query * p.q_token + (int64_t)head * p.q_head;
        const char* d = (const char*)p.dout + (int64_t)query * p.dout_token + (int64_t)head * p.dout_head;
        const bool one = begins && query == key;
        float weight = exp2_fast(__builtin_fmaf(dot_rows<T>(k, q, p.dim, h), scale, -p.lse[at] * kLog2e));
        if (one) weight = 1.f + (p.lse[at] - p.lse[at]);
        if (which == 1) {
          const float dp = dot_rows<T>(v, d, p.dim, h);
          weight *= dp - (one ? dp : p.delta[at] * one_over(k_scale));
        }
        if (sees) add_row<T, NB>(acc, 1.f, weight, which == 0 ? d : q, p.dim, h);
      }
    }
    if (key >= key_end) continue;
    const int64_t at = (int64_t)key * p.kv_heads + kv_head;
    float* const sums = which == 0 ? p.dv_sums : p.dk_sums;
    store_half<T, NB>(part >= 0 ? nullptr : (T*)(which == 0 ? p.dv : p.dk) + at * p.dim,
                      part >= 0 ? sums + ((int64_t)part * p.plan.tokens * p.kv_heads + at) * p.dim : nullptr, acc,
                      which == 0 ? 1.f : p.scale, p.dim, h);
  }
}

// ---- forward ------------------------------------------------------------------------------------
// One workgroup: 128 query tokens of one head; one wave: 32 of them, lane's token is column l & 31 of S^T = K Q^T, so
// the softmax of a row runs over a lane's own registers and its partner's, 32 lanes away, and P^T is the second operand of
// O^T = V^T P^T as it is.  The next tile of keys and values is on its way to LDS while this one is worked on.
//
// 16384 tokens, 16 heads of 128 on 2: 1.04 ms, 1.06 PFLOP/s, the matrix cores busy 57 % of the cycles; what is left is the
// exponentials between a wave's two products, which the other wave of its SIMD fills as far as it can.  1024 walks of up to
// 101 tokens, 8 heads of 64: 24 us, 89 MB (3.7 TB/s): two or three rounds a workgroup, bound by the latency of their loads.
template <class T, int NB>
__global__ __launch_bounds__(256, 2) void attention_forward_kernel(AttentionParams p) {
  constexpr int kChunks = HeadTile<NB>::kChunks, kSize = HeadTile<NB>::kSize;
  __shared__ u32x4 tiles[2][2][kSize];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), h = lane >> 5;
  int chunk, rank, head;
  chunk_tile_and_head(p.max_chunks, p.heads, chunk, rank, head);
  const int kv_head = uniform(head / p.group);
  int tile0, tile_end;
  if (p.plan.short_tiles > 0) {
    tile0 = uniform(p.plan.short_starts[rank]);
    tile_end = uniform(p.plan.short_starts[rank + 1]);
  } else {
    tile0 = uniform(p.plan.query_order[rank]) * kRows;
    tile_end = min(tile0 + kRows, p.plan.tokens);
  }
  const int end = min(tile_end, p.plan.covered);
  const int row0 = tile0 + wave * 32, row = row0 + (lane & 31);
  const bool there = row < end;
  f32x16 acc[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) acc[b] = f32x16{};
  float top = -INFINITY, sum = 0.f;  // sum: over the lane's own keys
  int chunks = 1, careful_begin = 0, careful_stop = 0;

  if (tile0 < p.plan.covered) {
    const int first_key = uniform(p.plan.first[tile0]);
    const int rounds = (end - first_key + kColumns - 1) / kColumns;
    chunks = uniform((int)chunks_of(rounds, p.chunk, p.max_chunks));
    if (chunk >= chunks) return;
    const int begin = first_key + uniform(rounds * chunk / chunks) * kColumns;
    const int stop = chunk + 1 < chunks ? first_key + uniform(rounds * (chunk + 1) / chunks) * kColumns : end;
    careful_begin = begin;
    careful_stop = stop;
    const TileLoader<NB> k(p.k, p.k_token, p.k_head, kv_head, p.dim), v(p.v, p.v_token, p.v_head, kv_head, p.dim);
    const uint32_t lds = lds_address(&tiles[0][0][0]) + wave * 1024;
    auto issue = [&](int half, int n0) {
      k.issue(lds + (2 * half) * kSize * 16, p.k_token, n0, end);
      v.issue(lds + (2 * half + 1) * kSize * 16, p.v_token, n0, end);
    };
    issue(0, begin);
    const int first = there ? p.plan.first[row] : row + 1;
    // of the wave's rows: the smallest and the largest `first`
    const int first_min = row0 < end ? uniform(first) : 0x7fffffff - kColumns;
    const int first_max = uniform(p.plan.first[min(row0 + 31, end - 1)]);
    u32x4 qf[2 * NB];
    load_rows<NB>(qf, (const char*)p.q + (int64_t)row * p.q_token + (int64_t)head * p.q_head, there, p.dim, h);
    if (p.flip) {
#pragma unroll
      for (int i = 0; i < 2 * NB; ++i) qf[i] ^= p.flip;
    }
    int half = 0;
    for (int n0 = begin; n0 < stop; n0 += kColumns, half ^= 1) {
      wait_for_loads_and_others();
      const bool more = n0 + kColumns < stop;
      // (wave-uniform) every key is later than the wave's rows, or before their sequences
      if (n0 > row0 + 31 || n0 + kColumns <= first_min) {
        if (more) issue(half ^ 1, n0 + kColumns);
        continue;
      }
      const u32x4 *keys = tiles[half][0], *values = tiles[half][1];
      f32x16 s[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        s[t] = f32x16{};
#pragma unroll
        for (int i = 0; i < 2 * NB; ++i)
          s[t] = product_32x32x16<T>(read_operand_by_rows<kChunks>(keys, 32 * t, i, lane), qf[i], s[t]);
      }
      // (asked for behind the first products and not before them, where the wave would wait for its loads to be taken: 38 for
      // 44 us with few workgroups, 2 % with many)
      if (more) issue(half ^ 1, n0 + kColumns);
      if (n0 + kColumns - 1 > row0 || n0 < first_max) {
        const int from = first - n0 - 4 * h, to = row - n0 - 4 * h;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int key = 32 * t + 8 * (i / 4) + i % 4;
            s[t][i] = key >= from && key <= to ? s[t][i] : -INFINITY;
          }
      }
      float m = s[0][0];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) m = fmaxf(m, s[t][i]);
      m = pair_max(m) * p.scale_log2;
      if (__builtin_amdgcn_ballot_w64(m > top + kTopSlack)) {  // (top: -inf before a row's first key)
        const float higher = fmaxf(m, top);
        const float shrink = higher == -INFINITY ? 0.f : exp2_fast(top - higher);
        top = higher;
        sum *= shrink;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[b][i] *= shrink;
      }
      // a row that has seen no key yet: exp2(-inf - 0) = 0 throughout
      const float base = top == -INFINITY ? 0.f : top;
      float part = 0.f;  // (a round's weights among themselves first: thousands of equal ones added to one sum are rounded alike)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          s[t][i] = exp2_fast(__builtin_fmaf(s[t][i], p.scale_log2, -base));
          part += s[t][i];
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const u32x4 pf = pack_operand<T>(s[t], j);
#pragma unroll
          for (int b = 0; b < NB; ++b)
            acc[b] = product_32x32x16<T>(read_operand_by_columns<kChunks, true>(values, 32 * t + 16 * j, 32 * b, lane), pf,
                                         acc[b]);
        }
      }
      sum += part;
    }
    __syncthreads();
  } else if (chunk > 0) {
    return;
  }
  if (row0 >= tile_end) return;
  if (row0 + 31 >= end && !there) {  // (tiles that all of the wave's sequences see are not masked)
    top = -INFINITY;
    sum = 0.f;
#pragma unroll
    for (int b = 0; b < NB; ++b) acc[b] = f32x16{};
  }
  sum = pair_sum(sum);
  if (__builtin_amdgcn_ballot_w64(!all_finite(acc)) != 0) {
    forward_carefully<T, NB>(p, head, kv_head, row, there ? p.plan.first[row] : row + 1, careful_begin, careful_stop, tile_end, chunk, chunks);
    return;
  }
  if (chunks > 1) {
    if (row >= tile_end) return;
    if (h == 0) p.row_tops[((int64_t)chunk * p.heads + head) * p.plan.tokens + row] = make_float2(top, sum);
    store_sums<NB>(p.row_sums + (((int64_t)chunk * p.plan.tokens + row) * p.heads + head) * p.dim, acc, 1.f, p.dim, h);
    return;
  }
  const float inverse = there ? 1.f / sum : 0.f;  // (a row of nothing but logits of -inf: 0 / 0, NaN as the formulas say)
  if (h == 0 && row < tile_end) p.lse[(int64_t)head * p.plan.tokens + row] = (top + log2f(sum)) * kLn2;
  store_rows<T, NB>((T*)p.out_w + ((int64_t)row0 * p.heads + head) * p.dim, (int64_t)p.heads * p.dim, tile_end - row0, acc, inverse,
                    p.dim, &tiles[0][0][0] + wave * 32 * kChunks);
}

// Joins the chunks of the rows of cut tiles: a lane has four columns of a row.  Bound by the sums it reads, which the caches
// mostly still hold (8.3 thousand tokens, 6 heads of 80, cut in up to four: 7 us).
template <class T>
__global__ __launch_bounds__(256) void attention_join_kernel(AttentionParams p, int64_t n) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  const int column = (int)(i % p.dim), head = (int)(i / p.dim % p.heads), row = (int)(i / p.dim / p.heads);
  const int tile0 = row / kRows * kRows;
  if (tile0 >= p.plan.covered) return;
  const int rounds = (min(tile0 + kRows, p.plan.covered) - p.plan.first[tile0] + kColumns - 1) / kColumns;
  const int chunks = (int)chunks_of(rounds, p.chunk, p.max_chunks);
  if (chunks == 1) return;
  const int64_t at = (int64_t)head * p.plan.tokens + row, step = (int64_t)p.heads * p.plan.tokens;
  float top = -INFINITY;
  for (int c = 0; c < chunks; ++c) top = fmaxf(top, p.row_tops[c * step + at].x);
  const float base = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  for (int c = 0; c < chunks; ++c) {
    const float2 one = p.row_tops[c * step + at];
    const float weight = exp2_fast(one.x - base);
    sum = __builtin_fmaf(one.y, weight, sum);
    const f32x4 part = *(const f32x4*)(p.row_sums + c * n + i);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = weight == 0.f ? v[j] : __builtin_fmaf(part[j], weight, v[j]);
  }
  const float inverse = row < p.plan.covered ? 1.f / sum : 0.f;
  u32x2 o;
  o[0] = pack_pair<T>(v[0] * inverse, v[1] * inverse);
  o[1] = pack_pair<T>(v[2] * inverse, v[3] * inverse);
  *(u32x2*)((T*)p.out_w + i) = o;
  if (column == 0) p.lse[at] = (top + log2f(sum)) * kLn2;
}

// ---- backward -----------------------------------------------------------------------------------
// dq: as the forward pass, with S^T and dP^T = V dO^T; dS^T is the second operand of dQ^T = K^T dS^T.  Leaves delta and lse
// in powers of two for the other kernel.
//
// delta_i = do_i . o_i comes from an o that is rounded to 16 bits, which shifts all of a row's ds by the same amount; the fewer
// keys a row has, the more that weighs.  Tiles of few keys go over them twice and take delta_i = sum_j p_ij (do_i . v_j), the
// same sum, in 32 bits.
//
// Three products to the forward pass's two, and no maxima: 5 sequences of 700 to 4096 tokens, 16 heads of 128: 229 us, 0.91
// PFLOP/s, the matrix cores busy 50 %; 23 sequences of 3 to 1999, 6 heads of 80: 48 us, bound by the rounds of a lone workgroup,
// 1.1 us each.
template <class T, int NB>
__global__ __launch_bounds__(256, 2) void attention_backward_query_kernel(AttentionParams p) {
  constexpr int kChunks = HeadTile<NB>::kChunks, kSize = HeadTile<NB>::kSize;
  __shared__ u32x4 tiles[2][2][kSize];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), h = lane >> 5;
  int chunk, rank, head;
  chunk_tile_and_head(p.max_chunks, p.heads, chunk, rank, head);
  const int tile0 = uniform(p.plan.query_order[rank]) * kRows, kv_head = uniform(head / p.group);
  const int row0 = tile0 + wave * 32, row = row0 + (lane & 31);
  const bool there = row < p.plan.covered;
  f32x16 acc[NB];
  int chunks = 1, careful_begin = 0, careful_stop = 0;
  float delta = 0.f, k_scale = 1.f;  // delta: times k_scale
  if (tile0 < p.plan.covered) {
    const int end = min(tile0 + kRows, p.plan.covered), first_key = uniform(p.plan.first[tile0]);
    const int rounds = (end - first_key + kColumns - 1) / kColumns;
    chunks = uniform((int)chunks_of(rounds, p.chunk, p.max_chunks));
    if (chunk >= chunks) return;
    const int begin = first_key + uniform(rounds * chunk / chunks) * kColumns;
    const int stop = chunk + 1 < chunks ? first_key + uniform(rounds * (chunk + 1) / chunks) * kColumns : end;
    careful_begin = begin;
    careful_stop = stop;
    const bool exact = chunks == 1 && rounds <= kExactDeltaRounds;
    const TileLoader<NB> k(p.k, p.k_token, p.k_head, kv_head, p.dim), v(p.v, p.v_token, p.v_head, kv_head, p.dim);
    const uint32_t lds = lds_address(&tiles[0][0][0]) + wave * 1024;
    auto issue = [&](int half, int n0) {
      k.issue(lds + (2 * half) * kSize * 16, p.k_token, n0, end);
      v.issue(lds + (2 * half + 1) * kSize * 16, p.v_token, n0, end);
    };
    issue(0, begin);
    const int first = there ? p.plan.first[row] : row + 1;
    const int first_min = row0 < p.plan.covered ? uniform(first) : 0x7fffffff - kColumns;
    const int first_max = uniform(p.plan.first[min(row0 + 31, p.plan.covered - 1)]);
    u32x4 qf[2 * NB], dof[2 * NB];
    load_rows<NB>(qf, (const char*)p.q + (int64_t)row * p.q_token + (int64_t)head * p.q_head, there, p.dim, h);
    load_rows<NB>(dof, (const char*)p.dout + (int64_t)row * p.dout_token + (int64_t)head * p.dout_head, there, p.dim, h);
    float lse2 = 0.f;
    {
      u32x4 of[2 * NB];
      load_rows<NB>(of, (const char*)p.out + ((int64_t)row * p.heads + head) * p.dim * 2, there, p.dim, h);
#pragma unroll
      for (int s = 0; s < 2 * NB; ++s)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          delta = __builtin_fmaf(unpack_low<T>(of[s][j]), unpack_low<T>(dof[s][j]), delta);
          delta = __builtin_fmaf(unpack_high<T>(of[s][j]), unpack_high<T>(dof[s][j]), delta);
        }
      k_scale = gradient_scale<T>(p);
      delta = pair_sum(delta) * k_scale;
      if (there) {
        const int64_t at = (int64_t)head * p.plan.tokens + row;
        const float lse = p.lse[at];
        lse2 = first == row ? one_key_lse2(lse) : lse * kLog2e - Held<T>::kShift;
        if (h == 0 && chunk == 0) {
          p.delta[at] = delta;
          p.lse2[at] = lse2;
        }
      }
    }
    if (p.flip) {
#pragma unroll
      for (int i = 0; i < 2 * NB; ++i) qf[i] ^= p.flip;
    }
    int half = 0;
    // one sweep over the keys; DELTA: the first of two, for delta (then the first tile is asked for again at its end)
    auto sweep = [&](auto delta_only) {
      constexpr bool DELTA = decltype(delta_only)::value;
      float sum = 0.f, weights = 0.f;
      for (int n0 = begin; n0 < stop; n0 += kColumns, half ^= 1) {
        wait_for_loads_and_others();
        const int next = n0 + kColumns < stop ? n0 + kColumns : DELTA ? begin : -1;
        if (n0 > row0 + 31 || n0 + kColumns <= first_min) {
          if (next >= 0) issue(half ^ 1, next);
          continue;
        }
        const u32x4 *keys = tiles[half][0], *values = tiles[half][1];
        const bool masked = n0 + kColumns - 1 > row0 || n0 < first_max;
        const int from = first - n0 - 4 * h, to = row - n0 - 4 * h;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          f32x16 s = {}, dp = {};
#pragma unroll
          for (int i = 0; i < 2 * NB; ++i) {
            s = product_32x32x16<T>(read_operand_by_rows<kChunks>(keys, 32 * t, i, lane), qf[i], s);
            dp = product_32x32x16<T>(read_operand_by_rows<kChunks>(values, 32 * t, i, lane), dof[i], dp);
          }
          if (t == 0 && next >= 0) issue(half ^ 1, next);
          if constexpr (DELTA) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int key = 32 * t + 8 * (i / 4) + i % 4;
              const bool sees = !masked || (key >= from && key <= to);
              const float weight = sees ? exp2_fast(__builtin_fmaf(s[i], p.scale_log2, -lse2)) : 0.f;
              sum += sees ? weight * dp[i] : 0.f;
              weights += weight;
            }
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = exp2_fast(__builtin_fmaf(s[i], p.scale_log2, -lse2)) * __builtin_fmaf(dp[i], k_scale, -delta);
            if (masked) {
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const int key = 32 * t + 8 * (i / 4) + i % 4;
                s[i] = key >= from && key <= to ? s[i] : 0.f;
              }
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const u32x4 dsf = pack_operand<T>(s, j);
#pragma unroll
              for (int b = 0; b < NB; ++b)
                acc[b] = product_32x32x16<T>(read_operand_by_columns<kChunks, true>(keys, 32 * t + 16 * j, 32 * b, lane), dsf,
                                             acc[b]);
            }
          }
        }
      }
      if constexpr (DELTA) {
        delta = delta_of<T>(pair_sum(sum), pair_sum(weights)) * k_scale;
        if (h == 0 && there) p.delta[(int64_t)head * p.plan.tokens + row] = delta;
      }
    };
    if (exact) sweep(std::true_type());
#pragma unroll
    for (int b = 0; b < NB; ++b) acc[b] = f32x16{};
    sweep(std::false_type());
    __syncthreads();
  } else if (chunk > 0) {
    return;
  } else {
#pragma unroll
    for (int b = 0; b < NB; ++b) acc[b] = f32x16{};
  }
  if (row0 + 31 >= p.plan.covered && !there) {
#pragma unroll
    for (int b = 0; b < NB; ++b) acc[b] = f32x16{};
  }
  if (row0 < p.plan.tokens && __builtin_amdgcn_ballot_w64(!all_finite(acc)) != 0) {
    dq_carefully<T, NB>(p, head, kv_head, row, there ? p.plan.first[row] : row + 1, careful_begin, careful_stop, p.plan.tokens, delta * one_over(k_scale),
                        chunk, chunks);
    return;
  }
  const float factor = p.scale * (1.f / Held<T>::kWeight) * one_over(k_scale);
  if (chunks > 1) {
    if (row < p.plan.tokens)
      store_sums<NB>(p.row_sums + (((int64_t)chunk * p.plan.tokens + row) * p.heads + head) * p.dim, acc, factor, p.dim, h);
    return;
  }
  if (row0 < p.plan.tokens)
    store_rows<T, NB>((T*)p.dq + ((int64_t)row0 * p.heads + head) * p.dim, (int64_t)p.heads * p.dim, p.plan.tokens - row0, acc, factor,
                      p.dim, &tiles[0][0][0] + wave * 32 * kChunks);
}

// dk, dv: one workgroup has 128 keys of one key head, a wave 32 of them (lane's key is a column of S = Q K^T), and goes
// over the query tiles that see them, for each head of its share of the group in turn: no sum is shared between
// workgroups.  Where keys and key heads are few for the GPU a group's heads are shared out; shares and chunks leave sums in
// 32 bits, which another kernel adds.
//
// Heads of up to 128: dk and dv of 32 keys take 128 registers and the keys 32; with the values in registers too a wave has
// to do without half of its 256 or run alone on its SIMD (long sequences of 4 x 128: 821 us with 43 registers spilled, 569
// alone).  They are read from LDS instead, and a round takes 32 queries, so that two workgroups fit a compute unit.
//
// Four products, two of them those of the dq kernel once more (taking dq here too would need atomics, or its sums for every tile
// of keys in memory).  The long sequences above, 4 key heads: 325 us, 0.86 PFLOP/s, matrix cores busy 44 %, 190 MB of sums and
// results written.
template <class T, int NB>
__global__ __launch_bounds__(256, 2) void attention_backward_key_kernel(AttentionParams p) {
  constexpr int kChunks = HeadTile<NB>::kChunks;
  constexpr bool kValuesInLds = NB == 4;
  constexpr int kRound = kValuesInLds ? 32 : 64, kSize = kRound * kChunks;
  __shared__ u32x4 tiles[2][2][kSize];
  __shared__ u32x4 values[kValuesInLds ? kRows * kChunks : 1];
  __shared__ float rows_of[2][2][64];  // lse2 and delta of a round's queries
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), h = lane >> 5;
  int chunk, rank, unit;
  chunk_tile_and_head(p.max_key_chunks, p.kv_heads * p.head_split, chunk, rank, unit);
  const int kv_head = uniform(unit / p.head_split), share = unit - kv_head * p.head_split, heads = uniform(p.group / p.head_split);
  const int tile0 = uniform(p.plan.key_order[rank]) * kRows;
  const int key0 = tile0 + wave * 32, key = key0 + (lane & 31);
  const bool there = key < p.plan.covered;
  f32x16 dk[NB], dv[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    dk[b] = f32x16{};
    dv[b] = f32x16{};
  }
  int chunks = 1, careful_begin = 0, careful_stop = 0, careful_rounds = 1, careful_end = 0;
  float k_scale = 1.f;
  if (tile0 < p.plan.covered) {
    const int end = uniform(p.plan.last[min(tile0 + kRows, p.plan.covered) - 1]);
    const int head0 = kv_head * p.group + share * heads, head_rounds = (end - tile0 + kRound - 1) / kRound, rounds = head_rounds * heads;
    chunks = uniform((int)chunks_of(rounds, p.key_chunk, p.max_key_chunks));
    if (chunk >= chunks) return;
    // round i: head i / head_rounds of the share, queries from tile0 + i % head_rounds * kRound on
    const int begin = uniform((int)((int64_t)rounds * chunk / chunks)), stop = uniform((int)((int64_t)rounds * (chunk + 1) / chunks));
    careful_begin = begin;
    careful_stop = stop;
    careful_rounds = head_rounds;
    careful_end = end;
    const TileLoader<NB, kRound> q(p.q, p.q_token, p.q_head, head0, p.dim), d(p.dout, p.dout_token, p.dout_head, head0, p.dim);
    const uint32_t lds = lds_address(&tiles[0][0][0]) + wave * 1024, rows_lds = lds_address(&rows_of[0][0][0]);
    auto issue = [&](int half, int head, int m0) {  // head: of the share
      TileLoader<NB, kRound> qh = q, dh = d;
      qh.base += head * p.q_head;
      dh.base += head * p.dout_head;
      qh.issue(lds + (2 * half) * kSize * 16, p.q_token, m0, end);
      dh.issue(lds + (2 * half + 1) * kSize * 16, p.dout_token, m0, end);
      if (wave < 2)
        load_words_to_lds((const char*)((wave == 0 ? p.lse2 : p.delta) + (int64_t)(head0 + head) * p.plan.tokens + m0),
                          min(lane, end - 1 - m0) * 4, rows_lds + (2 * half + wave) * 256);
    };
    if (kValuesInLds) {
      const TileLoader<NB, kRows> v(p.v, p.v_token, p.v_head, kv_head, p.dim);
      v.issue(lds_address(values) + wave * 1024, p.v_token, tile0, min(tile0 + kRows, p.plan.covered));
      if (p.dim < 8 * kChunks) {  // the other operand has a row's first columns past `dim`: 0 here
        wait_for_loads_and_others();
        for (int at = threadIdx.x; at < kRows * kChunks; at += 256)
          if (at % kChunks * 8 >= p.dim) values[tile_place<kChunks>(at / kChunks, at % kChunks)] = u32x4{0, 0, 0, 0};
      }
    }
    int head = uniform(begin / head_rounds), m0 = tile0 + uniform(begin % head_rounds) * kRound;
    issue(0, head, m0);
    k_scale = gradient_scale<T>(p);
    const int last = there ? p.plan.last[key] : key;
    const int one_at = there && p.plan.first[key] == key ? (lane & 31) - 4 * h : -32;
    // of the wave's keys: the smallest and the largest `last`
    const int last_min = key0 < p.plan.covered ? uniform(last) : 0;
    const int last_max = key0 < p.plan.covered ? uniform(p.plan.last[min(key0 + 31, p.plan.covered - 1)]) : 0;
    u32x4 kf[2 * NB], vf[kValuesInLds ? 1 : 2 * NB];
    load_rows<NB>(kf, (const char*)p.k + (int64_t)key * p.k_token + (int64_t)kv_head * p.k_head, there, p.dim, h);
    if constexpr (!kValuesInLds)
      load_rows<NB>(vf, (const char*)p.v + (int64_t)key * p.v_token + (int64_t)kv_head * p.v_head, there, p.dim, h);
    if (p.flip) {
#pragma unroll
      for (int i = 0; i < 2 * NB; ++i) kf[i] ^= p.flip;
    }
    int half = 0;
    for (int round = begin; round < stop; ++round) {
      int next_head = head, next = m0 + kRound;
      if (next >= end) {
        next = tile0;
        ++next_head;
      }
      wait_for_loads_and_others();
      if (round + 1 < stop) issue(half ^ 1, next_head, next);
      if (m0 + kRound > key0 && m0 < last_max) {  // (else no query of the tile sees a key of the wave)
        const u32x4 *queries = tiles[half][0], *douts = tiles[half][1];
        const bool masked = m0 < key0 + 31 || m0 + kRound > last_min;
        const int from = key - m0 - 4 * h, to = last - m0 - 4 * h;
#pragma unroll
        for (int t = 0; t < kRound / 32; ++t) {
          f32x16 s = {}, dp = {};
#pragma unroll
          for (int i = 0; i < 2 * NB; ++i) {
            s = product_32x32x16<T>(read_operand_by_rows<kChunks>(queries, 32 * t, i, lane), kf[i], s);
            dp = product_32x32x16<T>(read_operand_by_rows<kChunks>(douts, 32 * t, i, lane),
                                     kValuesInLds ? read_operand_by_rows<kChunks>(values, 32 * wave, i, lane) : vf[kValuesInLds ? 0 : i], dp);
          }
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const f32x4 lse2 = *(const f32x4*)&rows_of[half][0][32 * t + 8 * g + 4 * h];
            const f32x4 delta = *(const f32x4*)&rows_of[half][1][32 * t + 8 * g + 4 * h];
#pragma unroll
            for (int n = 0; n < 4; ++n) {
              const int i = 4 * g + n;
              s[i] = exp2_fast(__builtin_fmaf(s[i], p.scale_log2, -lse2[n]));
              dp[i] = s[i] * __builtin_fmaf(dp[i], k_scale, -delta[n]);
            }
          }
          if (masked) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int query = 32 * t + 8 * (i / 4) + i % 4;
              const bool sees = query >= from && query < to;
              s[i] = sees ? s[i] : 0.f;
              dp[i] = sees ? dp[i] : 0.f;
            }
          }
          if (m0 + 32 * t == key0) one_key_weight<T>(s, one_at);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const u32x4 pf = pack_operand<T>(s, j), dsf = pack_operand<T>(dp, j);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
              dv[b] = product_32x32x16<T>(read_operand_by_columns<kChunks, true>(douts, 32 * t + 16 * j, 32 * b, lane), pf,
                                          dv[b]);
              dk[b] = product_32x32x16<T>(read_operand_by_columns<kChunks, true>(queries, 32 * t + 16 * j, 32 * b, lane), dsf,
                                          dk[b]);
            }
          }
        }
      }
      head = next_head;
      m0 = next;
      half ^= 1;
    }
    __syncthreads();
  } else if (chunk > 0) {
    return;
  }
  if (key0 >= p.plan.tokens) return;
  if (__builtin_amdgcn_ballot_w64(!(all_finite(dk) && all_finite(dv))) != 0) {
    dk_dv_carefully<T, NB>(p, kv_head, kv_head * p.group + share * heads, key, there ? p.plan.last[key] : key, tile0, careful_end, kRound,
                           careful_rounds, careful_begin, careful_stop, p.plan.tokens,
                           chunks * p.head_split == 1 ? -1 : chunk * p.head_split + share, k_scale);
    return;
  }
  const int64_t row_elements = (int64_t)p.kv_heads * p.dim;
  const float dk_factor = p.scale * (1.f / Held<T>::kWeight) * one_over(k_scale), dv_factor = 1.f / Held<T>::kWeight;
  if (chunks * p.head_split == 1) {
    u32x4* part_lds = &tiles[0][0][0] + wave * 32 * kChunks;
    const int64_t at = ((int64_t)key0 * p.kv_heads + kv_head) * p.dim;
    store_rows<T, NB>((T*)p.dk + at, row_elements, p.plan.tokens - key0, dk, dk_factor, p.dim, part_lds);
    store_rows<T, NB>((T*)p.dv + at, row_elements, p.plan.tokens - key0, dv, dv_factor, p.dim, part_lds);
  } else if (key < p.plan.tokens) {
    const int64_t at = (((int64_t)(chunk * p.head_split + share) * p.plan.tokens + key) * p.kv_heads + kv_head) * p.dim;
    store_sums<NB>(p.dk_sums + at, dk, dk_factor, p.dim, h);
    store_sums<NB>(p.dv_sums + at, dv, dv_factor, p.dim, h);
  }
}

// Sequences of at most a tile: one workgroup has the whole sequences of a tile and one key head, so that it reads queries, keys,
// values and output gradients once and has all of dq, dk and dv.  Where tiles are few a group's heads are shared out, as in the
// dk, dv kernel.  Per head of the group each wave first has 32 queries, as in the dq kernel, then 32 keys, as in the other one;
// delta always comes from the weights themselves.
//
// 1024 walks of up to 101 tokens, 8 heads of 64: 57 us where the two kernels above take 97, 155 MB (2.7 TB/s), bound by the
// latency of one load of a tile and three sweeps over it.  8 heads of 128, walks of 20 to 101 spread over the logarithm: 349 us for
// 360; spread evenly 435 for 423; of 101 throughout, which leave a fifth of each tile empty, 798 for 716.
template <class T, int NB>
__global__ __launch_bounds__(256, NB <= 2 ? 2 : 1) void attention_backward_short_kernel(AttentionParams p) {
  constexpr int kChunks = HeadTile<NB>::kChunks, kSize = kRows * kChunks;
  __shared__ u32x4 keys[kSize], values[kSize], queries[kSize], douts[kSize];
  __shared__ float lse2s[kRows], deltas[kRows], factors[kRows];
  __shared__ uint32_t tops[4];
  // (what is computed from `lane` is computed anew after each empty asm: addresses kept from one part to the next cost 14 to 47
  // spilled registers, 66 and 397 us for 60 and 342 at heads of 64 and 128)
  int lane = threadIdx.x & 63;
  const int wave = uniform(threadIdx.x >> 6), h = lane >> 5;
  const int units = p.kv_heads * p.head_split, unit = uniform(blockIdx.x % units), tile = uniform(blockIdx.x / units);
  const int kv_head = uniform(unit / p.head_split), share = unit - kv_head * p.head_split, heads = uniform(p.group / p.head_split);
  const int head0 = kv_head * p.group + share * heads;
  const int tile0 = uniform(p.plan.short_starts[tile]), tile_end = uniform(p.plan.short_starts[tile + 1]);
  const int row0 = tile0 + wave * 32, row = row0 + (lane & 31);  // as queries and as keys
  u32x4* const part_lds = queries + wave * 32 * kChunks;
  const int64_t q_elements = (int64_t)p.heads * p.dim, k_elements = (int64_t)p.kv_heads * p.dim;
  f32x16 dk[NB], dv[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) dk[b] = dv[b] = f32x16{};
  const float dv_factor = 1.f / Held<T>::kWeight;
  float k_scale = 1.f;
  bool again = false;  // some head's dq is not finite: taken carefully at the end, where no sums are in registers

  if (tile0 < p.plan.covered) {
    // (such a tile ends at `covered` or before it)
    const bool there = row < tile_end, work = row0 < tile_end;
    const int first = there ? p.plan.first[row] : row + 1, last = there ? p.plan.last[row] : row;
    const int first_tile = work ? (uniform(first) - tile0) / 32 : 0;                                    // of the wave's keys
    const int last_tile = work ? (uniform(p.plan.last[min(row0 + 31, tile_end - 1)]) - 1 - tile0) / 32 : 0;  // of its queries
    const uint32_t part = wave * 1024;
    const TileLoader<NB, kRows> k(p.k, p.k_token, p.k_head, kv_head, p.dim), v(p.v, p.v_token, p.v_head, kv_head, p.dim);
    k.issue(lds_address(keys) + part, p.k_token, tile0, tile_end);
    v.issue(lds_address(values) + part, p.v_token, tile0, tile_end);
    for (int g = 0; g < heads; ++g) {
      const int head = head0 + g;
      if (g > 0) __syncthreads();  // (the last head's dq has left through `queries`)
      const TileLoader<NB, kRows> q(p.q, p.q_token, p.q_head, head, p.dim), d(p.dout, p.dout_token, p.dout_head, head, p.dim);
      q.issue(lds_address(queries) + part, p.q_token, tile0, tile_end);
      d.issue(lds_address(douts) + part, p.dout_token, tile0, tile_end);
      const float lse = there ? p.lse[(int64_t)head * p.plan.tokens + row] : 0.f, lse2 = lse * kLog2e - Held<T>::kShift;
      if (h == 0) lse2s[wave * 32 + (lane & 31)] = lse2;
      wait_for_loads_and_others();
      if (g == 0 && p.dim < 8 * kChunks) {  // the other operands have a row's first columns past `dim`: 0 here
        for (int at = threadIdx.x; at < kSize; at += 256)
          if (at % kChunks * 8 >= p.dim) {
            const int place = tile_place<kChunks>(at / kChunks, at % kChunks);
            keys[place] = values[place] = u32x4{0, 0, 0, 0};
          }
        __syncthreads();
      }
      if constexpr (std::is_same<T, _Float16>::value) {
        // k of what is in LDS and of the heads before (walks of up to 101, 8 heads of 64 and of 128: 57 and 464 us, 67 and 552 with the
        // launch before that reads all output gradients and values; 54 and 436 with neither)
        uint32_t top = 0, others = 0;
#pragma unroll
        for (int i = 0; i < kSize; i += 256) {
          const u32x4 a = douts[i + 64 * wave + lane], b = values[i + 64 * wave + lane];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            top = max_of_halves(top, a[j] & 0x7fff7fff);
            others = max_of_halves(others, b[j] & 0x7fff7fff);
          }
        }
        top = max(top & 0xffff, top >> 16) | max(others & 0xffff, others >> 16) << 16;
        if (__builtin_amdgcn_ballot_w64((top & 0xffff) >= 0x7c00 || top >= 0x7c000000) != 0) {  // (what is not finite does not count)
          top = 0;
#pragma unroll 1
          for (int at = 64 * wave + lane; at < kSize; at += 256) top = max_of_halves(top, top_of(douts[at]) | top_of(values[at]) << 16);
        }
        top = top_of_wave(top);
        if (lane == 0) tops[wave] = top;
        __syncthreads();
        const float k = scale_of_tops(max_of_halves(max_of_halves(tops[0], tops[1]), max_of_halves(tops[2], tops[3])), p.dim);
        asm volatile("" : "+v"(lane));
        if (g == 0 || k < k_scale) {
          const float ratio = g == 0 ? 1.f : k * one_over(k_scale);
#pragma unroll
          for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) dk[b][i] *= ratio;
          k_scale = k;
        }
      }
      f32x16 dq[NB];
#pragma unroll
      for (int b = 0; b < NB; ++b) dq[b] = f32x16{};
      if (work) {
        u32x4 qf[2 * NB], dof[2 * NB];
#pragma unroll
        for (int i = 0; i < 2 * NB; ++i) {
          qf[i] = read_operand_by_rows<kChunks>(queries, 32 * wave, i, lane) ^ p.flip;
          dof[i] = read_operand_by_rows<kChunks>(douts, 32 * wave, i, lane);
        }
        float delta = 0.f;
        const float factor = first == row ? 0.f : k_scale;
        if (h == 0) factors[wave * 32 + (lane & 31)] = factor;
        for (int sweep = 0; sweep < 2; ++sweep) {  // for delta, then for dq
          float sum = 0.f, weights = 0.f;
          for (int at = first_tile; at <= wave; ++at) {
            int t = at;
            asm volatile("" : "+s"(t));
            f32x16 s = {}, dp = {};
#pragma unroll
            for (int i = 0; i < 2 * NB; ++i) {
              s = product_32x32x16<T>(read_operand_by_rows<kChunks>(keys, 32 * t, i, lane), qf[i], s);
              dp = product_32x32x16<T>(read_operand_by_rows<kChunks>(values, 32 * t, i, lane), dof[i], dp);
            }
            const int from = first - tile0 - 32 * t - 4 * h, to = row - tile0 - 32 * t - 4 * h;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int key = 8 * (i / 4) + i % 4;
              const bool sees = key >= from && key <= to;
              s[i] = sees ? exp2_fast(__builtin_fmaf(s[i], p.scale_log2, -lse2)) : 0.f;
              dp[i] = sees ? __builtin_fmaf(dp[i], factor, -delta) : 0.f;
            }
            if (sweep == 0) {
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                weights += s[i];
                sum = __builtin_fmaf(s[i], dp[i], sum);
              }
              continue;
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] *= dp[i];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const u32x4 dsf = pack_operand<T>(s, j);
#pragma unroll
              for (int b = 0; b < NB; ++b)
                dq[b] = product_32x32x16<T>(read_operand_by_columns<kChunks, true>(keys, 32 * t + 16 * j, 32 * b, lane), dsf, dq[b]);
            }
          }
          asm volatile("" : "+v"(lane));
          if (sweep == 0) delta = delta_of<T>(pair_sum(sum), pair_sum(weights));
        }
        asm volatile("" : "+v"(lane));
        if (h == 0) {
          deltas[wave * 32 + (lane & 31)] = delta;
          if (there) p.delta[(int64_t)head * p.plan.tokens + row] = delta * one_over(k_scale);
        }
      }
      __syncthreads();
      if (work) {
        u32x4 kf[2 * NB], vf[2 * NB];
#pragma unroll
        for (int i = 0; i < 2 * NB; ++i) {
          kf[i] = read_operand_by_rows<kChunks>(keys, 32 * wave, i, lane) ^ p.flip;
          vf[i] = read_operand_by_rows<kChunks>(values, 32 * wave, i, lane);
        }
        for (int at = wave; at <= last_tile; ++at) {
          int t = at;
          asm volatile("" : "+s"(t));
          f32x16 s = {}, dp = {};
#pragma unroll
          for (int i = 0; i < 2 * NB; ++i) {
            s = product_32x32x16<T>(read_operand_by_rows<kChunks>(queries, 32 * t, i, lane), kf[i], s);
            dp = product_32x32x16<T>(read_operand_by_rows<kChunks>(douts, 32 * t, i, lane), vf[i], dp);
          }
          const int from = row - tile0 - 32 * t - 4 * h, to = last - tile0 - 32 * t - 4 * h;
#pragma unroll
          for (int q4 = 0; q4 < 4; ++q4) {
            const f32x4 lses = *(const f32x4*)&lse2s[32 * t + 8 * q4 + 4 * h], delta = *(const f32x4*)&deltas[32 * t + 8 * q4 + 4 * h];
            const f32x4 factor = *(const f32x4*)&factors[32 * t + 8 * q4 + 4 * h];
#pragma unroll
            for (int n = 0; n < 4; ++n) {
              const int i = 4 * q4 + n, query = 8 * q4 + n;
              const bool sees = query >= from && query < to;
              const float weight = exp2_fast(__builtin_fmaf(s[i], p.scale_log2, -lses[n]));
              s[i] = sees ? weight : 0.f;
              dp[i] = sees ? weight * __builtin_fmaf(dp[i], factor[n], -delta[n]) : 0.f;
            }
          }
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const u32x4 pf = pack_operand<T>(s, j), dsf = pack_operand<T>(dp, j);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
              dv[b] = product_32x32x16<T>(read_operand_by_columns<kChunks, true>(douts, 32 * t + 16 * j, 32 * b, lane), pf, dv[b]);
              dk[b] = product_32x32x16<T>(read_operand_by_columns<kChunks, true>(queries, 32 * t + 16 * j, 32 * b, lane), dsf, dk[b]);
            }
          }
        }
      }
      __syncthreads();
      again = again || __builtin_amdgcn_ballot_w64(!all_finite(dq)) != 0;
      if (work)
        store_rows<T, NB>((T*)p.dq + ((int64_t)row0 * p.heads + head) * p.dim, q_elements, tile_end - row0, dq,
                          p.scale * (1.f / Held<T>::kWeight) * one_over(k_scale), p.dim, part_lds);
    }
  } else if (row0 < tile_end) {  // tokens of no sequence
    for (int g = 0; g < heads; ++g)
      store_rows<T, NB>((T*)p.dq + ((int64_t)row0 * p.heads + head0 + g) * p.dim, q_elements, tile_end - row0, dk, 0.f, p.dim,
                        part_lds);
  }
  if (row0 >= tile_end) return;
  const float dk_factor = p.scale * (1.f / Held<T>::kWeight) * one_over(k_scale);
  if (__builtin_amdgcn_ballot_w64(!(all_finite(dk) && all_finite(dv))) != 0) {
    dk_dv_carefully<T, NB>(p, kv_head, head0, row, row < tile_end ? p.plan.last[row] : row, tile0, tile_end, kRows, 1, 0, heads, tile_end,
                           p.head_split == 1 ? -1 : share, 1.f);
  } else if (p.head_split == 1) {
    const int64_t at = ((int64_t)row0 * p.kv_heads + kv_head) * p.dim;
    store_rows<T, NB>((T*)p.dk + at, k_elements, tile_end - row0, dk, dk_factor, p.dim, part_lds);
    store_rows<T, NB>((T*)p.dv + at, k_elements, tile_end - row0, dv, dv_factor, p.dim, part_lds);
  } else if (row < tile_end) {
    const int64_t at = (((int64_t)share * p.plan.tokens + row) * p.kv_heads + kv_head) * p.dim;
    store_sums<NB>(p.dk_sums + at, dk, dk_factor, p.dim, h);
    store_sums<NB>(p.dv_sums + at, dv, dv_factor, p.dim, h);
  }
  if (!again) return;
#pragma unroll 1
  for (int g = 0; g < heads; ++g) {
    const int head = head0 + g;
    const bool there = row < tile_end;
    dq_carefully<T, NB>(p, head, kv_head, row, there ? p.plan.first[row] : row + 1, tile0, tile_end, tile_end,
                        there ? p.delta[(int64_t)head * p.plan.tokens + row] : 0.f, 0, 1);
  }
}

// Adds the chunks of cut tiles: dq (`which` 0), dk (1), dv (2); n values each, a lane has four.  Bound by the sums, which the
// last cache holds: 214 MB in 36 us (5.9 TB/s).
template <class T>
__global__ __launch_bounds__(256) void attention_add_kernel(AttentionParams p, int64_t n_rows, int64_t n_keys, int key_round) {
  const int which = blockIdx.y;
  const int64_t n = which == 0 ? n_rows : n_keys, i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= n || (which == 0 ? p.max_chunks : p.max_key_chunks * p.head_split) == 1) return;
  const int token = (int)(i / p.dim / (which == 0 ? p.heads : p.kv_heads)), tile0 = token / kRows * kRows;
  const int tile_end = min(tile0 + kRows, p.plan.covered);
  int chunks;
  if (tile0 >= p.plan.covered) chunks = 1;  // (of the zeros there each share has left its own)
  else if (which == 0) chunks = (int)chunks_of((tile_end - p.plan.first[tile0] + kColumns - 1) / kColumns, p.chunk, p.max_chunks);
  else
    chunks = (int)chunks_of((p.plan.last[tile_end - 1] - tile0 + key_round - 1) / key_round * (p.group / p.head_split), p.key_chunk, p.max_key_chunks);
  if (which > 0) chunks *= p.head_split;
  if (chunks == 1) return;
  const float* sums = which == 0 ? p.row_sums : which == 1 ? p.dk_sums : p.dv_sums;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  for (int c = 0; c < chunks; ++c) v += *(const f32x4*)(sums + c * n + i);
  u32x2 o;
  o[0] = pack_pair<T>(v[0], v[1]);
  o[1] = pack_pair<T>(v[2], v[3]);
  *(u32x2*)((T*)(which == 0 ? p.dq : which == 1 ? p.dk : p.dv) + i) = o;
}

// ---- host ---------------------------------------------------------------------------------------

int64_t round_up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }
int64_t tiles_of(int64_t tokens) { return (tokens + kRows - 1) / kRows; }

// The plan's parts, in words: first, last, query_order, key_order, short_starts (two tiles next to each other have more than kRows
// tokens).
struct PlanParts {
  int64_t last, query_order, key_order, short_starts, words;
};
PlanParts plan_parts(int64_t tokens) {
  PlanParts w;
  w.last = round_up(tokens, 4);
  w.query_order = 2 * w.last;
  w.key_order = w.query_order + round_up(tiles_of(tokens), 4);
  w.short_starts = w.key_order + round_up(tiles_of(tokens), 4);
  w.words = w.short_starts + round_up(2 * tiles_of(tokens) + 4, 4);
  return w;
}

// How the work is cut into chunks, and the parts of the workspace in bytes.  About kItems equal pieces of work fill the GPU
// (512 workgroups at a time) twice over; a tile with much more than its share of them is cut (one sequence of 8192 tokens and
// two heads: 128 tiles of up to 128 rounds).
// Chunks have no fewer than 8 rounds, or than 4 if even so they do not fill it once (both directions in us: 4 heads of 64, 2048
// tokens, 1088 rounds in all: 79 with 4, 92 with 8; 2 heads, 4096 tokens, 2112 rounds: 109 and 96).
constexpr int64_t kItems = 1024, kFewRounds = 1536;
constexpr int64_t kMostChunkBytes = (int64_t)1 << 30;
struct Cuts {
  int64_t chunk, max_chunks, key_chunk, max_key_chunks, head_split;
  int64_t delta, row_sums, row_tops, gradient_tops, dk_sums, dv_sums, bytes;
};
int64_t key_round_of(int dim) { return dim > 96 ? 32 : 64; }
Cuts cuts_of(const nd_packed_attention& a, bool backward) {
  Cuts w = {};
  auto most = [](int64_t largest, int64_t chunk, int64_t bytes_each) {
    return chunks_of(largest, chunk, std::max<int64_t>(1, kMostChunkBytes / std::max<int64_t>(bytes_each, 1)));
  };
  auto take = [&](int64_t bytes) {
    const int64_t at = w.bytes;
    w.bytes += round_up(bytes, 256);
    return at;
  };
  const int64_t row_bytes = a.n_tokens * a.heads * a.dim * 4, key_bytes = a.n_tokens * a.kv_heads * a.dim * 4;
  const int64_t work = a.rounds * a.heads;
  w.chunk = std::max<int64_t>(work <= kFewRounds ? 4 : 8, (work + kItems - 1) / kItems);
  w.max_chunks = most(a.most_rounds, w.chunk, row_bytes);
  w.max_key_chunks = w.key_chunk = w.head_split = 1;
  if (backward) {
    const int64_t finer = kColumns / key_round_of(a.dim), group = a.heads / a.kv_heads;
    const int64_t tiles = a.short_tiles > 0 ? 2 * a.short_tiles : tiles_of(a.n_tokens);  // (half the work to be worth a share)
    while (w.head_split < group && (group % w.head_split != 0 || tiles * a.kv_heads * w.head_split < kItems)) ++w.head_split;
    w.key_chunk = a.short_tiles > 0 ? 0x3fffffff : std::min<int64_t>(w.chunk * finer, 0x3fffffff);  // (whole tiles are not cut)
    w.max_key_chunks = most(a.most_rounds * finer * (group / w.head_split), w.key_chunk, key_bytes * w.head_split);
    take(a.n_tokens * a.heads * 4);  // lse2
    w.delta = take(a.n_tokens * a.heads * 4);
    if (a.dtype == ND_F16 && a.short_tiles == 0) w.gradient_tops = take(kTopParts * 4);
  }
  w.chunk = std::min<int64_t>(w.chunk, 0x3fffffff);
  if (w.max_chunks > 1) w.row_sums = take(w.max_chunks * row_bytes);
  if (w.max_chunks > 1 && !backward) w.row_tops = take(w.max_chunks * a.n_tokens * a.heads * (int64_t)sizeof(float2));
  if (w.max_key_chunks * w.head_split > 1) {
    w.dk_sums = take(w.max_key_chunks * w.head_split * key_bytes);
    w.dv_sums = take(w.max_key_chunks * w.head_split * key_bytes);
  }
  return w;
}

template <class T, int NB>
void launch_forward(const AttentionParams& p, hipStream_t stream) {
  const uint32_t tiles = p.plan.short_tiles > 0 ? p.plan.short_tiles : p.plan.tiles;
  attention_forward_kernel<T, NB><<<tiles * p.heads * p.max_chunks, 256, 0, stream>>>(p);
  if (p.max_chunks > 1) {
    const int64_t n = (int64_t)p.plan.tokens * p.heads * p.dim;
    attention_join_kernel<T><<<(uint32_t)((n / 4 + 255) / 256), 256, 0, stream>>>(p, n);
  }
}
template <class T, int NB>
void launch_backward(const AttentionParams& p, hipStream_t stream) {
  if (p.plan.short_tiles > 0) {
    attention_backward_short_kernel<T, NB><<<(uint32_t)p.plan.short_tiles * p.kv_heads * p.head_split, 256, 0, stream>>>(p);
  } else {
    if (std::is_same<T, _Float16>::value) attention_top_kernel<<<kTopParts, 1024, 0, stream>>>(p);
    attention_backward_query_kernel<T, NB><<<(uint32_t)p.plan.tiles * p.heads * p.max_chunks, 256, 0, stream>>>(p);
    attention_backward_key_kernel<T, NB><<<(uint32_t)p.plan.tiles * p.kv_heads * p.head_split * p.max_key_chunks, 256, 0, stream>>>(p);
  }
  const bool add_keys = p.max_key_chunks * p.head_split > 1;
  if (p.max_chunks > 1 || add_keys) {
    const int64_t n_rows = (int64_t)p.plan.tokens * p.heads * p.dim, n_keys = (int64_t)p.plan.tokens * p.kv_heads * p.dim;
    const int64_t n = p.max_chunks > 1 ? n_rows : n_keys;
    attention_add_kernel<T><<<dim3((uint32_t)((n / 4 + 255) / 256), add_keys ? 3 : 1), 256, 0, stream>>>(
        p, n_rows, n_keys, (int)key_round_of(p.dim));
  }
}

template <class T>
void launch(const AttentionParams& p, bool backward, hipStream_t stream) {
  switch ((p.dim + 31) / 32) {
    case 1: backward ? launch_backward<T, 1>(p, stream) : launch_forward<T, 1>(p, stream); break;
    case 2: backward ? launch_backward<T, 2>(p, stream) : launch_forward<T, 2>(p, stream); break;
    case 3: backward ? launch_backward<T, 3>(p, stream) : launch_forward<T, 3>(p, stream); break;
    default: backward ? launch_backward<T, 4>(p, stream) : launch_forward<T, 4>(p, stream); break;
  }
}

int check_attention(const nd_packed_attention* a, bool backward) {
  if (!a) return fail("packed attention: null argument");
  if (a->dtype != ND_F16 && a->dtype != ND_BF16) return fail("packed attention: 16-bit types only (ND_F16, ND_BF16)");
  if (a->n_tokens < 0 || a->n_tokens > ND_PACKED_MAX_TOKENS)
    return fail("packed attention: between 0 and " + std::to_string((int64_t)ND_PACKED_MAX_TOKENS) + " tokens, " +
                std::to_string(a->n_tokens) + " given");
  if (a->n_covered < 0 || a->n_covered > a->n_tokens) return fail("packed attention: more tokens in sequences than tokens");
  if (a->heads < 1 || a->kv_heads < 1 || a->heads % a->kv_heads != 0 || a->heads > 65535)
    return fail("packed attention: " + std::to_string(a->heads) + " heads do not share " + std::to_string(a->kv_heads) +
                " key heads evenly");
  if (a->dim < 8 || a->dim > ND_PACKED_MAX_DIM || a->dim % 8 != 0)
    return fail("packed attention: the head size is a multiple of 8 up to " + std::to_string(ND_PACKED_MAX_DIM) + ", " +
                std::to_string(a->dim) + " given");
  if (!isfinite(a->scale)) return fail("packed attention: the scale is not finite");
  if (a->n_tokens == 0) return 0;
  if (a->rounds < 0 || a->most_rounds < 0 || a->most_rounds > a->n_tokens / kColumns + 2 || a->short_tiles < 0 ||
      a->short_tiles > 2 * tiles_of(a->n_tokens) + 3)
    return fail("packed attention: a size that no plan of these tokens has");
  const void* in[] = {a->q, a->k, a->v, a->out, a->lse, a->plan, a->dout, a->dq, a->dk, a->dv};
  for (int i = 0; i < (backward ? 10 : 6); ++i) {
    if (!in[i]) return fail("packed attention: null array");
    if ((uintptr_t)in[i] & 15) return fail("packed attention: arrays are aligned to 16 bytes");
  }
  const int64_t strides[] = {a->q_token, a->q_head, a->k_token, a->k_head, a->v_token, a->v_head, a->dout_token, a->dout_head};
  for (int i = 0; i < (backward ? 8 : 6); ++i)
    if (strides[i] < 0 || strides[i] % 8 != 0 || (i % 2 == 0 && strides[i] > ND_PACKED_MAX_TOKEN_STRIDE))
      return fail("packed attention: strides are multiples of 8 elements, a token's at most " +
                  std::to_string(ND_PACKED_MAX_TOKEN_STRIDE));
  const Cuts cuts = cuts_of(*a, backward);
  if (std::max(a->short_tiles, tiles_of(a->n_tokens)) * a->heads * std::max(cuts.max_chunks, cuts.max_key_chunks) > 0xffffff)  // (of 256 threads)
    return fail("packed attention: more tokens and heads than one launch holds");
  if (a->workspace_bytes < cuts.bytes)
    return fail("packed attention: the workspace has " + std::to_string(a->workspace_bytes) + " bytes, " + std::to_string(cuts.bytes) +
                " needed");
  if (cuts.bytes > 0 && (!a->workspace || ((uintptr_t)a->workspace & 15)))
    return fail("packed attention: null workspace, or one not aligned to 16 bytes");
  return 0;
}

int run_attention(const nd_packed_attention* a, bool backward, void* stream) {
  const int rc = check_attention(a, backward);
  if (rc != 0 || a->n_tokens == 0) return rc;
  AttentionParams p = {};
  const PlanParts parts = plan_parts(a->n_tokens);
  p.plan.first = (const int32_t*)a->plan;
  p.plan.last = p.plan.first + parts.last;
  p.plan.query_order = p.plan.first + parts.query_order;
  p.plan.key_order = p.plan.first + parts.key_order;
  p.plan.short_starts = p.plan.first + parts.short_starts;
  p.plan.short_tiles = (int32_t)a->short_tiles;
  p.plan.tokens = (int32_t)a->n_tokens;
  p.plan.covered = (int32_t)a->n_covered;
  p.plan.tiles = (int32_t)tiles_of(a->n_tokens);
  p.q = a->q;
  p.k = a->k;
  p.v = a->v;
  p.out = p.out_w = a->out;
  p.dout = a->dout;
  p.dq = a->dq;
  p.dk = a->dk;
  p.dv = a->dv;
  p.lse = a->lse;
  const Cuts w = cuts_of(*a, backward);
  char* work = (char*)a->workspace;
  p.lse2 = (float*)work;
  p.delta = (float*)(work + w.delta);
  p.row_sums = (float*)(work + w.row_sums);
  p.row_tops = (float2*)(work + w.row_tops);
  p.gradient_tops = (uint32_t*)(work + w.gradient_tops);
  p.dk_sums = (float*)(work + w.dk_sums);
  p.dv_sums = (float*)(work + w.dv_sums);
  p.chunk = (int32_t)w.chunk;
  p.max_chunks = (int32_t)w.max_chunks;
  p.key_chunk = (int32_t)w.key_chunk;
  p.max_key_chunks = (int32_t)w.max_key_chunks;
  p.head_split = (int32_t)w.head_split;
  p.q_token = a->q_token * 2;
  p.q_head = a->q_head * 2;
  p.k_token = a->k_token * 2;
  p.k_head = a->k_head * 2;
  p.v_token = a->v_token * 2;
  p.v_head = a->v_head * 2;
  p.dout_token = a->dout_token * 2;
  p.dout_head = a->dout_head * 2;
  p.heads = a->heads;
  p.kv_heads = a->kv_heads;
  p.group = a->heads / a->kv_heads;
  p.dim = a->dim;
  p.scale = a->scale;
  // (a scale of 0 as the smallest one: -inf x 0 would be NaN where a key is masked)
  p.scale_log2 = fmaxf(fabsf(a->scale) * kLog2e, 1e-37f);
  p.flip = a->scale < 0.f ? 0x80008000u : 0u;
  if (a->dtype == ND_BF16) launch<__bf16>(p, backward, (hipStream_t)stream);
  else launch<_Float16>(p, backward, (hipStream_t)stream);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(std::string("packed attention: ") + hipGetErrorString(e));
  return 0;
}

}  // namespace
}  // namespace nd

extern "C" {

int64_t nd_packed_plan_bytes(int64_t n_tokens) {
  if (n_tokens < 0 || n_tokens > ND_PACKED_MAX_TOKENS) return -1;
  return nd::plan_parts(n_tokens).words * (int64_t)sizeof(int32_t);
}

int nd_packed_plan(const int32_t* starts, int64_t n_sequences, int64_t n_tokens, const int32_t* d_starts, void* d_plan,
                   int64_t sizes[3], void* stream) {
  return nd::guarded([&]() -> int {
    if (n_tokens < 0 || n_tokens > ND_PACKED_MAX_TOKENS || n_sequences < 0 || n_sequences > ND_PACKED_MAX_TOKENS)
      return nd::fail("packed sequences: between 0 and " + std::to_string((int64_t)ND_PACKED_MAX_TOKENS) + " tokens and sequences");
    if (!starts) return nd::fail("packed sequences: null array");
    if (starts[0] != 0) return nd::fail("packed sequences: the first one starts at token " + std::to_string(starts[0]) + ", not 0");
    for (int64_t i = 0; i < n_sequences; ++i)
      if (starts[i + 1] < starts[i])
        return nd::fail("packed sequences: sequence " + std::to_string(i) + " ends before it starts");
    if (starts[n_sequences] > n_tokens)
      return nd::fail("packed sequences: " + std::to_string(starts[n_sequences]) + " tokens in sequences, " +
                      std::to_string(n_tokens) + " tokens");
    if (!sizes) return nd::fail("packed sequences: null array");
    sizes[0] = sizes[1] = sizes[2] = 0;
    int64_t of = 0;  // the sequence that a tile's first token is in
    for (int64_t t = 0; t < starts[n_sequences]; t += nd::kRows) {
      while (starts[of + 1] <= t) ++of;
      const int64_t end = std::min<int64_t>(t + nd::kRows, starts[n_sequences]);
      const int64_t one = (end - starts[of] + nd::kColumns - 1) / nd::kColumns;
      sizes[0] += one;
      // as a tile of queries, and as one of keys (whose last token's sequence may end after it)
      const int32_t* after = std::upper_bound(starts + of + 1, starts + n_sequences + 1, (int32_t)(end - 1));
      sizes[1] = std::max(sizes[1], std::max(one, (*after - t + nd::kColumns - 1) / nd::kColumns));
    }
    // whole sequences to a tile, if none is longer
    std::vector<int32_t> cuts;
    int64_t longest = 0;
    for (int64_t i = 0; i < n_sequences; ++i) longest = std::max<int64_t>(longest, starts[i + 1] - starts[i]);
    if (longest <= nd::kRows) {
      cuts.push_back(0);
      for (int64_t i = 1; i <= n_sequences; ++i)
        if (starts[i] - cuts.back() > nd::kRows) cuts.push_back(starts[i - 1]);
      if (starts[n_sequences] > cuts.back()) cuts.push_back(starts[n_sequences]);
      while (cuts.back() < n_tokens) cuts.push_back((int32_t)std::min<int64_t>((int64_t)cuts.back() + nd::kRows, n_tokens));
      sizes[2] = (int64_t)cuts.size() - 1;
    }
    if (n_tokens == 0) return 0;
    if (!d_starts || !d_plan || ((uintptr_t)d_plan & 15)) return nd::fail("packed sequences: null or misaligned device array");
    int32_t* first = (int32_t*)d_plan;
    const nd::PlanParts parts = nd::plan_parts(n_tokens);
    nd::packed_plan_kernel<<<(uint32_t)((n_tokens + nd::kPlanThreads - 1) / nd::kPlanThreads), nd::kPlanThreads, 0,
                             (hipStream_t)stream>>>(d_starts, (int32_t)n_sequences, (int32_t)n_tokens, first, first + parts.last);
    nd::packed_order_kernel<<<2, nd::kOrderThreads, 0, (hipStream_t)stream>>>(
        first, first + parts.last, (int32_t)n_tokens, starts[n_sequences], (int32_t)nd::tiles_of(n_tokens), first + parts.query_order,
        first + parts.key_order);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && sizes[2] > 0)  // (from pageable memory: done with it when the call returns)
      e = hipMemcpyAsync(first + parts.short_starts, cuts.data(), cuts.size() * sizeof(int32_t), hipMemcpyHostToDevice,
                         (hipStream_t)stream);
    if (e != hipSuccess) return nd::fail(std::string("packed sequences: ") + hipGetErrorString(e));
    return 0;
  });
}

int64_t nd_packed_attention_workspace(const nd_packed_attention* a, int backward) {
  if (!a || a->n_tokens < 0 || a->n_tokens > ND_PACKED_MAX_TOKENS || a->rounds < 0 || a->most_rounds < 0 || a->kv_heads < 1 ||
      a->heads < a->kv_heads || a->heads % a->kv_heads != 0 || a->dim < 1 || a->dim > ND_PACKED_MAX_DIM)
    return -1;
  return nd::cuts_of(*a, backward != 0).bytes;
}

int nd_packed_attention_forward(const nd_packed_attention* a, void* stream) {
  return nd::guarded([&]() -> int { return nd::run_attention(a, false, stream); });
}

int nd_packed_attention_backward(const nd_packed_attention* a, void* stream) {
  return nd::guarded([&]() -> int { return nd::run_attention(a, true, stream); });
}

}  // extern "C"

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

#include "nd_errors.hpp"
#include "nd_matrix.hpp"

namespace nd {
namespace {

constexpr int kPlanThreads = 256;
constexpr int kQueryTile = 128;  // rows of a workgroup: four waves of 32
constexpr int kKeyTile = 64;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct PackedPlan {
  const int32_t* first;  // of the sequence a token belongs to; tokens from `covered` on belong to none
  const int32_t* last;   // one past it
  int32_t tokens, covered;
};

struct AttentionParams {
  PackedPlan plan;
  const void *q, *k, *v, *out, *dout;
  void *out_w, *dq, *dk, *dv;
  float *lse, *delta;  // [heads][tokens]
  int64_t q_token, q_head, k_token, k_head, v_token, v_head, dout_token, dout_head;  // in elements
  int32_t heads, kv_heads, group, dim;
  float scale, scale_log2;
};

__global__ __launch_bounds__(kPlanThreads) void packed_plan_kernel(const int32_t* starts, int32_t sequences,
                                                                   int32_t tokens, int32_t* first, int32_t* last) {
  const int64_t t = (int64_t)blockIdx.x * kPlanThreads + threadIdx.x;
  if (t >= tokens) return;
  // the last sequence that starts at or before t (empty ones start where the next does)
  int32_t lo = 0, hi = sequences;
  while (hi - lo > 1) {
    const int32_t mid = (lo + hi) >> 1;
    if (starts[mid] <= t) lo = mid;
    else hi = mid;
  }
  const bool in = sequences > 0 && t < starts[sequences];
  // (the bounds are those of a checked array; whatever a caller has on the device, no token outside is ever read)
  first[t] = in ? min(max(starts[lo], 0), (int32_t)t) : (int32_t)t;
  last[t] = in ? max(min(starts[lo + 1], tokens), (int32_t)t + 1) : (int32_t)t;
}

// Rows row0 .. row0 + ROWS - 1 (those below `end`) of a matrix of `dim` columns into a tile; the rest is zero.
template <int ROWS, int CHUNKS>
__device__ __forceinline__ void load_tile(u32x4* tile, const char* base, int64_t row_bytes, int row0, int end, int dim) {
  for (int i = threadIdx.x; i < ROWS * CHUNKS; i += 256) {
    const int r = i / CHUNKS, c = i % CHUNKS;
    u32x4 v = {0, 0, 0, 0};
    if (row0 + r < end && c * 8 < dim) v = *(const u32x4*)(base + (int64_t)(row0 + r) * row_bytes + c * 16);
    tile[tile_place<CHUNKS>(r, c)] = v;
  }
}

template <class T, int NB>
struct HeadTile {
  static constexpr int kChunks = NB == 1 ? 4 : NB == 2 ? 8 : 16;
  static constexpr int kSlices = 2 * NB;  // of 16 columns
};

// A wave's 32 rows as operands: lane's row, columns 16 s + 8 h .. + 7.
template <int NB>
__device__ __forceinline__ void load_rows(u32x4 (&frag)[2 * NB], const char* row, bool there, int dim, int h) {
#pragma unroll
  for (int s = 0; s < 2 * NB; ++s) {
    const int c = 2 * s + h;
    frag[s] = u32x4{0, 0, 0, 0};
    if (there && c * 8 < dim) frag[s] = *(const u32x4*)(row + c * 16);
  }
}

// Result rows = columns of a head, result column = token: four consecutive columns of the lane's token at a time.
template <class T, int NB>
__device__ __forceinline__ void store_rows(T* row, const f32x16 (&acc)[NB], float factor, int dim, int h) {
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int c = 32 * b + 8 * g + 4 * h;
      u32x2 v;
      v[0] = pack_pair<T>(acc[b][4 * g] * factor, acc[b][4 * g + 1] * factor);
      v[1] = pack_pair<T>(acc[b][4 * g + 2] * factor, acc[b][4 * g + 3] * factor);
      if (c < dim) *(u32x2*)(row + c) = v;
    }
}

// ---- forward ------------------------------------------------------------------------------------
// One workgroup: 128 query tokens of one head; one wave: 32 of them, lane's token is column l & 31 of S^T = K Q^T, so
// the softmax of a row runs over a lane's own registers and its partner's, 32 lanes away.
template <class T, int NB>
__global__ __launch_bounds__(256) void attention_forward_kernel(AttentionParams p) {
  constexpr int kChunks = HeadTile<T, NB>::kChunks;
  __shared__ u32x4 keys[kKeyTile * kChunks], values[kKeyTile * kChunks];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
  const int tile0 = (int)(gridDim.x - 1 - blockIdx.x) * kQueryTile;
  const int head = blockIdx.y, kv_head = head / p.group;
  const int row0 = tile0 + wave * 32, row = row0 + (lane & 31);
  const bool there = row < p.plan.covered;
  const int first = there ? p.plan.first[row] : row + 1;
  u32x4 qf[2 * NB];
  load_rows<NB>(qf, (const char*)p.q + ((int64_t)row * p.q_token + (int64_t)head * p.q_head) * 2, there, p.dim, h);
  f32x16 acc[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) acc[b] = f32x16{};
  float top = -INFINITY, sum = 0.f;

  if (tile0 < p.plan.covered) {
    const int end = min(tile0 + kQueryTile, p.plan.covered);
    const char* kbase = (const char*)p.k + (int64_t)kv_head * p.k_head * 2;
    const char* vbase = (const char*)p.v + (int64_t)kv_head * p.v_head * 2;
    for (int n0 = p.plan.first[tile0]; n0 < end; n0 += kKeyTile) {
      __syncthreads();
      load_tile<kKeyTile, kChunks>(keys, kbase, p.k_token * 2, n0, end, p.dim);
      load_tile<kKeyTile, kChunks>(values, vbase, p.v_token * 2, n0, end, p.dim);
      __syncthreads();
      if (n0 > row0 + 31) continue;  // (wave-uniform) every key is later than the wave's rows
      f32x16 s[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        s[t] = f32x16{};
#pragma unroll
        for (int i = 0; i < 2 * NB; ++i)
          s[t] = product_32x32x16<T>(read_operand_by_rows<kChunks>(keys, 32 * t, i, lane), qf[i], s[t]);
      }
      float m = -INFINITY;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int key = n0 + 32 * t + 8 * (i / 4) + 4 * h + i % 4;
          s[t][i] = key >= first && key <= row ? s[t][i] * p.scale_log2 : -INFINITY;
          m = fmaxf(m, s[t][i]);
        }
      m = fmaxf(pair_max(m), top);
      // a row that has seen no key yet: its top stays -inf, and exp2(-inf - 0) = 0 throughout
      const float base = m == -INFINITY ? 0.f : m;
      const float shrink = exp2_fast(top - base);
      top = m;
      float part = 0.f;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          s[t][i] = exp2_fast(s[t][i] - base);
          part += s[t][i];
        }
      sum = sum * shrink + part;
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[b][i] *= shrink;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const u32x4 pf = pack_operand<T>(s[t], j);
#pragma unroll
          for (int b = 0; b < NB; ++b)
            acc[b] = product_32x32x16<T>(read_operand_by_columns<kChunks, true>(values, 32 * t + 16 * j, 32 * b, lane), pf,
                                         acc[b]);
        }
    }
  }
  if (row >= p.plan.tokens) return;
  sum = pair_sum(sum);
  const float inverse = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;  // (NaN stays NaN)
  store_rows<T, NB>((T*)p.out_w + ((int64_t)row * p.heads + head) * p.dim, acc, inverse, p.dim, h);
  if (h == 0) p.lse[(int64_t)head * p.plan.tokens + row] = (top + log2f(sum)) * kLn2;
}

// ---- backward -----------------------------------------------------------------------------------
// dq: as the forward pass, with S^T and dP^T = V dO^T; dS^T is the second operand of dQ^T = K^T dS^T.  Leaves delta.
template <class T, int NB>
__global__ __launch_bounds__(256) void attention_backward_query_kernel(AttentionParams p) {
  constexpr int kChunks = HeadTile<T, NB>::kChunks;
  __shared__ u32x4 keys[kKeyTile * kChunks], values[kKeyTile * kChunks];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
  const int tile0 = (int)(gridDim.x - 1 - blockIdx.x) * kQueryTile;
  const int head = blockIdx.y, kv_head = head / p.group;
  const int row0 = tile0 + wave * 32, row = row0 + (lane & 31);
  const bool there = row < p.plan.covered;
  const int first = there ? p.plan.first[row] : row + 1;
  u32x4 qf[2 * NB], dof[2 * NB];
  load_rows<NB>(qf, (const char*)p.q + ((int64_t)row * p.q_token + (int64_t)head * p.q_head) * 2, there, p.dim, h);
  load_rows<NB>(dof, (const char*)p.dout + ((int64_t)row * p.dout_token + (int64_t)head * p.dout_head) * 2, there, p.dim, h);
  float delta = 0.f, lse2 = 0.f;
  {
    u32x4 of[2 * NB];
    load_rows<NB>(of, (const char*)p.out + ((int64_t)row * p.heads + head) * p.dim * 2, there, p.dim, h);
#pragma unroll
    for (int s = 0; s < 2 * NB; ++s)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        delta += unpack_low<T>(of[s][j]) * unpack_low<T>(dof[s][j]);
        delta += unpack_high<T>(of[s][j]) * unpack_high<T>(dof[s][j]);
      }
    delta = pair_sum(delta);
    if (there) {
      lse2 = p.lse[(int64_t)head * p.plan.tokens + row] * kLog2e;
      if (h == 0) p.delta[(int64_t)head * p.plan.tokens + row] = delta;
    }
  }
  f32x16 acc[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) acc[b] = f32x16{};

  if (tile0 < p.plan.covered) {
    const int end = min(tile0 + kQueryTile, p.plan.covered);
    const char* kbase = (const char*)p.k + (int64_t)kv_head * p.k_head * 2;
    const char* vbase = (const char*)p.v + (int64_t)kv_head * p.v_head * 2;
    for (int n0 = p.plan.first[tile0]; n0 < end; n0 += kKeyTile) {
      __syncthreads();
      load_tile<kKeyTile, kChunks>(keys, kbase, p.k_token * 2, n0, end, p.dim);
      load_tile<kKeyTile, kChunks>(values, vbase, p.v_token * 2, n0, end, p.dim);
      __syncthreads();
      if (n0 > row0 + 31) continue;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        f32x16 s = {}, dp = {};
#pragma unroll
        for (int i = 0; i < 2 * NB; ++i) {
          s = product_32x32x16<T>(read_operand_by_rows<kChunks>(keys, 32 * t, i, lane), qf[i], s);
          dp = product_32x32x16<T>(read_operand_by_rows<kChunks>(values, 32 * t, i, lane), dof[i], dp);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int key = n0 + 32 * t + 8 * (i / 4) + 4 * h + i % 4;
          const float weight = exp2_fast(s[i] * p.scale_log2 - lse2);
          s[i] = key >= first && key <= row ? weight * (dp[i] - delta) : 0.f;
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
  if (row < p.plan.tokens)
    store_rows<T, NB>((T*)p.dq + ((int64_t)row * p.heads + head) * p.dim, acc, p.scale, p.dim, h);
}

// dk, dv: one workgroup has 128 keys of one key head, a wave 32 of them (lane's key is a column of S = Q K^T), and goes
// over the query tiles that see them, for each head of the group in turn: no sum is shared between workgroups.
template <class T, int NB>
__global__ __launch_bounds__(256) void attention_backward_key_kernel(AttentionParams p) {
  constexpr int kChunks = HeadTile<T, NB>::kChunks;
  __shared__ u32x4 queries[kKeyTile * kChunks], douts[kKeyTile * kChunks];
  __shared__ float lse2[kKeyTile], deltas[kKeyTile];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
  const int tile0 = (int)blockIdx.x * kQueryTile, kv_head = blockIdx.y;
  const int key0 = tile0 + wave * 32, key = key0 + (lane & 31);
  const bool there = key < p.plan.covered;
  const int last = there ? p.plan.last[key] : key;
  u32x4 kf[2 * NB], vf[2 * NB];
  load_rows<NB>(kf, (const char*)p.k + ((int64_t)key * p.k_token + (int64_t)kv_head * p.k_head) * 2, there, p.dim, h);
  load_rows<NB>(vf, (const char*)p.v + ((int64_t)key * p.v_token + (int64_t)kv_head * p.v_head) * 2, there, p.dim, h);
  f32x16 dk[NB], dv[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    dk[b] = f32x16{};
    dv[b] = f32x16{};
  }
  if (tile0 < p.plan.covered) {
    const int end = p.plan.last[min(tile0 + kQueryTile, p.plan.covered) - 1];
    for (int head = kv_head * p.group; head < (kv_head + 1) * p.group; ++head) {
      const char* qbase = (const char*)p.q + (int64_t)head * p.q_head * 2;
      const char* dobase = (const char*)p.dout + (int64_t)head * p.dout_head * 2;
      for (int m0 = tile0; m0 < end; m0 += kKeyTile) {
        __syncthreads();
        load_tile<kKeyTile, kChunks>(queries, qbase, p.q_token * 2, m0, end, p.dim);
        load_tile<kKeyTile, kChunks>(douts, dobase, p.dout_token * 2, m0, end, p.dim);
        if (threadIdx.x < kKeyTile) {
          const int64_t at = (int64_t)head * p.plan.tokens + m0 + threadIdx.x;
          const bool in = m0 + (int)threadIdx.x < end;
          lse2[threadIdx.x] = in ? p.lse[at] * kLog2e : 0.f;
          deltas[threadIdx.x] = in ? p.delta[at] : 0.f;
        }
        __syncthreads();
        if (m0 + kKeyTile <= key0) continue;  // every query is earlier than the wave's keys
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          f32x16 s = {}, dp = {};
#pragma unroll
          for (int i = 0; i < 2 * NB; ++i) {
            s = product_32x32x16<T>(read_operand_by_rows<kChunks>(queries, 32 * t, i, lane), kf[i], s);
            dp = product_32x32x16<T>(read_operand_by_rows<kChunks>(douts, 32 * t, i, lane), vf[i], dp);
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int at = 32 * t + 8 * (i / 4) + 4 * h + i % 4, query = m0 + at;
            const bool sees = query >= key && query < last;
            const float weight = sees ? exp2_fast(s[i] * p.scale_log2 - lse2[at]) : 0.f;
            dp[i] = sees ? weight * (dp[i] - deltas[at]) : 0.f;
            s[i] = weight;
          }
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
    }
  }
  if (key < p.plan.tokens) {
    const int64_t at = ((int64_t)key * p.kv_heads + kv_head) * p.dim;
    store_rows<T, NB>((T*)p.dk + at, dk, p.scale, p.dim, h);
    store_rows<T, NB>((T*)p.dv + at, dv, 1.f, p.dim, h);
  }
}

// ---- host ---------------------------------------------------------------------------------------

template <class T, int NB>
void launch_forward(const AttentionParams& p, hipStream_t stream) {
  const dim3 grid((p.plan.tokens + kQueryTile - 1) / kQueryTile, p.heads);
  attention_forward_kernel<T, NB><<<grid, 256, 0, stream>>>(p);
}
template <class T, int NB>
void launch_backward(const AttentionParams& p, hipStream_t stream) {
  const int tiles = (p.plan.tokens + kQueryTile - 1) / kQueryTile;
  attention_backward_query_kernel<T, NB><<<dim3(tiles, p.heads), 256, 0, stream>>>(p);
  attention_backward_key_kernel<T, NB><<<dim3(tiles, p.kv_heads), 256, 0, stream>>>(p);
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
  const void* in[] = {a->q, a->k, a->v, a->out, a->lse, a->plan, a->dout, a->dq, a->dk, a->dv, a->delta};
  for (int i = 0; i < (backward ? 11 : 6); ++i) {
    if (!in[i]) return fail("packed attention: null array");
    if ((uintptr_t)in[i] & 15) return fail("packed attention: arrays are aligned to 16 bytes");
  }
  const int64_t strides[] = {a->q_token, a->q_head, a->k_token, a->k_head, a->v_token, a->v_head, a->dout_token, a->dout_head};
  for (int i = 0; i < (backward ? 8 : 6); ++i)
    if (strides[i] < 0 || strides[i] % 8 != 0) return fail("packed attention: strides are multiples of 8 elements");
  return 0;
}

int run_attention(const nd_packed_attention* a, bool backward, void* stream) {
  const int rc = check_attention(a, backward);
  if (rc != 0 || a->n_tokens == 0) return rc;
  AttentionParams p;
  p.plan.first = (const int32_t*)a->plan;
  p.plan.last = p.plan.first + (a->n_tokens + 3) / 4 * 4;
  p.plan.tokens = (int32_t)a->n_tokens;
  p.plan.covered = (int32_t)a->n_covered;
  p.q = a->q;
  p.k = a->k;
  p.v = a->v;
  p.out = p.out_w = a->out;
  p.dout = a->dout;
  p.dq = a->dq;
  p.dk = a->dk;
  p.dv = a->dv;
  p.lse = a->lse;
  p.delta = a->delta;
  p.q_token = a->q_token;
  p.q_head = a->q_head;
  p.k_token = a->k_token;
  p.k_head = a->k_head;
  p.v_token = a->v_token;
  p.v_head = a->v_head;
  p.dout_token = a->dout_token;
  p.dout_head = a->dout_head;
  p.heads = a->heads;
  p.kv_heads = a->kv_heads;
  p.group = a->heads / a->kv_heads;
  p.dim = a->dim;
  p.scale = a->scale;
  p.scale_log2 = a->scale * kLog2e;
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
  return 2 * ((n_tokens + 3) / 4 * 4) * (int64_t)sizeof(int32_t);
}

int nd_packed_plan(const int32_t* starts, int64_t n_sequences, int64_t n_tokens, const int32_t* d_starts, void* d_plan,
                   void* stream) {
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
    if (n_tokens == 0) return 0;
    if (!d_starts || !d_plan || ((uintptr_t)d_plan & 15)) return nd::fail("packed sequences: null or misaligned device array");
    int32_t* first = (int32_t*)d_plan;
    nd::packed_plan_kernel<<<(uint32_t)((n_tokens + nd::kPlanThreads - 1) / nd::kPlanThreads), nd::kPlanThreads, 0,
                             (hipStream_t)stream>>>(d_starts, (int32_t)n_sequences, (int32_t)n_tokens, first,
                                                    first + (n_tokens + 3) / 4 * 4);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return nd::fail(std::string("packed sequences: ") + hipGetErrorString(e));
    return 0;
  });
}

int nd_packed_attention_forward(const nd_packed_attention* a, void* stream) {
  return nd::guarded([&]() -> int { return nd::run_attention(a, false, stream); });
}

int nd_packed_attention_backward(const nd_packed_attention* a, void* stream) {
  return nd::guarded([&]() -> int { return nd::run_attention(a, true, stream); });
}

}  // extern "C"

// The kernels of nd_linear.hpp and the two that go with them, for one type of values.
#pragma once

#include "nd_linear.hpp"

namespace nd {

// ---- few rows: the weights are what there is to read -----------------------------------------------------------

__device__ __forceinline__ f32x4 product_16x16x32(u32x4 a, u32x4 b, f32x4 c, __bf16) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 product_16x16x32(u32x4 a, u32x4 b, f32x4 c, _Float16) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// A workgroup makes 16 columns of C (gated: 16 pairs) for up to 16 ROW_BLOCKS rows.  Its waves share out the sum, 64 places at a
// time, and read the weights straight to registers: lane l has row l & 15, places 8 (l >> 4) .. + 7 of 32, so two products use
// whole lines of 128 bytes.  x is the same for all workgroups and comes from the caches.  Bound by the latency of one chain: launch,
// weights, the waves' sums, what is added (1 x 1024 -> 4096: 8.4 MB in 4.2 us, 2.7 being what the smallest kernel takes; 16 x 1024 ->
// 2 x 2816: 11.5 MB in 6.0).
template <class T, int ROW_BLOCKS, After AFTER, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void few_rows_kernel(LinearParams a) {
  constexpr int kSides = AFTER == After::kGated ? 2 : 1, kAhead = ROW_BLOCKS == 1 && kSides == 1 ? 8 : 4;  // slices asked for at once
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), column0 = blockIdx.x * 16;
  __shared__ float part[WAVES][kSides * ROW_BLOCKS][16][17];
  f32x4 sum[kSides][ROW_BLOCKS];
#pragma unroll
  for (int s = 0; s < kSides; ++s)
#pragma unroll
    for (int b = 0; b < ROW_BLOCKS; ++b) sum[s][b] = f32x4{0.f, 0.f, 0.f, 0.f};
  const char *weight[kSides], *row[ROW_BLOCKS];
  const int own = (lane >> 4) * 16;  // bytes into 64 of a row
#pragma unroll
  for (int s = 0; s < kSides; ++s) weight[s] = (const char*)a.p + (int64_t)(s * a.n + min(column0 + (lane & 15), a.n - 1)) * a.p_bytes + own;
#pragma unroll
  for (int b = 0; b < ROW_BLOCKS; ++b) row[b] = (const char*)a.q + (int64_t)min(16 * b + (lane & 15), a.m - 1) * a.q_bytes + own;
  const int bytes = a.k * 2;
  // slices of 32 places: wave w has pairs of them w, w + WAVES, ...
  auto get = [&](const char* from, int at) {
    u32x4 v = {0, 0, 0, 0};
    if (at + own < bytes) v = *(const u32x4*)(from + at);
    return v;
  };
  for (int base = wave * 128; base < bytes; base += 128 * WAVES * (kAhead / 2)) {
    u32x4 w[kAhead][kSides], x[kAhead][ROW_BLOCKS];
#pragma unroll
    for (int t = 0; t < kAhead; ++t) {
      const int at = base + (t / 2) * 128 * WAVES + (t & 1) * 64;
#pragma unroll
      for (int s = 0; s < kSides; ++s) w[t][s] = get(weight[s], at);
#pragma unroll
      for (int b = 0; b < ROW_BLOCKS; ++b) x[t][b] = get(row[b], at);
    }
#pragma unroll
    for (int t = 0; t < kAhead; ++t)
#pragma unroll
      for (int s = 0; s < kSides; ++s)
#pragma unroll
        for (int b = 0; b < ROW_BLOCKS; ++b) sum[s][b] = product_16x16x32(w[t][s], x[t][b], sum[s][b], T());
  }
  // lane: row l & 15, columns 4 (l >> 4) .. + 3
#pragma unroll
  for (int s = 0; s < kSides; ++s)
#pragma unroll
    for (int b = 0; b < ROW_BLOCKS; ++b)
#pragma unroll
      for (int e = 0; e < 4; ++e) part[wave][s * ROW_BLOCKS + b][lane & 15][4 * (lane >> 4) + e] = sum[s][b][e];
  __syncthreads();
  // the waves' sums, one value to a lane; then eight columns of a row
  for (int t = threadIdx.x; t < 256 * kSides * ROW_BLOCKS; t += 64 * WAVES) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) v += part[w][t >> 8][(t >> 4) & 15][t & 15];
    part[0][t >> 8][(t >> 4) & 15][t & 15] = v;  // (read by this lane only)
  }
  __syncthreads();
  for (int t = threadIdx.x; t < 32 * ROW_BLOCKS; t += 64 * WAVES) {
    const int r = t >> 1, c = (t & 1) * 8;
    if (r >= a.m || column0 + c >= a.n) continue;
    float v[8], u[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] = part[0][r >> 4][r & 15][c + e];
      if (kSides == 2) u[e] = part[0][ROW_BLOCKS * (kSides - 1) + (r >> 4)][r & 15][c + e];
    }
    finish<T, AFTER>(a, r, column0 + c, v, u);
  }
}

constexpr int kLongSum = 2048;  // places from which on a sum has 16 waves: one turn of loads to each

template <class T, After AFTER>
hipError_t launch_few_rows_of(const LinearParams& a, hipStream_t stream) {
  const dim3 grid((a.n + 15) / 16);
  if (a.m <= 16) {
    if (a.k >= kLongSum) few_rows_kernel<T, 1, AFTER, 16><<<grid, 1024, 0, stream>>>(a);
    else few_rows_kernel<T, 1, AFTER, 8><<<grid, 512, 0, stream>>>(a);
  } else if (a.m <= 32) {
    few_rows_kernel<T, 2, AFTER, 8><<<grid, 512, 0, stream>>>(a);
  } else {
    few_rows_kernel<T, 4, AFTER, 8><<<grid, 512, 0, stream>>>(a);
  }
  return hipGetLastError();
}
template <class T>
hipError_t launch_few_rows(const LinearParams& a, After after, hipStream_t stream) {
  return after == After::kGated ? launch_few_rows_of<T, After::kGated>(a, stream) : launch_few_rows_of<T, After::kForward>(a, stream);
}

// ---- dz = dy a'(z) of a linear map, and the sums of the rows of dz ------------------------------------------------

// Workgroups of 64 columns, 8 lanes of 8 values, 32 rows at a time.  Bound by memory: 8192 x 4096, 200 MB: 43 us, 4.7 TB/s, and
// 47 behind a forward pass.
template <class T>
__global__ __launch_bounds__(256) void slope_kernel(LinearParams a, const void* dout, int64_t dout_bytes, float* sums, T* total_out, int64_t rows_per_share, float* parts) {
  __shared__ float part[32][kSlopeColumns + 4];
  const int c = blockIdx.x * kSlopeColumns + (threadIdx.x & 7) * 8, r0 = threadIdx.x >> 3;
  float total[8], most = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) total[i] = 0.f;
  const float factor = a.parts ? scale_of_slopes(a.parts, a.n_parts, threadIdx.x & 63) : 1.f;
  if (a.parts && blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *a.unscale = 1.f / factor;
  static_assert(kExponents == 256, "a word to a thread");
  if (a.found && blockIdx.x == 0 && blockIdx.y == 0) a.found[threadIdx.x] = 0;
  if (c < a.n) {
    const int64_t begin = blockIdx.y * rows_per_share, end = min(begin + rows_per_share, (int64_t)a.m);
#pragma unroll 4
    for (int64_t row = begin + r0; row < end; row += 32) {
      u32x4 w = *(const u32x4*)((const char*)dout + row * dout_bytes + (int64_t)c * 2);
      float d[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        d[2 * i] = unpack_low<T>(w[i]);
        d[2 * i + 1] = unpack_high<T>(w[i]);
      }
      if (parts) {
#pragma unroll
        for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(d[i]) < INFINITY ? fabsf(d[i]) : 0.f);
      }
      if (a.z) {
        // (the sums are of dz as it is, not as it is held)
        const u32x4 wz = *(const u32x4*)((const char*)a.z + (row * a.n + c) * 2);
        float z[8], s[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          z[2 * i] = unpack_low<T>(wz[i]);
          z[2 * i + 1] = unpack_high<T>(wz[i]);
        }
        activate_with_slope(a.activation, z, s);
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] *= s[i];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = pack_pair<T>(d[2 * i] * factor, d[2 * i + 1] * factor);
        *(u32x4*)((char*)a.out + (row * a.n + c) * 2) = w;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) total[i] += d[i];
    }
  }
  if (parts) {
    __shared__ float largest[4];
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) most = fmaxf(most, __shfl_xor(most, d));
    if ((threadIdx.x & 63) == 0) largest[threadIdx.x >> 6] = most;
    __syncthreads();
    if (threadIdx.x == 0) parts[blockIdx.y * gridDim.x + blockIdx.x] = fmaxf(fmaxf(largest[0], largest[1]), fmaxf(largest[2], largest[3]));
  }
  if (!sums && !total_out) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) part[r0][(threadIdx.x & 7) * 8 + i] = total[i];
  __syncthreads();
  const int column = blockIdx.x * kSlopeColumns + threadIdx.x;
  if (threadIdx.x < kSlopeColumns && column < a.n) {
    float sum = 0.f;
#pragma unroll
    for (int r = 0; r < 32; ++r) sum += part[r][threadIdx.x];
    if (total_out) total_out[column] = (T)sum;
    else sums[(int64_t)blockIdx.y * a.n + column] = sum;
  }
}

template <class T>
hipError_t launch_slope(const LinearParams& a, const void* dout, int64_t dout_bytes, float* sums, void* total, int64_t shares, float* parts, hipStream_t stream) {
  const int64_t rows_per_share = (a.m + shares - 1) / shares;
  slope_kernel<T><<<dim3((a.n + kSlopeColumns - 1) / kSlopeColumns, (uint32_t)shares), 256, 0, stream>>>(a, dout, dout_bytes, sums, (T*)total, rows_per_share, parts);
  return hipGetLastError();
}

// ---- tiles ----------------------------------------------------------------------------------------------------

template <class S>
Tiles tiles_of(const LinearParams& a, int columns = S::kTileM) {
  return {(a.m + S::kTileN - 1) / S::kTileN, (a.n + columns - 1) / columns};
}
template <class S>
bool too_many(int64_t blocks) {  // for one launch
  return blocks * S::kThreads >> 32;
}

template <class T, class S, Layout LAYOUT, After AFTER>
hipError_t launch_tiles(const LinearParams& a, hipStream_t stream) {
  const Tiles t = tiles_of<S>(a, AFTER == After::kGated ? S::kTileM / 2 : S::kTileM);
  const int64_t blocks = (int64_t)t.m * t.n * a.shares;
  if (too_many<S>(blocks)) return hipErrorInvalidConfiguration;
  linear_kernel<T, S, LAYOUT, AFTER><<<(uint32_t)blocks, S::kThreads, 0, stream>>>(a, t);
  return hipGetLastError();
}
template <class T, Layout LAYOUT, After AFTER>
hipError_t launch_shape(const LinearParams& a, int shape, hipStream_t stream) {
  if (shape == 0) return launch_tiles<T, Large, LAYOUT, AFTER>(a, stream);
  if (shape == 1) return launch_tiles<T, Medium, LAYOUT, AFTER>(a, stream);
  if constexpr (AFTER != After::kGated && AFTER != After::kSlope) {  // (those have columns in pairs of 32)
    if (shape == 3) return launch_tiles<T, Narrow, LAYOUT, AFTER>(a, stream);
  }
  return launch_tiles<T, Small, LAYOUT, AFTER>(a, stream);
}
template <class T, After AFTER>
hipError_t launch_join(const LinearParams& a, hipStream_t stream) {
  const int64_t groups = (int64_t)a.m * (a.n / 8);
  // (64 x 256 values of 16 shares: 7.5 us with a lane to eight values, for the reads of one lane follow each other; 3.9 with eight)
  if (groups <= 1 << 14 && a.shares >= 4) linear_join_kernel<T, AFTER, 8><<<(uint32_t)((groups + 31) / 32), 256, 0, stream>>>(a);
  else linear_join_kernel<T, AFTER, 1><<<(uint32_t)((groups + 255) / 256), 256, 0, stream>>>(a);
  return hipGetLastError();
}

template <class T>
hipError_t launch_linear(const LinearParams& a, Layout layout, After after, const LinearPlan& plan, hipStream_t stream) {
  LinearParams p = a;
  if (plan.rows > 0) {
    p.m = plan.rows;
    const hipError_t e = launch_linear<T>(p, layout, after, {plan.shape, 1, plan.share}, stream);
    if (e != hipSuccess) return e;
    auto behind = [&](auto*& at, int64_t row_bytes) {
      if (at) at = (std::remove_reference_t<decltype(at)>)((uintptr_t)at + plan.rows * row_bytes);
    };
    const int64_t n_bytes = (int64_t)a.n * 2;
    behind(p.q, layout == Layout::kColumns ? 2 : a.q_bytes);
    behind(p.residual, a.residual_bytes);
    behind(p.out, n_bytes);
    behind(p.z, after == After::kGated ? 3 * n_bytes : n_bytes);
    p.m = a.m - plan.rows;
    return launch_linear<T>(p, layout, after, {plan.rest, 1, plan.share}, stream);
  }
  p.shares = plan.shares;
  p.share = plan.share;
  if (after == After::kPlain)
    return layout == Layout::kWeightColumns ? launch_shape<T, Layout::kWeightColumns, After::kPlain>(p, plan.shape, stream)
                                            : launch_shape<T, Layout::kColumns, After::kPlain>(p, plan.shape, stream);
  if (after == After::kSlope) return launch_shape<T, Layout::kWeightColumns, After::kSlope>(p, plan.shape, stream);
  if (plan.shares == 1)
    return after == After::kForward ? launch_shape<T, Layout::kRows, After::kForward>(p, plan.shape, stream)
                                    : launch_shape<T, Layout::kRows, After::kGated>(p, plan.shape, stream);
  p.n = after == After::kGated ? 2 * a.n : a.n;
  const hipError_t e = launch_shape<T, Layout::kRows, After::kSums>(p, plan.shape, stream);
  if (e != hipSuccess) return e;
  p.n = a.n;
  return after == After::kForward ? launch_join<T, After::kForward>(p, stream) : launch_join<T, After::kGated>(p, stream);
}

template <class T, class S>
hipError_t launch_again_of(const LinearParams& a, hipStream_t stream) {
  const Tiles t = tiles_of<S>(a);
  const int64_t blocks = (int64_t)t.m * t.n;
  if (too_many<S>(blocks)) return hipErrorInvalidConfiguration;
  again_kernel<T, S><<<(uint32_t)blocks, S::kThreads, 0, stream>>>(a, t);
  return hipGetLastError();
}
template <class T>
hipError_t launch_again(const LinearParams& a, const LinearPlan& plan, hipStream_t stream) {
  LinearParams p = a;
  p.shares = plan.shares;
  p.share = plan.share;
  p.again = true;
  if (plan.shape == 0) return launch_again_of<T, Large>(p, stream);
  return plan.shape == 1 ? launch_again_of<T, Medium>(p, stream) : launch_again_of<T, Small>(p, stream);
}

template <class T, class S, After FIRST>
hipError_t launch_pair_of(const LinearParams& a, const LinearParams& b, hipStream_t stream) {
  Pair p = {tiles_of<S>(a), tiles_of<S>(b)};
  const int64_t a_blocks = (int64_t)p.a_tiles.m * p.a_tiles.n * a.shares, b_blocks = (int64_t)p.b_tiles.m * p.b_tiles.n * b.shares;
  if (too_many<S>(a_blocks + b_blocks + 16)) return hipErrorInvalidConfiguration;
  p.a_blocks = (uint32_t)a_blocks;
  p.b_blocks = (uint32_t)b_blocks;
  p.a_turns = (p.a_blocks + 7) / 8;
  p.b_turns = (p.b_blocks + 7) / 8;
  p.b_first = (b.shares > 1 ? b.share : b.k) > (a.shares > 1 ? a.share : a.k);
  pair_kernel<T, S, FIRST><<<8 * (p.a_turns + p.b_turns), S::kThreads, 0, stream>>>(a, b, p);
  return hipGetLastError();
}
template <class T>
hipError_t launch_pair(const LinearParams& a, After after, const LinearPlan& a_plan, const LinearParams& b, const LinearPlan& b_plan, hipStream_t stream) {
  LinearParams p = a, q = b;
  p.shares = a_plan.shares;
  p.share = a_plan.share;
  q.shares = b_plan.shares;
  q.share = b_plan.share;
  if (after == After::kSlope)
    return a_plan.shape == 1 ? launch_pair_of<T, Medium, After::kSlope>(p, q, stream) : launch_pair_of<T, Small, After::kSlope>(p, q, stream);
  return a_plan.shape == 1 ? launch_pair_of<T, Medium, After::kPlain>(p, q, stream) : launch_pair_of<T, Small, After::kPlain>(p, q, stream);
}

template <class T>
hipError_t launch_joins(const Joins& joins, uint32_t blocks, hipStream_t stream) {
  joins_kernel<T><<<blocks, 256, 0, stream>>>(joins);
  return hipGetLastError();
}

}  // namespace nd

// Linear maps with what follows them (C entries: nd_linear_*, nd_mlp_*): what their kernels share.
//
//   linear:  z = x W^T + b,  y = a(z) + r;     dz = dy a'(z),  dx = dz W,  dW = dz^T x,  db = sum of the rows of dz
//   mlp:     [g, u] = x U^T + b,  h = a(g) u (gated) or a(g),  y = h D^T + d + r
//            dh = dy D,  dg = dh u a'(g),  du = dh a(g),  then as above with dz = [dg, du]
//
// Three products of the same tiles (nd_product.hpp): both operands by rows (forward), the weights by columns (gradient of x),
// both by columns (gradient of the weights).  What follows a product is done to its results before they leave the registers.
// Sums are held in 32 bits; z, h and dz, which the next product or the backward pass reads, are rounded to 16 bits once, as
// the results are; but the z of a gated part, of which g and u are both factors of dz, keeps the upper 24 bits of 32: rounded to
// bfloat16 they had brought the gradients' error from 2.4e-3 to 3.0e-3 (1.7e-3 is that of rounding them alone).  float16: dz is held
// times a power of two, so that the small gradients of a mean over many rows are not lost below 2^-14, nor large ones above 65504: see
// scale_of.  What is made of it is divided by that in 32 bits.
#pragma once

#include <algorithm>

#include "nd_activation.hpp"
#include "nd_product.hpp"

namespace nd {

enum class After { kSums, kForward, kGated, kPlain, kSlope };  // (kPlain: sums too, where there are shares)

constexpr int kExponents = 256;

struct LinearParams {
  // C [m][n], sums over k; gated: n counts pairs, and P has 2 n rows
  const void *p, *q;
  int64_t p_bytes, q_bytes;  // of a row
  int32_t m, n, k;
  int32_t activation, gated;
  const void *bias, *residual;
  int64_t residual_bytes;  // of a row
  void* out;
  void* z;  // forward: written unless null; backward: read.  [m][n]; gated: rows of 6 n bytes, see Upper24
  bool z_later;  // forward: z is written past the caches
  // float16: what dz is held times.  parts: the largest finite |dout| of workgroups, null: 1.  Who makes dz finds the scale in them and
  // leaves one over it in *unscale, with which the sums of kPlain are multiplied (null: 1).  kSlope: found
  // [kExponents], 0 before, see there; again: the scale comes from that.
  const float* parts;
  int64_t n_parts;
  float* unscale;
  uint32_t* found;
  bool again;
  // shares of the sum: share s has places s * share .. and leaves [m][n] values (gated: [m][2 n]) in 32 bits
  float* sums;
  int32_t shares, share;
  float* column_sums;  // kSlope, unless null: sums of 32 kN rows of dz, [share of the rows][columns of dz]
};

// Rows of z of a gated part: the upper 16 bits of g (n of them), of u, and of every 8 places 16 bytes with the next 8 bits: four
// of g, four of u, and of the other four places the same.
struct Upper24 {
  static __device__ __forceinline__ u32x2 upper(const float* v) {
    u32x2 w;
    w[0] = __builtin_amdgcn_perm(__float_as_uint(v[1]), __float_as_uint(v[0]), 0x07060302);
    w[1] = __builtin_amdgcn_perm(__float_as_uint(v[3]), __float_as_uint(v[2]), 0x07060302);
    return w;
  }
  static __device__ __forceinline__ uint32_t next(const float* v) {
    const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(v[1]), __float_as_uint(v[0]), 0x0c0c0501);
    const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(v[3]), __float_as_uint(v[2]), 0x0c0c0501);
    return __builtin_amdgcn_perm(hi, lo, 0x05040100);
  }
  static __device__ __forceinline__ void value(u32x2 upper, uint32_t next, float* v) {
    v[0] = __uint_as_float(__builtin_amdgcn_perm(upper[0], next, 0x0504000c));
    v[1] = __uint_as_float(__builtin_amdgcn_perm(upper[0], next, 0x0706010c));
    v[2] = __uint_as_float(__builtin_amdgcn_perm(upper[1], next, 0x0504020c));
    v[3] = __uint_as_float(__builtin_amdgcn_perm(upper[1], next, 0x0706030c));
  }
};

// What dz is held times, for all lanes of a wave: a power of two that takes the largest finite |dout|, of all parts, to 2^TO or more
// and below twice that; but no less than LEAST.
template <int TO>
__device__ __forceinline__ float scale_of(const float* parts, int64_t n, int lane, float least) {
  float most = 0.f;
#pragma unroll 4
  for (int64_t i = lane; i < n; i += 64) most = fmaxf(most, parts[i]);
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) most = fmaxf(most, __shfl_xor(most, d));
  if (most == 0.f) return 1.f;
  return fmaxf(least, ldexpf(1.f, TO - ilogbf(most)));
}
// dz = dout a'(z): no slope is above 1.13, so the largest dz is at most 1.13 2^15.
__device__ __forceinline__ float scale_of_slopes(const float* parts, int64_t n, int lane) { return scale_of<14>(parts, n, lane, 0.f); }
// dz of a feed-forward part is dh, a product with weights, times a slope and u: it may be any number of times dout.  The largest |dout|
// is taken to 2^9 where it is less, so that 64 times that is still held, and 2^-23 of it with all its bits.  Where the largest dz turns out
// to be above 65504, an infinity, or below 1, where smaller rows lose their last bits, dz is made again with the largest at 2^14: smaller
// rows are then off by 2^-39 of it, less than the results' own rounding where its gradients are numbers of 16 bits.
__device__ __forceinline__ float scale_of_products(const float* parts, int64_t n, int lane) { return scale_of<9>(parts, n, lane, 1.f); }
// Each wave marks the exponent of the largest finite |dz| that it would hold: a store that no other wave's can spoil.  (With an atomic
// maximum, of one word or of 64, the kernel took 2 to 12 us longer.)
__device__ __forceinline__ void mark(uint32_t* found, float most) {
  // (what is 65473 or more counts with what is 2^16 or more)
  found[__float_as_uint(__builtin_fmaf(most, 0x1p-10f, most)) >> 23] = 1;
}
// The largest of the exponents that are marked, for all lanes of a wave; as they are in a float's bits, 0 if there is none.
__device__ __forceinline__ int largest_of(const uint32_t* found, int lane) {
  int largest = 0;
#pragma unroll
  for (int i = lane; i < kExponents; i += 64) largest = found[i] ? i : largest;
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) largest = max(largest, __shfl_xor(largest, d));
  return largest;
}
__device__ __forceinline__ bool leaves_range(int exponent) { return exponent > 0 && (exponent < 127 || exponent > 127 + 15); }
// (2^48: dh, at most 2^52, stays a finite number of 32 bits before it is multiplied with a slope)
__device__ __forceinline__ float scale_again(float scale, int exponent) { return fminf(ldexpf(scale, 127 + 14 - exponent), 0x1p48f); }

// The largest |v| (NaN aside) of the first `quarters` quarters of a lane's values; what of v is finite, where there are others.
__device__ __forceinline__ float most_of(const float (&v)[16], int quarters) {
  float most = 0.f;
  if (quarters >= 4) {
#pragma unroll
    for (int e = 0; e < 16; ++e) most = fmaxf(most, fabsf(v[e]));
  } else {
#pragma unroll
    for (int e = 0; e < 12; ++e) most = fmaxf(most, e / 4 < quarters ? fabsf(v[e]) : 0.f);
  }
  return most;
}
__device__ __forceinline__ float finite_most_of(const float (&v)[16], int quarters) {
  float finite[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) finite[e] = fabsf(v[e]) < INFINITY ? v[e] : 0.f;
  return most_of(finite, quarters);
}

// z as it is kept.  float16: what is positive stays so, for that is what a relu's slope is read from (below 2^-25 it was rounded to 0: one
// in 10^8 of normal values, and with it a slope of 0 for 1).
template <class T, int N>
__device__ __forceinline__ void keep_sign(int activation, const float (&v)[N], float (&z)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) z[i] = v[i];
  if (!std::is_same_v<T, _Float16> || activation != ND_RELU) return;
#pragma unroll
  for (int i = 0; i < N; ++i) z[i] = v[i] > 0.f ? fmaxf(v[i], 0x1p-24f) : v[i];
}

// The sums of 16 values over the 32 lanes of a half: lane l has that of value l & 15.  Each step sends half of the values on.
__device__ __forceinline__ float sums_of_rows(const float (&v)[16], int lane) {
  auto other = [](float x, auto how) { return __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x), decltype(how)::value, 0xf, 0xf, true)); };
  float a[8], b[4], c[2];
#pragma unroll
  for (int i = 0; i < 8; ++i) a[i] = (lane & 8 ? v[8 + i] : v[i]) + other(lane & 8 ? v[i] : v[8 + i], std::integral_constant<int, 0x140>());  // lane 15 - l
#pragma unroll
  for (int i = 0; i < 4; ++i) b[i] = (lane & 4 ? a[4 + i] : a[i]) + other(lane & 4 ? a[i] : a[4 + i], std::integral_constant<int, 0x141>());  // 7 - l
#pragma unroll
  for (int i = 0; i < 2; ++i) c[i] = (lane & 2 ? b[2 + i] : b[i]) + other(lane & 2 ? b[i] : b[2 + i], std::integral_constant<int, 0x4e>());  // l ^ 2
  const float d = (lane & 1 ? c[1] : c[0]) + other(lane & 1 ? c[0] : c[1], std::integral_constant<int, 0xb1>());  // l ^ 1
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(d), __float_as_uint(d), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// What follows the sums v (gated: and u) of columns c .. c + 7 of a row of a forward pass.
template <class T, After AFTER>
__device__ __forceinline__ void finish(const LinearParams& a, int row, int c, float (&v)[8], float (&u)[8]) {
  auto unpack = [](const u32x4& w, float(&x)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = unpack_low<T>(w[i]);
      x[2 * i + 1] = unpack_high<T>(w[i]);
    }
  };
  auto pack = [](const float(&x)[8]) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = pack_pair<T>(x[2 * i], x[2 * i + 1]);
    return w;
  };
  auto at = [&](const void* matrix, int64_t row_bytes, int column) { return (u32x4*)((char*)matrix + row * row_bytes + (int64_t)column * 2); };
  static_assert(AFTER == After::kForward || AFTER == After::kGated, "");
  const int64_t n_bytes = (int64_t)a.n * 2;
  float x[8];
  if (a.bias) {
    unpack(*at(a.bias, 0, c), x);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += x[i];
    if (AFTER == After::kGated) {
      unpack(*at(a.bias, 0, a.n + c), x);
#pragma unroll
      for (int i = 0; i < 8; ++i) u[i] += x[i];
    }
  }
  if (AFTER == After::kForward) {
    if (a.z) {
      keep_sign<T>(a.activation, v, x);
      *at(a.z, n_bytes, c) = pack(x);
    }
    activate(a.activation, v);
    if (a.residual) {
      unpack(*at(a.residual, a.residual_bytes, c), x);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] += x[i];
    }
  } else {
    if (a.z) {
      const u32x2 g0 = Upper24::upper(v), g1 = Upper24::upper(v + 4), u0 = Upper24::upper(u), u1 = Upper24::upper(u + 4);
      *at(a.z, 3 * n_bytes, c) = u32x4{g0[0], g0[1], g1[0], g1[1]};
      *at(a.z, 3 * n_bytes, a.n + c) = u32x4{u0[0], u0[1], u1[0], u1[1]};
      *at(a.z, 3 * n_bytes, 2 * a.n + c) = u32x4{Upper24::next(v), Upper24::next(u), Upper24::next(v + 4), Upper24::next(u + 4)};
    }
    activate(a.activation, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= u[i];
  }
  *at(a.out, n_bytes, c) = pack(v);
}

// ---- a tile of C to a workgroup ---------------------------------------------------------------------------

// 256 x 256, eight waves with 4 x 2 results each, alone on a compute unit; 256 rows of C x 192 columns, which leaves fewer compute
// units without work at the end of some sizes; 128 x 128 and 64 x 64, two and three of which share a compute unit.  Turns of large
// tiles run at 1.25 to 1.37 PFLOP/s (8192 x 8192 x 8192: 785 to 807 us; the library's large product: 1.55 to 1.6 by rows), with the matrix
// cores busy 66 to 80 % of the time, LDS a third of it, at 1.5 to 1.7 GHz (the library's: 86 to 90 %, half of it, 1.66 GHz): neither power
// nor LDS is short, what the loop waits for has not been found.  What follows a tile is not hidden: all workgroups store at once (8192 x
// 1024 -> 4096: 66 us, 78 with a gelu, 85 with z too, on the same operands again and again; 76, 82 and 92 on others; 104 for the last
// between the backward passes of a training step).  Within 2 % either way: four waves with 4 x 4 results, a third stage for P, two
// stages of small tiles, other spans of the reads and loads; workgroups set apart in time: 3 to 10 % slower.
using Large = product::Shape<2, 4, 4, 2, 64, 2, 1, 4, 16, 2>;
using Narrow = product::Shape<2, 4, 3, 2, 64, 2, 1, 4, 12, 2>;
using Medium = product::Shape<2, 2, 2, 2, 64, 2, 2, 4, 8, 2>;
using Small = product::Shape<1, 2, 2, 1, 64, 3, 2, 2, 4, 1>;

enum class Layout { kRows, kWeightColumns, kColumns };  // both operands by rows; P by columns; both by columns

// Chunks of LDS of a wave.  (What follows a product wants room for its results: two regions, and five of 64 columns where a slope
// is read.)
template <class S, After AFTER>
constexpr int kWaveChunks = std::max(S::kTileChunks / (S::kThreads / 64), AFTER == After::kSlope ? 5 * product::Region<8>::kSize : S::kWaveResults);

// Tile `block` of C, of share 0, then of share 1 and so on.  tiles: kWaveChunks for each wave.
template <class T, class S, Layout LAYOUT, After AFTER>
__device__ __forceinline__ void make_tile(const LinearParams& a, uint32_t block, int m_tiles, int n_tiles, u32x4* tiles) {
  constexpr bool kGated = AFTER == After::kGated;
  constexpr int kColumns = kGated ? S::kTileM / 2 : S::kTileM;  // of C to a tile
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  // Bands of eight tiles of rows, in a band column after column: the tiles that a die works on at a time (32 or more) share few rows
  // of both operands.
  const int per_share = m_tiles * n_tiles, share = uniform(block / per_share);
  block -= share * per_share;
  const int band = uniform(block / (8 * n_tiles)), in_band = block - band * 8 * n_tiles, width = min(8, m_tiles - band * 8);
  const int column0 = uniform(in_band / width) * kColumns, row0 = (band * 8 + uniform(in_band % width)) * S::kTileN;
  const int place0 = share * a.share, place_end = share + 1 < a.shares ? place0 + a.share : a.k;
  f32x16 acc[S::kM][S::kN];
  if constexpr (LAYOUT == Layout::kRows) {
    using P = product::ByRows<S::kTileM, S::kDepth, S::kThreads, kGated>;
    using Q = product::ByRows<S::kTileN, S::kDepth, S::kThreads>;
    product::multiply<T, S>(acc, P(a.p, a.p_bytes, column0, a.n, place_end, a.n * a.p_bytes), Q(a.q, a.q_bytes, row0, a.m, place_end), place0, place_end, tiles);
  } else if constexpr (LAYOUT == Layout::kWeightColumns) {
    using P = product::ByColumns<S::kTileM, S::kDepth, S::kThreads>;
    using Q = product::ByRows<S::kTileN, S::kDepth, S::kThreads>;
    product::multiply<T, S>(acc, P(a.p, a.p_bytes, column0, a.n, place_end), Q(a.q, a.q_bytes, row0, a.m, place_end), place0, place_end, tiles);
  } else {
    using P = product::ByColumns<S::kTileM, S::kDepth, S::kThreads>;
    using Q = product::ByColumns<S::kTileN, S::kDepth, S::kThreads>;
    product::multiply<T, S>(acc, P(a.p, a.p_bytes, column0, a.n, place_end), Q(a.q, a.q_bytes, row0, a.m, place_end), place0, place_end, tiles);
  }
  product::meet();
  // ---- the results: wave's rows from wave_row0 on, columns from wave_column0 on
  constexpr int kRoom = kWaveChunks<S, AFTER>;
  u32x4* mine = tiles + wave * kRoom;
  const int wave_row0 = row0 + wave % S::kWavesN * 32 * S::kN, wave_column0 = column0 + wave / S::kWavesN * (kColumns / S::kWavesM);
  const int h = lane >> 5;
  const int64_t n_bytes = (int64_t)a.n * 2;
  if (AFTER == After::kSums || (AFTER == After::kPlain && a.shares > 1)) {
    // blocks of 32 columns, 128 bytes of a row
    float* sums = a.sums + (int64_t)share * a.m * a.n;
#pragma unroll
    for (int j = 0; j < S::kN; ++j)
#pragma unroll
      for (int i = 0; i < S::kM; ++i) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int r = lane & 31;
          f32x4 v;
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = acc[i][j][4 * q + e];
          *(f32x4*)(mine + r * 8 + ((2 * q + h) ^ (r & 7))) = v;
        }
        asm volatile("" ::: "memory");
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const int r = t * 8 + lane / 8, c = lane % 8, row = wave_row0 + 32 * j + r, column = wave_column0 + 32 * i + 4 * c;
          const f32x4 v = *(const f32x4*)(mine + r * 8 + (c ^ (r & 7)));
          if (row < a.m && column < a.n) *(f32x4*)(sums + (int64_t)row * a.n + column) = v;
        }
        asm volatile("" ::: "memory");
      }
    return;
  }
  // A lane has 16 values of a result: its row, columns 8 q + 4 h .. + 3 of block i in registers 4 q .. 4 q + 3.
  auto unpack = [](u32x2 w, float* v) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      v[2 * e] = unpack_low<T>(w[e]);
      v[2 * e + 1] = unpack_high<T>(w[e]);
    }
  };
  auto read = [&](const auto& region, int i, float(&v)[16]) {
#pragma unroll
    for (int q = 0; q < 4; ++q) unpack(region.piece(4 * i + q, lane), v + 4 * q);
  };
  auto write = [&](const auto& region, int i, const float(&v)[16]) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      u32x2 w;
      w[0] = pack_pair<T>(v[4 * q], v[4 * q + 1]);
      w[1] = pack_pair<T>(v[4 * q + 2], v[4 * q + 3]);
      region.piece(4 * i + q, lane) = w;
    }
  };
  // (of a block of 32 columns of C; columns past the end have no bias, and are not stored)
  struct Bias {
    u32x2 w[4];
  };
  auto bias_of = [&](int first, int past) {
    Bias b;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int column = first + 8 * q + 4 * h;
      b.w[q] = u32x2{0, 0};
      if (column < a.n) b.w[q] = *(const u32x2*)((const char*)a.bias + (int64_t)(past + column) * 2);
    }
    return b;
  };
  auto add_bias = [&](const Bias& b, float(&v)[16]) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float x[4];
      unpack(b.w[q], x);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[4 * q + e] += x[e];
    }
  };
  auto put_z = [&](const auto& region, void* to, auto... where) {
    if (a.z_later) region.template put<true>(to, where...);
    else region.put(to, where...);
  };
  auto values = [](const f32x16& c, float(&v)[16]) {
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = c[e];
  };
  if constexpr (AFTER == After::kGated) {
    using Out = product::Region<2 * S::kM>;
    const Out gates{mine}, others{mine + Out::kSize}, next{mine + 2 * Out::kSize}, products{mine + 3 * Out::kSize};
    static_assert(4 * Out::kSize <= kRoom, "");
    Bias bias[S::kM];
    if (a.bias) {
#pragma unroll
      for (int i = 0; i < S::kM; ++i) bias[i] = bias_of(wave_column0 + i / 2 * 32, i % 2 * a.n);
    }
#pragma unroll
    for (int j = 0; j < S::kN; ++j) {
      const int at = wave_row0 + 32 * j;
#pragma unroll
      for (int i = 0; i < S::kM / 2; ++i) {
        float g[16], u[16];
        values(acc[2 * i][j], g);
        values(acc[2 * i + 1][j], u);
        if (a.bias) {
          add_bias(bias[2 * i], g);
          add_bias(bias[2 * i + 1], u);
        }
        if (a.z) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            gates.piece(4 * i + q, lane) = Upper24::upper(g + 4 * q);
            others.piece(4 * i + q, lane) = Upper24::upper(u + 4 * q);
            next.piece(4 * i + q, lane) = u32x2{Upper24::next(g + 4 * q), Upper24::next(u + 4 * q)};
          }
        }
        activate(a.activation, g);
#pragma unroll
        for (int e = 0; e < 16; ++e) g[e] *= u[e];
        write(products, i, g);
      }
      if (a.z) {
        put_z(gates, a.z, 3 * n_bytes, at, a.m, wave_column0, a.n, lane);
        put_z(others, (char*)a.z + n_bytes, 3 * n_bytes, at, a.m, wave_column0, a.n, lane);
        put_z(next, (char*)a.z + 2 * n_bytes, 3 * n_bytes, at, a.m, wave_column0, a.n, lane);
      }
      products.put(a.out, n_bytes, at, a.m, wave_column0, a.n, lane);
    }
  } else if constexpr (AFTER == After::kSlope) {
    // Parts of 32 rows x 64 columns one after another: what is read of the next is on its way while one is worked on, and dz
    // goes out from where z was.
    using Part = product::Region<8>;
    constexpr int kParts = S::kM / 2 * S::kN;
    constexpr bool kHeld = std::is_same_v<T, _Float16>;
    static_assert(S::kM % 2 == 0 && 5 * Part::kSize <= kRoom, "");
    const bool slope = a.z, gated = a.gated;  // (without a z, dz is what the product gives)
    const bool whole = wave_row0 + 32 * S::kN <= a.m && wave_column0 + 32 * S::kM <= a.n;
    const int64_t z_bytes = gated ? 3 * n_bytes : n_bytes, out_bytes = gated ? 2 * n_bytes : n_bytes;
    const Part next{mine + 4 * Part::kSize};
    auto region = [&](int part, int which) { return Part{mine + ((part & 1) * 2 + which) * Part::kSize}; };
    auto row_of = [&](int part) { return wave_row0 + 32 * (part % S::kN); };
    auto column_of = [&](int part) { return wave_column0 + 64 * (part / S::kN); };
    auto bring = [&](int part) {
      if (slope) region(part, 0).bring(a.z, z_bytes, row_of(part), a.m, column_of(part), a.n, lane);
      if (gated) region(part, 1).bring((const char*)a.z + n_bytes, z_bytes, row_of(part), a.m, column_of(part), a.n, lane);
    };
    auto bring_next = [&](int part) {
      if (gated) next.bring((const char*)a.z + 2 * n_bytes, z_bytes, row_of(part), a.m, column_of(part), a.n, lane);
    };
    float factor = a.parts ? scale_of_products(a.parts, a.n_parts, lane) : 1.f, most = 0.f;
    if (kHeld && a.again) factor = scale_again(factor, largest_of(a.found, lane));
    const bool look = kHeld && a.parts && !a.again;
    if (a.parts && block == 0 && share == 0 && threadIdx.x == 0) *a.unscale = 1.f / factor;
    bring(0);
    bring_next(0);
    float own_sums[2], other_sums[2];
#pragma unroll
    for (int part = 0; part < kParts; ++part) {
      const int j = part % S::kN, first = part / S::kN * 2;
      // (behind the loads only the stores of the part before this one; all of them are there if the tile is whole)
      if (part == 0 || !whole) product::wait_for_loads<0>();
      else if (gated) product::wait_for_loads<2 * Part::kTurns>();
      else product::wait_for_loads<Part::kTurns>();
      if (part + 1 < kParts) bring(part + 1);
      const Part mine0 = region(part, 0), mine1 = region(part, 1);
      const bool counts = row_of(part) + (lane & 31) < a.m;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float v[16], x[16], s[16], u[16];
        values(acc[first + i][j], v);
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] *= factor;
        if (slope) {
          if (gated) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const u32x2 low = next.piece(4 * i + q, lane);
              Upper24::value(mine0.piece(4 * i + q, lane), low[0], x + 4 * q);
              Upper24::value(mine1.piece(4 * i + q, lane), low[1], u + 4 * q);
            }
          } else {
            read(mine0, i, x);
          }
          activate_with_slope(a.activation, x, s);
          if (gated) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              x[e] *= v[e];
              s[e] *= u[e];
            }
            write(mine1, i, x);
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) v[e] *= s[e];
        }
        if (look) {  // (rows past the end are the last one again, with its z; of 8 columns all are there or none)
          const int quarters = row_of(part) < a.m ? (a.n - column_of(part) - 32 * i) / 8 : 0;
          float here = most_of(v, quarters);
          if (gated) here = fmaxf(here, most_of(x, quarters));
          if (here == INFINITY) {
            here = finite_most_of(v, quarters);
            if (gated) here = fmaxf(here, finite_most_of(x, quarters));
          }
          most = fmaxf(most, here);
        }
        write(mine0, i, v);
        if (a.column_sums) {  // of dz before it is rounded, over the parts with these columns
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            v[e] = counts ? v[e] : 0.f;
            x[e] = counts ? x[e] : 0.f;
          }
          const float own = sums_of_rows(v, lane);
          own_sums[i] = j == 0 ? own : own_sums[i] + own;
          if (gated) {
            const float other = sums_of_rows(x, lane);
            other_sums[i] = j == 0 ? other : other_sums[i] + other;
          }
        }
      }
      if (part + 1 < kParts) bring_next(part + 1);
      mine0.put(a.out, out_bytes, row_of(part), a.m, column_of(part), a.n, lane);
      if (gated) mine1.put((char*)a.out + n_bytes, out_bytes, row_of(part), a.m, column_of(part), a.n, lane);
      if (a.column_sums && j == S::kN - 1) {
        const int64_t share_of_rows = (int64_t)(row0 / S::kTileN) * S::kWavesN + wave % S::kWavesN;
        float* sums = a.column_sums + share_of_rows * (gated ? 2 * a.n : a.n);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int column = column_of(part) + 32 * i + 8 * ((lane & 15) / 4) + 4 * h + (lane & 3);
          if (lane & 16 || column >= a.n) continue;
          sums[column] = own_sums[i];
          if (gated) sums[a.n + column] = other_sums[i];
        }
      }
    }
    if (look) {
#pragma unroll
      for (int d = 32; d > 0; d >>= 1) most = fmaxf(most, __shfl_xor(most, d));
      if (lane == 0) mark(a.found, most);
    }
  } else if constexpr (AFTER != After::kSums) {
    using Out = product::Region<4 * S::kM>;
    constexpr int kRegions = kRoom / Out::kSize;
    static_assert(kRegions >= 2 && kRegions >= S::kN, "");
    const bool residual = AFTER == After::kForward && a.residual, keep = AFTER == After::kForward && a.z;
    // Regions of rows j: what is read, and goes out again in the same place; with z one region further.  All rows are asked for
    // at once where there are regions enough.
    const int step = keep ? 2 : 1;
    const bool ahead = step * S::kN <= kRegions;
    auto bring = [&](int j) {
      if (residual) Out{mine + (ahead ? step * j : 0) * Out::kSize}.bring(a.residual, a.residual_bytes, wave_row0 + 32 * j, a.m, wave_column0, a.n, lane);
    };
    const float factor = AFTER == After::kPlain && a.unscale ? *a.unscale : 1.f;
    Bias bias[S::kM];
    if (AFTER == After::kForward && a.bias) {
#pragma unroll
      for (int i = 0; i < S::kM; ++i) bias[i] = bias_of(wave_column0 + 32 * i, 0);
    }
    if (ahead) {
#pragma unroll
      for (int j = 0; j < S::kN; ++j) bring(j);
      if (residual) product::wait_for_loads<0>();
    }
#pragma unroll
    for (int j = 0; j < S::kN; ++j) {
      const int at = wave_row0 + 32 * j;
      if (!ahead) {
        bring(j);
        if (residual) product::wait_for_loads<0>();
      }
      const Out first{mine + (ahead ? step * j : 0) * Out::kSize}, second{first.at + Out::kSize};
#pragma unroll
      for (int i = 0; i < S::kM; ++i) {
        float v[16], x[16];
        values(acc[i][j], v);
        if (AFTER == After::kForward) {
          if (a.bias) add_bias(bias[i], v);
          if (keep) {
            keep_sign<T>(a.activation, v, x);
            write(second, i, x);
          }
          activate(a.activation, v);
          if (residual) {
            read(first, i, x);
#pragma unroll
            for (int e = 0; e < 16; ++e) v[e] += x[e];
          }
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) v[e] *= factor;
        }
        write(first, i, v);
      }
      if (keep) put_z(second, a.z, n_bytes, at, a.m, wave_column0, a.n, lane);
      first.put(a.out, n_bytes, at, a.m, wave_column0, a.n, lane);
    }
  }
}

struct Tiles {
  int m, n;  // of one share
};

template <class T, class S, Layout LAYOUT, After AFTER>
__global__ __launch_bounds__(S::kThreads, S::kWavesPerSimd) void linear_kernel(LinearParams a, Tiles t) {
  __shared__ u32x4 tiles[kWaveChunks<S, AFTER> * (S::kThreads / 64)];
  make_tile<T, S, LAYOUT, AFTER>(a, block_by_die(), t.m, t.n, tiles);
}

// float16: kSlope once more where dz leaves its range, with the scale that it takes; else nothing but the launch, 4 to 5 us.
template <class T, class S>
__global__ __launch_bounds__(S::kThreads, S::kWavesPerSimd) void again_kernel(LinearParams a, Tiles t) {
  __shared__ u32x4 tiles[kWaveChunks<S, After::kSlope> * (S::kThreads / 64)];
  if (leaves_range(largest_of(a.found, threadIdx.x & 63))) make_tile<T, S, Layout::kWeightColumns, After::kSlope>(a, block_by_die(), t.m, t.n, tiles);
}

// Two products in one launch, neither of which fills the GPU: dx (or dz) and a gradient of weights; first the one whose workgroups take
// longer.  Each die (consecutive workgroups go to the eight in turn) has an eighth of either.  1021 rows, 520 -> 1000: 13 us for 9.4
// and 9.5 one after another, and a launch less.
struct Pair {
  Tiles a_tiles, b_tiles;
  uint32_t a_blocks, b_blocks, a_turns, b_turns;  // turns: blocks of one die
  bool b_first;
};
template <class T, class S, After FIRST>
__global__ __launch_bounds__(S::kThreads, S::kWavesPerSimd) void pair_kernel(LinearParams a, LinearParams b, Pair p) {
  __shared__ u32x4 tiles[std::max(kWaveChunks<S, FIRST>, kWaveChunks<S, After::kPlain>) * (S::kThreads / 64)];
  const uint32_t die = blockIdx.x % 8, turn = blockIdx.x / 8;
  const bool is_b = p.b_first ? turn < p.b_turns : turn >= p.a_turns;
  const uint32_t before = is_b == p.b_first ? 0 : is_b ? p.a_turns : p.b_turns;
  const uint32_t block = die * (is_b ? p.b_turns : p.a_turns) + turn - before;
  if (block >= (is_b ? p.b_blocks : p.a_blocks)) return;
  if (is_b) make_tile<T, S, Layout::kColumns, After::kPlain>(b, block, p.b_tiles.m, p.b_tiles.n, tiles);
  else make_tile<T, S, Layout::kWeightColumns, FIRST>(a, block, p.a_tiles.m, p.a_tiles.n, tiles);
}

// The shares' sums of a forward pass added up, and what follows: eight columns of a row to LANES lanes, which share out the shares
// where there are few rows and columns.
template <class T, After AFTER, int LANES>
__global__ __launch_bounds__(256) void linear_join_kernel(LinearParams a) {
  constexpr int kGroups = 256 / LANES, kSides = AFTER == After::kGated ? 2 : 1;
  __shared__ float part[LANES > 1 ? LANES : 1][LANES > 1 ? kGroups : 1][8 * kSides + 1];
  const int64_t groups = a.n / 8;
  const int own = threadIdx.x % kGroups, lane = threadIdx.x / kGroups;
  const int64_t at = (int64_t)blockIdx.x * kGroups + own;
  const bool there = at < groups * a.m;
  const int row = there ? (int)(at / groups) : 0, c = there ? (int)(at % groups) * 8 : 0;
  float v[8], u[8];
  auto total = [&](int column, float(&x)[8], int side) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = 0.f;
    if (there) {
      const int64_t width = kSides * (int64_t)a.n;
      const float* from = a.sums + ((int64_t)lane * a.m + row) * width + column;
#pragma unroll 4
      for (int s = lane; s < a.shares; s += LANES, from += LANES * a.m * width) {
        const f32x4 lo = *(const f32x4*)from, hi = *(const f32x4*)(from + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[i] += lo[i];
          x[4 + i] += hi[i];
        }
      }
    }
    if (LANES > 1) {
#pragma unroll
      for (int i = 0; i < 8; ++i) part[lane][own][side * 8 + i] = x[i];
    }
  };
  total(c, v, 0);
  if (AFTER == After::kGated) total(a.n + c, u, kSides - 1);
  if (LANES > 1) {
    __syncthreads();
    if (lane > 0) return;
    for (int l = 1; l < LANES; ++l)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] += part[l][own][i];
        if (kSides == 2) u[i] += part[l][own][8 * (kSides - 1) + i];
      }
  }
  if (there) finish<T, AFTER>(a, row, c, v, u);
}

// Sums of shares added up: groups * 8 values in a row, out = (the sum of sums[share][value]) * *factor.  Several such jobs in one launch,
// `lanes` lanes to eight values.
struct Join {
  const float* sums;
  void* out;
  const float* factor;  // null: 1
  int64_t groups;
  int32_t shares, lanes;
  uint32_t first_block;
};
struct Joins {
  static constexpr int kMost = 5;
  Join job[kMost];
  int n;
};
template <class T>
__global__ __launch_bounds__(256) void joins_kernel(Joins joins) {
  __shared__ float part[256][9];
  int which = 0;
  while (which + 1 < joins.n && blockIdx.x >= joins.job[which + 1].first_block) ++which;
  const Join& a = joins.job[which];
  const int here = 256 / a.lanes, own = threadIdx.x % here, lane = threadIdx.x / here;
  const int64_t at = (int64_t)(blockIdx.x - a.first_block) * here + own;
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = 0.f;
  if (at < a.groups) {
#pragma unroll 4
    for (int s = lane; s < a.shares; s += a.lanes) {
      const float* from = a.sums + (s * a.groups + at) * 8;
      const f32x4 lo = *(const f32x4*)from, hi = *(const f32x4*)(from + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] += lo[i];
        x[4 + i] += hi[i];
      }
    }
  }
  if (a.lanes > 1) {
#pragma unroll
    for (int i = 0; i < 8; ++i) part[threadIdx.x][i] = x[i];
    __syncthreads();
    if (lane > 0) return;
    for (int l = 1; l < a.lanes; ++l)
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] += part[l * here + own][i];
  }
  if (at >= a.groups) return;
  const float factor = a.factor ? *a.factor : 1.f;
  u32x4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = pack_pair<T>(x[2 * i] * factor, x[2 * i + 1] * factor);
  ((u32x4*)a.out)[at] = w;
}

// ---- launches (nd_linear_types.hpp, compiled for each type by itself) -----------------------------------------

struct LinearPlan {
  int shape;  // 0 large, 1 medium, 2 small, 3 narrow
  int shares, share;
  int rows, rest;  // with one share: if rows > 0, that many rows of C are made so, and those behind them with shape `rest`
};
// kPlain with shares: leaves sums.
template <class T>
hipError_t launch_linear(const LinearParams& a, Layout layout, After after, const LinearPlan& plan, hipStream_t stream);
// The first by columns of the weights, kPlain or kSlope, the second by columns, kPlain; of one shape, medium or small.
template <class T>
hipError_t launch_pair(const LinearParams& a, After after, const LinearPlan& a_plan, const LinearParams& b, const LinearPlan& b_plan, hipStream_t stream);
// Behind either of them, float16 only: a product of kSlope made again if it has to be.
template <class T>
hipError_t launch_again(const LinearParams& a, const LinearPlan& plan, hipStream_t stream);
template <class T>
hipError_t launch_joins(const Joins& joins, uint32_t blocks, hipStream_t stream);
template <class T>
hipError_t launch_few_rows(const LinearParams& a, After after, hipStream_t stream);
// dz = dout a'(z), held times its scale, if there is a z, and unless they are null sums of its rows (times 1; with one share
// to `total`, rounded), and the largest finite |dout| of each workgroup, with zeros in `found` unless that is null.
template <class T>
hipError_t launch_slope(const LinearParams& a, const void* dout, int64_t dout_bytes, float* sums, void* total, int64_t shares, float* parts, hipStream_t stream);
constexpr int kSlopeColumns = 64;  // of a workgroup there

constexpr int kFewRows = 64;  // at most: a kernel of its own, which reads the weights once and keeps a sum in many waves

}  // namespace nd

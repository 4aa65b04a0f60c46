// Tiles of short rows (up to 128 16-bit columns: the heads of attention, the vectors of a vocabulary) for kernels that keep
// 32 rows of one side in a wave's registers and bring the other side to LDS, 64 rows at a time, by workgroups of 256.
#pragma once

#include "nd_matrix.hpp"

namespace nd {

constexpr int kColumns = 64;  // rows of a tile (columns of the product that reads them)

// Rows of up to 32 * NB columns.
template <int NB>
struct HeadTile {
  static constexpr int kChunks = NB == 1 ? 4 : NB == 2 ? 8 : NB <= 4 ? 16 : 32;  // of a row in LDS
  static constexpr int kSize = kColumns * kChunks;                // of a tile
};

// Brings tiles of ROWS rows of one matrix of heads to LDS.  Columns past `dim` are the row's first ones again (the other operand
// is 0 there, or the result's column is not stored), rows past the last one that one again (they are masked).
template <int NB, int ROWS = kColumns>
struct TileLoader {
  static constexpr int kTurns = ROWS * HeadTile<NB>::kChunks / 256;
  static_assert(kTurns >= 1, "");
  const char* base;
  uint32_t row_bytes;
  uint32_t offset[kTurns];
  __device__ __forceinline__ TileLoader(const void* matrix, int64_t token_bytes, int64_t head_bytes, int head, int dim)
      : base((const char*)matrix + head * head_bytes), row_bytes((uint32_t)token_bytes) {
    constexpr int kChunks = HeadTile<NB>::kChunks;
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
      const int at = threadIdx.x + 256 * i, r = at / kChunks, c = (at % kChunks) ^ tile_swizzle<kChunks>(r);
      offset[i] = r * row_bytes + (c * 8 < dim ? c * 16 : 0);
    }
  }
  __device__ __forceinline__ void issue(uint32_t wave_lds, int64_t token_bytes, int row0, int end) const {
    const char* at = base + row0 * token_bytes;
    if (row0 + ROWS <= end) {
#pragma unroll
      for (int i = 0; i < kTurns; ++i) load_to_lds(at, offset[i], wave_lds + 4096 * i);
    } else {
#pragma unroll
      for (int i = 0; i < kTurns; ++i) {
        const int r = (threadIdx.x + 256 * i) / HeadTile<NB>::kChunks;
        load_to_lds(at, offset[i] - max(r - (end - 1 - row0), 0) * row_bytes, wave_lds + 4096 * i);
      }
    }
  }
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

// A wave's 32 rows x NB * 32 columns: result rows = columns of a head, result column = the lane's token.  Rounded, turned
// through the wave's part of LDS (16 x HeadTile::kChunks x 32 bytes) and stored 16 bytes a lane.
template <class T, int NB>
__device__ __forceinline__ void store_rows(T* first_row, int64_t row_elements, int rows, const f32x16 (&acc)[NB], float factor, int dim,
                                           u32x4* part) {
  constexpr int kChunks = HeadTile<NB>::kChunks;
  const int lane = threadIdx.x & 63, h = lane >> 5, r = lane & 31;
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      u32x2 v;
      v[0] = pack_pair<T>(acc[b][4 * g] * factor, acc[b][4 * g + 1] * factor);
      v[1] = pack_pair<T>(acc[b][4 * g + 2] * factor, acc[b][4 * g + 3] * factor);
      ((u32x2*)(part + tile_place<kChunks>(r, 4 * b + g)))[h] = v;
    }
  // (one wave's LDS operations are done in order)
#pragma unroll
  for (int i = 0; i < kChunks / 2; ++i) {
    const int at = lane + 64 * i, rr = at / kChunks, c = at % kChunks;
    if (c >= 4 * NB) continue;
    const u32x4 v = part[tile_place<kChunks>(rr, c)];
    if (rr < rows && c * 8 < dim) *(u32x4*)(first_row + rr * row_elements + c * 8) = v;
  }
}

// The same of the lane's token as they are, in 32 bits.
template <int NB>
__device__ __forceinline__ void store_sums(float* row, const f32x16 (&acc)[NB], float factor, int dim, int h) {
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int c = 32 * b + 8 * g + 4 * h;
      f32x4 v;
#pragma unroll
      for (int n = 0; n < 4; ++n) v[n] = acc[b][4 * g + n] * factor;
      if (c < dim) *(f32x4*)(row + c) = v;
    }
}

}  // namespace nd

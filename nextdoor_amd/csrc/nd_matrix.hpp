// Matrix-core building blocks of the training operators: 16-byte fragments, the 32x32x16 products of
// gfx950, reads of LDS tiles by rows and by columns, and the roundings to 16 bits.
//
// Layouts (wave64; l = lane, h = l >> 5):
//   operand of a 32x32x16 product: row (or column) l & 31, places 8 h .. 8 h + 7 of the 16 summed over;
//   result: column l & 31, register i holds row 8 (i / 4) + 4 h + i % 4.
// A sum does not depend on the order of its places as long as both operands agree, so the registers
// 8 s .. 8 s + 7 of a result, rounded to 16 bits, are an operand of the next product as they are: its
// places are then rows 16 s + 4 h + 0..3 and 16 s + 8 + 4 h + 0..3 (the PAIRED order below).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace nd {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

template <class T>
__device__ __forceinline__ f32x16 product_32x32x16(u32x4 a, u32x4 b, f32x16 c);
template <>
__device__ __forceinline__ f32x16 product_32x32x16<__bf16>(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x16 product_32x32x16<_Float16>(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Two values rounded to the nearest 16-bit ones (ties to even), the first in the low half.
template <class T>
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack_pair<__bf16>(float lo, float hi) {
  bf16x2 v;
  v[0] = (__bf16)lo;
  v[1] = (__bf16)hi;
  return __builtin_bit_cast(uint32_t, v);
}
template <>
__device__ __forceinline__ uint32_t pack_pair<_Float16>(float lo, float hi) {
  f16x2 v;
  v[0] = (_Float16)lo;
  v[1] = (_Float16)hi;
  return __builtin_bit_cast(uint32_t, v);
}

template <class T>
__device__ __forceinline__ float unpack_low(uint32_t pair);
template <class T>
__device__ __forceinline__ float unpack_high(uint32_t pair);
template <>
__device__ __forceinline__ float unpack_low<__bf16>(uint32_t pair) { return __uint_as_float(pair << 16); }
template <>
__device__ __forceinline__ float unpack_high<__bf16>(uint32_t pair) { return __uint_as_float(pair & 0xffff0000u); }
template <>
__device__ __forceinline__ float unpack_low<_Float16>(uint32_t pair) { return (float)__builtin_bit_cast(f16x2, pair)[0]; }
template <>
__device__ __forceinline__ float unpack_high<_Float16>(uint32_t pair) { return (float)__builtin_bit_cast(f16x2, pair)[1]; }

// Registers 8 s .. 8 s + 7 of a result as an operand in the PAIRED order.
template <class T>
__device__ __forceinline__ u32x4 pack_operand(const f32x16& c, int s) {
  u32x4 out;
#pragma unroll
  for (int j = 0; j < 4; ++j) out[j] = pack_pair<T>(c[8 * s + 2 * j], c[8 * s + 2 * j + 1]);
  return out;
}

// ---- LDS tiles ----------------------------------------------------------------------------------
// A tile is rows of CHUNKS 16-byte chunks (4, 8, 16 or 32: 64 to 512 bytes).  Chunk c of row r is kept at
// place c ^ tile_swizzle(r): sixteen consecutive rows read at one chunk (an operand by rows) and the 64 bytes of
// four consecutive rows (an operand by columns) then both lie in different banks.
template <int CHUNKS>
__device__ __forceinline__ constexpr int tile_swizzle(int r) {
  return CHUNKS >= 16  ? ((r & 3) << 2) | ((r >> 2) & 3)
         : CHUNKS == 8 ? (((r >> 1) & 1) << 2) | ((r >> 2) & 3)
                       : (r >> 2) & 3;
}
template <int CHUNKS>
__device__ __forceinline__ constexpr int tile_place(int r, int c) {
  return r * CHUNKS + (c ^ tile_swizzle<CHUNKS>(r));
}

// Operand by columns: four 16-bit values of one column from four consecutive rows.  The sixteen lanes of a group
// point at 4 rows x 16 columns (lane i: row i / 4, columns 4 (i % 4) .. + 3) and lane i gets column i.
__device__ __forceinline__ u32x2 read_columns(const void* lds) {
  typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)lds));
}

// An operand of 32 columns (from `column`, a multiple of 32, on) and 16 rows (from `row`, a multiple of 16, on) of a
// tile; lane: column l & 31.  PAIRED: the rows in the order above, else lane's rows are 8 h .. 8 h + 7.
template <int CHUNKS, bool PAIRED>
__device__ __forceinline__ u32x4 read_operand_by_columns(const u32x4* tile, int row, int column, int lane) {
  const int h = lane >> 5, at = (lane & 15) >> 2;
  const int chunk = (column >> 3) + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
  const int r0 = row + (PAIRED ? 4 * h : 8 * h) + at, r1 = r0 + (PAIRED ? 8 : 4);
  const u32x2 a = read_columns((const char*)(tile + tile_place<CHUNKS>(r0, chunk)) + (lane & 1) * 8);
  const u32x2 b = read_columns((const char*)(tile + tile_place<CHUNKS>(r1, chunk)) + (lane & 1) * 8);
  u32x4 out;
  out[0] = a[0];
  out[1] = a[1];
  out[2] = b[0];
  out[3] = b[1];
  return out;
}

// An operand of 32 rows and 16 columns (chunks 2 s and 2 s + 1); lane: row l & 31, columns 16 s + 8 h .. + 7.
template <int CHUNKS>
__device__ __forceinline__ u32x4 read_operand_by_rows(const u32x4* tile, int row, int s, int lane) {
  return tile[tile_place<CHUNKS>(row + (lane & 31), 2 * s + (lane >> 5))];
}

// ---- loads straight to LDS --------------------------------------------------------------------------
// Each lane's 16 bytes at base + offset go to `lds` + 16 * lane (an LDS address, the same for the wave).  Written as a
// statement of its own and not with the builtin: the compiler makes every read of LDS wait for all loads to LDS that it
// knows of, also those of the other half of a double buffer, which are to stay in flight.  Nothing is returned in
// registers; wait_for_loads() and a barrier stand between the load and whoever reads the tile.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // (m0 is reserved; it is set and used in here only)
__device__ __forceinline__ void load_to_lds(const char* base, uint32_t offset, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(offset), "s"(base) : "memory", "m0");
}
// The same with 4 bytes a lane.
__device__ __forceinline__ void load_words_to_lds(const char* base, uint32_t offset, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(lds), "v"(offset), "s"(base) : "memory", "m0");
}
#pragma clang diagnostic pop
// A value that is the same for the whole wave, in a scalar register (what divisions leave is not).
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ uint32_t lds_address(const void* p) {
  typedef __attribute__((address_space(3))) const void lds_void;
  return (uint32_t)(uintptr_t)(lds_void*)p;
}
// Loads and LDS writes of this wave have arrived; then all waves'.
__device__ __forceinline__ void wait_for_loads_and_others() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// The block's index such that blocks with neighbouring results run on one of the eight dies, whose L2 they share:
// consecutive workgroups go to the dies in turn.
__device__ __forceinline__ uint32_t block_by_die(uint32_t block, uint32_t n) {
  const uint32_t die = block % 8, turn = block / 8;
  return die * (n / 8) + min(die, n % 8) + turn;
}
__device__ __forceinline__ uint32_t block_by_die() { return block_by_die(blockIdx.x, gridDim.x); }

// Over the two lanes 32 apart.
__device__ __forceinline__ float pair_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float pair_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

}  // namespace nd

// Products of 16-bit matrices, C[m][n] = sum over k of P[n][k] Q[m][k]: tiles brought to LDS behind the matrix
// instructions, and tiles of results brought back through LDS so that memory sees whole lines.
//
// P is the operand whose rows are the result's columns: registers 4 q .. 4 q + 3 of a 32 x 32 result then hold four
// neighbours of a row of C.  Either operand may be kept by rows ([row][place of the sum]) or by columns ([place][row]).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "nd_matrix.hpp"

namespace nd {
namespace product {

// kWavesM x kWavesN waves, each with kM x kN results of 32 x 32 (M counts rows of P, N those of Q), kDepth places a round,
// kStages rounds' tiles in LDS.  A wave reads the operands of a slice of 16 places kAhead slices before it multiplies them, among
// the first kReadSpan products of a slice; the loads of a round are issued among the first kLoadSpan products behind the
// barrier that frees their tile.
template <int WAVES_M, int WAVES_N, int M, int N, int DEPTH, int STAGES, int AHEAD, int READ_SPAN, int LOAD_SPAN, int WAVES_PER_SIMD>
struct Shape {
  static constexpr int kAhead = AHEAD;
  static constexpr int kWavesM = WAVES_M, kWavesN = WAVES_N, kM = M, kN = N, kDepth = DEPTH, kStages = STAGES;
  static constexpr int kReadSpan = READ_SPAN, kLoadSpan = LOAD_SPAN, kWavesPerSimd = WAVES_PER_SIMD;
  static constexpr int kThreads = 64 * WAVES_M * WAVES_N;
  static constexpr int kTileM = 32 * WAVES_M * M, kTileN = 32 * WAVES_N * N;
  static constexpr int kTileChunks = STAGES * (kTileM + kTileN) * DEPTH / 8;
  static constexpr int kWaveResults = 2 * 32 * (M > 2 ? 16 : 8);  // chunks of two regions of a wave's results
  static_assert(DEPTH == 64 && AHEAD >= 1 && AHEAD <= 3 && LOAD_SPAN <= 3 * M * N && STAGES >= 2, "");
};

// ---- operands -----------------------------------------------------------------------------------------
// ROWS rows, DEPTH places of the sum a round, brought to LDS by THREADS threads: load(i) asks for one of kTurns parts of a
// round's tile.  Of a tile that is not WHOLE what lies past the last place is some value of the matrix, until clear(), by the
// thread that asked for it, makes it 0; what lies past the last row is some row.  Offsets are 32 bits wide: ROWS (or DEPTH) rows of
// a matrix lie within 4 GiB.

// [row][place].  GATED: blocks of 32 rows come in turn from the first half of the matrix and, `other_bytes` further, from the second;
// row0 and row_end count those of one half.
template <int ROWS, int DEPTH, int THREADS, bool GATED = false>
struct ByRows {
  static constexpr int kRowChunks = DEPTH / 8, kChunks = ROWS * kRowChunks, kTurns = kChunks / THREADS;
  static_assert(kChunks % THREADS == 0 && THREADS / kRowChunks % 16 == 0 && 64 / kRowChunks <= 32, "");
  const char* base;
  int64_t other_bytes;
  uint32_t offset[kTurns];
  int places, chunk;
  __device__ __forceinline__ ByRows(const void* matrix, int64_t row_bytes, int row0, int row_end, int places_, int64_t other_bytes_ = 0)
      : base((const char*)matrix + row0 * row_bytes), other_bytes(other_bytes_), places(places_) {
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
      const int at = threadIdx.x + THREADS * i, r = at / kRowChunks, c = (at % kRowChunks) ^ tile_swizzle<kRowChunks>(r);
      offset[i] = (uint32_t)(min(GATED ? (r >> 6) * 32 + (r & 31) : r, row_end - 1 - row0) * row_bytes + c * 16);
      chunk = c;  // (the same in every turn)
    }
  }
  template <bool WHOLE>
  __device__ __forceinline__ void load(int i, uint32_t wave_lds, int place0) const {
    const uint32_t past = WHOLE || place0 + chunk * 8 < places ? 0 : chunk * 16;  // (the round's first place is there)
    // (a wave's rows are of one half)
    const bool second = GATED && ((uniform(threadIdx.x >> 6) * (64 / kRowChunks) + THREADS / kRowChunks * i) & 32);
    load_to_lds(base + (int64_t)place0 * 2 + (second ? other_bytes : 0), offset[i] - past, wave_lds + THREADS * 16 * i);
  }
  __device__ __forceinline__ void clear(u32x4* tile, int place0) const {
    if (place0 + chunk * 8 < places) return;
#pragma unroll
    for (int i = 0; i < kTurns; ++i) tile[threadIdx.x + THREADS * i] = u32x4{0, 0, 0, 0};
  }
  __device__ __forceinline__ static u32x4 operand(const u32x4* tile, int row, int s, int lane) {
    return read_operand_by_rows<kRowChunks>(tile, row, s, lane);
  }
};

// [place][row]; rows end at a multiple of 8.
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
  template <bool WHOLE>
  __device__ __forceinline__ void load(int i, uint32_t wave_lds, int place0) const {
    const int past = WHOLE ? 0 : max(place0 + (int)(threadIdx.x + THREADS * i) / kRowChunks - (places - 1), 0);
    load_to_lds(base + place0 * row_bytes, offset[i] - (uint32_t)(past * row_bytes), wave_lds + THREADS * 16 * i);
  }
  __device__ __forceinline__ void clear(u32x4* tile, int place0) const {
#pragma unroll
    for (int i = 0; i < kTurns; ++i)
      if (place0 + (int)(threadIdx.x + THREADS * i) / kRowChunks >= places) tile[threadIdx.x + THREADS * i] = u32x4{0, 0, 0, 0};
  }
  __device__ __forceinline__ static u32x4 operand(const u32x4* tile, int row, int s, int lane) {
    return read_operand_by_columns<kRowChunks, false>(tile, 16 * s, row, lane);
  }
};

// ---- the product ---------------------------------------------------------------------------------------

// At most N loads of this wave are still on their way, its reads and writes of LDS are done.
template <int N>
__device__ __forceinline__ void wait_for_loads() {
  static_assert(N < 64, "");
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
}
// The same for `tiles` (at most MOST) times EACH loads.
template <int EACH, int MOST>
__device__ __forceinline__ void wait_for_tiles(int tiles) {
  if constexpr (MOST <= 0) {
    wait_for_loads<0>();
  } else {
    if (tiles >= MOST) wait_for_loads<EACH * MOST>();
    else wait_for_tiles<EACH, MOST - 1>(tiles);
  }
}
// All waves are here.
__device__ __forceinline__ void meet() {
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// acc = P Q^T over the places place0 .. place_end - 1 (place0 a multiple of kDepth; only the last round may end inside).
// One barrier a round, kAhead slices before its end: every wave has the last slices' operands in registers then, so the
// round's tile is free, and the next round's tile, asked for kStages - 1 rounds ago, has arrived.
// `tiles` has room for S::kTileChunks; the caller may use it again after meet().
template <class T, class S, class P, class Q>
__device__ __forceinline__ void multiply(f32x16 (&acc)[S::kM][S::kN], const P& p, const Q& q, int place0, int place_end, u32x4* tiles) {
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int m0 = wave / S::kWavesN * 32 * S::kM, n0 = wave % S::kWavesN * 32 * S::kN;
#pragma unroll
  for (int i = 0; i < S::kM; ++i)
#pragma unroll
    for (int j = 0; j < S::kN; ++j) acc[i][j] = f32x16{};
  constexpr int kStage = P::kChunks + Q::kChunks, kLoads = P::kTurns + Q::kTurns, kSlices = S::kDepth / 16;
  constexpr int kProducts = S::kM * S::kN, kReads = S::kM + S::kN, kSets = S::kAhead == 1 ? 2 : 4, kMeet = kSlices - S::kAhead;
  // loads issued between the barrier and the round's end; the others follow in the next round
  constexpr int kAtOnce = (kLoads * kProducts * S::kAhead + S::kLoadSpan - 1) / S::kLoadSpan, kFirst = kAtOnce < kLoads ? kAtOnce : kLoads;
  const uint32_t lds = lds_address(tiles) + wave * 1024;
  const int rounds = (place_end - place0 + S::kDepth - 1) / S::kDepth;
  if (rounds <= 0) return;
  auto load = [&](int n, int stage, int round, auto whole) {
    constexpr bool kWhole = decltype(whole)::value;
    const uint32_t at = lds + stage * kStage * 16;
    const int place = place0 + round * S::kDepth;
    if (n < P::kTurns) p.template load<kWhole>(n, at, place);
    else q.template load<kWhole>(n - P::kTurns, at + P::kChunks * 16, place);
  };
  auto load_some = [&](int first, int end, int stage, int round) {  // the last round's tile may not be whole
    if (round + 1 < rounds) {
#pragma unroll
      for (int n = 0; n < kLoads; ++n)
        if (n >= first && n < end) load(n, stage, round, std::true_type());
    } else if (round < rounds) {
#pragma unroll
      for (int n = 0; n < kLoads; ++n)
        if (n >= first && n < end) load(n, stage, round, std::false_type());
    }
  };
  // This wave's part of a tile has arrived; of the last one, what lies past the end is cleared.
  auto finish_tile = [&](int round, int stage) {
    if (round + 1 == rounds && place0 + rounds * S::kDepth > place_end) {
      p.clear(tiles + stage * kStage, place0 + round * S::kDepth);
      q.clear(tiles + stage * kStage + P::kChunks, place0 + round * S::kDepth);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
  };
#pragma unroll
  for (int t = 0; t < S::kStages; ++t) load_some(0, t == S::kStages - 1 ? kFirst : kLoads, t, t);
  u32x4 fp[kSets][S::kM], fq[kSets][S::kN];
  if (rounds >= S::kStages) wait_for_loads<(S::kStages - 2) * kLoads + kFirst>();
  else wait_for_tiles<kLoads, S::kStages - 2>(rounds - 1);
  finish_tile(0, 0);
  meet();
#pragma unroll
  for (int s = 0; s < S::kAhead; ++s) {
#pragma unroll
    for (int j = 0; j < S::kN; ++j) fq[s][j] = Q::operand(tiles + P::kChunks, n0 + 32 * j, s, lane);
#pragma unroll
    for (int i = 0; i < S::kM; ++i) fp[s][i] = P::operand(tiles, m0 + 32 * i, s, lane);
  }
  int stage = 0;
  auto round = [&](int t, auto steady) {
    constexpr bool kSteady = decltype(steady)::value;
    const int next = stage + 1 == S::kStages ? 0 : stage + 1, before = stage == 0 ? S::kStages - 1 : stage - 1;
#pragma unroll
    for (int s = 0; s < kSlices; ++s) {
      const u32x4* from = tiles + (s >= kMeet ? next : stage) * kStage;
      const int slice = (s + S::kAhead) % kSlices, with = s % kSets, into = (s + S::kAhead) % kSets;
      if (s == kMeet) {  // the next tile has arrived, those behind it are on their way
        if (kSteady) {
          wait_for_loads<(S::kStages - 2) * kLoads>();
        } else {
          wait_for_tiles<kLoads, S::kStages - 2>(min(t + S::kStages - 1, rounds - 1) - (t + 1));
          finish_tile(t + 1, next);
        }
        meet();
      }
      if (!kSteady) {
        if (s == 0) load_some(kFirst, kLoads, before, t + S::kStages - 1);
        if (s == kMeet) load_some(0, kFirst, stage, t + S::kStages);
      }
#pragma unroll
      for (int n = 0; n < kProducts; ++n) {
        acc[n / S::kN][n % S::kN] = product_32x32x16<T>(fp[with][n / S::kN], fq[with][n % S::kN], acc[n / S::kN][n % S::kN]);
#pragma unroll
        for (int r = 0; r < kReads; ++r)
          if (r * S::kReadSpan / kReads == n) {
            if (r < S::kN) fq[into][r] = Q::operand(from + P::kChunks, n0 + 32 * r, slice, lane);
            else fp[into][r - S::kN] = P::operand(from, m0 + 32 * (r - S::kN), slice, lane);
          }
        if (kSteady) {
          const int slot = ((s + S::kAhead) % kSlices) * kProducts + n;
#pragma unroll
          for (int l = 0; l < kLoads; ++l)
            if (l * S::kLoadSpan / kLoads == slot) load(l, s >= kMeet ? stage : before, t + S::kStages - (s >= kMeet ? 0 : 1), std::true_type());
        }
        __builtin_amdgcn_sched_barrier(0);  // (this order: a load or a read behind each product)
      }
    }
    stage = next;
  };
  int t = 0;
  for (; t + S::kStages + 1 < rounds; ++t) round(t, std::true_type());
  for (; t < rounds; ++t) round(t, std::false_type());
}

// ---- results through LDS -----------------------------------------------------------------------------------
// A wave's 32 rows of C by CHUNKS chunks of 8 values (16 bits) in rows of kRow places, chunk c of row r at place c ^ (r mod kRow).
// Lane l of a result has row l & 31 and, of chunk 4 i + q, the values 4 h .. 4 h + 3.  Only the wave itself uses a region.
template <int CHUNKS>
struct Region {
  static constexpr int kRow = CHUNKS <= 4 ? 4 : CHUNKS <= 8 ? 8 : 16, kSize = 32 * kRow, kTurns = kSize / 64;
  static_assert(CHUNKS <= 16, "");
  u32x4* at;
  __device__ __forceinline__ u32x2& piece(int chunk, int lane) const {
    const int r = lane & 31;
    return *((u32x2*)(at + r * kRow + (chunk ^ (r & (kRow - 1)))) + (lane >> 5));
  }
  // Rows row0 .. row0 + 31 and columns column0 .. of a matrix with rows of row_bytes, which ends at row_end and column_end (a
  // multiple of 8): past them some values of the matrix.  wait_for_loads() before they are used.
  __device__ __forceinline__ void bring(const void* matrix, int64_t row_bytes, int row0, int row_end, int column0, int column_end, int lane) const {
    if (row0 >= row_end || column0 >= column_end) return;
    const char* base = (const char*)matrix + row0 * row_bytes + (int64_t)column0 * 2;
    const uint32_t lds = uniform((int)lds_address(at));
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (loads to LDS do not queue behind reads of it)
#pragma unroll
    for (int t = 0; t < kTurns; ++t) {
      const int p = t * 64 + lane, r = p / kRow, c = (p % kRow) ^ (r & (kRow - 1));
      const bool there = c < CHUNKS && column0 + c * 8 < column_end;
      load_to_lds(base, (uint32_t)(min(r, row_end - 1 - row0) * row_bytes) + (there ? c * 16 : 0), lds + t * 1024);
    }
  }
  // LATER: written past the caches, for what is read by another kernel and after much else (z for the backward pass: kept in the
  // caches it drives out the operands of the tiles that are being made).
  template <bool LATER = false>
  __device__ __forceinline__ void put(void* matrix, int64_t row_bytes, int row0, int row_end, int column0, int column_end, int lane) const {
    asm volatile("" ::: "memory");  // (what other lanes wrote is read: LDS serves a wave in order)
#pragma unroll
    for (int t = 0; t < kTurns; ++t) {
      const int p = t * 64 + lane, r = p / kRow, c = p % kRow;
      const u32x4 v = at[r * kRow + (c ^ (r & (kRow - 1)))];
      if (row0 + r < row_end && c < CHUNKS && column0 + c * 8 < column_end) {
        u32x4* to = (u32x4*)((char*)matrix + (row0 + r) * row_bytes + (int64_t)(column0 + c * 8) * 2);
        if (LATER) __builtin_nontemporal_store(v, to);
        else *to = v;
      }
    }
    asm volatile("" ::: "memory");
  }
};

}  // namespace product
}  // namespace nd

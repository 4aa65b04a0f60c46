// Sums over the rows of a matrix, the gradients of what is added to or multiplied with every row: each workgroup of the kernel
// that reads the rows leaves sums of its share, in 32 bits, and one more kernel adds those.  No atomics: the same call
// gives the same bytes.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace nd {

// The sum of sums[s][c] over the shares, for column c: to first[c], or from column `split` on to
// second[c - split]; either may be null.  32 columns to a workgroup, 32 lanes to a column: bound by the latency of one lane's reads
// (256 shares, 8 each: 4 to 5 us with the launch).
template <class T>
__global__ __launch_bounds__(1024) void column_join_kernel(const float* sums, int64_t shares, int64_t columns, T* first, int64_t split,
                                                           T* second) {
  __shared__ float part[32][33];
  const int lane = threadIdx.x & 31, at = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;
  float sum = 0.f;
  if (c < columns)
    for (int64_t s = at; s < shares; s += 32) sum += sums[s * columns + c];
  part[at][lane] = sum;
  __syncthreads();
  if (at == 0 && c < columns) {
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) sum += part[i][lane];
    if (c < split) {
      if (first) first[c] = (T)sum;
    } else if (second) {
      second[c - split] = (T)sum;
    }
  }
}
template <class T>
hipError_t column_join(const float* sums, int64_t shares, int64_t columns, void* first, int64_t split, void* second, hipStream_t stream) {
  column_join_kernel<T><<<(uint32_t)((columns + 31) / 32), 1024, 0, stream>>>(sums, shares, columns, (T*)first, split, (T*)second);
  return hipGetLastError();
}

}  // namespace nd

// Sums over the rows of a matrix, second half: a kernel leaves one row of partial sums for
// each of its CTAs, and this one adds them, always in the same order.
#pragma once
#include "layers.cuh"

namespace hipress {

// part [parts][cols]; the first `split` columns go to `first`, the others to `second` (either
// may be NULL).  32 columns to a CTA of 32 warps, which share the rows.
static __global__ void __launch_bounds__(1024) column_sums_kernel(const float* part, int parts, int64_t cols, int64_t split,
                                                                  void* first, void* second, int type) {
  __shared__ float sums[32][33];
  const int64_t col = (int64_t)blockIdx.x * 32 + threadIdx.x;
  dependents_may_start();
  wait_for_kernel_before();
  float s = 0.f;
  if (col < cols)
#pragma unroll 4
    for (int r = threadIdx.y; r < parts; r += 32) s += part[r * cols + col];
  sums[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  s = warp_sum(sums[threadIdx.x][threadIdx.y]);
  const int64_t c = (int64_t)blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && c < cols) {
    if (c < split) {
      if (first) store_any(first, c, s, type);
    } else if (second) {
      store_any(second, c - split, s, type);
    }
  }
}

inline int column_sums(const float* part, int parts, int64_t cols, int64_t split, void* first, void* second, int type,
                       cudaStream_t s) {
  return launch_behind(column_sums_kernel, dim3((unsigned)((cols + 31) / 32)), dim3(32, 32), 0, s, part, parts, cols, split,
                       first, second, type);
}

}  // namespace hipress

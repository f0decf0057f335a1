// Zeros by a kernel of the caller's stream (a captured memset node is none).
#pragma once

#include <algorithm>

#include "common.h"
#include "enqueue.h"

namespace tilec {

namespace {

template <typename T>
__global__ __launch_bounds__(256) void zeros_kernel(T* __restrict__ p, int64_t rows, int64_t cols, int64_t ld) {
  for (int64_t r = blockIdx.y; r < rows; r += gridDim.y)
    for (int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x; c < cols; c += (int64_t)gridDim.x * 256) p[r * ld + c] = T(0);
}

// Zeros in a [rows, cols] matrix of row stride ld, whatever its size: a grid of at most
// 2^16 x 2^12 workgroups, whose loops stride over the rest.
template <typename T>
hipError_t enqueue_zeros(T* p, int64_t rows, int64_t cols, int64_t ld, hipStream_t stream) {
  if (rows <= 0 || cols <= 0) return hipSuccess;
  if (rows == 1 || ld == cols) cols *= rows, rows = 1;
  const dim3 grid((unsigned)std::min<int64_t>(cdiv(cols, 256), 1 << 16), (unsigned)std::min<int64_t>(rows, 1 << 12));
  return enqueue(zeros_kernel<T>, grid, dim3(256), stream, p, rows, cols, ld);
}

}  // namespace

}  // namespace tilec

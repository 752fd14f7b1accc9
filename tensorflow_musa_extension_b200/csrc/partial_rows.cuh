// Second level of a column sum: partial rows to one row.
#pragma once

#include "common.cuh"

namespace musa_b200 {

// Column sums of [count, n] fp32 partial rows, in a fixed order, in fp64.  CTA: 32 columns,
// eight row lanes.
template <typename T>
__global__ void __launch_bounds__(256)
    AddPartialRowsKernel(const float* __restrict__ partial, int count, int64_t n, T* out) {
  __shared__ double sums[8][32];
  GridDepWait();
  GridDepLaunch();
  const int lane = threadIdx.x % 32, part = threadIdx.x / 32;
  const int64_t col = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  double t = 0.0;
  if (col < n) {
#pragma unroll 8
    for (int r = part; r < count; r += 8) t += partial[r * n + col];
  }
  sums[part][lane] = t;
  __syncthreads();
  if (part == 0 && col < n) {
    for (int r = 1; r < 8; ++r) t += sums[r][lane];
    out[col] = FromF32<T>(static_cast<float>(t));
  }
}

template <typename T>
cudaError_t LaunchAddPartialRows(bool programmatic, const float* partial, int count, int64_t n,
                                 void* out, cudaStream_t stream) {
  return LaunchChained(programmatic, AddPartialRowsKernel<T>,
                       dim3(static_cast<unsigned>(CeilDiv(n, 32))), dim3(256), 0, stream, partial,
                       count, n, static_cast<T*>(out));
}

}  // namespace musa_b200

// Second level of a column sum: partial rows to one row.
#pragma once

#include "common.cuh"

namespace musa_b200 {

// Column sums of [count, n] fp32 partial rows, in a fixed order, in fp64.  CTA: 32 columns,
// 32 row lanes (with eight the 444 partial rows of a [16384,256] gradient took 8 us).
template <typename T>
__global__ void __launch_bounds__(1024)
    AddPartialRowsKernel(const float* __restrict__ partial, int count, int64_t n, T* out) {
  __shared__ double sums[32][33];
  GridDepWait();
  GridDepLaunch();
  const int lane = threadIdx.x % 32, part = threadIdx.x / 32;
  const int64_t col = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  double t = 0.0;
  if (col < n) {
#pragma unroll 4
    for (int r = part; r < count; r += 32) t += partial[r * n + col];
  }
  sums[part][lane] = t;
  __syncthreads();
  // Warp `part` adds the lanes of one column.
  t = sums[lane][part];
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) t += __shfl_xor_sync(0xffffffffu, t, m);
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 32 + part;
  if (lane == 0 && at < n) out[at] = FromF32<T>(static_cast<float>(t));
}

template <typename T>
cudaError_t LaunchAddPartialRows(bool programmatic, const float* partial, int count, int64_t n,
                                 void* out, cudaStream_t stream) {
  return LaunchChained(programmatic, AddPartialRowsKernel<T>,
                       dim3(static_cast<unsigned>(CeilDiv(n, 32))), dim3(1024), 0, stream, partial,
                       count, n, static_cast<T*>(out));
}

}  // namespace musa_b200

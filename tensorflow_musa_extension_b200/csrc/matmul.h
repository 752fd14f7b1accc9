// Parameters of the matrix-product kernels (matmul.cu).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace musa_b200 {

// One factor of a product: op(X) is [rows, depth]; `rows_contiguous` says that memory
// holds [depth, rows] (the factor is stored transposed), else [rows, depth]; `ld`
// elements from line to line of what memory holds.
struct Factor {
  const void* p;
  int64_t ld;
  bool rows_contiguous;
};

// z = product * a_scale[row] * b_scale[column] + bias[column];  y = act(z) + residual.
struct Epilogue {
  const void* bias;       // [n], type of y, or null
  const void* residual;   // [m, n], type of y, or null
  const float* a_scale;   // [m], 8-bit factors
  const float* b_scale;   // [n], 8-bit factors
  void* y;                // [m, n]
  void* z;                // [m, n], type of y, or null
  int act;
};

}  // namespace musa_b200

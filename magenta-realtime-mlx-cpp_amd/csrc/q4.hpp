// Products with 4-bit weights (q4.hip).
#pragma once

#include "common.hpp"

namespace mrt {

// w (n, k / 8): eight 4-bit codes a word, the first in the low bits; scales, biases
// (n, k / group) in the activations' type: weight = scale * code + bias.
struct Q4Weights {
  const uint32_t* w = nullptr;
  const void* scales = nullptr;
  const void* biases = nullptr;
  int n = 0, k = 0, group = 0;
};

// y (rows, n) = x (rows, k) W^T, row strides ldx, ldy.
void q4_matmul(DType dt, const Q4Weights& w, const void* x, int64_t ldx, int rows, void* y, int64_t ldy, hipStream_t s);
// Codes, scales and biases of src (n, k) with row stride ld.
void q4_quantize(DType dt, const void* src, int64_t ld, int n, int k, int group, uint32_t* w, void* scales, void* biases,
                 hipStream_t s);

}  // namespace mrt

// Products in 8-bit integers (i8.hip).
#pragma once

#include "common.hpp"

namespace mrt {

// Codes and scales of the rows of src (rows, k), row stride ld: scale = max |x| / 127.
void i8_quantize(DType dt, const void* src, int64_t ld, int rows, int k, int8_t* codes, int64_t ldc, float* scales,
                 hipStream_t s);

struct I8Args {
  const int8_t* x = nullptr;       // (rows, k), row stride ldx
  const float* x_scale = nullptr;  // (rows)
  const int8_t* w = nullptr;       // (n, k), row stride ldw
  const float* w_scale = nullptr;  // (n)
  const void* add = nullptr;       // (rows, n) of the output's type, row stride lda, or nullptr
  void* out = nullptr;             // (rows, n), row stride ldo
  int64_t ldx = 0, ldw = 0, lda = 0, ldo = 0;
  int rows = 0, n = 0, k = 0;
};
// out = (x w^T) x_scale w_scale + add
void i8_matmul(DType dt, const I8Args& a, hipStream_t s);

}  // namespace mrt

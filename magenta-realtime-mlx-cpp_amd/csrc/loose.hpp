// Vectors of words in memory at the alignment of an element of T, for rows that begin
// anywhere: memory takes such accesses whole.
#pragma once

#include <stdint.h>

#include <hip/hip_runtime.h>

namespace mrt {

template <typename T, int WORDS>
struct Loose {
  typedef uint32_t Word __attribute__((ext_vector_type(WORDS)));
  typedef Word Any __attribute__((aligned(sizeof(T))));
  typedef __attribute__((address_space(1))) Any Global;
  __device__ __forceinline__ static Word load(const T* p) { return *(const Global*)p; }
  __device__ __forceinline__ static void store(T* p, Word w) { *(Global*)p = w; }
};

}  // namespace mrt

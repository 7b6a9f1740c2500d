// Verification of drafted tokens against the target's probabilities (verify.hip).
#pragma once

#include "kv_cache.hpp"

namespace mrt {

// Slot 0 is what follows the cache, slot t + 1 what follows node t.  target (rows, nodes +
// 1, vocab): the target's probabilities at each slot; draft (rows, nodes, vocab): those that
// a slot's children were drawn from, or nullptr.  Element strides, the vocabulary contiguous.
struct VerifyArgs {
  const void* target = nullptr;
  const void* draft = nullptr;
  int64_t t_row = 0, t_slot = 0, d_row = 0, d_slot = 0;
  const int* tokens = nullptr;   // (rows, nodes)
  const int* parents = nullptr;  // (rows, nodes), or nullptr: a chain
  int64_t parents_stride = 0;    // 0: one tree for every sequence
  const float* uniforms = nullptr;  // (rows, nodes + 1)
  int* accepted = nullptr;          // (rows, nodes)
  int* count = nullptr;             // (rows)
  int* token = nullptr;             // (rows)
  int rows = 0, nodes = 0, vocab = 0;
};
// Bytes of workspace that draft_verify wants (0: none).
size_t draft_verify_workspace(const VerifyArgs& a);
void draft_verify(DType dt, const VerifyArgs& a, void* ws, hipStream_t s);

}  // namespace mrt

// Operators over caller-owned K/V caches: attention of a tree of drafted tokens
// (tree_attn.hip), the commit of the accepted path and eviction (cache_ops.hip).
#pragma once

#include "common.hpp"

namespace mrt {

constexpr int kMaxNodes = 64;   // drafted tokens of a sequence in one call: a bit each in a 64-bit ancestor mask
constexpr int kMaxHeadDim = 256;

// A cache of `rows` sequences: k and v (rows, kv_heads, capacity, d) of one dtype,
// d contiguous, with the same element strides; sequence b holds length[b] entries
// in slots 0.. of every KV head.  pos (rows, kv_heads, capacity): each entry's
// position, or nullptr where an entry's slot is its position; next_pos (rows): the
// next token's position (length where pos is nullptr).
struct KvCache {
  void* k = nullptr;
  void* v = nullptr;
  int64_t row_stride = 0, head_stride = 0, slot_stride = 0;
  const int* length = nullptr;
  int* pos = nullptr;
  const int* next_pos = nullptr;
  const float* score = nullptr;
  int rows = 0, kv_heads = 0, capacity = 0, d = 0;
  DType dt = DType::F32;
};

// A (rows, nodes, heads, d) operand: element strides, d contiguous.
struct NodeRows {
  void* p = nullptr;
  int64_t row_stride = 0, node_stride = 0, head_stride = 0;
};

struct TreeAttnArgs {
  NodeRows q, k_new, v_new, out;
  const int* parents = nullptr;  // (rows, nodes)
  int64_t parents_stride = 0;    // 0: one tree for every sequence
  float* lse = nullptr;          // (rows, nodes, heads) or nullptr
  const float* bias = nullptr;   // (heads, buckets) by distance, or nullptr
  int buckets = 0, nodes = 0, heads = 0;
  float scale = 1.f;
};
// Whether a launch has threads enough for these sizes.
bool tree_attention_fits(const KvCache& c, int heads, int nodes);
// Bytes of workspace that tree_attention wants (0: none).
size_t tree_attention_workspace(const KvCache& c, int heads, int nodes);
void tree_attention(const KvCache& c, const TreeAttnArgs& a, void* ws, hipStream_t s);

struct CommitArgs {
  NodeRows k_new, v_new, q;       // q.p nullptr: no weights
  const int* accepted = nullptr;  // (rows, accepted_n)
  int64_t accepted_stride = 0;
  const float* lse = nullptr;     // (rows, nodes, heads)
  const float* bias = nullptr;
  float* score_out = nullptr;     // (rows, kv_heads, capacity)
  int* length_out = nullptr;      // (rows)
  int* next_out = nullptr;        // (rows), with pos
  int accepted_n = 0, nodes = 0, heads = 0, buckets = 0;
  float scale = 1.f;
};
void cache_commit(const KvCache& c, const CommitArgs& a, hipStream_t s);

struct EvictArgs {
  float* score_out = nullptr;  // (rows, kv_heads, capacity)
  int* pos_out = nullptr;      // the same
  int* length_out = nullptr;   // (rows)
  int keep = 0, recent = 0, sinks = 0;
};
size_t cache_evict_workspace(const KvCache& c, int keep);
void cache_evict(const KvCache& c, const EvictArgs& a, void* ws, hipStream_t s);

}  // namespace mrt

// Operators over caches in pages: new entries written, quantised on the way, and read
// back (paged_store.hip), attention of new tokens (paged_attn.hip).
#pragma once

#include "kv_cache.hpp"

namespace mrt {

constexpr int kPageUnit = 16;  // entries of a page: a multiple of this, so that 16 keys in a row share a page

// k and v: pools (pages, kv_heads, page_size, d) with the same element strides, d
// contiguous, of `dt`, or, with `codes`, int8 and fp32 scales (pages, kv_heads, page_size).
// table (rows, row_pages): page x of sequence b, entries x page_size .., or an id outside
// [0, pages) where there is none.  length (rows): entries in use.
struct PagedCache {
  void* k = nullptr;
  void* v = nullptr;
  float* k_scale = nullptr;
  float* v_scale = nullptr;
  const int* table = nullptr;
  const int* length = nullptr;
  int64_t page_stride = 0, head_stride = 0, slot_stride = 0, table_stride = 0;
  int pages = 0, rows = 0, row_pages = 0, kv_heads = 0, page_size = 0, d = 0;
  bool codes = false;
  DType dt = DType::F32;  // of the pages; not with codes
  int capacity() const { return row_pages * page_size; }
};

// Division of numbers below 2^31 by a constant: n / d = (n mul) >> (31 + shift), mul the
// quotient of 2^(31 + shift) by d rounded up, 2^(shift - 1) < d <= 2^shift, so mul is in [2^31, 2^32].
struct Divide {
  uint32_t mul = 0;
  int shift = 0;
  Divide() = default;
  explicit Divide(int d) {
    while ((1ll << shift) < d) ++shift;
    mul = (uint32_t)(((1ull << (31 + shift)) + d - 1) / d);
  }
  __host__ __device__ int operator()(int n) const { return (int)(((uint64_t)(uint32_t)n * mul) >> (31 + shift)); }
};

struct PagedStoreArgs {
  NodeRows k, v;               // (rows, tokens, kv_heads, d) of `dt`
  const int* fresh = nullptr;  // (rows) tokens that are there, or nullptr: all
  const int* start = nullptr;  // (rows) first entry read, or nullptr: 0
  int* length_out = nullptr;   // (rows) or nullptr
  int tokens = 0;
  DType dt = DType::F32;
};
void paged_write(const PagedCache& c, const PagedStoreArgs& a, hipStream_t s);
void paged_read(const PagedCache& c, const PagedStoreArgs& a, hipStream_t s);

struct PagedAttnArgs {
  NodeRows q, out;              // (rows, tokens, heads, d) of `dt`
  const int* fresh = nullptr;   // (rows) or nullptr
  float* lse = nullptr;         // (rows, tokens, heads) or nullptr
  const float* bias = nullptr;  // (heads, buckets) by distance, or nullptr
  int buckets = 0, tokens = 0, heads = 0;
  DType dt = DType::F32;
  float scale = 1.f;
};
// Whether a launch has threads enough for these sizes.
bool paged_attention_fits(const PagedCache& c, int heads, int tokens);
// Bytes of workspace that paged_attention wants (0: none).
size_t paged_attention_workspace(const PagedCache& c, int heads, int tokens);
void paged_attention(const PagedCache& c, const PagedAttnArgs& a, void* ws, hipStream_t s);

}  // namespace mrt

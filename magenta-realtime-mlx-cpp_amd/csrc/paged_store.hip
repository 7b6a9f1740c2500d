// Entries of a paged cache: written, quantised to 8 bits on the way where the pages hold
// codes, and read back.
//
// A vector is one entry's d values of one K/V head, of K or of V; codes8.hpp says how it is
// quantised.  Every vector has its own scale, so a new entry never changes what others stand
// for.  A vector with an infinity or NaN has scale NaN: 8 bits cannot hold what it was, and
// nothing that reads it may pass it off as finite.
//
// LP lanes (the power of two from d / 16 on) take a vector, 16 elements each: to quantise, 16
// in a row, so that codes move in 16-byte pieces and the maximum needs log2 LP exchanges; else
// 16-byte pieces of the values, LP in a row, so that what a store covers is contiguous (codes
// to fp32, 16 x 2000 tokens of 8 heads of d 128: 96 us with 64 bytes a lane, 63 so).  Bound by
// bytes; consecutive vectors are consecutive entries of a head, which lie together in a page.
// 16 x 4001 tokens in fp16: written in 80 us, read in 84, 4.9 and 4.7 TB/s, as a large copy.
// Several vectors a lane group do not help: 97, 106 and 124 us with one, two and four (when a
// write took 97).
#include <algorithm>

#include "codes8.hpp"
#include "device_utils.hpp"
#include "paged.hpp"

namespace mrt {
namespace {

struct MoveArgs {
  char* pool[2];
  float* scale[2];
  char* rows_p[2];  // (rows, tokens, kv_heads, d) operand of K and of V
  int64_t r_row[2], r_node[2], r_head[2];
  int64_t page_stride, head_stride, slot_stride, table_stride, vectors;
  const int *table, *length, *fresh, *start;
  int* length_out;
  int pages, kv_heads, page_size, capacity, tokens, D;
  Divide by_page, by_inner, by_outer;  // vector = (b outer + x) inner + y
  int inner, outer;
  bool tokens_inner;
};

// 16 values.
template <typename T>
__device__ __forceinline__ void load16(const T* p, float (&v)[16]) {
  constexpr int kPer = 16 / sizeof(T);
#pragma unroll
  for (int x = 0; x < 16 / kPer; ++x) {
    union {
      uint4 w;
      T e[kPer];
    } u;
    u.w = ld_g16(p + x * kPer);
#pragma unroll
    for (int j = 0; j < kPer; ++j) v[x * kPer + j] = St<T>::ld(u.e[j]);
  }
}

// blockIdx.y: K or V.  CODES: the pages hold 8-bit codes, else values of T.
template <typename T, bool CODES, bool WRITE, int LP>
__global__ __launch_bounds__(256) void k_paged_move(const MoveArgs a) {
  const int64_t vec = (int64_t)blockIdx.x * (256 / LP) + threadIdx.x / LP;
  const int part = threadIdx.x % LP, x = blockIdx.y;
  if (vec >= a.vectors) return;  // all lanes of a vector alike
  const int at = a.by_inner((int)vec), y = (int)vec - at * a.inner, b = a.by_outer(at), z = at - b * a.outer;
  const int t = a.tokens_inner ? y : z, h = a.tokens_inner ? z : y;
  const int len = min(max(a.length[b], 0), a.capacity);
  T* row = reinterpret_cast<T*>(a.rows_p[x]) + b * a.r_row[x] + t * a.r_node[x] + h * a.r_head[x];
  constexpr int kPer = 16 / sizeof(T), kPieces = 16 / kPer;  // elements of 16 bytes
  [[maybe_unused]] float v[16] = {};
  [[maybe_unused]] uint4 piece[kPieces];
  auto at_of = [&](int p) { return (p * LP + part) * kPer; };  // first element of the lane's piece p
  if constexpr (WRITE && CODES) {
    if (part * 16 < a.D) load16(row + part * 16, v);
  } else if constexpr (WRITE) {
#pragma unroll
    for (int p = 0; p < kPieces; ++p)
      if (at_of(p) < a.D) piece[p] = ld_g16(row + at_of(p));
  }
  int entry;
  bool there;
  if constexpr (WRITE) {
    const int n = a.fresh != nullptr ? min(max(a.fresh[b], 0), a.tokens) : a.tokens;
    entry = len + t;  // below 2^31: capacity and tokens are at most 2^30
    there = t < n && entry < a.capacity;
    if (a.length_out != nullptr && x == 0 && h == 0 && t == 0 && part == 0) a.length_out[b] = min(len + n, a.capacity);
  } else {
    const int64_t e = (int64_t)(a.start != nullptr ? a.start[b] : 0) + t;
    there = e >= 0 && e < len;
    entry = there ? (int)e : 0;
  }
  const int page = a.by_page(entry), slot = entry - page * a.page_size;
  const int id = there ? a.table[b * a.table_stride + page] : -1;
  if (id < 0 || id >= a.pages) return;
  const int64_t to = id * a.page_stride + h * a.head_stride + slot * a.slot_stride;
  [[maybe_unused]] float* scale = CODES ? a.scale[x] + ((int64_t)id * a.kv_heads + h) * a.page_size + slot : nullptr;

  if constexpr (WRITE && CODES) {
    uint32_t top = 0;  // bits of |x| order as the values do, NaN above all
#pragma unroll
    for (int j = 0; j < 16; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
#pragma unroll
    for (int o = 1; o < LP; o <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
    const float s = codes_scale(top);
    if (part * 16 < a.D) *reinterpret_cast<uint4*>(a.pool[x] + to + part * 16) = codes16(v, s);
    if (part == 0) *scale = s;
  } else if constexpr (WRITE) {
#pragma unroll
    for (int p = 0; p < kPieces; ++p)
      if (at_of(p) < a.D) *reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.pool[x]) + to + at_of(p)) = piece[p];
  } else if constexpr (CODES) {
    const float s = ld_g(scale);
    uint32_t w[kPieces][kPer / 4];
#pragma unroll
    for (int p = 0; p < kPieces; ++p) {
      const char* from = a.pool[x] + to + min(at_of(p), a.D - kPer);
      if constexpr (kPer == 8) {
        const uint64_t u = ld_g(reinterpret_cast<const uint64_t*>(from));
        w[p][0] = (uint32_t)u, w[p][1] = (uint32_t)(u >> 32);
      } else {
        w[p][0] = ld_g(reinterpret_cast<const uint32_t*>(from));
      }
    }
#pragma unroll
    for (int p = 0; p < kPieces; ++p) {
      union {
        T e[kPer];
        uint4 w4;
      } u;
#pragma unroll
      for (int j = 0; j < kPer; ++j) u.e[j] = St<T>::st((float)(int8_t)(w[p][j / 4] >> (8 * (j % 4))) * s);
      if (at_of(p) < a.D) *reinterpret_cast<uint4*>(row + at_of(p)) = u.w4;
    }
  } else {
#pragma unroll
    for (int p = 0; p < kPieces; ++p)
      if (at_of(p) < a.D) piece[p] = ld_g16(reinterpret_cast<const T*>(a.pool[x]) + to + at_of(p));
#pragma unroll
    for (int p = 0; p < kPieces; ++p)
      if (at_of(p) < a.D) *reinterpret_cast<uint4*>(row + at_of(p)) = piece[p];
  }
}

template <typename T, bool CODES, bool WRITE>
void launch(const MoveArgs& a, hipStream_t s) {
  auto go = [&](auto lanes) {
    constexpr int LP = decltype(lanes)::value;
    const dim3 grid((unsigned)((a.vectors + 256 / LP - 1) / (256 / LP)), 2);
    hipLaunchKernelGGL((k_paged_move<T, CODES, WRITE, LP>), grid, dim3(256), 0, s, a);
  };
  if (a.D <= 16) go(std::integral_constant<int, 1>{});
  else if (a.D <= 32) go(std::integral_constant<int, 2>{});
  else if (a.D <= 64) go(std::integral_constant<int, 4>{});
  else if (a.D <= 128) go(std::integral_constant<int, 8>{});
  else go(std::integral_constant<int, 16>{});
}

template <bool WRITE>
void move(const PagedCache& c, const PagedStoreArgs& p, hipStream_t s) {
  MoveArgs a{};
  a.pool[0] = static_cast<char*>(c.k), a.pool[1] = static_cast<char*>(c.v);
  a.scale[0] = c.k_scale, a.scale[1] = c.v_scale;
  const NodeRows* rows[2] = {&p.k, &p.v};
  for (int x = 0; x < 2; ++x) {
    a.rows_p[x] = static_cast<char*>(rows[x]->p);
    a.r_row[x] = rows[x]->row_stride, a.r_node[x] = rows[x]->node_stride, a.r_head[x] = rows[x]->head_stride;
  }
  a.page_stride = c.page_stride, a.head_stride = c.head_stride, a.slot_stride = c.slot_stride;
  a.table_stride = c.table_stride, a.table = c.table, a.length = c.length, a.fresh = p.fresh, a.start = p.start;
  a.length_out = p.length_out, a.pages = c.pages, a.kv_heads = c.kv_heads, a.page_size = c.page_size;
  a.capacity = c.capacity(), a.tokens = p.tokens, a.D = c.d;
  a.vectors = (int64_t)c.rows * p.tokens * c.kv_heads;
  // entries of a head in turn, unless a page has its heads side by side
  a.tokens_inner = c.head_stride >= c.slot_stride;
  a.inner = a.tokens_inner ? p.tokens : c.kv_heads, a.outer = a.tokens_inner ? c.kv_heads : p.tokens;
  a.by_page = Divide(c.page_size), a.by_inner = Divide(a.inner), a.by_outer = Divide(a.outer);
  MRT_DTYPE_DISPATCH(p.dt, {
    if (c.codes) launch<T, true, WRITE>(a, s);
    else launch<T, false, WRITE>(a, s);
  });
  MRT_HIP_CHECK(hipGetLastError());
}

}  // namespace

void paged_write(const PagedCache& c, const PagedStoreArgs& a, hipStream_t s) { move<true>(c, a, s); }
void paged_read(const PagedCache& c, const PagedStoreArgs& a, hipStream_t s) { move<false>(c, a, s); }

}  // namespace mrt

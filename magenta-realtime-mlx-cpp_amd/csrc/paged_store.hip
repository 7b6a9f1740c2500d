// Entries of a paged cache: written, quantised to 8 bits on the way where the pages hold
// codes, and read back.
//
// A vector is one entry's d values of one K/V head, of K or of V; codes8.hpp says how it is
// quantised.  Every vector has its own scale, so a new entry never changes what others stand
// for.  A vector with an infinity or NaN has scale NaN: 8 bits cannot hold what it was, and
// nothing that reads it may pass it off as finite.
//
// LP lanes (the power of two from d / 16 on) take a vector, 16 elements each, so that
// codes move in 16-byte pieces and the maximum needs log2 LP exchanges.  Bound by bytes;
// consecutive vectors are consecutive entries of a head, which lie together in a page.
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

template <typename T>
__device__ __forceinline__ void load8(const T* p, float* v) {
  if constexpr (sizeof(T) == 4) {
    const uint4 a = ld_g16(p), b = ld_g16(p + 4);
    v[0] = __uint_as_float(a.x), v[1] = __uint_as_float(a.y), v[2] = __uint_as_float(a.z), v[3] = __uint_as_float(a.w);
    v[4] = __uint_as_float(b.x), v[5] = __uint_as_float(b.y), v[6] = __uint_as_float(b.z), v[7] = __uint_as_float(b.w);
  } else {
    const uint4 a = ld_g16(p);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) v[2 * j] = St<T>::unbits(w[j] & 0xffffu), v[2 * j + 1] = St<T>::unbits(w[j] >> 16);
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float* v) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = St<T>::bits(v[2 * j]) | (St<T>::bits(v[2 * j + 1]) << 16);
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
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
  const int d0 = part * 16;
  float v[16] = {};
  if constexpr (WRITE) {
#pragma unroll
    for (int c = 0; c < 2; ++c)
      if (d0 + c * 8 < a.D) load8(row + d0 + c * 8, v + c * 8);
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
    if (d0 < a.D) *reinterpret_cast<uint4*>(a.pool[x] + to + d0) = codes16(v, s);
    if (part == 0) *scale = s;
  } else if constexpr (WRITE) {
#pragma unroll
    for (int c = 0; c < 2; ++c)
      if (d0 + c * 8 < a.D) store8(reinterpret_cast<T*>(a.pool[x]) + to + d0 + c * 8, v + c * 8);
  } else {
    if constexpr (CODES) {
      if (d0 >= a.D) return;
      const float s = ld_g(scale);
      const uint4 c = ld_g16(a.pool[x] + to + d0);
      const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) v[4 * j + k] = (float)(int8_t)(w[j] >> (8 * k)) * s;
    } else {
#pragma unroll
      for (int c = 0; c < 2; ++c)
        if (d0 + c * 8 < a.D) load8(reinterpret_cast<const T*>(a.pool[x]) + to + d0 + c * 8, v + c * 8);
    }
#pragma unroll
    for (int c = 0; c < 2; ++c)
      if (d0 + c * 8 < a.D) store8(row + d0 + c * 8, v + c * 8);
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

// Attention of a sequence's newest tokens over a cache in pages.
//
// Query t of a sequence's n new tokens sees the entries 0 .. length + t, its own among
// them:
//   s_tj = scale q_t . k_j + bias[h, min(length + t - j, M - 1)],  out_t = softmax(s_t) V.
// One pass over the keys with the running maximum and sum of the softmax.  Few query rows
// meet each key (a K/V head, a unit, has R = tokens heads / kv_heads of them), so reading the
// keys is what it costs: straight from memory to registers, the waves of a block taking
// steps in turn.  Pages are multiples of 16 entries, so the 16 keys of a matrix tile share a
// page: a wave looks up its next 64 tiles in its lanes at once and then needs a scalar for
// each.
//
// Pages of the operands' type: the fragments of attn_frag.hpp, 32 keys a step.
//
// Pages of 8-bit codes: 64 keys a step.  For operands of 16 bits both products are in integers:
// converting codes to 16 bits would cost a vector instruction for two of them; instead the few
// query rows and weights become three digits of 8 bits,
//   x = f (65536 a + 256 b + c),  a, b, c in [-128, 127],
// f a power of two for the row (of weights: for the row and step) by which its largest
// magnitude is in [2^21, 2^22), so that x is within 2^-22 of that magnitude; sums of products
// with codes are exact.  Scales of keys multiply scores, those of values the weights.  S^T = K Q^T leaves
// lane (i, g) with keys 16 t + 4 g + r of the four tiles, just the 16 keys whose codes of one
// dimension, transposed in registers by byte permutations, are its operand of
// O^T = V^T P^T.
//
// Digits are relative to a row's largest magnitude.  Beside a channel of q 1000 times the others,
// in which keys have little, the others keep 12 bits: enough for operands of 16 bits, which have
// no more than 11.  Outputs of fp32 operands were 1.5e-4 off there, 5e-7 with plain fp32
// products.  So q and the weights of fp32 are three bf16 parts each, which hold any value whole,
// and codes become bf16, which holds them exactly: every product is exact in fp32, as over fp32
// pages.  It costs the conversion, one and a half vector instructions a code: 48 x 8 heads of up
// to 8191 of d 128 111 us (digits 96, the fp32 matrix instruction 172), 4 x 32000 of d 128 with 4
// tokens of 4 heads 72 (63, 108), with 16 161 (131, 363), 16 x 16000 of d 256 51 (44, 83).
//
// Bound by bytes but for many rows a K/V head (16 new tokens of 4 heads on one over 8-bit pages
// of 4 x 32000 entries, d 128: 127 us for 63 with 4, by vector instructions on the digits and the
// softmax).  One pass, us (bytes at the rate of a large copy): 64 x 16 heads of 1006 entries of
// d 64 in 8 bits 37 (30), 48 x 8 heads of up to 8191 of d 128 in bf16 156 (172), 3 x 8 heads of
// up to 131000 in 8 bits, 4 tokens of 4 heads each, 99 (101).  Vector instructions take 42, 19
// and 36 % of the SIMDs' cycles there, the matrix cores 5 to 9 %, and waves wait for 35 to 47 %
// of theirs.
//
// As many blocks run as the card holds.  Long caches: the units' steps, one after the other,
// are cut into equal shares, on the device, from the lengths, which the host never sees; a
// share may end and begin inside units, whose parts leave (maximum, sum, output) in fp32, and
// k_paged_join sums them in order, so a result does not depend on timing.  Short ones: a block
// takes whole units in turn.  Either way the next unit's first keys are requested before
// this one's waves join.
#include <algorithm>
#include <climits>
#include <type_traits>

#include "attn_frag.hpp"
#include "mfma_ring.hpp"
#include "paged.hpp"

namespace mrt {
namespace {

constexpr int kBiasLds = 4096;  // floats of the bias by distance kept in LDS

// Row tiles a wave holds at most: what one more takes in registers costs more than reading
// the keys again from the L2.  With 16 rows or fewer there is one.
constexpr int row_tiles(size_t elt, int dp) { return elt == 2 && dp <= 64 ? 2 : 1; }
// Waves of a block, and blocks that a CU holds (by their registers).
constexpr int waves_of(size_t elt, int dp) { return elt == 2 && dp == 128 ? 8 : 4; }
constexpr int blocks_of_cu(size_t elt, int dp, int nr) {
  return elt == 1 ? (dp == 256 ? 1 : 2) : elt == 4 ? (dp == 32 ? 4 : dp == 64 ? 2 : 1)
                                                   : dp == 32 ? 4 / nr : dp == 64 ? (nr == 1 ? 3 : 2) : 1;
}
#define MRT_ATTN_BOUNDS(elt, nr) \
  __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(blocks_of_cu(elt, DP, nr) * W / 4)))
typedef int i32x4_t __attribute__((ext_vector_type(4)));

struct PageArgs {
  const void *q, *k, *v;
  void* out;
  const float *k_scale, *v_scale, *bias;
  const int *table, *length, *fresh;
  float* lse;
  float* part;      // (slots, R, D) outputs of the parts
  float2* part_ml;  // (slots, R) maximum (in log2 units) and sum
  int64_t q_row, q_node, q_head, o_row, o_node, o_head, page_stride, head_stride, slot_stride, table_stride;
  Divide by_tiles;  // 16-key tiles of a page
  int page_tiles, row_pages, pages, rows, kv_heads, heads, tokens, D, buckets;
  int teams;   // blocks that take a share each
  int least;   // steps that a share has at least
  int unit;    // steps that beginning and ending a unit counts as; 0: units are not cut
  int row_blocks;
  float scale;
};

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t uniform(int64_t v) {
  return (int64_t)((uint64_t)(uint32_t)uniform((int)(v >> 32)) << 32 | (uint32_t)uniform((int)v));
}

// Entries before the new tokens, and new tokens, of sequence b.
__device__ __forceinline__ int capacity_of(const PageArgs& a) { return a.row_pages * a.page_tiles * kPageUnit; }
__device__ __forceinline__ int length_of(const PageArgs& a, int b) { return min(max(a.length[b], 0), capacity_of(a)); }
__device__ __forceinline__ int fresh_of(const PageArgs& a, int b) {
  return a.fresh != nullptr ? min(max(a.fresh[b], 0), a.tokens) : a.tokens;
}
// Steps of a unit of sequence b: none where it has no new token.
template <int KEYS>
__device__ __forceinline__ int steps_of(const PageArgs& a, int b) {
  const int n = fresh_of(a, b);
  return n == 0 ? 0 : (min(length_of(a, b) + n, capacity_of(a)) + KEYS - 1) / KEYS;
}

// Positions of all units' steps in a row, each unit's after `unit` of its own, cut into `teams`
// shares of `total`: share t is [t total / teams, (t + 1) total / teams), rounded down.
struct Shares {
  int64_t total;
  int teams;
  __device__ __forceinline__ int64_t begin(int t) const { return t * total / teams; }
  __device__ __forceinline__ int of(int64_t at) const { return (int)(((at + 1) * teams + total - 1) / total) - 1; }
};
__device__ __forceinline__ int64_t wave_sum64(int64_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return uniform(v);
}
// first: the steps of a unit of row `lane`.
template <int KEYS>
__device__ __forceinline__ Shares shares_of(const PageArgs& a, int lane, int first) {
  int64_t steps = first;
  for (int b = lane + 64; b < a.rows; b += 64) steps += steps_of<KEYS>(a, b);
  steps = wave_sum64(steps) * a.kv_heads;
  Shares s;
  s.total = steps + (int64_t)a.unit * a.rows * a.kv_heads;
  s.teams = (int)max((int64_t)1, min((int64_t)a.teams, s.total / a.least));
  return s;
}

// One unit's part: steps s0 .. s1 - 1 of its `steps`.  Whole units of short caches leave s1
// and steps open, so that no key waits for the length.
struct Part {
  int b, kvh, s0, s1, steps;
  int64_t slot;  // of its result, if the unit is cut: unit + team, which are all different
  bool open, all;
};

// The parts of a team, one after the other.
template <int KEYS>
struct Walk {
  int64_t at, from, to;  // cut: where the next unit begins, the share
  int team, b, kvh, steps;
  __device__ __forceinline__ Walk(const PageArgs& a, int lane, int team_)
      : at(0), from(0), to(0), team(team_), b(0), kvh(0), steps(0) {
    if (a.unit == 0) {
      b = team / a.kv_heads, kvh = team - b * a.kv_heads;
      return;
    }
    int own_steps = lane < a.rows ? steps_of<KEYS>(a, lane) : 0;
    const Shares s = shares_of<KEYS>(a, lane, own_steps);
    if (team >= s.teams) return;
    from = s.begin(team), to = s.begin(team + 1);
    int64_t base = 0;
    for (int b0 = 0; b0 < a.rows; b0 += 64) {  // the row that holds position `from`
      if (b0 > 0) own_steps = b0 + lane < a.rows ? steps_of<KEYS>(a, b0 + lane) : 0;
      const int64_t own = b0 + lane < a.rows ? (int64_t)(own_steps + a.unit) * a.kv_heads : 0;
      int64_t incl = own;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int64_t x = __shfl_up(incl, o, 64);
        if (lane >= o) incl += x;
      }
      const uint64_t past = __ballot(base + incl > from);
      if (past != 0) {
        const int l = __ffsll((unsigned long long)past) - 1;
        base += uniform((int64_t)__shfl(incl - own, l, 64));
        b = b0 + l, steps = uniform(__shfl(own_steps, l, 64));
        kvh = (int)((from - base) / (steps + a.unit));
        at = base + (int64_t)kvh * (steps + a.unit);
        return;
      }
      base += uniform((int64_t)__shfl(incl, 63, 64));
    }
  }
  __device__ __forceinline__ bool next(const PageArgs& a, Part& w) {
    if (a.unit == 0) {
      if (b >= a.rows) return false;
      w.b = b, w.kvh = kvh, w.s0 = 0, w.s1 = w.steps = 0, w.slot = 0, w.open = w.all = true;
      const int64_t u = (int64_t)b * a.kv_heads + kvh + a.teams;
      b = (int)(u / a.kv_heads), kvh = (int)(u - (int64_t)b * a.kv_heads);
      return true;
    }
    while (at < to) {
      const int64_t first = at + a.unit;  // of the unit's steps
      w.b = b, w.kvh = kvh, w.steps = steps, w.open = false;
      w.s0 = (int)max((int64_t)0, from - first), w.s1 = (int)min((int64_t)steps, to - first);
      w.slot = (int64_t)b * a.kv_heads + kvh + team;
      // a unit without steps, whose outputs are zeros, falls to the share with its beginning
      w.all = steps == 0 || (w.s0 == 0 && w.s1 == steps);
      const bool mine = steps == 0 ? at >= from : w.s0 < w.s1;
      at = first + steps;
      if (++kvh == a.kv_heads) {
        kvh = 0, ++b;
        steps = b < a.rows ? uniform(steps_of<KEYS>(a, b)) : 0;
      }
      if (mine) return true;
    }
    return false;
  }
};

// The team of this block, and its first query row; row blocks of a team share keys and follow
// each other on one XCD.
__device__ __forceinline__ int team_of(const PageArgs& a, int rows_of_block, int& row0) {
  if (a.row_blocks == 1) {
    row0 = 0;
    return blockIdx.x;
  }
  const int x = blockIdx.x >> 3, rb = x % a.row_blocks;
  row0 = rb * rows_of_block;
  return (x / a.row_blocks) * 8 + (blockIdx.x & 7);
}

// The page and place in it of a wave's next tiles, one a lane.
template <int TILES>
struct TileLookup {
  int page, place;  // page -1: not there
  // lane l: tile l % TILES of the wave's step `first + every (l / TILES)`
  __device__ __forceinline__ void fetch(const PageArgs& a, const int* table, int first, int every, int lane) {
    const int tile = (first + every * (lane / TILES)) * TILES + lane % TILES, at = a.by_tiles(tile);
    place = (tile - at * a.page_tiles) * kPageUnit;
    page = -1;
    if (at < a.row_pages) {
      const int id = ld_g(table + at);
      page = id >= 0 && id < a.pages ? id : -1;
    }
  }
  static constexpr int kSteps = 64 / TILES;  // that a fetch is good for
};

// E consecutive outputs of row r from dimension d on: to `out`, or, of a part, to its slot.
template <typename T, int E>
__device__ __forceinline__ void emit(const PageArgs& a, bool whole, int64_t slot, int b, int kvh, int r, int d,
                                     const float (&v)[E], float top, float sum, bool there) {
  const int n = a.heads / a.kv_heads, node = r / n, h = kvh * n + r - node * n;
  if (whole) {
    there = there && sum != 0.f;
    const float inv = there ? 1.f / sum : 0.f;
    T* dst = static_cast<T*>(a.out) + b * a.o_row + node * a.o_node + h * a.o_head + d;
    union {
      T x[E];
      uint4 w4[(E * sizeof(T) + 15) / 16];
      uint2 w2;
      uint32_t w1;
    } u;
#pragma unroll
    for (int e = 0; e < E; ++e) u.x[e] = St<T>::st(there ? v[e] * inv : 0.f);
    if constexpr (E * sizeof(T) >= 16) {
#pragma unroll
      for (int w = 0; w < (int)(E * sizeof(T) / 16); ++w)
        if (d + w * (int)(16 / sizeof(T)) < a.D) reinterpret_cast<uint4*>(dst)[w] = u.w4[w];
    } else if (d < a.D) {
      if constexpr (E * sizeof(T) == 8) *reinterpret_cast<uint2*>(dst) = u.w2;
      else *reinterpret_cast<uint32_t*>(dst) = u.w1;
    }
    if (a.lse != nullptr && d == 0)
      a.lse[((size_t)b * a.tokens + node) * a.heads + h] = there ? fmaf(top, kLn2, logf(sum)) : -INFINITY;
  } else {
    const size_t at = slot * (size_t)(a.tokens * n) + r;
    float* dst = a.part + at * a.D + d;
    if constexpr (E % 4 == 0) {
#pragma unroll
      for (int e = 0; e < E; e += 4)
        if (d + e < a.D) *reinterpret_cast<float4*>(dst + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
    } else if (d < a.D) {
      *reinterpret_cast<float2*>(dst) = make_float2(v[0], v[1]);
    }
    if (d == 0) a.part_ml[at] = make_float2(top, sum);
  }
}

// Whether a row's sum and outputs are numbers.
template <int E>
__device__ __forceinline__ bool all_finite(float l, const f32x4_t (&o)[E]) {
  float top = fabsf(l);
#pragma unroll
  for (int e = 0; e < E; ++e)
#pragma unroll
    for (int r = 0; r < 4; ++r) top = fmaf(0.f, o[e][r], top);  // NaN from either
  return top < INFINITY;
}

// ---- fragments of 8-bit pages ----------------------------------------------------------

// The power of two that brings a magnitude (as bits, finite) into [2^21, 2^22), and its
// inverse.  Magnitudes below 2^-104, whose power would not be finite, count as 0.
constexpr uint32_t kLeastBits = 23u << 23;
__device__ __forceinline__ float to_digits(uint32_t size) {
  return size >= kLeastBits ? __uint_as_float((275u << 23) - (size & 0x7f800000u)) : 0.f;
}
__device__ __forceinline__ float from_digits(uint32_t size) {  // NaN for what is not finite
  return size >= 0x7f800000u ? NAN : size >= kLeastBits ? __uint_as_float((size & 0x7f800000u) - (21u << 23)) : 0.f;
}

// Bytes 0, 1 and 2 of four words.
__device__ __forceinline__ void bytes_of(const uint32_t (&y)[4], uint32_t& b0, uint32_t& b1, uint32_t& b2) {
  const uint32_t p = __builtin_amdgcn_perm(y[1], y[0], 0x05010400u), q = __builtin_amdgcn_perm(y[3], y[2], 0x05010400u);
  b0 = __builtin_amdgcn_perm(q, p, 0x05040100u);
  b1 = __builtin_amdgcn_perm(q, p, 0x07060302u);
  b2 = __builtin_amdgcn_perm(__builtin_amdgcn_perm(y[3], y[2], 0x0c0c0602u), __builtin_amdgcn_perm(y[1], y[0], 0x0c0c0602u),
                             0x05040100u);
}

__device__ __forceinline__ i32x4_t mma8(uint4 a, uint4 b, i32x4_t c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4_t, a), __builtin_bit_cast(i32x4_t, b), c, 0, 0, 0);
}
// 65536 a + 256 b + c of three sums, each below 2^23.
__device__ __forceinline__ float join_digits(int a, int b, int c) { return fmaf((float)a, 65536.f, (float)((b << 8) + c)); }

__device__ __forceinline__ uint32_t max_bits_over_groups(uint32_t x) {  // of lanes i, i + 16, i + 32, i + 48
  auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  x = max((uint32_t)r[0], (uint32_t)r[1]);
  r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  return max((uint32_t)r[0], (uint32_t)r[1]);
}

// Fragments of head dimension DP (64, 128 or 256; D <= DP, a multiple of 16).
template <int DP>
struct CodeFrag {
  static constexpr int KC = DP / 64;  // 16-byte loads of a key row, a lane
  static constexpr int E = DP / 16;   // codes of a V row, a lane
  static constexpr int VW = E / 4;    // the same in registers
  // The lane's byte offsets from a tile's first row on, of K and of V (j: row 4 g + j).  What
  // lies past D is read from the row's start: queries have digits 0 there, outputs no place.
  struct Offsets {
    uint32_t k[KC], v[4];
    __device__ __forceinline__ Offsets(uint32_t slot, int i, int g, int D) {
#pragma unroll
      for (int c = 0; c < KC; ++c) k[c] = i * slot + ((c * 4 + g) * 16 < D ? (c * 4 + g) * 16 : 0);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = (4 * g + j) * slot + (i * E < D ? i * E : 0);
    }
  };
  // Widened where it is used, an offset needs no registers for 64 bits: the load adds it to
  // the uniform base.
  __device__ __forceinline__ static uint32_t here(uint32_t at) {
    asm volatile("" : "+v"(at));
    return at;
  }
  __device__ __forceinline__ static void load_row(const char* base, const Offsets& at, uint4 (&f)[KC]) {
#pragma unroll
    for (int c = 0; c < KC; ++c) f[c] = ld_g16(base + here(at.k[c]));
  }
  __device__ __forceinline__ static void load_v(const char* base, uint32_t at, uint32_t (&f)[VW]) {
    at = here(at);
    if constexpr (VW == 4) {
      const uint4 x = ld_g16(base + at);
      f[0] = x.x, f[1] = x.y, f[2] = x.z, f[3] = x.w;
    } else if constexpr (VW == 2) {
      const uint64_t x = ld_g(reinterpret_cast<const uint64_t*>(base + at));
      f[0] = (uint32_t)x, f[1] = (uint32_t)(x >> 32);
    } else {
      f[0] = ld_g(reinterpret_cast<const uint32_t*>(base + at));
    }
  }
  // Operands of 16 values: three digits, of fp32 three bf16 parts of each eight.
  template <typename T>
  static constexpr int kParts = sizeof(T) == 4 ? 6 : 3;
  // Eight fp32 values as three bf16 operands, whose sum they are (bits below 2^-133 are lost).
  __device__ __forceinline__ static void split(const float* x, uint4 (&p)[3]) {
    uint32_t w[3][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float a = x[2 * j], b = x[2 * j + 1];
#pragma unroll
      for (int e = 0; e < 3; ++e) {
        w[e][j] = Mma<bf16>::pack(a, b);
        a -= Mma<bf16>::low(w[e][j]), b -= Mma<bf16>::high(w[e][j]);
      }
    }
#pragma unroll
    for (int e = 0; e < 3; ++e) p[e] = make_uint4(w[e][0], w[e][1], w[e][2], w[e][3]);
  }
  // One query row: lane group g's 16 KC values in units of f, as digits or in parts, and f.
  template <typename T>
  __device__ __forceinline__ static float query(const T* row, int g, int D, uint4 (&q)[KC][kParts<T>]) {
    float x[KC][16];
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < KC; ++k) {
      const int d = (k * 4 + g) * 16;
      constexpr int kPer = 16 / sizeof(T);
#pragma unroll
      for (int w = 0; w < 16 / kPer; ++w) {
        const uint4 u = d < D ? ld_g16(row + d + w * kPer) : make_uint4(0, 0, 0, 0);
        const uint32_t r[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (sizeof(T) == 4) x[k][w * 4 + j] = __uint_as_float(r[j]);
          else x[k][w * 8 + 2 * j] = Mma<T>::low(r[j]), x[k][w * 8 + 2 * j + 1] = Mma<T>::high(r[j]);
        }
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) top = max(top, __float_as_uint(x[k][j]) & 0x7fffffffu);
    }
    top = max_bits_over_groups(top);
    const float up = top < 0x7f800000u ? to_digits(top) : 0.f;
#pragma unroll
    for (int k = 0; k < KC; ++k) {
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < 16; ++j) x[k][j] *= up;
        uint4 p[3];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          split(x[k] + 8 * h, p);
#pragma unroll
          for (int e = 0; e < 3; ++e) q[k][3 * h + e] = p[e];
        }
      } else {
        uint32_t p[3][4];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          uint32_t y[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) y[j] = (uint32_t)((int)rintf(x[k][w * 4 + j] * up) + 0x808080);  // each digit and 128
          bytes_of(y, p[2][w], p[1][w], p[0][w]);
        }
#pragma unroll
        for (int e = 0; e < 3; ++e)
          q[k][e] = make_uint4(p[e][0] ^ 0x80808080u, p[e][1] ^ 0x80808080u, p[e][2] ^ 0x80808080u, p[e][3] ^ 0x80808080u);
      }
    }
    return from_digits(top);
  }
  // Two codes, byte ea of a and byte eb of b, in bf16, which holds them exactly: the upper halves
  // of their fp32 values.
  __device__ __forceinline__ static uint32_t pair(uint32_t a, int ea, uint32_t b, int eb) {
    const float x = (float)(int8_t)(a >> (8 * ea)), y = (float)(int8_t)(b >> (8 * eb));
    return __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302u);
  }
  __device__ __forceinline__ static uint4 codes8(uint32_t a, uint32_t b) {
    return make_uint4(pair(a, 0, a, 1), pair(a, 2, a, 3), pair(b, 0, b, 1), pair(b, 2, b, 3));
  }
  // Products of the step's four tiles of keys with a row in parts, in units of f; the lane's operand
  // x is at parts[64 x].  Products of parts are exact in fp32; the small ones, below 2^-8 of the others, have sums of
  // their own.
  __device__ __forceinline__ static void scores(const uint4 (&k)[4][KC], const uint4* parts, f32x4_t (&s)[4]) {
    f32x4_t low[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) s[t] = low[t] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < KC; ++c) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint4 q[3];
#pragma unroll
        for (int e = 0; e < 3; ++e) q[e] = parts[(c * 6 + 3 * h + e) * 64];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const uint4 x = h == 0 ? codes8(k[t][c].x, k[t][c].y) : codes8(k[t][c].z, k[t][c].w);
          s[t] = Mma<bf16>::mma(x, q[0], s[t]);
          low[t] = Mma<bf16>::mma(x, q[1], low[t]);
          low[t] = Mma<bf16>::mma(x, q[2], low[t]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) s[t] += low[t];
  }
  // 16 weights, not negative and below 2^22 by `up`: the digits, in the order of the
  // keys.  In [2^23, 2^24) a float's low bits count ones; 0x8080 adds 128 to two digits.
  __device__ __forceinline__ static void digits(const float (&w)[16], float up, uint4& a, uint4& b, uint4& c) {
    uint32_t q[3][4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      uint32_t y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] = __float_as_uint(fmaf(w[t * 4 + j], up, 8388608.f + 32896.f));
      bytes_of(y, q[2][t], q[1][t], q[0][t]);
    }
    a = make_uint4(q[0][0], q[0][1], q[0][2], q[0][3]);
    b = make_uint4(q[1][0] ^ 0x80808080u, q[1][1] ^ 0x80808080u, q[1][2] ^ 0x80808080u, q[1][3] ^ 0x80808080u);
    c = make_uint4(q[2][0] ^ 0x80808080u, q[2][1] ^ 0x80808080u, q[2][2] ^ 0x80808080u, q[2][3] ^ 0x80808080u);
  }
  // o += V^T P^T of fp32 weights: 16 keys of the lane's dimensions, v[4 t + j] and p[4 t + j] of
  // key 16 t + 4 g + j.
  __device__ __forceinline__ static void add_pv(const uint32_t (&v)[16][VW], const float (&p)[16], f32x4_t (&o)[E]) {
    uint4 w[2][3];
#pragma unroll
    for (int h = 0; h < 2; ++h) split(p + 8 * h, w[h]);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      f32x4_t low = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = pair(v[8 * h + 2 * j][e / 4], e % 4, v[8 * h + 2 * j + 1][e / 4], e % 4);
        const uint4 a = make_uint4(x[0], x[1], x[2], x[3]);
        o[e] = Mma<bf16>::mma(a, w[h][0], o[e]);
        low = Mma<bf16>::mma(a, w[h][1], low);
        low = Mma<bf16>::mma(a, w[h][2], low);
      }
      o[e] += low;
      if (e & 1) __builtin_amdgcn_sched_barrier(0);  // values of all dimensions do not fit the registers
    }
  }
  // Codes of dimensions 4 w .. 4 w + 3 of the lane, all 16 keys: operands of the four
  // output tiles.  v[4 t + j]: key 16 t + 4 g + j.
  __device__ __forceinline__ static void transpose(const uint32_t (&v)[16][VW], int w, uint4 (&out)[4]) {
    uint32_t o[4][4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const uint32_t p = __builtin_amdgcn_perm(v[4 * t + 1][w], v[4 * t][w], 0x05010400u);
      const uint32_t q = __builtin_amdgcn_perm(v[4 * t + 3][w], v[4 * t + 2][w], 0x05010400u);
      const uint32_t r = __builtin_amdgcn_perm(v[4 * t + 1][w], v[4 * t][w], 0x07030602u);
      const uint32_t s = __builtin_amdgcn_perm(v[4 * t + 3][w], v[4 * t + 2][w], 0x07030602u);
      o[0][t] = __builtin_amdgcn_perm(q, p, 0x05040100u), o[1][t] = __builtin_amdgcn_perm(q, p, 0x07060302u);
      o[2][t] = __builtin_amdgcn_perm(s, r, 0x05040100u), o[3][t] = __builtin_amdgcn_perm(s, r, 0x07060302u);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) out[e] = make_uint4(o[e][0], o[e][1], o[e][2], o[e][3]);
  }
};

// ---- what both kernels share ------------------------------------------------------------

// The bias by distance of a K/V head's heads: in LDS where it fits, else in memory.
struct BiasTable {
  const float* lds;
  const float* mem;
  int last;  // column of the furthest distances
  bool small;
  __device__ __forceinline__ BiasTable(const PageArgs& a, float* buf, int kvh, int n)
      : lds(buf), mem(a.bias + (size_t)kvh * n * a.buckets), last(a.buckets - 1), small(n * a.buckets <= kBiasLds) {}
  // By the whole block; true if a barrier is due.
  __device__ __forceinline__ bool fill(float* buf, int n, int threads) const {
    if (!small) return false;
    for (int x = threadIdx.x; x < n * (last + 1); x += threads) buf[x] = mem[x];
    return true;
  }
  // use(j, value, in log2 units) for the distances far - off(j), j < J, of query head hq.
  template <int J, class Off, class Use>
  __device__ __forceinline__ void each(int hq, int far, Off&& off, Use&& use) const {
    const int row = hq * (last + 1);
    if (small) {
#pragma unroll
      for (int j = 0; j < J; ++j) use(j, lds[row + min(max(far - off(j), 0), last)] * kLog2e);
    } else {
#pragma unroll
      for (int j = 0; j < J; ++j) use(j, ld_g(mem + row + min(max(far - off(j), 0), last)) * kLog2e);
    }
  }
};

// Joins the waves' outputs at the common maximum and stores the rows.  l: the lane's own
// sums.  In two halves, so that the buffer holds half of the waves' outputs.  No barrier
// waits for loads: those of the next part are on their way.
template <typename T, int W, int NR, int E>
__device__ __forceinline__ void join_waves(const PageArgs& a, const Part& w, int row0, int there_rows, char* lds,
                                           float2 (*ml)[16 * NR], const float (&m)[NR], float (&l)[NR], f32x4_t (&o)[NR][E]) {
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, g = lane >> 4;
  constexpr int H = W / 2;
  f32x4_t* buf = reinterpret_cast<f32x4_t*>(lds);
#pragma unroll
  for (int t = 0; t < NR; ++t) {
    l[t] = sum_over_groups(l[t]);
    if (g == 0) ml[wid][t * 16 + i] = make_float2(m[t], l[t]);
  }
  ring_barrier();  // and the bias in LDS has been read
  float top[NR], sum[NR];
#pragma unroll
  for (int t = 0; t < NR; ++t) {
    top[t] = kNone, sum[t] = 0.f;
#pragma unroll
    for (int x = 0; x < W; ++x) top[t] = fmaxf(top[t], ml[x][t * 16 + i].x);
#pragma unroll
    for (int x = 0; x < W; ++x) sum[t] = fmaf(ml[x][t * 16 + i].y, fade(ml[x][t * 16 + i].x - top[t]), sum[t]);
    const float f = fade(m[t] - top[t]);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      o[t][e] *= f;
      if (wid >= H) buf[((wid - H) * NR * E + t * E + e) * 64 + lane] = o[t][e];
    }
  }
  ring_barrier();
  if (wid < H) {
#pragma unroll
    for (int t = 0; t < NR; ++t)
#pragma unroll
      for (int e = 0; e < E; ++e) buf[(wid * NR * E + t * E + e) * 64 + lane] += o[t][e];
  }
  ring_barrier();
  const int R = a.tokens * (a.heads / a.kv_heads);
#pragma unroll
  for (int t = 0; t < NR; ++t) {
    if (wid / 4 != t % (W / 4)) continue;  // wave x: register x % 4 of every W / 4 th row tile
    const int r = row0 + t * 16 + i, reg = wid & 3, d = (4 * g + reg) * E;
    if (r >= R) continue;
    float v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      v[e] = 0.f;
#pragma unroll
      for (int x = 0; x < H; ++x) v[e] += reinterpret_cast<const float*>(&buf[(x * NR * E + t * E + e) * 64 + lane])[reg];
    }
    emit<T, E>(a, w.all, w.slot, w.b, w.kvh, r, d, v, top[t], sum[t], r < there_rows);
  }
  ring_barrier();  // the buffer is free
}

template <typename T, int DP, int NR, int W>
__global__ MRT_ATTN_BOUNDS(sizeof(T), NR) void k_paged(const PageArgs a) {
  using F = AttnFrag<T, DP>;
  constexpr int E = F::E, VW = F::VW, KC = F::KC, KEYS = 32;
  using Lookup = TileLookup<2>;
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i = lane & 15, g = lane >> 4, D = a.D;
  int row0;
  Walk<KEYS> walk(a, lane, team_of(a, 16 * NR, row0));
  Part w;
  if (!walk.next(a, w)) return;
  const int n = a.heads / a.kv_heads, R = a.tokens * n;
  const int* table;
  const T *kc, *vc;

  // Nothing here needs the length: what lies past it is masked, and so is what has no page,
  // which is read from page 0.
  Lookup look;
  int looked;  // the step of the lookup's first tile
  uint4 kf[2][KC];
  uint32_t vf[8][VW];
  int page[2], place[2];
  auto find = [&](int st) {
    const int x = (st - looked) / W * 2;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      page[h] = __builtin_amdgcn_readlane(look.page, x + h);
      place[h] = __builtin_amdgcn_readlane(look.place, x + h);
    }
  };
  auto load_k = [&] {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      F::load_row(kc + max(page[h], 0) * a.page_stride + (int64_t)(place[h] + i) * a.slot_stride, g, D, kf[h]);
  };
  auto load_v = [&] {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const T* base = vc + max(page[h], 0) * a.page_stride + (int64_t)place[h] * a.slot_stride;
#pragma unroll
      for (int j = 0; j < 4; ++j) F::load_v(base + (4 * g + j) * a.slot_stride, i, D, vf[h * 4 + j]);
    }
  };
  auto request = [&] {  // the first keys of part w
    table = a.table + w.b * a.table_stride;
    kc = static_cast<const T*>(a.k) + w.kvh * a.head_stride;
    vc = static_cast<const T*>(a.v) + w.kvh * a.head_stride;
    looked = w.s0 + wid;
    look.fetch(a, table, looked, W, lane);
    find(looked);
    load_k();
    load_v();
  };
  request();

  for (;;) {
    const int b = w.b, kvh = w.kvh;
    const int len = length_of(a, b), fresh = fresh_of(a, b), end = min(len + fresh, capacity_of(a));
    if (w.open) w.s1 = w.steps = steps_of<KEYS>(a, b);

    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ float2 ml[W][16 * NR];
    float* btab = reinterpret_cast<float*>(lds);  // the bias of this K/V head's heads, until the waves join
    const BiasTable table_of(a, btab, kvh, n);
    uint4 q[NR][KC];
    int last[NR], head[NR];  // the newest entry that the row sees, -1: the row is not there; its query head of the K/V head's
#pragma unroll
    for (int t = 0; t < NR; ++t) {
      const int r = min(row0 + t * 16 + i, R - 1), node = r / n, hq = r - node * n;
      F::load_row(static_cast<const T*>(a.q) + b * a.q_row + node * a.q_node + (int64_t)(kvh * n + hq) * a.q_head, g, D, q[t]);
      last[t] = node < fresh ? len + node : -1, head[t] = hq;
    }
    if (a.bias != nullptr && table_of.fill(btab, n, 64 * W)) ring_barrier();  // does not wait for the loads of the first step

    f32x4_t o[NR][E];
    float m[NR], l[NR];
    auto begin = [&] {
#pragma unroll
      for (int t = 0; t < NR; ++t) {
        m[t] = kNone, l[t] = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) o[t][e] = {0.f, 0.f, 0.f, 0.f};
      }
    };
    begin();
    const float scale2 = a.scale * kLog2e;
    // fp16 weights reach up to 2^15, so that those far below the maximum keep their bits.
    constexpr float kShift = std::is_same_v<T, f16> ? 15.f : 0.f;

    // One step; next() requests the keys of the wave's next one.  A matrix product makes NaN
    // of 0 * inf: infinities and NaN in values that some rows do not see (the new tokens', and
    // with `exact` all) are left out of it and added by class.
    auto step = [&](int st, auto exact, auto&& next) {
      const int base = st * KEYS;
      const bool in[2] = {page[0] >= 0, page[1] >= 0};
      const bool whole = base + KEYS <= len + 1 && fresh > 0 && in[0] && in[1];
      const bool apart = exact.value || (fresh > 1 && base + KEYS > len + 1);
      const int page_v[2] = {page[0], page[1]}, place_v[2] = {place[0], place[1]};
      if (!whole) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int x = 0; x < VW; ++x) vf[j][x] = in[j >> 2] && base + lane_key(g, j) < end ? vf[j][x] : 0u;
      }
      float p[NR][8];
#pragma unroll
      for (int t = 0; t < NR; ++t) {
        const f32x4_t x = F::scores(kf[0], q[t]), y = F::scores(kf[1], q[t]);
        const float s[8] = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
        if (a.bias != nullptr) {
          table_of.template each<8>(head[t], last[t] - base - 4 * g, [](int j) { return lane_key(0, j); }, [&](int j, float by) {
            p[t][j] = by < kNone ? -INFINITY : fmaf(s[j], scale2, by);  // a masked key may hold anything
          });
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) p[t][j] = s[j] * scale2;
        }
        if (!whole) {
          const int most[2] = {in[0] ? last[t] - base - 4 * g : -1, in[1] ? last[t] - base - 4 * g : -1};
#pragma unroll
          for (int j = 0; j < 8; ++j) p[t][j] = lane_key(0, j) <= most[j >> 2] ? p[t][j] : -INFINITY;
        }
      }
      next();
      uint32_t seen[NR];  // the keys that the row does not mask, a bit each
      if (apart) {
#pragma unroll
        for (int t = 0; t < NR; ++t) {
          seen[t] = 0;
#pragma unroll
          for (int j = 0; j < 8; ++j) seen[t] |= p[t][j] < kNone ? 0u : 1u << j;
        }
      }
      running_softmax<NR, E>(p, m, l, o, kShift);
      if (!apart) {
        F::template add_pv<NR>(vf, p, o);
      } else {
        uint32_t diff = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int x = 0; x < VW; ++x) {
            const uint32_t y = F::finite_part(vf[j][x]);
            diff |= y ^ vf[j][x];
            vf[j][x] = y;
          }
        F::template add_pv<NR>(vf, p, o);
        if (__builtin_expect(__any(diff != 0), 0)) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int h = j >> 2;
            const bool have = page_v[h] >= 0 && base + lane_key(g, j) < end;
            if (page_v[h] >= 0)
              F::load_v(vc + page_v[h] * a.page_stride + (int64_t)(place_v[h] + 4 * g + (j & 3)) * a.slot_stride, i, D, vf[j]);
#pragma unroll
            for (int x = 0; x < VW; ++x) vf[j][x] = have ? F::classes(vf[j][x]) : 0u;
          }
#pragma unroll
          for (int t = 0; t < NR; ++t) {
            float one[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) one[j] = (seen[t] >> j) & 1 ? 1.f : 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e) {
              const f32x4_t c = F::count(vf, one, e);
#pragma unroll
              for (int r = 0; r < 4; ++r) o[t][e][r] += F::class_value(c[r]);
            }
          }
        }
      }
    };
    auto steps = [&](auto exact) {
      for (int st = w.s0 + wid; st < w.s1; st += W) {
        const bool more = st + W < w.s1;
        step(st, exact, [&] {
          if (!more) return;
          if (st + W - looked >= Lookup::kSteps * W) {
            looked = st + W;
            look.fetch(a, table, looked, W, lane);
          }
          find(st + W);
          load_k();
        });
        if (more) load_v();
      }
    };
    steps(std::false_type{});
    bool odd = false;
#pragma unroll
    for (int t = 0; t < NR; ++t) odd |= !all_finite<E>(l[t], o[t]) && last[t] >= 0;
    if (__builtin_expect(__any(odd), 0)) {  // rare: this wave's steps once more
      begin();
      request();
      steps(std::true_type{});
    }
    const Part done = w;
    const bool more = walk.next(a, w);
    if (more) request();
    join_waves<T, W, NR, E>(a, done, row0, fresh * n, lds, ml, m, l, o);
    if (!more) break;
  }
}

template <typename T, int DP, int W>
__global__ MRT_ATTN_BOUNDS(1, 1) void k_paged_codes(const PageArgs a) {
  using F = CodeFrag<DP>;
  constexpr int E = F::E, VW = F::VW, KC = F::KC, KEYS = 64, NR = row_tiles(1, DP);
  using Lookup = TileLookup<4>;
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i = lane & 15, g = lane >> 4, D = a.D;
  int row0;
  Walk<KEYS> walk(a, lane, team_of(a, 16 * NR, row0));
  Part w;
  if (!walk.next(a, w)) return;
  const int n = a.heads / a.kv_heads, R = a.tokens * n, page_size = a.page_tiles * kPageUnit;
  const int* table;
  const char *kc, *vc;

  Lookup look;
  int looked;
  uint4 kf[4][KC];
  uint32_t vf[16][VW];
  float ks, vs;  // the scales of key `lane` of the step, of K and of V
  int page[4], place[4];
  auto find = [&](int st) {
    const int x = (st - looked) / W * 4;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      page[t] = __builtin_amdgcn_readlane(look.page, x + t);
      place[t] = __builtin_amdgcn_readlane(look.place, x + t);
    }
  };
  const typename F::Offsets at((uint32_t)a.slot_stride, i, g, D);
  // Keys whose page is not there are read from page 0, and masked.
  auto load_k = [&](int st) {
    const int x = (st - looked) / W * 4 + g;  // of the lane's own key, 16 g + i
    const int pg = __shfl(look.page, x, 64), pl = __shfl(look.place, x, 64);
    const int64_t own = ((int64_t)max(pg, 0) * a.kv_heads + w.kvh) * page_size + pl + i;
    ks = ld_g(a.k_scale + own);
    vs = ld_g(a.v_scale + own);
#pragma unroll
    for (int t = 0; t < 4; ++t) F::load_row(kc + max(page[t], 0) * a.page_stride + place[t] * a.slot_stride, at, kf[t]);
  };
  auto load_v = [&] {
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const char* base = vc + max(page[t], 0) * a.page_stride + place[t] * a.slot_stride;
#pragma unroll
      for (int j = 0; j < 4; ++j) F::load_v(base, at.v[j], vf[4 * t + j]);
    }
  };
  auto request = [&] {
    table = a.table + w.b * a.table_stride;
    kc = static_cast<const char*>(a.k) + w.kvh * a.head_stride;
    vc = static_cast<const char*>(a.v) + w.kvh * a.head_stride;
    looked = w.s0 + wid;
    look.fetch(a, table, looked, W, lane);
    find(looked);
    load_k(looked);
    load_v();
  };
  request();

  for (;;) {
    const int b = w.b, kvh = w.kvh;
    const int len = length_of(a, b), fresh = fresh_of(a, b);
    if (w.open) w.s1 = w.steps = steps_of<KEYS>(a, b);

    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ float2 ml[W][16 * NR];
    __shared__ __attribute__((aligned(16))) float sc[W][128];  // the scales of a wave's step
    float* btab = reinterpret_cast<float*>(lds);
    const BiasTable table_of(a, btab, kvh, n);
    constexpr int kParts = F::template kParts<T>;
    uint4 q[NR][KC][kParts];
    [[maybe_unused]] __shared__ uint4 parts[sizeof(T) == 4 ? NR * KC * kParts * 64 : 1];  // q of fp32, for all waves
    float qf[NR];
    int last[NR], head[NR];
#pragma unroll
    for (int t = 0; t < NR; ++t) {
      const int r = min(row0 + t * 16 + i, R - 1), node = r / n, hq = r - node * n;
      qf[t] = F::query(static_cast<const T*>(a.q) + b * a.q_row + node * a.q_node + (int64_t)(kvh * n + hq) * a.q_head, g, D,
                       q[t]) * a.scale * kLog2e;
      last[t] = node < fresh ? len + node : -1, head[t] = hq;
    }
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int x = 0; x < NR * KC * kParts; ++x)
        if (x % W == wid) parts[x * 64 + lane] = q[x / (KC * kParts)][x / kParts % KC][x % kParts];
    }
    // does not wait for the loads of the first step
    if ((a.bias != nullptr && table_of.fill(btab, n, 64 * W)) || sizeof(T) == 4) ring_barrier();

    f32x4_t o[NR][E];
    float m[NR], l[NR];
#pragma unroll
    for (int t = 0; t < NR; ++t) {
      m[t] = kNone, l[t] = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) o[t][e] = {0.f, 0.f, 0.f, 0.f};
    }
    [[maybe_unused]] const i32x4_t zero = {0, 0, 0, 0};
    // Keys at distances beyond the table's have its last value, unless that is a mask.
    float far[NR];
    bool plain = true;
#pragma unroll
    for (int t = 0; t < NR; ++t) {
      far[t] = 0.f;
      if (a.bias != nullptr)
        table_of.template each<1>(head[t], INT_MAX, [](int) { return 0; }, [&](int, float by) { far[t] = by; });
      plain = plain && far[t] >= kNone;
    }
    const int near = a.bias == nullptr ? INT_MAX : __all(plain) ? len - a.buckets + 2 : 0;  // from here on the table is read

    for (int st = w.s0 + wid; st < w.s1; st += W) {
      const int base = st * KEYS;
      const bool there = page[0] >= 0 && page[1] >= 0 && page[2] >= 0 && page[3] >= 0;
      const bool masks = !there || fresh == 0 || base + KEYS > min(near, len + 1);
      const bool in[4] = {page[0] >= 0, page[1] >= 0, page[2] >= 0, page[3] >= 0};
      const bool more = st + W < w.s1;
      sc[wid][lane] = ks, sc[wid][64 + lane] = vs;  // read by the wave's lanes alone, in order
      __builtin_amdgcn_wave_barrier();
      float p[NR][16];
#pragma unroll
      for (int t = 0; t < NR; ++t) {
        [[maybe_unused]] f32x4_t all[4];
        if constexpr (sizeof(T) == 4) F::scores(kf, parts + t * KC * kParts * 64 + lane, all);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          [[maybe_unused]] i32x4_t x = zero, y = zero, z = zero;
          if constexpr (sizeof(T) != 4) {
#pragma unroll
            for (int c = 0; c < KC; ++c) {
              x = mma8(kf[k][c], q[t][c][0], x);
              y = mma8(kf[k][c], q[t][c][1], y);
              z = mma8(kf[k][c], q[t][c][2], z);
            }
          }
          const float4 s = *reinterpret_cast<const float4*>(&sc[wid][k * 16 + 4 * g]);
          const float by_key[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            if constexpr (sizeof(T) == 4) p[t][4 * k + r] = all[k][r] * qf[t] * by_key[r];
            else p[t][4 * k + r] = join_digits(x[r], y[r], z[r]) * qf[t] * by_key[r];
            asm volatile("" : "+v"(p[t][4 * k + r]));  // here: the sums of all tiles do not fit the registers
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      if (more) {
        if (st + W - looked >= Lookup::kSteps * W) {
          looked = st + W;
          look.fetch(a, table, looked, W, lane);
        }
        find(st + W);
        load_k(st + W);
      }
      [[maybe_unused]] uint4 wa[NR], wb[NR], wc[NR];
      [[maybe_unused]] float wf[NR];
#pragma unroll
      for (int t = 0; t < NR; ++t) {
        float sv[16];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float4 s = *reinterpret_cast<const float4*>(&sc[wid][64 + k * 16 + 4 * g]);
          sv[4 * k] = s.x, sv[4 * k + 1] = s.y, sv[4 * k + 2] = s.z, sv[4 * k + 3] = s.w;
        }
        if (masks) {
          const int upto = last[t] - base - 4 * g;  // the row's newest key, from the lane's first on
          auto key = [](int j) { return (j >> 2) * 16 + (j & 3); };
          if (a.bias != nullptr)
            table_of.template each<16>(head[t], upto, key, [&](int j, float by) {
              p[t][j] = by < kNone ? -INFINITY : p[t][j] + by;
            });
          const int most[4] = {in[0] ? upto : -1, in[1] ? upto : -1, in[2] ? upto : -1, in[3] ? upto : -1};
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const bool out = key(j) > most[j >> 2] || p[t][j] < kNone;
            p[t][j] = out ? -INFINITY : p[t][j];
            sv[j] = out ? 0.f : sv[j];  // a masked entry's scale may be NaN
          }
        } else if (a.bias != nullptr) {
#pragma unroll
          for (int j = 0; j < 16; ++j) p[t][j] += far[t];
        }
        float top = p[t][0];
#pragma unroll
        for (int j = 1; j < 16; ++j) top = fmaxf(top, p[t][j]);
        top = max_over_groups(top);
        if (__any(top > m[t])) {
          asm volatile("");  // a branch: most steps leave the output alone
          const float mn = fmaxf(m[t], top), f = __builtin_amdgcn_exp2f(m[t] - mn);
          m[t] = mn;
          l[t] *= f;
#pragma unroll
          for (int e = 0; e < E; ++e) o[t][e] *= f;
        }
        uint32_t size = 0;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float x = __builtin_amdgcn_exp2f(p[t][j] - m[t]);
          l[t] += x;
          p[t][j] = x * sv[j];
          size = max(size, __float_as_uint(p[t][j]));  // bits of what is not negative order as the values do, NaN above all
        }
        if constexpr (sizeof(T) == 4) {
          F::add_pv(vf, p[t], o[t]);
        } else {
          size = max_bits_over_groups(size);
          F::digits(p[t], to_digits(size), wa[t], wb[t], wc[t]);
          wf[t] = from_digits(size);
        }
      }
      if constexpr (sizeof(T) != 4) {
#pragma unroll
        for (int x = 0; x < VW; ++x) {
          uint4 op[4];
          F::transpose(vf, x, op);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
#pragma unroll
            for (int t = 0; t < NR; ++t) {
              const i32x4_t u = mma8(op[e], wa[t], zero), v = mma8(op[e], wb[t], zero), y = mma8(op[e], wc[t], zero);
#pragma unroll
              for (int r = 0; r < 4; ++r) o[t][4 * x + e][r] = fmaf(join_digits(u[r], v[r], y[r]), wf[t], o[t][4 * x + e][r]);
              asm volatile("" : "+v"(o[t][4 * x + e]));
            }
            if (e & 1) __builtin_amdgcn_sched_barrier(0);
          }
        }
      }
      if (more) load_v();
    }
    const Part done = w;
    const bool again = walk.next(a, w);
    if (again) request();
    join_waves<T, W, NR, E>(a, done, row0, fresh * n, lds, ml, m, l, o);
    if (!again) break;
  }
}

// ---- joining parts ------------------------------------------------------------------------

// A block a row: the row's parts at their common maximum.  `cols` lanes (a power of two, 4
// cols >= D) take a part's outputs, four each; groups of lanes take parts in turn, and are
// summed in order.
template <typename T, int KEYS>
__global__ __launch_bounds__(256) void k_paged_join(const PageArgs a, int cols) {
  const int tid = threadIdx.x, lane = tid & 63, n = a.heads / a.kv_heads, R = a.tokens * n;
  const int unit = blockIdx.x / R, r = blockIdx.x - unit * R, b = unit / a.kv_heads, kvh = unit - b * a.kv_heads;
  // steps of the units of this row, and of all and those before it
  const int own = lane < a.rows ? steps_of<KEYS>(a, lane) : 0, steps = steps_of<KEYS>(a, b);
  if (steps == 0) return;
  const Shares sh = shares_of<KEYS>(a, lane, own);
  int64_t first = lane < b ? a.unit + own : 0;
  for (int x = lane + 64; x < b; x += 64) first += a.unit + steps_of<KEYS>(a, x);
  first = wave_sum64(first) * a.kv_heads + (int64_t)kvh * (a.unit + steps) + a.unit;  // the unit's first step
  const int t0 = sh.of(first), parts = sh.of(first + steps - 1) - t0 + 1;
  if (parts == 1) return;  // written by its block
  first = unit + t0;
  const float2* ml = a.part_ml + first * R + r;
  const int groups = 256 / cols, group = tid / cols, d = tid % cols * 4;
  const float* part = a.part + (first * R + r) * a.D + min(d, a.D - 4);
  float top = kNone;
  for (int s = lane; s < parts; s += 64) top = fmaxf(top, ml[(size_t)s * R].x);
  top = wave_max(top);
  float sum = 0.f;
  for (int s0 = 0; s0 < parts; s0 += 64) {
    const float2 y = s0 + lane < parts ? ml[(size_t)(s0 + lane) * R] : make_float2(kNone, 0.f);
    sum += wave_sum(y.y * fade(y.x - top));
  }
  float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = group; s < parts; s += groups) {
    const float w = fade(ml[(size_t)s * R].x - top);
    const float4 z = *reinterpret_cast<const float4*>(part + (size_t)s * R * a.D);
    v[0] = fmaf(z.x, w, v[0]), v[1] = fmaf(z.y, w, v[1]), v[2] = fmaf(z.z, w, v[2]), v[3] = fmaf(z.w, w, v[3]);
  }
  __shared__ float4 sums[256];
  sums[tid] = make_float4(v[0], v[1], v[2], v[3]);
  __syncthreads();
  if (tid >= cols) return;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = 0.f;
  for (int x = 0; x < groups; ++x) {
    const float4 z = sums[x * cols + tid];
    v[0] += z.x, v[1] += z.y, v[2] += z.z, v[3] += z.w;
  }
  if (d < a.D) emit<T, 4>(a, true, 0, b, kvh, r, d, v, top, sum, r / n < fresh_of(a, b));
}

// ---- host -----------------------------------------------------------------------------------

// Cutting units costs 4 to 8 us: the walk over the lengths, a second join in most blocks, the
// launch of k_paged_join.  Whole units leave a wave up to (rounds of units over the blocks less
// units a block) x steps / waves more steps to read, one after the other, about 10 us for 84 KB.
// So units are cut where it is more than that (codes of d 64 take as long as those of d 128), by
// the table's room, as lengths are not known here.  One token, whole / cut (us): 16 heads of
// d 64 in bf16, 2 sequences of 1000 entries 13.0 / 15.0, of 2400 26.9 / 15.5; 24 of 2400 45.8 /
// 54.0; 8-bit pages, 2 of 1000 12.5 / 15.3, of 2400 24.2 / 15.7; 24 of 2400 33.9 / 39.1.  With
// many units a block they even out: 100 x 16 heads of up to 2400 114.1 / 115.2.
//
// A share has a step a wave at least (two: 2 sequences of 2400, 8 heads of d 128, 8-bit pages,
// 17.8 us for 15.9; 8 of 5000 23.7 for 25.2), and a unit counts as two more (one: 24 sequences of
// up to 8000 62 us, two 54, four 56; in bf16 105, 86, 86).
constexpr int64_t kMoreBytes = 84000;

struct Plan {
  int keys, tiles, row_blocks, teams, least, unit;
};

Plan plan(const PagedCache& c, int heads, int tokens) {
  const int R = tokens * (heads / c.kv_heads), dp = c.d <= 32 && !c.codes ? 32 : c.d <= 64 ? 64 : c.d <= 128 ? 128 : 256;
  const size_t elt = c.codes ? 1 : dtype_size(c.dt);
  Plan p;
  p.keys = c.codes ? 64 : 32;
  p.tiles = std::min(row_tiles(elt, dp), R <= 16 ? 1 : 2);
  p.row_blocks = (R + 16 * p.tiles - 1) / (16 * p.tiles);
  const int64_t units = std::max<int64_t>(1, (int64_t)c.rows * c.kv_heads);
  const int64_t steps = ((int64_t)c.capacity() + p.keys - 1) / p.keys;
  const int waves = waves_of(elt, dp), teams = std::max(8, 256 * blocks_of_cu(elt, dp, p.tiles) / p.row_blocks / 8 * 8);
  p.least = waves;
  const int64_t rounds = (units + teams - 1) / teams, bytes = (int64_t)p.keys * (c.codes ? std::max(dp, 128) : dp) * (int)elt * 2;
  const bool whole = (rounds * steps * teams - units * steps) * bytes <= kMoreBytes * waves * teams || units >= 8 * teams;
  p.unit = whole ? 0 : 2 * waves;
  p.teams = p.unit == 0 ? (int)std::min<int64_t>((units + 7) / 8 * 8, teams) : teams;
  return p;
}

size_t slots_of(const PagedCache& c, const Plan& p) { return (size_t)p.teams + (size_t)c.rows * c.kv_heads; }

template <typename K>
void start(K kernel, int threads, size_t lds, const PageArgs& a, hipStream_t s) {
  lds = std::max(lds, a.bias != nullptr ? (size_t)kBiasLds * 4 : size_t{0});
  allow_dynamic_lds(reinterpret_cast<const void*>(kernel), 96 * 1024);
  hipLaunchKernelGGL(kernel, dim3((unsigned)(a.teams * a.row_blocks)), dim3(threads), lds, s, a);
}

template <typename T, int DP, int NR>
void launch(const PageArgs& a, bool codes, hipStream_t s) {
  if constexpr (NR <= row_tiles(sizeof(T), DP)) {
    if (codes) {
      if constexpr (DP >= 64 && NR <= row_tiles(1, DP)) {
        constexpr int W = waves_of(1, DP);
        start(&k_paged_codes<T, DP, W>, 64 * W, (size_t)W / 2 * NR * (DP / 16) * 1024, a, s);
      }
    } else {
      constexpr int W = waves_of(sizeof(T), DP);
      start(&k_paged<T, DP, NR, W>, 64 * W, (size_t)W / 2 * NR * (DP / 16) * 1024, a, s);
    }
  }
}

}  // namespace

bool paged_attention_fits(const PagedCache& c, int heads, int tokens) {
  const Plan p = plan(c, heads, tokens);
  const int64_t units = (int64_t)c.rows * c.kv_heads, most = (1ll << 32) - 1;  // threads of a launch
  const int R = tokens * (heads / c.kv_heads);
  return (int64_t)p.teams * p.row_blocks * 512 <= most && units * R * 256 <= most;
}

size_t paged_attention_workspace(const PagedCache& c, int heads, int tokens) {
  const Plan p = plan(c, heads, tokens);
  return p.unit == 0 ? 0 : slots_of(c, p) * (size_t)(heads / c.kv_heads * tokens) * (c.d + 2) * 4;
}

void paged_attention(const PagedCache& c, const PagedAttnArgs& t, void* ws, hipStream_t s) {
  const Plan p = plan(c, t.heads, t.tokens);
  PageArgs a{};
  a.q = t.q.p, a.k = c.k, a.v = c.v, a.out = t.out.p, a.k_scale = c.k_scale, a.v_scale = c.v_scale, a.bias = t.bias;
  a.table = c.table, a.length = c.length, a.fresh = t.fresh, a.lse = t.lse;
  a.q_row = t.q.row_stride, a.q_node = t.q.node_stride, a.q_head = t.q.head_stride;
  a.o_row = t.out.row_stride, a.o_node = t.out.node_stride, a.o_head = t.out.head_stride;
  a.page_stride = c.page_stride, a.head_stride = c.head_stride, a.slot_stride = c.slot_stride, a.table_stride = c.table_stride;
  a.page_tiles = c.page_size / kPageUnit, a.by_tiles = Divide(a.page_tiles), a.row_pages = c.row_pages, a.pages = c.pages;
  a.rows = c.rows, a.kv_heads = c.kv_heads, a.heads = t.heads, a.tokens = t.tokens, a.D = c.d, a.buckets = t.buckets;
  a.teams = p.teams, a.unit = p.unit, a.least = p.least, a.row_blocks = p.row_blocks, a.scale = t.scale;
  const int R = t.tokens * (t.heads / c.kv_heads);
  if (p.unit > 0) {
    a.part = static_cast<float*>(ws);
    a.part_ml = reinterpret_cast<float2*>(a.part + slots_of(c, p) * R * c.d);
  }
  MRT_DTYPE_DISPATCH(t.dt, {
    auto tiles = [&](auto width) {
      constexpr int DP = decltype(width)::value;
      if (p.tiles == 1) launch<T, DP, 1>(a, c.codes, s);
      else launch<T, DP, 2>(a, c.codes, s);
    };
    if (c.d <= 32 && !c.codes) tiles(std::integral_constant<int, 32>{});
    else if (c.d <= 64) tiles(std::integral_constant<int, 64>{});
    else if (c.d <= 128) tiles(std::integral_constant<int, 128>{});
    else tiles(std::integral_constant<int, 256>{});
  });
  MRT_HIP_CHECK(hipGetLastError());
  if (p.unit > 0) {
    const int cols = c.d <= 32 ? 8 : c.d <= 64 ? 16 : c.d <= 128 ? 32 : 64;
    const dim3 grid((unsigned)((size_t)c.rows * c.kv_heads * R));
    MRT_DTYPE_DISPATCH(t.dt, {
      if (c.codes) hipLaunchKernelGGL((k_paged_join<T, 64>), grid, dim3(256), 0, s, a, cols);
      else hipLaunchKernelGGL((k_paged_join<T, 32>), grid, dim3(256), 0, s, a, cols);
    });
    MRT_HIP_CHECK(hipGetLastError());
  }
}

}  // namespace mrt

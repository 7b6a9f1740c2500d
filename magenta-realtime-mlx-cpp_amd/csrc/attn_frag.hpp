// Register fragments of attention over cached keys: 32 keys a step, straight from
// memory to the matrix cores without LDS.
//
// A wave holds scores transposed, S^T = K Q^T (keys down, query rows across), so
// that lane (i, g), i = lane & 15, g = lane >> 4, of the two 16-key tiles of a step
// has the scores of query row i with keys 4g .. 4g + 3 (first tile) and 16 + 4g .. 16 +
// 4g + 3 (second).  These eight are just what the second product O^T = V^T P^T reads
// from that lane for the 32 keys, in every type, so P never moves between lanes: the
// order of keys inside that product is free.  V's operand wants eight keys of one
// dimension in a lane; lane (i, g) loads dimensions i E .. i E + E - 1 (E = DP / 16)
// of its eight keys and pairs them with one byte permutation a register: output
// tile t then has dimension i E + t in row i.
//
// The order of dimensions inside Q K^T is free as long as both operands share it.
#pragma once

#include "device_utils.hpp"

namespace mrt {

typedef float f32x4_t __attribute__((ext_vector_type(4)));
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kStepKeys = 32;
// Running maximum before any key, in log2 units: finite, so exp2(-inf - kNone) is 0.  Logits
// and biases below it count as masked, and a row whose sum is 0 has nothing left.
constexpr float kNone = -1e30f;

__device__ __forceinline__ float max_over_groups(float x) {  // of lanes i, i + 16, i + 32, i + 48
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_over_groups(float x) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// Sum over the 16 lanes of a group, in every one of them.
__device__ __forceinline__ float sum_in_group(float v) {
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xB1, 0xf, 0xf, true));   // quad [1,0,3,2]
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4E, 0xf, 0xf, true));   // quad [2,3,0,1]
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x141, 0xf, 0xf, true));  // row_half_mirror
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x140, 0xf, 0xf, true));  // row_mirror
  return v;
}

template <typename T>
struct Mma;
template <>
struct Mma<bf16> {
  typedef __bf16 v8 __attribute__((ext_vector_type(8)));
  __device__ __forceinline__ static f32x4_t mma(uint4 a, uint4 b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
  static constexpr uint32_t kExp = 0x7f80u;  // all ones: infinite or NaN
  // Two values to the type and back, the first in the low half.
  __device__ __forceinline__ static uint32_t pack(float x, float y) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    const f2 v = {x, y};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, b2));
  }
  __device__ __forceinline__ static float low(uint32_t w) { return __uint_as_float(w << 16); }
  __device__ __forceinline__ static float high(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
};
template <>
struct Mma<f16> {
  typedef _Float16 v8 __attribute__((ext_vector_type(8)));
  __device__ __forceinline__ static f32x4_t mma(uint4 a, uint4 b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
  static constexpr uint32_t kExp = 0x7c00u;
  __device__ __forceinline__ static uint32_t pack(float x, float y) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const f2 v = {x, y};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, h2));
  }
  __device__ __forceinline__ static float low(uint32_t w) {
    return (float)__builtin_bit_cast(_Float16, (unsigned short)(w & 0xffffu));
  }
  __device__ __forceinline__ static float high(uint32_t w) {
    return (float)__builtin_bit_cast(_Float16, (unsigned short)(w >> 16));
  }
};
template <>
struct Mma<float> {
  // Four dimensions of each of the four lane groups: exact fp32 products.
  __device__ __forceinline__ static f32x4_t mma(uint4 a, uint4 b, f32x4_t c) {
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.x), __uint_as_float(b.x), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.y), __uint_as_float(b.y), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.z), __uint_as_float(b.z), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.w), __uint_as_float(b.w), c, 0, 0, 0);
  }
};

// Fragments of head dimension DP (32, 64, 128 or 256; D <= DP, a multiple of 8: what
// lies past D is zero).
template <typename T, int DP>
struct AttnFrag {
  static constexpr int kElt = 16 / sizeof(T);           // elements of a 16-byte load
  static constexpr int KC = DP / (4 * kElt);            // 16-byte loads of a key or query row, a lane
  static constexpr int E = DP / 16;                     // V elements of a key, a lane
  static constexpr int VW = E * (int)sizeof(T) / 4;     // the same in registers

  // One key or query row's part of lane group g.
  __device__ __forceinline__ static void load_row(const T* row, int g, int D, uint4 (&f)[KC]) {
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      const int d = (c * 4 + g) * kElt;
      f[c] = (D == DP || d < D) ? ld_g16(row + d) : make_uint4(0, 0, 0, 0);
    }
  }
  // 16 key rows as the cache's lines are read best, four lanes to 64 bytes of a row: lane l
  // loads with load_row(row l / 4, l % 4), and spread() hands each lane (i, g) its part of
  // row i.  Read as the lanes need them, each load asks the L1 for 64 lines instead of 16.
  __device__ __forceinline__ static void spread(uint4 (&f)[KC], int lane) {
    const int from = ((lane & 15) * 4 + (lane >> 4)) * 4;
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      f[c].x = __builtin_amdgcn_ds_bpermute(from, f[c].x), f[c].y = __builtin_amdgcn_ds_bpermute(from, f[c].y);
      f[c].z = __builtin_amdgcn_ds_bpermute(from, f[c].z), f[c].w = __builtin_amdgcn_ds_bpermute(from, f[c].w);
    }
  }
  __device__ __forceinline__ static f32x4_t scores(const uint4 (&k)[KC], const uint4 (&q)[KC]) {
    f32x4_t a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < KC; ++c) a = Mma<T>::mma(k[c], q[c], a);
    return a;
  }
  // Lane i's E elements of a V row.
  __device__ __forceinline__ static void load_v(const T* row, int i, int D, uint32_t (&f)[VW]) {
    const T* p = row + i * E;
    if constexpr (VW >= 4) {
#pragma unroll
      for (int w = 0; w < VW; w += 4) {
        const bool in = D == DP || i * E + w * 4 / (int)sizeof(T) < D;
        const uint4 x = in ? ld_g16(p + w * 4 / sizeof(T)) : make_uint4(0, 0, 0, 0);
        f[w] = x.x, f[w + 1] = x.y, f[w + 2] = x.z, f[w + 3] = x.w;
      }
    } else if constexpr (VW == 2) {
      const bool in = D == DP || i * E < D;
      const uint64_t x = in ? ld_g(reinterpret_cast<const uint64_t*>(p)) : 0ull;
      f[0] = (uint32_t)x, f[1] = (uint32_t)(x >> 32);
    } else {
      f[0] = D == DP || i * E < D ? ld_g(reinterpret_cast<const uint32_t*>(p)) : 0u;
    }
  }
  // Eight weights as a high and a low operand.
  __device__ __forceinline__ static void split(const float (&p)[8], uint4& h, uint4& l) {
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      hi[j] = Mma<T>::pack(p[2 * j], p[2 * j + 1]);
      lo[j] = Mma<T>::pack(p[2 * j] - Mma<T>::low(hi[j]), p[2 * j + 1] - Mma<T>::high(hi[j]));
    }
    h = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    l = make_uint4(lo[0], lo[1], lo[2], lo[3]);
  }
  // o[r][t] += V^T P^T of the lane's eight keys, for every row tile r.  16-bit types:
  // P in two parts, high and low, since rounding P alone to 16 bits would add as much
  // error as the output's own rounding; the parts' sum is within 2^-17 (bf16) of P.
  template <int NR>
  __device__ __forceinline__ static void add_pv(const uint32_t (&v)[8][VW], const float (&p)[NR][8],
                                                f32x4_t (&o)[NR][E]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int t = 0; t < E; ++t)
#pragma unroll
          for (int r = 0; r < NR; ++r)
            o[r][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(v[j][t]), p[r][j], o[r][t], 0, 0, 0);
    } else {
      uint4 ph[NR], pl[NR];
#pragma unroll
      for (int r = 0; r < NR; ++r) split(p[r], ph[r], pl[r]);
#pragma unroll
      for (int t = 0; t < E; ++t) {
        const uint4 a = v_operand(v, t);
#pragma unroll
        for (int r = 0; r < NR; ++r) o[r][t] = Mma<T>::mma(a, ph[r], o[r][t]);
#pragma unroll
        for (int r = 0; r < NR; ++r) o[r][t] = Mma<T>::mma(a, pl[r], o[r][t]);
      }
    }
  }
  // Eight keys of dimension i E + t (16-bit types).
  __device__ __forceinline__ static uint4 v_operand(const uint32_t (&v)[8][VW], int t) {
    const uint32_t sel = t & 1 ? 0x07060302u : 0x05040100u;
    return make_uint4(__builtin_amdgcn_perm(v[1][t / 2], v[0][t / 2], sel),
                      __builtin_amdgcn_perm(v[3][t / 2], v[2][t / 2], sel),
                      __builtin_amdgcn_perm(v[5][t / 2], v[4][t / 2], sel),
                      __builtin_amdgcn_perm(v[7][t / 2], v[6][t / 2], sel));
  }
  // A register of V without its infinities and NaN (zero in their place) ...
  __device__ __forceinline__ static uint32_t finite_part(uint32_t w) {
    if constexpr (sizeof(T) == 4) {
      return (w & 0x7f800000u) == 0x7f800000u ? 0u : w;
    } else {
      constexpr uint32_t hi = Mma<T>::kExp << 16;
      return ((w & Mma<T>::kExp) == Mma<T>::kExp ? 0u : w & 0xffffu) | ((w & hi) == hi ? 0u : w & 0xffff0000u);
    }
  }
  // ... and their classes in the same places: 1 for +inf, 64 for -inf, 4096 for NaN,
  // 0 for the rest.
  __device__ __forceinline__ static uint32_t classes(uint32_t w) {
    if constexpr (sizeof(T) == 4) {
      if ((w & 0x7f800000u) != 0x7f800000u) return 0u;
      return __float_as_uint((w & 0x7fffffu) ? 4096.f : (w >> 31) ? 64.f : 1.f);
    } else {
      uint32_t c = 0;
#pragma unroll
      for (int h = 0; h < 32; h += 16) {
        const uint32_t x = (w >> h) & 0xffffu;
        const bool nan = (x & (0x7fffu & ~Mma<T>::kExp)) != 0;
        if ((x & Mma<T>::kExp) == Mma<T>::kExp) c |= St<T>::bits(nan ? 4096.f : (x >> 15) ? 64.f : 1.f) << h;
      }
      return c;
    }
  }
  // Output tile t of classes times what each row sees (0 or 1): exact counts.
  __device__ __forceinline__ static f32x4_t count(const uint32_t (&cls)[8][VW], const float (&one)[8], int t) {
    f32x4_t c = {0.f, 0.f, 0.f, 0.f};
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(cls[j][t]), one[j], c, 0, 0, 0);
    } else {
      uint32_t b[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) b[j] = St<T>::bits(one[2 * j]) | (St<T>::bits(one[2 * j + 1]) << 16);
      c = Mma<T>::mma(v_operand(cls, t), make_uint4(b[0], b[1], b[2], b[3]), c);
    }
    return c;
  }
  // What a sum over keys with these classes (counted in fp32) adds to an output.
  __device__ __forceinline__ static float class_value(float count) {
    const int n = (int)count;
    const float a = n & 63 ? INFINITY : 0.f, b = (n >> 6) & 63 ? -INFINITY : 0.f;
    return n >= 4096 ? NAN : a + b;
  }
};

// Key (of a step's 32) of row i of its first (half 0) or second 16-key tile, and of
// element j of lane group g's eight scores.
__device__ __forceinline__ int step_key(int i, int half) { return i + 16 * half; }
__device__ __forceinline__ int lane_key(int g, int j) { return 4 * g + (j & 3) + (j >> 2) * 16; }

// Column of the bias by distance: positions may lie further apart than 31 bits count.
__device__ __forceinline__ int bucket(int from, int to, int buckets) {
  return min(max(__builtin_elementwise_sub_sat(from, to), 0), buckets - 1);
}

// The factor 2^x, x <= 0, by which sums and outputs follow a larger maximum.  At least the
// smallest normal number: 0 would make NaN of an infinite value, whose weight is small but
// not 0; finite sums, of at least 2^-8, take in 2^-126 of others without a trace.
__device__ __forceinline__ float fade(float x) { return fmaxf(__builtin_amdgcn_exp2f(x), 0x1p-126f); }

// One step of the running softmax of NR row tiles: s, the logits in log2 units (-inf
// where masked), become weights exp2(s - m); m, l and o follow.  m is the maximum less
// `shift`, uniform over the lanes of a row; l stays a sum of the lane's own keys.
template <int NR, int E>
__device__ __forceinline__ void running_softmax(float (&s)[NR][8], float (&m)[NR], float (&l)[NR], f32x4_t (&o)[NR][E],
                                                float shift) {
#pragma unroll
  for (int t = 0; t < NR; ++t) {
    float top = s[t][0];
#pragma unroll
    for (int j = 1; j < 8; ++j) top = fmaxf(top, s[t][j]);
    top = max_over_groups(top) - shift;
    if (__any(top > m[t])) {
      const float mn = fmaxf(m[t], top), f = fade(m[t] - mn);
      m[t] = mn;
      l[t] *= f;
#pragma unroll
      for (int e = 0; e < E; ++e) o[t][e] *= f;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      s[t][j] = __builtin_amdgcn_exp2f(s[t][j] - m[t]);
      l[t] += s[t][j];
    }
  }
}

}  // namespace mrt

// Matrix-vector products with 4-bit weights: y = x W^T, W[n][k] = s[n][g] code + b[n][g]
// for groups of 32, 64 or 128 k.
//
// Few rows of x meet each weight once, so the weights' bytes bound the product and
// the codes go to the matrix cores as they are:
//   y_n = sum_g s_g sum_k (16 + code_k) x_k + (b_g - 16 s_g) sum_k x_k
// 16 + code is exact in bf16 and fp16 and costs one shift and one and-or for two codes
// (in [16, 32) a step of 1 is the bits 3..6 of bf16, 6..9 of fp16), products with x
// are exact in fp32, and a group's sum is scaled in fp32; the sums of x come from the
// same instruction with an operand of ones, in the lanes that need them.
//
// The two terms cancel where x has a mean: one as large as its deviation puts y off by 8e-6
// (norm-wise; k 2048, groups of 128), a product with the weights in fp32 by 3e-7.  Rounding y
// to bf16 takes 240 times that, to fp16 30 times, but fp32 results have codes around 0,
//   y_n = sum_g s_g sum_k (code_k - 7.5) x_k + (b_g + 7.5 s_g) sum_k x_k
// from tables of bytes (18 instructions for eight codes instead of 7), which puts y off by
// 4e-7: 5 x 1024 by 29824 13.0 us instead of 12.2.  fp32 rows are split exactly into three bf16
// parts.  In bf16 and fp32 the codes, and so all sums, are 2^-12 or 2^-11 of what they stand
// for until the end, so that terms that cancel do not overflow where y does not (and y below
// 2^-114 loses bits).
//
// A block takes 16 NT output columns (matrix-core rows), its waves chunks of 128 k in
// turn, summed through LDS in order.  A lane loads 32 codes (16 bytes) of one row; two
// exchanges between lane halves and two between quarters turn that into the operand
// order in which each instruction's 32 k are consecutive, so within one group.
// Reached: 2 x 1024 by 5632 (3.3 MB, bf16) 5 us, most of it one trip to memory and the sums
// of the waves; 5 x 1024 by 29824 in fp32 (23.5 MB) 13 us; 9 x 8192 by 28672 (125 MB) 38 us,
// 3.3 TB/s: a block a CU (its registers), whose loads and products take turns.  Two blocks
// by fewer registers spill (47 us), codes two slabs ahead gain nothing (43).
#include <algorithm>
#include <type_traits>

#include "attn_frag.hpp"
#include "mfma_ring.hpp"
#include "q4.hpp"

namespace mrt {
namespace {

constexpr int kQ4Waves = 8;
constexpr int kChunk = 128;
constexpr int kSlab = kQ4Waves * kChunk;      // k in LDS at a time: a chunk a wave
// LDS up to which a second slab saves a barrier, two blocks to a CU: 9 x 8192 by 28672 38.3
// us instead of 40.7, 16 x 4096 by 8192 9.1 instead of 10.0.
constexpr size_t kTwoSlabs = 80 * 1024;
// Blocks that fill the card; with more, a block takes two or four column tiles and x is
// read less often: 2 x 1024 by 8192 with one / two / four tiles 4.9 / 4.4 / 5.7 us, by 29824
// one / four 13.3 / 9.7, 9 x 8192 by 28672 47.7 / 38.8, 40 x 4096 by 16384 one / two 57 / 44.
constexpr int kFill = 256;

struct Q4Args {
  const uint32_t* w;
  const void *scales, *biases, *x;
  void* y;
  int64_t ldx, ldy;
  int n, k, groups, rows;
  int bufs;   // slabs of x in LDS
  bool wide;  // y rows take 4-element stores
};

// Operands of the matrix instruction: parts of x (1, or 3 bf16 parts of fp32) in the
// order of the codes: 0 4 1 5 2 6 3 7 of eight consecutive k, in fp32 0 2 4 6 1 3 5 7.
template <typename T>
struct Q4Op {
  static constexpr int kParts = 1;
  static constexpr uint32_t kOnes = std::is_same_v<T, f16> ? 0x3c003c00u : 0x39803980u;  // 1, 2^-12
  static constexpr float kUp = std::is_same_v<T, f16> ? 1.f : 4096.f;
  static constexpr float kOffset = -16.f;  // of a code, from what its operand stands for
  typedef uint4 Raw;  // eight values of x as they are in memory
  using M = Mma<T>;
  struct X {
    uint4 part[1];
  };
  // 16 (in bf16 2^-8) in both halves, in a register: one and-or instead of two instructions with literals.
  __device__ __forceinline__ static uint32_t offset() {
    uint32_t v = std::is_same_v<T, f16> ? 0x4c004c00u : 0x3b803b80u;
    asm("" : "+v"(v));
    return v;
  }
  __device__ __forceinline__ static uint4 codes(uint32_t w, uint32_t o) {
    if constexpr (std::is_same_v<T, f16>) {
      uint32_t m = 0x03c003c0u;
      asm("" : "+s"(m));
      return make_uint4(((w << 6) & m) | o, ((w << 2) & m) | o, ((w >> 2) & m) | o, ((w >> 6) & m) | o);
    } else {
      uint32_t m = 0x00780078u;
      asm("" : "+s"(m));
      return make_uint4(((w << 3) & m) | o, ((w >> 1) & m) | o, ((w >> 5) & m) | o, ((w >> 9) & m) | o);
    }
  }
  __device__ __forceinline__ static Raw raw(const T* p, bool in) { return in ? ld_g16(p) : make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ static X split(const Raw& v) {
    X x;
    x.part[0] = make_uint4(__builtin_amdgcn_perm(v.z, v.x, 0x05040100u), __builtin_amdgcn_perm(v.z, v.x, 0x07060302u),
                           __builtin_amdgcn_perm(v.w, v.y, 0x05040100u), __builtin_amdgcn_perm(v.w, v.y, 0x07060302u));
    return x;
  }
};
template <>
struct Q4Op<float> {
  static constexpr int kParts = 3;
  static constexpr uint32_t kOnes = 0x3a003a00u;  // 2^-11
  static constexpr float kUp = 2048.f;
  static constexpr float kOffset = 7.5f;
  struct Raw {
    uint4 a, b;
  };
  using M = Mma<bf16>;
  struct X {
    uint4 part[3];
  };
  __device__ __forceinline__ static uint32_t offset() { return 0; }
  // (code - 7.5) 2^-11 = (2 code - 15) 2^-12 in bf16: sign, exponent and significant bits of the
  // odd numbers 1 .. 15 from tables of their two bytes, by l = (magnitude - 1) / 2, which is the
  // code's low three bits, and below 8 those inverted.
  __device__ __forceinline__ static uint4 codes(uint32_t w, uint32_t) {
    const uint32_t neg = ~w & 0x88888888u, l = w ^ (neg - (neg >> 3));
    uint32_t v[4];
#pragma unroll
    for (int odd = 0; odd < 2; ++odd) {
      const uint32_t at = (odd ? l >> 4 : l) & 0x07070707u;
      const uint32_t high = __builtin_amdgcn_perm(0x3b3b3b3bu, 0x3a3a3a39u, at) | ((odd ? neg : neg << 4) & 0x80808080u);
      const uint32_t low = __builtin_amdgcn_perm(0x70503010u, 0xe0a04080u, at);
      v[2 * odd] = __builtin_amdgcn_perm(high, low, 0x05010400u);
      v[2 * odd + 1] = __builtin_amdgcn_perm(high, low, 0x07030602u);
    }
    return make_uint4(v[0], v[1], v[2], v[3]);
  }
  __device__ __forceinline__ static Raw raw(const float* p, bool in) {
    return {in ? ld_g16(p) : make_uint4(0, 0, 0, 0), in ? ld_g16(p + 4) : make_uint4(0, 0, 0, 0)};
  }
  // Three times the upper 8 of the significant bits that are left.
  __device__ __forceinline__ static X split(const Raw& r) {
    uint4 a = r.a, b = r.b;
    X o;
#pragma unroll
    for (int c = 0; c < 3; ++c) {
      o.part[c] = make_uint4(__builtin_amdgcn_perm(a.z, a.x, 0x07060302u), __builtin_amdgcn_perm(b.z, b.x, 0x07060302u),
                             __builtin_amdgcn_perm(a.w, a.y, 0x07060302u), __builtin_amdgcn_perm(b.w, b.y, 0x07060302u));
      a = make_uint4(rest(a.x), rest(a.y), rest(a.z), rest(a.w)), b = make_uint4(rest(b.x), rest(b.y), rest(b.z), rest(b.w));
    }
    return o;
  }
  __device__ __forceinline__ static uint32_t rest(uint32_t x) {
    return __float_as_uint(__uint_as_float(x) - __uint_as_float(x & 0xffff0000u));
  }
};

__device__ __forceinline__ void swap32(uint32_t& a, uint32_t& b) {
  const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
  a = r[0], b = r[1];
}
__device__ __forceinline__ void swap16(uint32_t& a, uint32_t& b) {
  const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
  a = r[0], b = r[1];
}

// What a thread loads for a slab, a slab ahead: its lane's codes (16 bytes of row l / 4,
// so that four lanes share 64 consecutive bytes), and its shares of the scales, biases and
// x, which the block puts into LDS.
template <typename T, int MT, int G, int NT>
struct Q4Load {
  static constexpr int S = (16 * NT * kQ4Waves * G + 64 * kQ4Waves - 1) / (64 * kQ4Waves);
  static constexpr int X = MT * 16 * (kSlab / 8) / (64 * kQ4Waves);
  uint4 w[NT];
  T s[S], b[S];
  typename Q4Op<T>::Raw x[X];
};

// GT: instructions (32 k) a group.  MT: 16-row tiles of x.
template <typename T, int MT, int GT, int NT>
__global__ __launch_bounds__(64 * kQ4Waves) void k_q4(const Q4Args a) {
  using Op = Q4Op<T>;
  constexpr int G = 4 / GT, P = Op::kParts;  // groups of a chunk; parts of x
  constexpr int kThreads = 64 * kQ4Waves, kRows = 16 * NT;
  using Load = Q4Load<T, MT, G, NT>;
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i = lane & 15, g = lane >> 4, n0 = blockIdx.x * kRows, m0 = blockIdx.y * 16 * MT;
  const int words = a.k / 8, chunks = (a.k + kChunk - 1) / kChunk, cols = min(a.rows - m0, 16 * MT);
  const int slab_chunks = min(kQ4Waves, chunks), pieces = slab_chunks * kChunk / 8;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  // LDS, `bufs` times: x as operands, 16 bytes of (instruction, part, row, lane group);
  // scale and offset of (group of the slab, row).
  const int x16 = pieces / 4 * P * cols * 4, buf16 = x16 + kQ4Waves * G * kRows / 2;

  const uint32_t* wrow[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) wrow[t] = a.w + (int64_t)min(n0 + t * 16 + (lane >> 2), a.n - 1) * words;
  auto load = [&](int c0) {
    Load l;
    // past the end: the row's last codes, against zeros of x
    const int at = min((c0 + wid) * 16 + (lane & 3) * 4, words - 4);
#pragma unroll
    for (int z = 0; z < Load::S; ++z) {
      const int e = tid + z * kThreads, row = e / (slab_chunks * G), gi = c0 * G + e - row * (slab_chunks * G);
      const int64_t from = (int64_t)min(n0 + min(row, kRows - 1), a.n - 1) * a.groups + min(gi, a.groups - 1);
      l.s[z] = ld_g(static_cast<const T*>(a.scales) + from);
      l.b[z] = ld_g(static_cast<const T*>(a.biases) + from);
    }
#pragma unroll
    for (int z = 0; z < Load::X; ++z) {
      const int e = tid + z * kThreads, m = e / pieces, k = c0 * kChunk + (e - m * pieces) * 8;
      l.x[z] = Op::raw(static_cast<const T*>(a.x) + (int64_t)(m0 + m) * a.ldx + k, m < cols && k < a.k);
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) l.w[t] = ld_nt16(wrow[t] + at);
    return l;
  };
  Load next = load(0);

  f32x4_t y[NT][MT];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int m = 0; m < MT; ++m) y[t][m] = {0.f, 0.f, 0.f, 0.f};
  const uint4 ones = make_uint4(Op::kOnes, Op::kOnes, Op::kOnes, Op::kOnes);
  const uint32_t offset = Op::offset();
  const int pull = (i * 4 + g) * 4;  // the lane with row i's codes of lane group g

  int buf = 0;
  for (int c0 = 0; c0 < chunks; c0 += kQ4Waves) {
    uint4* xl = reinterpret_cast<uint4*>(lds) + buf * buf16;
    float2* sc = reinterpret_cast<float2*>(xl + x16);
    if (c0 > 0 && a.bufs == 1) ring_barrier();
#pragma unroll
    for (int z = 0; z < Load::S; ++z) {
      const int e = tid + z * kThreads, row = e / (slab_chunks * G), q = e - row * (slab_chunks * G);
      const float s = St<T>::ld(next.s[z]), b = St<T>::ld(next.b[z]);
      if (row < kRows) sc[q * kRows + row] = make_float2(s, fmaf(Op::kOffset, s, b));
    }
#pragma unroll
    for (int z = 0; z < Load::X; ++z) {
      const int e = tid + z * kThreads, m = e / pieces, p = e - m * pieces;
      const typename Op::X x = Op::split(next.x[z]);
      if (m < cols) {
#pragma unroll
        for (int c = 0; c < P; ++c) xl[((p / 4 * P + c) * cols + m) * 4 + (p & 3)] = x.part[c];
      }
    }
    uint32_t wd[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t) wd[t][0] = next.w[t].x, wd[t][1] = next.w[t].y, wd[t][2] = next.w[t].z, wd[t][3] = next.w[t].w;
    if (c0 + kQ4Waves < chunks) next = load(c0 + kQ4Waves);
    ring_barrier();
    if (c0 + wid < chunks) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int z = 0; z < 4; ++z) wd[t][z] = __builtin_amdgcn_ds_bpermute(pull, wd[t][z]);
        swap32(wd[t][0], wd[t][2]);
        swap32(wd[t][1], wd[t][3]);
        swap16(wd[t][0], wd[t][1]);
        swap16(wd[t][2], wd[t][3]);
      }
      const uint4* xw[MT];
#pragma unroll
      for (int m = 0; m < MT; ++m) xw[m] = xl + wid * 4 * P * cols * 4 + min(m * 16 + i, cols - 1) * 4 + g;
#pragma unroll
      for (int q = 0; q < G; ++q) {
        f32x4_t p[NT][MT], sum[MT];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          sum[m] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int t = 0; t < NT; ++t) p[t][m] = {0.f, 0.f, 0.f, 0.f};
        }
#pragma unroll
        for (int z = 0; z < GT; ++z) {
          const int step = q * GT + z;
          uint4 code[NT];
#pragma unroll
          for (int t = 0; t < NT; ++t) code[t] = Op::codes(wd[t][step], offset);
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int c3 = 0; c3 < P; ++c3) {
              const uint4 x = xw[m][(step * P + c3) * cols * 4];
              sum[m] = Op::M::mma(ones, x, sum[m]);
#pragma unroll
              for (int t = 0; t < NT; ++t) p[t][m] = Op::M::mma(code[t], x, p[t][m]);
            }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const float4* at = reinterpret_cast<const float4*>(sc + (wid * G + q) * kRows + t * 16 + g * 4);
          const float4 u = at[0], v = at[1];
          const float s[4] = {u.x, u.z, v.x, v.z}, o[4] = {u.y, u.w, v.y, v.w};
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int r = 0; r < 4; ++r) y[t][m][r] += fmaf(s[r], p[t][m][r], o[r] * sum[m][r]);
        }
      }
    }
    buf ^= a.bufs - 1;
  }

  ring_barrier();
  f32x4_t* sums = reinterpret_cast<f32x4_t*>(lds);
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int m = 0; m < MT; ++m) sums[((wid * NT + t) * MT + m) * 64 + lane] = y[t][m];
  ring_barrier();
  for (int z = wid; z < NT * MT; z += kQ4Waves) {
    const int t = z / MT, m = z - t * MT, row = m0 + m * 16 + i, col = n0 + t * 16 + g * 4;
    f32x4_t v = sums[z * 64 + lane];
#pragma unroll
    for (int w = 1; w < kQ4Waves; ++w) v += sums[(w * NT * MT + z) * 64 + lane];
    if (row >= a.rows) continue;
    T* dst = static_cast<T*>(a.y) + row * a.ldy + col;
    union {
      T x[4];
      uint4 w4;
      uint2 w2;
    } u;
#pragma unroll
    for (int r = 0; r < 4; ++r) u.x[r] = St<T>::st(v[r] * Op::kUp);
    if (a.wide && col + 4 <= a.n) {
      if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(dst) = u.w4;
      else *reinterpret_cast<uint2*>(dst) = u.w2;
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (col + r < a.n) dst[r] = u.x[r];
    }
  }
}

template <typename T, int MT, int GT, int NT>
void launch(Q4Args a, hipStream_t s) {
  const size_t slab = (size_t)std::min(kSlab, (a.k + kChunk - 1) / kChunk * kChunk) * std::min(a.rows, 16 * MT) * 2 * Q4Op<T>::kParts +
                      (size_t)kQ4Waves * (4 / GT) * 16 * NT * 8;
  a.bufs = a.k > kSlab && 2 * slab <= kTwoSlabs ? 2 : 1;
  const size_t lds = std::max((size_t)kQ4Waves * NT * MT * 64 * 16, slab * a.bufs);
  const dim3 grid((a.n + 16 * NT - 1) / (16 * NT), (a.rows + 16 * MT - 1) / (16 * MT));
  allow_dynamic_lds(reinterpret_cast<const void*>(&k_q4<T, MT, GT, NT>), 160 * 1024);
  hipLaunchKernelGGL((k_q4<T, MT, GT, NT>), grid, dim3(64 * kQ4Waves), lds, s, a);
}

template <typename T, int MT, int NT>
void launch_group(const Q4Args& a, int group, hipStream_t s) {
  if (group == 32) launch<T, MT, 1, NT>(a, s);
  else if (group == 64) launch<T, MT, 2, NT>(a, s);
  else launch<T, MT, 4, NT>(a, s);
}

template <typename T, int MT>
void launch_tiles(const Q4Args& a, int group, hipStream_t s) {
  const int tiles = (a.n + 15) / 16;
  if constexpr (MT == 1)
    if (tiles >= 4 * kFill) return launch_group<T, MT, 4>(a, group, s);
  if (tiles >= 2 * kFill) launch_group<T, MT, 2>(a, group, s);
  else launch_group<T, MT, 1>(a, group, s);
}

// Eight weights a thread, group / 8 threads a group: bias = least weight, scale = a
// 15th of the range, both rounded to the type before the codes are taken.  Codes cannot hold
// infinities or NaN: a group with any is NaN.
template <typename T>
__global__ __launch_bounds__(256) void k_q4_quantize(const T* src, int64_t ld, int64_t total, int k, int group,
                                                     uint32_t* w, T* scales, T* biases) {
  using S = St<T>;
  const int64_t word = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int words = k / 8, span = group / 8;
  const int64_t at = min(word, total - 1), row = at / words;
  const int c = (int)(at - row * words);
  float v[8], lo = INFINITY, hi = -INFINITY;
  int odd = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    v[j] = S::ld(src[row * ld + c * 8 + j]);
    lo = fminf(lo, v[j]), hi = fmaxf(hi, v[j]), odd |= !(fabsf(v[j]) < INFINITY);
  }
  for (int o = 1; o < span; o <<= 1)
    lo = fminf(lo, __shfl_xor(lo, o, 64)), hi = fmaxf(hi, __shfl_xor(hi, o, 64)), odd |= __shfl_xor(odd, o, 64);
  const float scale = odd ? NAN : S::rnd((hi - lo) / 15.f), bias = odd ? NAN : S::rnd(lo);
  uint32_t code = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float q = scale > 0.f ? fminf(fmaxf(rintf((v[j] - bias) / scale), 0.f), 15.f) : 0.f;
    code |= (uint32_t)q << (4 * j);
  }
  if (word >= total) return;
  w[word] = code;
  if (c % span == 0) {
    scales[row * (k / group) + c / span] = S::st(scale);
    biases[row * (k / group) + c / span] = S::st(bias);
  }
}

}  // namespace

void q4_matmul(DType dt, const Q4Weights& w, const void* x, int64_t ldx, int rows, void* y, int64_t ldy, hipStream_t s) {
  Q4Args a{};
  a.w = w.w, a.scales = w.scales, a.biases = w.biases, a.x = x, a.y = y, a.ldx = ldx, a.ldy = ldy;
  a.n = w.n, a.k = w.k, a.groups = w.k / w.group, a.rows = rows;
  const size_t unit = 4 * dtype_size(dt);
  a.wide = reinterpret_cast<uintptr_t>(y) % unit == 0 && ldy % 4 == 0;
  MRT_DTYPE_DISPATCH(dt, {
    if constexpr (std::is_same_v<T, float>) {
      launch_tiles<T, 1>(a, w.group, s);
    } else {
      if (rows <= 16) launch_tiles<T, 1>(a, w.group, s);
      else if (rows <= 32) launch_tiles<T, 2>(a, w.group, s);
      else launch_tiles<T, 4>(a, w.group, s);
    }
  });
  MRT_HIP_CHECK(hipGetLastError());
}

void q4_quantize(DType dt, const void* src, int64_t ld, int n, int k, int group, uint32_t* w, void* scales, void* biases,
                 hipStream_t s) {
  const int64_t total = (int64_t)n * (k / 8);
  const dim3 grid((unsigned)((total + 255) / 256));
  MRT_DTYPE_DISPATCH(dt, hipLaunchKernelGGL(k_q4_quantize<T>, grid, dim3(256), 0, s, (const T*)src, ld, total, k, group, w,
                                            (T*)scales, (T*)biases));
  MRT_HIP_CHECK(hipGetLastError());
}

}  // namespace mrt

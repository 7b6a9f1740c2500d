// Matrix-vector products with 4-bit weights: y = x W^T, W[n][k] = s[n][g] code + b[n][g]
// for groups of 32, 64 or 128 k.
//
// Few rows of x meet each weight once, so the weights' bytes bound the product and
// the codes go to the matrix cores as they are:
//   y_n = sum_g s_g sum_k (16 + code_k) x_k + (b_g - 16 s_g) sum_k x_k
// 16 + code is exact in bf16 and fp16 and costs one shift and one and-or for two codes
// (in [16, 32) a step of 1 is the bits 3..6 of bf16, 6..9 of fp16), products with x
// are exact in fp32, and a group's sum is scaled in fp32; the sums of x come from the
// same instruction with an operand of ones, in the lanes that need them.  The offset
// makes a group's sum about 5 times its part without it: 2 bits of the 24.
// fp32 activations are split exactly into three bf16 parts.
//
// A block takes 16 NT output columns (matrix-core rows), its waves chunks of 128 k in
// turn, summed through LDS in order.  A lane loads 32 codes (16 bytes) of one row; two
// exchanges between lane halves and two between quarters turn that into the operand
// order in which each instruction's 32 k are consecutive, so within one group.
#include <algorithm>

#include "attn_frag.hpp"
#include "q4.hpp"

namespace mrt {
namespace {

constexpr int kQ4Waves = 8;
constexpr int kChunk = 128;

struct Q4Args {
  const uint32_t* w;
  const void *scales, *biases, *x;
  void* y;
  int64_t ldx, ldy;
  int n, k, groups, rows;
  bool wide;  // y rows take 4-element stores
};

// Operands of the matrix instruction: parts of x (1, or 3 bf16 parts of fp32) in the
// order of the codes: 0 4 1 5 2 6 3 7 of eight consecutive k.
template <typename T>
struct Q4Op {
  static constexpr int kParts = 1;
  static constexpr uint32_t kOnes = sizeof(T) == 2 && std::is_same_v<T, f16> ? 0x3c003c00u : 0x3f803f80u;
  typedef T Raw;
  using M = Mma<T>;
  struct X {
    uint4 part[1];
  };
  __device__ __forceinline__ static uint4 codes(uint32_t w) {
    if constexpr (std::is_same_v<T, f16>)
      return make_uint4(((w << 6) & 0x03c003c0u) | 0x4c004c00u, ((w << 2) & 0x03c003c0u) | 0x4c004c00u,
                        ((w >> 2) & 0x03c003c0u) | 0x4c004c00u, ((w >> 6) & 0x03c003c0u) | 0x4c004c00u);
    else
      return make_uint4(((w << 3) & 0x00780078u) | 0x41804180u, ((w >> 1) & 0x00780078u) | 0x41804180u,
                        ((w >> 5) & 0x00780078u) | 0x41804180u, ((w >> 9) & 0x00780078u) | 0x41804180u);
  }
  __device__ __forceinline__ static X load(const T* p, bool in) {
    const uint4 v = in ? ld_g16(p) : make_uint4(0, 0, 0, 0);
    X x;
    x.part[0] = make_uint4(__builtin_amdgcn_perm(v.z, v.x, 0x05040100u), __builtin_amdgcn_perm(v.z, v.x, 0x07060302u),
                           __builtin_amdgcn_perm(v.w, v.y, 0x05040100u), __builtin_amdgcn_perm(v.w, v.y, 0x07060302u));
    return x;
  }
};
template <>
struct Q4Op<float> {
  static constexpr int kParts = 3;
  static constexpr uint32_t kOnes = 0x3f803f80u;
  using M = Mma<bf16>;
  struct X {
    uint4 part[3];
  };
  __device__ __forceinline__ static uint4 codes(uint32_t w) { return Q4Op<bf16>::codes(w); }
  __device__ __forceinline__ static X load(const float* p, bool in) {
    const uint4 a = in ? ld_g16(p) : make_uint4(0, 0, 0, 0), b = in ? ld_g16(p + 4) : make_uint4(0, 0, 0, 0);
    const uint32_t lo[4] = {a.x, a.y, a.z, a.w}, hi[4] = {b.x, b.y, b.z, b.w};
    uint32_t out[3][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float x = __uint_as_float(lo[j]), y = __uint_as_float(hi[j]);
#pragma unroll
      for (int c = 0; c < 3; ++c) {
        const uint32_t u = f2bf(x), v = f2bf(y);
        out[c][j] = u | (v << 16);
        x -= bf2f(u), y -= bf2f(v);
      }
    }
    X r;
#pragma unroll
    for (int c = 0; c < 3; ++c) r.part[c] = make_uint4(out[c][0], out[c][1], out[c][2], out[c][3]);
    return r;
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

// GT: instructions (32 k) a group.  MT: 16-row tiles of x.
template <typename T, int MT, int GT, int NT>
__global__ __launch_bounds__(64 * kQ4Waves) void k_q4(const Q4Args a) {
  using Op = Q4Op<T>;
  constexpr int G = 4 / GT;  // groups of a chunk
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i = lane & 15, g = lane >> 4, n0 = blockIdx.x * 16 * NT, m0 = blockIdx.y * 64;
  const int words = a.k / 8, chunks = (a.k + kChunk - 1) / kChunk;
  __shared__ float2 sc[kQ4Waves][NT][4][16];  // scale and offset of a wave's chunk: group, row
  __shared__ f32x4_t buf[kQ4Waves][NT][MT][64];

  const uint32_t* wrow[NT];
  const T *srow[NT], *brow[NT], *xrow[MT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int64_t row = min(n0 + t * 16 + i, a.n - 1);
    wrow[t] = a.w + row * words + g * 4;
    srow[t] = static_cast<const T*>(a.scales) + row * a.groups;
    brow[t] = static_cast<const T*>(a.biases) + row * a.groups;
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) xrow[t] = static_cast<const T*>(a.x) + (int64_t)min(m0 + t * 16 + i, a.rows - 1) * a.ldx + g * 8;

  f32x4_t y[NT][MT];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int m = 0; m < MT; ++m) y[t][m] = {0.f, 0.f, 0.f, 0.f};
  const uint4 ones = make_uint4(Op::kOnes, Op::kOnes, Op::kOnes, Op::kOnes);

  for (int c = wid; c < chunks; c += kQ4Waves) {
    const int k0 = c * kChunk;
    uint4 w[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) w[t] = k0 + g * 32 < a.k ? ld_nt16(wrow[t] + k0 / 8) : make_uint4(0, 0, 0, 0);
    __builtin_amdgcn_wave_barrier();
    const int gi = min(k0 / 32 / GT + min(g, G - 1), a.groups - 1);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const float s = St<T>::ld(ld_g(srow[t] + gi)), b = St<T>::ld(ld_g(brow[t] + gi));
      sc[wid][t][g][i] = make_float2(s, fmaf(-16.f, s, b));
    }
    // the wave's own LDS, which serves it in order: only the compiler is held
    __builtin_amdgcn_wave_barrier();
    uint32_t wd[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      wd[t][0] = w[t].x, wd[t][1] = w[t].y, wd[t][2] = w[t].z, wd[t][3] = w[t].w;
      swap32(wd[t][0], wd[t][2]);
      swap32(wd[t][1], wd[t][3]);
      swap16(wd[t][0], wd[t][1]);
      swap16(wd[t][2], wd[t][3]);
    }
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
        const int step = q * GT + z, k = k0 + step * 32;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const typename Op::X x = Op::load(xrow[m] + k, k + g * 8 < a.k);
#pragma unroll
          for (int c3 = 0; c3 < Op::kParts; ++c3) {
            sum[m] = Op::M::mma(ones, x.part[c3], sum[m]);
#pragma unroll
            for (int t = 0; t < NT; ++t) p[t][m] = Op::M::mma(Op::codes(wd[t][step]), x.part[c3], p[t][m]);
          }
        }
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const float4 u = *reinterpret_cast<const float4*>(&sc[wid][t][q][g * 4]);
        const float4 v = *reinterpret_cast<const float4*>(&sc[wid][t][q][g * 4 + 2]);
        const float s[4] = {u.x, u.z, v.x, v.z}, o[4] = {u.y, u.w, v.y, v.w};
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int r = 0; r < 4; ++r) y[t][m][r] += fmaf(s[r], p[t][m][r], o[r] * sum[m][r]);
      }
    }
  }

#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int m = 0; m < MT; ++m) buf[wid][t][m][lane] = y[t][m];
  __syncthreads();
  for (int z = wid; z < NT * MT; z += kQ4Waves) {
    const int t = z / MT, m = z - t * MT, row = m0 + m * 16 + i, col = n0 + t * 16 + g * 4;
    f32x4_t v = buf[0][t][m][lane];
#pragma unroll
    for (int w = 1; w < kQ4Waves; ++w) v += buf[w][t][m][lane];
    if (row >= a.rows) continue;
    T* dst = static_cast<T*>(a.y) + row * a.ldy + col;
    union {
      T x[4];
      uint4 w4;
      uint2 w2;
    } u;
#pragma unroll
    for (int r = 0; r < 4; ++r) u.x[r] = St<T>::st(v[r]);
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

template <typename T, int MT, int NT>
void launch(const Q4Args& a, int group, hipStream_t s) {
  const dim3 grid((a.n + 16 * NT - 1) / (16 * NT), (a.rows + 63) / 64), block(64 * kQ4Waves);
  if (group == 32) hipLaunchKernelGGL((k_q4<T, MT, 1, NT>), grid, block, 0, s, a);
  else if (group == 64) hipLaunchKernelGGL((k_q4<T, MT, 2, NT>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((k_q4<T, MT, 4, NT>), grid, block, 0, s, a);
}

// Eight weights a thread, group / 8 threads a group: bias = least weight, scale = a
// 15th of the range, both rounded to the type before the codes are taken.
template <typename T>
__global__ __launch_bounds__(256) void k_q4_quantize(const T* src, int64_t ld, int64_t total, int k, int group,
                                                     uint32_t* w, T* scales, T* biases) {
  using S = St<T>;
  const int64_t word = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int words = k / 8, span = group / 8;
  const int64_t at = min(word, total - 1), row = at / words;
  const int c = (int)(at - row * words);
  float v[8], lo = INFINITY, hi = -INFINITY;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    v[j] = S::ld(src[row * ld + c * 8 + j]);
    lo = fminf(lo, v[j]), hi = fmaxf(hi, v[j]);
  }
  for (int o = 1; o < span; o <<= 1) lo = fminf(lo, __shfl_xor(lo, o, 64)), hi = fmaxf(hi, __shfl_xor(hi, o, 64));
  const float scale = S::rnd((hi - lo) / 15.f), bias = S::rnd(lo);
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
  const int mt = (std::min(rows, 64) + 15) / 16;
  MRT_DTYPE_DISPATCH(dt, {
    if (mt == 1) launch<T, 1, 1>(a, w.group, s);
    else if (mt == 2) launch<T, 2, 1>(a, w.group, s);
    else launch<T, 4, 1>(a, w.group, s);
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

// 8-bit codes of a vector of values: scale s = max |x| (1 / 127) in fp32, codes the whole
// numbers nearest to the fp32 quotients x / s (ties to even).
#pragma once

#include <math.h>
#include <stdint.h>

#include <hip/hip_runtime.h>

namespace mrt {

// The scale of a vector with this largest magnitude (as bits); NaN where it is not finite.
__device__ __forceinline__ float codes_scale(uint32_t top) {
  return top >= 0x7f800000u ? NAN : __uint_as_float(top) * (1.f / 127.f);
}

// Codes of 16 values of it, by the scale s.
//
// The quotient is rounded to fp32 before it is rounded to a whole number, so it has to be that
// one: with r = 1 / s rounded to nearest, y = x r is within 1.5 units of its last place, and each
// y + (x - y s) r in fused steps corrects it: to less than one, then, by Markstein's theorem
// (Computation of elementary functions on the IBM RISC System/6000 processor, 1990), to the
// quotient rounded to nearest.  That takes 5 instructions of a division's 10: 16 x 4001 tokens
// of 8 heads of d 128 in fp16 are written in 80 us, not 97.  Where s is below 2^-60 remainders
// may lose bits and the division itself is used; the least scales are rounded down by so much
// that quotients are beyond 127.
__device__ __forceinline__ uint4 codes16(const float (&x)[16], float s) {
  uint32_t w[4];
  if (s >= 0x1p-60f) {
    const float r = 1.f / s;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float v = x[4 * j + e];
        float q = v * r;
        q = fmaf(fmaf(-q, s, v), r, q);
        q = fmaf(fmaf(-q, s, v), r, q);
        y[e] = __float_as_uint(q + 12582912.f);  // 1.5 2^23: the low bits count ones
      }
      const uint32_t lo = __builtin_amdgcn_perm(y[1], y[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(y[3], y[2], 0x0c0c0400u);
      w[j] = __builtin_amdgcn_perm(hi, lo, 0x05040100u);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      w[j] = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float q = s > 0.f ? fminf(fmaxf(rintf(x[4 * j + e] / s), -127.f), 127.f) : 0.f;
        w[j] |= ((uint32_t)(int)q & 0xffu) << (8 * e);
      }
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

}  // namespace mrt

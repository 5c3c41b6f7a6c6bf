// Int8 codes of a token in fp32 arithmetic, shared by everything that makes them:
//   symmetric   s = max(max |x|, 1e-5) / 127         q = clamp(rint(x / s), -128, 127)
//   asymmetric  s = max(max x - min x, 1e-5) / 255   z = clamp(-128 - rint(min x / s), -128, 127)
//               q = clamp(rint(x / s) + z, -128, 127)
//   given scale q = clamp(rint(x / s), -128, 127)
#pragma once
#include "divisor.h"

namespace lcq {

struct TokenCodes {
  Divisor d;
  float lo, hi;                                     // quotients outside are clamped (so that the codes are: z is whole)
  int z;
  bool clamp;
  __device__ __forceinline__ TokenCodes(float s, float z_, bool bounded, bool clamp_) : d(s), lo(-128.0f - z_), hi(127.0f - z_), z((int)z_), clamp(clamp_) {
    d.fast = d.fast && bounded;
  }
  __device__ __forceinline__ static TokenCodes given(float s) { return TokenCodes(s, 0.0f, false, true); }  // x / s may overflow: divides
  // (|x| / s <= 127 up to its rounding: nothing to clamp)
  __device__ __forceinline__ static TokenCodes symmetric(float most) { return TokenCodes(nan_max(most, 1e-5f) / 127.0f, 0.0f, true, false); }
  __device__ __forceinline__ static TokenCodes asymmetric(float lo, float hi) {
    const float s = nan_max(hi - lo, 1e-5f) / 255.0f;
    // (s >= 1e-5 / 255: x / s overflows only for a narrow range far from zero)
    return TokenCodes(s, fminf(fmaxf(-128.0f - rintf(lo / s), -128.0f), 127.0f), fmaxf(fabsf(hi), fabsf(lo)) < 1e30f, true);
  }
  // N codes, four to a word, the first in the lowest byte; the wave holds one token, so the branches are the wave's.
  // A quotient q within +-2^22 plus 1.5 2^23 is rounded to a whole number, ties to even, as rint rounds it, and leaves it in the sum's low bits.
  template <int N>
  __device__ __forceinline__ void codes(const float* x, uint32_t* w) const {
    float t[N];
    if (__builtin_amdgcn_readfirstlane((int)d.fast)) {
      #pragma unroll
      for (int j = 0; j < N; ++j) t[j] = d.fast_quotient(x[j]);
    } else {
      #pragma unroll
      for (int j = 0; j < N; ++j) t[j] = x[j] / d.s;
    }
    if (__builtin_amdgcn_readfirstlane((int)clamp)) {
      #pragma unroll
      for (int j = 0; j < N; ++j) t[j] = __builtin_amdgcn_fmed3f(t[j], lo, hi);
    }
    #pragma unroll
    for (int p = 0; p < N / 4; ++p) {
      uint32_t q[4];
      #pragma unroll
      for (int j = 0; j < 4; ++j) q[j] = f2u(t[4 * p + j] + 12582912.0f);
      // bytes 0 of the four words, then of pairs of them
      const uint32_t ab = __builtin_amdgcn_perm(q[1], q[0], 0x0c0c0400u), cd = __builtin_amdgcn_perm(q[3], q[2], 0x04000c0cu);
      w[p] = ab | cd;
      if (__builtin_amdgcn_readfirstlane(z)) {      // + z in every byte, without carries between them
        const uint32_t zz = (uint32_t)(z & 255) * 0x01010101u;
        w[p] = ((w[p] & 0x7f7f7f7fu) + (zz & 0x7f7f7f7fu)) ^ ((w[p] ^ zz) & 0x80808080u);
      }
    }
  }
};

}  // namespace lcq

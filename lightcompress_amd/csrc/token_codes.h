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
  float z;
  __device__ __forceinline__ TokenCodes(float s, float z_, bool bounded) : d(s), z(z_) { d.fast = d.fast && bounded; }
  __device__ __forceinline__ static TokenCodes given(float s) { return TokenCodes(s, 0.0f, false); }        // x / s may overflow: divides
  __device__ __forceinline__ static TokenCodes symmetric(float most) { return TokenCodes(nan_max(most, 1e-5f) / 127.0f, 0.0f, true); }
  __device__ __forceinline__ static TokenCodes asymmetric(float lo, float hi) {
    const float s = nan_max(hi - lo, 1e-5f) / 255.0f;
    // (s >= 1e-5 / 255: x / s overflows only for a narrow range far from zero)
    return TokenCodes(s, fminf(fmaxf(-128.0f - rintf(lo / s), -128.0f), 127.0f), fmaxf(fabsf(hi), fabsf(lo)) < 1e30f);
  }
  __device__ __forceinline__ int clamped(float quotient) const { return (int)fminf(fmaxf(rintf(quotient) + z, -128.0f), 127.0f); }
  __device__ __forceinline__ int code(float x) const { return clamped(d.quotient(x)); }
  // eight of them, the first in the lowest byte; the wave holds one token (one branch, not one per value)
  __device__ __forceinline__ u32x2 codes(const float* x) const {
    int q[8];
    if (__builtin_amdgcn_readfirstlane((int)d.fast)) {
      #pragma unroll
      for (int j = 0; j < 8; ++j) q[j] = clamped(d.fast_quotient(x[j]));
    } else {
      #pragma unroll
      for (int j = 0; j < 8; ++j) q[j] = clamped(x[j] / d.s);
    }
    u32x2 w;
    #pragma unroll
    for (int p = 0; p < 2; ++p)
      w[p] = (uint32_t)(q[4 * p] & 255) | (uint32_t)(q[4 * p + 1] & 255) << 8 | (uint32_t)(q[4 * p + 2] & 255) << 16 | (uint32_t)q[4 * p + 3] << 24;
    return w;
  }
};

}  // namespace lcq

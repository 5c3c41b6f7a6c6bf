// Division of many fp32 values by one, correctly rounded.
#pragma once
#include "common.h"

namespace lcq {

// x / s for a divisor that many elements share, correctly rounded without the division sequence: with y = RN(1/s) the product
// q0 = x y is within 2 ulp, one residual step makes it faithful and a second one exact (Markstein, IBM J. R&D 34(1), 1990;
// the residuals are exact).  Five full-rate instructions; a guarded product needs as many to find out whether it may stay, and
// values below the minimum normal, where the grid's midpoints are not a bit pattern, went through the division sequence.
// Scales outside 2^-60 .. 2^60 (an infinite or NaN block, a block of subnormals) divide.
struct Divisor {
  float s, y;
  bool fast;
  __device__ __forceinline__ explicit Divisor(float s_) : s(s_), fast(s_ > 8.6736174e-19f && s_ < 1.1529215e18f) {
    const float y0 = __builtin_amdgcn_rcpf(s);
    y = __builtin_fmaf(__builtin_fmaf(-s, y0, 1.0f), y0, y0);
  }
  __device__ __forceinline__ float fast_quotient(float x) const {            // where `fast`
    float q = x * y;                                         // (s q - x taken off, not x - s q added: that way -0 / s stays -0)
    q = __builtin_fmaf(-__builtin_fmaf(s, q, -x), y, q);
    return __builtin_fmaf(-__builtin_fmaf(s, q, -x), y, q);
  }
  __device__ __forceinline__ float quotient(float x) const {
    if (__builtin_expect(!fast, 0)) return x / s;
    return fast_quotient(x);
  }
};

}  // namespace lcq

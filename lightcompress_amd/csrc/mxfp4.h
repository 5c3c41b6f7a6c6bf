// Blocks of 32 four-bit numbers with a shared power of two (OCP microscaling, MXFP4).
//   codes   e2m1: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign (bit 3); two to a byte, the lower half first
//   scale   E8M0: byte s stands for 2^(s - 127), 255 for NaN
// A row of K values has B = ceil(K / 32) blocks: 16 B bytes of codes (zeros behind K) and B of scales.
#pragma once
#include "rowquant.h"

namespace lcq {

// The scale of a block whose largest magnitude has the fp32 bits `most`: 2^(floor(log2 most) - 2), so that the largest code is 4 or 6.
// An infinity or a NaN makes the block NaN.
__device__ __forceinline__ uint32_t mx_scale(uint32_t most) {
  const uint32_t e = most >> 23;
  return e == 255 ? 255u : e < 2 ? 0u : e - 2;
}
// the same byte as the conversions take it: they look at the exponent alone
__device__ __forceinline__ float mx_factor(uint32_t scale) { return u2f(scale << 23); }

// eight values -> eight codes, each the nearest, a tie the even one, saturated at 6 (v_cvt_scalef32_pk_fp4_f32); a NaN block: 0
__device__ __forceinline__ uint32_t mx_codes(const float* v, uint32_t scale) {
  const float s = mx_factor(scale);
  uint32_t p = 0;
  p = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(p, v[0], v[1], s, 0);
  p = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(p, v[2], v[3], s, 1);
  p = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(p, v[4], v[5], s, 2);
  p = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(p, v[6], v[7], s, 3);
  return scale == 255 ? 0u : p;
}

__device__ __forceinline__ uint32_t mx_max_bits(const float* v) {
  uint32_t m = 0;
  #pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t u = f2u(v[e]) & 0x7fffffffu;
    m = u > m ? u : m;
  }
  return m;
}
// the largest of four neighbouring lanes
__device__ __forceinline__ uint32_t mx_quad_max(uint32_t m) {
  const uint32_t a = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xf, 0xf, true);
  m = a > m ? a : m;
  const uint32_t b = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xf, 0xf, true);
  return b > m ? b : m;
}

typedef u32x4 u32x4_anywhere __attribute__((aligned(2)));      // rows may start on any element
// 16 bytes that go past the caches.  (The asm keeps the store from being made one with the same store on another path, which would lose that.)
__device__ __forceinline__ void mx_store_past(void* to, u32x4 v) {
  asm volatile("");
  __builtin_nontemporal_store(v, (u32x4_anywhere*)to);
  asm volatile("");
}

// Eight values of a row of XT, from element k on; what lies behind K is 0.  Rows may start on any element.
template <int XT>
__device__ __forceinline__ void mx_load8(const char* row, int64_t k, int64_t K, float* v) {
  if (k + 8 <= K) {
    u32x4 raw[XT == ROW_F32 ? 2 : 1];
    __builtin_memcpy(raw, row + k * (XT == ROW_F32 ? 4 : 2), sizeof raw);
    unpack<XT>(raw[0], v);
    if constexpr (XT == ROW_F32) unpack<XT>(raw[1], v + 4);
  } else {
    #pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = k + e < K ? load_scalar<XT>(row, k + e) : 0.0f;
  }
}

}  // namespace lcq

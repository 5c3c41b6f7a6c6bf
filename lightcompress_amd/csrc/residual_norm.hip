// The end of one block and the start of the next, one pass over a token's row:
//
//   b = x                 or  norm(x; post_weight, post_bias)
//   h = residual + scale * (gate * b)                              -> the residual stream
//   y = norm(h; weight, bias)                                      -> the next block's input, as values or as int8 codes
//   rms:   norm(v) = v / sqrt(mean v^2 + eps) * (w + offset) + bias
//   layer: norm(v) = (v - mean) / sqrt(mean (v - mean)^2 + eps) * (w + offset) + bias
//
// and the int8 codes of a token by themselves (lcq_quant_tokens: the same rows without norm and residual; token_codes.h).
//
// Everything between the loads and the stores is in 32 bits: y is taken from h before h is rounded to the stream's type, codes
// from y before any rounding.  The quantizer arithmetic is IntegerQuantizer's (quant.py:544-558, 698-716) on fp32 rows with
// granularity per_token, codes moved to int8 (its unsigned codes less 128).
//
// A row stays in the registers of 64 to 1024 lanes, 16 values per lane for most widths, so every operand is read once.  Bound by HBM: 8192 x 4096
// bf16 with residual and weight 46 us (5.8 TB/s read and written; a copy runs at 5.1), with codes for values 45, the codes alone 20 one after another (24 to 26 a launch by itself); 16384 x 4096 with
// two norms and a gate 119 us (5.6 TB/s).  Rows of 4096 on one wave took 60 us for these 46, on two 51; nontemporal loads 51.
#include "rowquant.h"
#include "token_codes.h"

namespace {
using namespace lcq;

struct NormArgs {
  const void *x, *residual, *gate, *post_weight, *post_bias, *weight, *bias;
  const float* scale_in;
  void *h, *out;
  int8_t* codes;
  float* scales;
  int32_t* zeros;
  int64_t T, ldx, ldr, ldg, first;                  // (first: the first row of a launch)
  int K, flags;
  float scale, eps, offset;
};

constexpr int NORM = 1 << 20;                       // (internal: y is a norm of h; without it y = h)

// n <= V consecutive elements at index i of a row of type BF, or of fp32 where f32 says so; rows may start anywhere.  Those past n are 0.
template <int BF, int V>
__device__ __forceinline__ void load_v(const void* p, int64_t i, bool f32, float* v, int n) {
  if (n == V) {
    if (BF == ROW_F32 || f32) {
      #pragma unroll
      for (int q = 0; q < V / 4; ++q) {
        u32x4 r;
        __builtin_memcpy(&r, (const float*)p + i + 4 * q, 16);
        unpack<ROW_F32>(r, v + 4 * q);
      }
    } else {
      u32x4 r;
      __builtin_memcpy(&r, (const uint16_t*)p + i, 16);
      unpack<BF>(r, v);
    }
  } else {
    #pragma unroll
    for (int j = 0; j < V; ++j) v[j] = j < n ? f32 ? ((const float*)p)[i + j] : load_scalar<BF>(p, i + j) : 0.0f;
  }
}
template <int BF, int V>
__device__ __forceinline__ void store_v(void* p, int64_t i, bool f32, const float* v, int n) {
  if (n == V) {
    if (BF == ROW_F32 || f32) {
      #pragma unroll
      for (int q = 0; q < V / 4; ++q) {
        const u32x4 r = pack<ROW_F32>(v + 4 * q);
        __builtin_memcpy((float*)p + i + 4 * q, &r, 16);
      }
    } else {
      const u32x4 r = pack_rne<BF>(v);
      __builtin_memcpy((uint16_t*)p + i, &r, 16);
    }
  } else {
    #pragma unroll
    for (int j = 0; j < V; ++j)
      if (j < n) {
        if (f32) ((float*)p)[i + j] = v[j];
        else store_scalar<BF>(p, i + j, rnd<BF>(v[j]));
      }
  }
}

// TEAM lanes share a row: 64 (a wave, four rows per workgroup) or the whole workgroup.  A sum or a maximum over the row in a fixed order.
template <int TEAM>
struct Row {
  float* sm;                                        // one float per wave
  template <int OP>                                 // 0 sum, 1 maximum, 2 minimum (both NaN where an element is)
  __device__ __forceinline__ float reduce(float v) const {
    if constexpr (OP == 0) v = team_sum<64>(v);
    else v = team_reduce<64, OP == 1>(v);
    if constexpr (TEAM > 64) {
      __syncthreads();
      if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = v;
      __syncthreads();
      v = sm[0];
      #pragma unroll
      for (int w = 1; w < TEAM / 64; ++w) v = OP == 0 ? v + sm[w] : OP == 1 ? nan_max(v, sm[w]) : nan_min(v, sm[w]);
    }
    return v;
  }
};

// One row per TEAM lanes, CH pieces of V elements (16 bytes) per lane in registers.
template <int BF, int TEAM, int CH>
__global__ __launch_bounds__(TEAM == 64 ? 256 : TEAM) void residual_norm_kernel(NormArgs a) {
  constexpr int V = Vec<BF>::N;
  __shared__ float sm[TEAM / 64];
  const Row<TEAM> row_{sm};
  const int t = threadIdx.x % TEAM;
  const int64_t r = a.first + (TEAM == 64 ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : (int64_t)blockIdx.x);
  if (r >= a.T) return;                             // (whole waves, and no barriers where TEAM is a wave)
  const int K = a.K, flags = a.flags;
  const float rK = 1.0f / (float)K;
  float v[CH][V];
  const auto each = [&](auto&& f) {                 // f(index, elements, how many of them are in the row)
    #pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int i = (t + c * TEAM) * V;
      if (i < K) f(i, v[c], K - i < V ? K - i : V);
    }
  };
  each([&](int i, float* e, int n) { load_v<BF, V>(a.x, r * a.ldx + i, false, e, n); });
  const auto norm = [&](const void* w, bool w32, const void* b, bool b32) {
    float sum = 0.0f, mean = 0.0f;
    if (flags & LCQ_NORM_LAYER) {
      each([&](int, float* e, int) {
        #pragma unroll
        for (int j = 0; j < V; ++j) sum += e[j];
      });
      mean = row_.template reduce<0>(sum) * rK;
      sum = 0.0f;
      each([&](int, float* e, int n) {
        #pragma unroll
        for (int j = 0; j < V; ++j) e[j] = j < n ? e[j] - mean : 0.0f;
      });
    }
    each([&](int, float* e, int) {
      #pragma unroll
      for (int j = 0; j < V; ++j) sum = __builtin_fmaf(e[j], e[j], sum);
    });
    const float inv = 1.0f / sqrtf(row_.template reduce<0>(sum) * rK + a.eps);
    each([&](int i, float* e, int n) {
      float f[V];
      if (w) {
        load_v<BF, V>(w, i, w32, f, n);
        #pragma unroll
        for (int j = 0; j < V; ++j) e[j] = e[j] * inv * (f[j] + a.offset);
      } else {
        #pragma unroll
        for (int j = 0; j < V; ++j) e[j] *= inv;
      }
      if (b) {
        load_v<BF, V>(b, i, b32, f, n);
        #pragma unroll
        for (int j = 0; j < V; ++j) e[j] += f[j];
      }
    });
  };

  if (a.post_weight) norm(a.post_weight, flags & LCQ_NORM_POST_WEIGHT_F32, a.post_bias, flags & LCQ_NORM_POST_BIAS_F32);
  if (a.gate) {
    each([&](int i, float* e, int n) {
      float f[V];
      load_v<BF, V>(a.gate, r * a.ldg + i, false, f, n);
      #pragma unroll
      for (int j = 0; j < V; ++j) e[j] *= f[j];
    });
  }
  if (a.residual) {
    each([&](int i, float* e, int n) {
      float f[V];
      load_v<BF, V>(a.residual, r * a.ldr + i, flags & LCQ_NORM_RESIDUAL_F32, f, n);
      #pragma unroll
      for (int j = 0; j < V; ++j) e[j] = __builtin_fmaf(a.scale, e[j], f[j]);
    });
  } else if (flags & NORM) {
    each([&](int, float* e, int) {
      #pragma unroll
      for (int j = 0; j < V; ++j) e[j] *= a.scale;
    });
  }
  if (a.h) each([&](int i, float* e, int n) { store_v<BF, V>(a.h, r * K + i, flags & LCQ_NORM_RESIDUAL_F32, e, n); });
  if (flags & NORM) norm(a.weight, flags & LCQ_NORM_WEIGHT_F32, a.bias, flags & LCQ_NORM_BIAS_F32);
  if (a.out) each([&](int i, float* e, int n) { store_v<BF, V>(a.out, r * K + i, flags & LCQ_NORM_OUT_F32, e, n); });
  if (!a.codes) return;

  const auto make = [&]() -> TokenCodes {
    if (a.scale_in) return TokenCodes::given(a.scale_in[0]);
    if (flags & LCQ_NORM_ASYM) {
      float hi = -__builtin_inff(), lo = __builtin_inff();
      each([&](int, float* e, int n) {
        #pragma unroll
        for (int j = 0; j < V; ++j) {
          const float x = j < n ? e[j] : e[0];
          hi = nan_max(hi, x);
          lo = nan_min(lo, x);
        }
      });
      hi = row_.template reduce<1>(hi);
      return TokenCodes::asymmetric(row_.template reduce<2>(lo), hi);
    }
    float m = 0.0f;
    each([&](int, float* e, int n) {
      #pragma unroll
      for (int j = 0; j < V; ++j) m = nan_max(m, j < n ? fabsf(e[j]) : 0.0f);
    });
    return TokenCodes::symmetric(row_.template reduce<1>(m));
  };
  const TokenCodes q = make();
  each([&](int i, float* e, int n) {
    uint32_t w[V / 4];
    q.template codes<V>(e, w);
    int8_t* const to = a.codes + r * K + i;
    if (n == V) {
      __builtin_memcpy(to, w, V);
    } else {
      #pragma unroll
      for (int j = 0; j < V; ++j)
        if (j < n) to[j] = (int8_t)(w[j / 4] >> 8 * (j % 4));
    }
  });
  if (t == 0 && a.scales) a.scales[r] = q.d.s;
  if (t == 0 && a.zeros) a.zeros[r] = q.z;
}

constexpr int64_t ROWS_OF_A_LAUNCH = 1 << 21;       // (a launch has fewer than 2^32 lanes)

// E elements per lane
template <int BF, int TEAM, int E>
void launch(const NormArgs& a, hipStream_t st) {
  constexpr int rows = TEAM == 64 ? 4 : 1;
  NormArgs part = a;
  for (part.first = 0; part.first < a.T; part.first += ROWS_OF_A_LAUNCH) {
    const int64_t left = a.T - part.first, n = left < ROWS_OF_A_LAUNCH ? left : ROWS_OF_A_LAUNCH;
    residual_norm_kernel<BF, TEAM, E / Vec<BF>::N><<<dim3((unsigned)((n + rows - 1) / rows)), dim3(TEAM == 64 ? 256 : TEAM), 0, st>>>(part);
  }
}
template <int BF>
void launch_rows(const NormArgs& a, hipStream_t st) {
  if (a.K <= 512) launch<BF, 64, 8>(a, st);
  else if (a.K <= 1024) launch<BF, 64, 16>(a, st);
  else if (a.K <= 2048) launch<BF, 256, 8>(a, st);
  else if (a.K <= 4096) launch<BF, 256, 16>(a, st);
  else if (a.K <= 8192) launch<BF, 512, 16>(a, st);
  else if (a.K <= 16384) launch<BF, 1024, 16>(a, st);
  else if (a.K <= 32768) launch<BF, 1024, 32>(a, st);
  else launch<BF, 1024, 64>(a, st);
}

constexpr int64_t MOST_COLS = 65536;                // a row stays in the registers of 1024 lanes

int run(const NormArgs& a, int dtype, hipStream_t st) {
  if (dtype == LCQ_BF16) launch_rows<ROW_BF16>(a, st);
  else if (dtype == LCQ_F16) launch_rows<ROW_F16>(a, st);
  else launch_rows<ROW_F32>(a, st);
  LCQ_CHECK_LAUNCH();
  return LCQ_OK;
}

bool known_dtype(int dtype) { return dtype == LCQ_F32 || dtype == LCQ_BF16 || dtype == LCQ_F16; }

}  // namespace

extern "C" {

int lcq_residual_norm(const void* x, int dtype, int64_t T, int64_t K, int64_t ldx, const void* residual, int64_t ldr, const void* gate,
                      int64_t ldg, const void* post_weight, const void* post_bias, const void* weight, const void* bias, float scale,
                      float eps, float weight_offset, int flags, void* h, void* out, int8_t* codes, float* scales, int32_t* zeros,
                      void* stream) {
  if (!x || !h || T <= 0 || K <= 0 || T > 0x7fffffff || (!out && !codes) || (codes && !scales)) return LCQ_EINVAL;
  if ((post_bias && !post_weight) || ldx < 0 || ldr < 0 || ldg < 0) return LCQ_EINVAL;
  if ((flags & LCQ_NORM_ASYM) && codes && !zeros) return LCQ_EINVAL;
  if (flags & ~255) return LCQ_EINVAL;
  if (!known_dtype(dtype)) return LCQ_EDTYPE;
  if (K > MOST_COLS) return LCQ_ESIZE;
  NormArgs a = {};
  a.x = x; a.residual = residual; a.gate = gate; a.post_weight = post_weight; a.post_bias = post_bias; a.weight = weight; a.bias = bias;
  a.h = h; a.out = out; a.codes = codes; a.scales = scales; a.zeros = zeros;
  a.T = T; a.ldx = ldx; a.ldr = ldr; a.ldg = ldg; a.K = (int)K; a.flags = flags | NORM;
  a.scale = scale; a.eps = eps; a.offset = weight_offset;
  return run(a, dtype, (hipStream_t)stream);
}

int lcq_quant_tokens(const void* x, int dtype, int64_t T, int64_t K, int64_t ldx, int asym, const float* scale, int8_t* codes,
                     float* scales, int32_t* zeros, void* stream) {
  if (!x || !codes || T <= 0 || K <= 0 || T > 0x7fffffff || ldx < 0 || (!scale && !scales)) return LCQ_EINVAL;
  if (asym && (scale || !zeros)) return LCQ_EINVAL;
  if (!known_dtype(dtype)) return LCQ_EDTYPE;
  if (K > MOST_COLS) return LCQ_ESIZE;
  NormArgs a = {};
  a.x = x; a.scale_in = scale; a.codes = codes; a.scales = scale ? nullptr : scales; a.zeros = asym ? zeros : nullptr;
  a.T = T; a.ldx = ldx; a.K = (int)K; a.flags = asym ? LCQ_NORM_ASYM : 0; a.scale = 1.0f;
  return run(a, dtype, (hipStream_t)stream);
}

}  // extern "C"

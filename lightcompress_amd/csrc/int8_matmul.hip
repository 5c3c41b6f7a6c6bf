// Product of int8 codes with a scale for each token and each channel:
//   y[m, n] = as[m] ws[n] (sum_k a[m, k] w[n, k] - az[m] sum_k w[n, k]) + bias[n]
// The sums are exact in 32-bit integers for K <= 65536 (|a - az| <= 255, |w| <= 128: 255 * 128 * 65536 < 2^31).
#include "rowquant.h"

namespace {
using namespace lcq;

typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((ext_vector_type(16))) int i32x16;

struct MatmulArgs {
  const int8_t *a, *w;
  const float* as;
  const int32_t* az;
  const void *ws, *bias;
  void* y;
  int64_t M, N;
  int K, ws_dtype, bias_dtype, dtype, a_scalar, w_scalar;
};

__device__ __forceinline__ float load_any(const void* p, int dtype, int64_t i) {
  return dtype == LCQ_F32 ? load_scalar<ROW_F32>(p, i) : dtype == LCQ_BF16 ? load_scalar<ROW_BF16>(p, i) : load_scalar<ROW_F16>(p, i);
}

// 64 x 64 outputs per workgroup, a quarter of the rows per wave; 64 codes of K at a time through LDS.
__global__ __launch_bounds__(256) void int8_matmul_kernel(MatmulArgs g) {
  __shared__ __attribute__((aligned(16))) int8_t sa[64][80], sw[64][80];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t m0 = (int64_t)blockIdx.y * 64, n0 = (int64_t)blockIdx.x * 64;
  i32x4 acc[4] = {};
  int sums[4] = {};
  for (int k0 = 0; k0 < g.K; k0 += 64) {
    __syncthreads();
    for (int i = tid; i < 64 * 64; i += 256) {
      const int r = i >> 6, k = k0 + (i & 63);
      sa[r][i & 63] = m0 + r < g.M && k < g.K ? g.a[(m0 + r) * g.K + k] : 0;
      sw[r][i & 63] = n0 + r < g.N && k < g.K ? g.w[(n0 + r) * g.K + k] : 0;
    }
    __syncthreads();
    const i32x4 fa = *(const i32x4*)&sa[wave * 16 + (lane & 15)][(lane >> 4) * 16];
    #pragma unroll
    for (int j = 0; j < 4; ++j) {
      const i32x4 fw = *(const i32x4*)&sw[j * 16 + (lane & 15)][(lane >> 4) * 16];
      acc[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fa, fw, acc[j], 0, 0, 0);
      if (g.az) {
        #pragma unroll
        for (int q = 0; q < 4; ++q) sums[j] = __builtin_amdgcn_sdot4(fw[q], 0x01010101, sums[j], false);
      }
    }
  }
  #pragma unroll
  for (int j = 0; j < 4; ++j) {
    sums[j] += __shfl_xor(sums[j], 16);
    sums[j] += __shfl_xor(sums[j], 32);
    const int64_t n = n0 + j * 16 + (lane & 15);
    if (n >= g.N) continue;
    const float sw_n = load_any(g.ws, g.ws_dtype, g.w_scalar ? 0 : n), b = g.bias ? load_any(g.bias, g.bias_dtype, n) : 0.0f;
    #pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int64_t m = m0 + wave * 16 + (lane >> 4) * 4 + r;
      if (m >= g.M) continue;
      const int s = acc[j][r] - (g.az ? g.az[m] * sums[j] : 0);
      const float v = (float)s * (g.as[g.a_scalar ? 0 : m] * sw_n) + b;
      if (g.dtype == LCQ_F32) ((float*)g.y)[m * g.N + n] = v;
      else if (g.dtype == LCQ_BF16) store_scalar<ROW_BF16>(g.y, m * g.N + n, rnd<ROW_BF16>(v));
      else store_scalar<ROW_F16>(g.y, m * g.N + n, v);
    }
  }
}

}  // namespace

extern "C" {

int64_t lcq_int8_matmul_workspace_bytes(int64_t M, int64_t N, int64_t K) { (void)M; (void)N; (void)K; return 0; }

int lcq_int8_matmul(const int8_t* a, const float* as, int a_scalar, const int32_t* az, const int8_t* w, const void* ws, int ws_dtype,
                    int w_scalar, const void* bias, int bias_dtype, int64_t M, int64_t N, int64_t K, void* y, int dtype,
                    void* workspace, void* stream) {
  (void)workspace;
  if (!a || !as || !w || !ws || !y || M <= 0 || N <= 0 || K <= 0) return LCQ_EINVAL;
  const auto known = [](int d) { return d == LCQ_F32 || d == LCQ_BF16 || d == LCQ_F16; };
  if (!known(dtype) || !known(ws_dtype) || (bias && !known(bias_dtype))) return LCQ_EDTYPE;
  if (K > 65536 || (M + 63) / 64 > 65535) return LCQ_ESIZE;
  MatmulArgs g = {a, w, as, az, ws, bias, y, M, N, (int)K, ws_dtype, bias_dtype, dtype, a_scalar, w_scalar};
  int8_matmul_kernel<<<dim3((unsigned)((N + 63) / 64), (unsigned)((M + 63) / 64)), dim3(256), 0, (hipStream_t)stream>>>(g);
  LCQ_CHECK_LAUNCH();
  return LCQ_OK;
}

}  // extern "C"

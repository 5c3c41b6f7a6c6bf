// Log probabilities of given tokens, entropy and best alternatives of logits x [T, V]:
//   m = max x,  S = sum exp(x - m),  U = sum exp(x - m) (x - m)
//   log sum exp x = m + log S;   logprob of a token t = (x_t - m) - log S;   entropy = log S - U / S
#include "rowquant.h"

namespace {
using namespace lcq;

struct LogprobArgs {
  const void* x;
  const int64_t* tokens;
  float *logprobs, *entropy, *top_logprobs;
  int64_t* top_tokens;
  int64_t T, V, ldx, m, ignore;
  int k;
};

// A whole number that orders logits by value and, among equal ones, by the lowest index; a NaN is above everything, -0 equals +0.
// 0 is below every logit's.
__device__ __forceinline__ uint64_t key_of(float x, uint32_t index) {
  uint32_t u = x == x ? f2u(x + 0.0f) : 0x7fc00000u;
  u = (u & 0x80000000u) ? ~u : u | 0x80000000u;
  return (uint64_t)u << 32 | (0xffffffffu - index);
}
__device__ __forceinline__ float logit_of(uint64_t key) {
  const uint32_t u = (uint32_t)(key >> 32);
  return u2f((u & 0x80000000u) ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ uint32_t index_of(uint64_t key) { return 0xffffffffu - (uint32_t)key; }

// One workgroup per row: a pass for the maximum, one for the sums, one for each alternative.
template <int BF>
__global__ __launch_bounds__(256) void logprobs_kernel(LogprobArgs a) {
  __shared__ float sf[256];
  __shared__ uint64_t sk[256];
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x, base = row * a.ldx;
  const auto fold = [&](float v, auto&& f) {
    __syncthreads();
    sf[tid] = v;
    __syncthreads();
    for (int d = 128; d; d >>= 1) {
      if (tid < d) sf[tid] = f(sf[tid], sf[tid + d]);
      __syncthreads();
    }
    return sf[0];
  };
  float m = -3.4028234663852886e38f;
  for (int64_t v = tid; v < a.V; v += 256) m = nan_max(m, load_scalar<BF>(a.x, base + v));
  m = fold(m, [](float p, float q) { return nan_max(p, q); });
  float S = 0.0f, U = 0.0f;
  for (int64_t v = tid; v < a.V; v += 256) {
    const float d = load_scalar<BF>(a.x, base + v) - m, e = expf(d);
    S += e;
    U += e * nan_max(d, -150.0f);
  }
  S = fold(S, [](float p, float q) { return p + q; });
  U = fold(U, [](float p, float q) { return p + q; });
  const float l = logf(S);
  if (tid == 0 && a.entropy) a.entropy[row] = l - U / S;
  for (int64_t j = tid; j < a.m; j += 256) {
    const int64_t t = a.tokens[row * a.m + j];
    a.logprobs[row * a.m + j] = t == a.ignore ? 0.0f : t < 0 || t >= a.V ? __builtin_nanf("") : (load_scalar<BF>(a.x, base + t) - m) - l;
  }
  uint64_t last = ~0ull;
  for (int j = 0; j < a.k; ++j) {
    uint64_t best = 0;
    for (int64_t v = tid; v < a.V; v += 256) {
      const uint64_t key = key_of(load_scalar<BF>(a.x, base + v), (uint32_t)v);
      if (key < last && key > best) best = key;
    }
    __syncthreads();
    sk[tid] = best;
    __syncthreads();
    for (int d = 128; d; d >>= 1) {
      if (tid < d && sk[tid + d] > sk[tid]) sk[tid] = sk[tid + d];
      __syncthreads();
    }
    last = sk[0];
    if (tid == 0) {
      a.top_logprobs[row * a.k + j] = (logit_of(last) - m) - l;
      a.top_tokens[row * a.k + j] = index_of(last);
    }
  }
}

}  // namespace

extern "C" {

int64_t lcq_token_logprobs_workspace_bytes(int64_t T, int64_t V, int k) { (void)T; (void)V; (void)k; return 0; }

int lcq_token_logprobs(const void* logits, int dtype, int64_t T, int64_t V, int64_t ldx, const int64_t* tokens, int64_t m,
                       int64_t ignore, float* logprobs, float* entropy, int k, float* top_logprobs, int64_t* top_tokens,
                       void* workspace, void* stream) {
  (void)workspace;
  if (!logits || T <= 0 || V <= 0 || ldx < 0 || m < 0 || k < 0 || k > 64 || k > V) return LCQ_EINVAL;
  if ((m > 0 && (!tokens || !logprobs)) || (k > 0 && (!top_logprobs || !top_tokens))) return LCQ_EINVAL;
  if (dtype != LCQ_F32 && dtype != LCQ_BF16 && dtype != LCQ_F16) return LCQ_EDTYPE;
  if (T > 0x7fffffff || V > 0x7fffffff) return LCQ_ESIZE;
  const LogprobArgs a = {logits, tokens, logprobs, entropy, top_logprobs, top_tokens, T, V, ldx, m, ignore, k};
  const dim3 grid((unsigned)T);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == LCQ_BF16) logprobs_kernel<ROW_BF16><<<grid, dim3(256), 0, st>>>(a);
  else if (dtype == LCQ_F16) logprobs_kernel<ROW_F16><<<grid, dim3(256), 0, st>>>(a);
  else logprobs_kernel<ROW_F32><<<grid, dim3(256), 0, st>>>(a);
  LCQ_CHECK_LAUNCH();
  return LCQ_OK;
}

}  // extern "C"

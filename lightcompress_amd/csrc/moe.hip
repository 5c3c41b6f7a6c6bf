// A mixture-of-experts layer for a few tokens, on experts of microscaled 4-bit numbers:
//   y[t] = sum_s w[t, s] (down_e h + down_bias_e),   h = act(gate_e x[t] + b) * (up_e x[t] + b),   e = experts[t, s]
// Tokens that chose the same expert share one pass over its bytes, which is what bounds the layer: a plan (tokens by expert), gate and up, down, the
// weighted sum, a kernel each, as each needs all of the one in front.  7168 x 2048, 8 of 256 experts: 1 token 6.5 + 27.6 + 14.4 + 3.8 us (gate and up
// 3 of launch, 2.9 to the first stage, 18.2 at the memory's rate, 1.2 of results), 16 tokens 10.9 + 250 + 140 + 5.2 (6.2 TB/s in a row).
//
// The activations keep their precision.  A lane takes a block of a weight row, 16 bytes, and the conversion to bf16 applies its scale: that is
// exact, so the products are those of the stored numbers.  bf16 tokens go into the matrix pipe as they are, fp32 ones as sums of three bf16 planes, and so
// does h, which stays within the layer: 24 bits are three times eight, so nothing of an fp32 number is lost (above 2^-110).  fp16 tokens go as they are too, with the
// weights' blocks as fp16, which is exact for scales of 2^-23 .. 2^13; stages with others, beside blocks of zeros, take the tokens apart into two bf16 numbers (gate and up of 50 tokens, 2 of 8
// experts 4090 x 14336: 129 us, as two planes throughout 161; of 96 tokens 4096 x 4096 45 and 66).
#include "mxfp4.h"
#include <type_traits>

namespace {
using namespace lcq;

typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;

template <int I> using Int = std::integral_constant<int, I>;

constexpr int MOST_EXPERTS = 1024, MOST_TOP = 32, MOST_PASS = 128;           // tokens of a pass
constexpr int MOST_GROUP = 32, COUNTERS = 1024;
constexpr int MOST_DOWN = 16;                       // slots of a group of down
constexpr int PLANES = 3;                           // bf16 numbers that an fp32 number is the sum of
constexpr uint32_t OUTSIDE = 0x80000000u;

__device__ __forceinline__ float load_any(const void* p, int dtype, int64_t i) {
  return dtype == LCQ_F32 ? load_scalar<ROW_F32>(p, i) : dtype == LCQ_BF16 ? load_scalar<ROW_BF16>(p, i) : load_scalar<ROW_F16>(p, i);
}

// ---- the router ---------------------------------------------------------------------------------------------------
struct RouterArgs {
  const void* logits;
  const float* correction;
  int64_t ldl;
  int dtype, E, top, flags;
  float scale;
};

// a number that orders as the floats do, a NaN above all, 0 below all
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t u = f2u(v + 0.0f);
  return v != v ? 0xffffffffu : (int)u < 0 ? ~u : u | 0x80000000u;
}
// the largest of a wave's, by lane permutations alone
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  const auto take = [&](auto ctrl, auto rows) {
    const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, decltype(ctrl)::value, decltype(rows)::value, 0xf, false);
    v = o > v ? o : v;
  };
  take(Int<0xB1>{}, Int<0xf>{});                    // neighbours, pairs, fours, eights: rows of 16
  take(Int<0x4E>{}, Int<0xf>{});
  take(Int<0x141>{}, Int<0xf>{});
  take(Int<0x140>{}, Int<0xf>{});
  take(Int<0x142>{}, Int<0xa>{});                   // the last of a row into the next
  take(Int<0x143>{}, Int<0xc>{});
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ double wave_sum(double v) {
  #pragma unroll
  for (int m = 1; m < 64; m *= 2) v += __shfl_xor(v, m);
  return v;
}

// One token by one wave: lane s < top gets the s-th choice.  A lane looks at NL consecutive experts.
//  softmax: e^(l - max) / sum;  sigmoid: 1 / (1 + e^-l).  Chosen by the logits (both grow with them), or, with a correction, by
//  fp32(score) + correction, the scores from 64 bits, so that they are the numbers they should be to the last bit.
// -inf is chosen last and weighs 0.  Scores that are divided by their sum and are too small for 32 bits are taken times e^-(their largest logit).
template <int NL>
__device__ __forceinline__ void route_token(const RouterArgs& r, int64_t t, int& expert, float& weight) {
  const int lane = threadIdx.x & 63;
  float x[NL], score[NL], correction[NL];
  uint32_t key[NL], raw[NL];
  const float none = -__builtin_inff();
  float m = none;
  #pragma unroll
  for (int j = 0; j < NL; ++j) {                    // (all loads before the first use)
    const int e = lane * NL + j < r.E ? lane * NL + j : 0;
    raw[j] = r.dtype == LCQ_F32 ? ((const uint32_t*)r.logits)[t * r.ldl + e] : (uint32_t)((const uint16_t*)r.logits)[t * r.ldl + e];
  }
  #pragma unroll
  for (int j = 0; j < NL; ++j) correction[j] = r.correction ? r.correction[lane * NL + j < r.E ? lane * NL + j : 0] : 0.0f;
  #pragma unroll
  for (int j = 0; j < NL; ++j) {
    x[j] = r.dtype == LCQ_F32 ? u2f(raw[j]) : r.dtype == LCQ_BF16 ? u2f(raw[j] << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)raw[j]);
    if (lane * NL + j >= r.E) x[j] = none;
    m = nan_max(m, x[j]);
  }
  m = team_reduce<64, true>(m);
  const bool sigmoid = r.flags & LCQ_ROUTE_SIGMOID, renormalize = r.flags & LCQ_ROUTE_RENORMALIZE;
  if (r.correction) {
    double s[NL], sum = 0;
    #pragma unroll
    for (int j = 0; j < NL; ++j) {
      s[j] = exp(sigmoid ? -(double)x[j] : (double)x[j] - (double)m);
      if (!sigmoid && x[j] == none) s[j] = 0.0;
      sum += s[j];
    }
    sum = wave_sum(sum);
    #pragma unroll
    for (int j = 0; j < NL; ++j) {
      const double over = sigmoid ? 1.0 + s[j] : sum;
      score[j] = (float)(over == 0.0 ? 0.0 : (sigmoid ? 1.0 : s[j]) / over);
      key[j] = lane * NL + j >= r.E ? 0u : ordered(x[j] == none ? none : score[j] + correction[j]);
    }
  } else {
    float sum = 0;
    bool small = false;
    #pragma unroll
    for (int j = 0; j < NL; ++j) {
      score[j] = expf(sigmoid ? -x[j] : x[j] - m);
      if (!sigmoid && x[j] == none) score[j] = 0.0f;
      sum += score[j];
      key[j] = lane * NL + j < r.E ? ordered(x[j]) : 0u;
      small = small || (x[j] < -60.0f && x[j] != none);
    }
    sum = team_sum<64>(sum);
    #pragma unroll
    for (int j = 0; j < NL; ++j) {
      const float over = sigmoid ? 1.0f + score[j] : sum;
      score[j] = over == 0.0f ? 0.0f : (sigmoid ? 1.0f : score[j]) / over;
    }
    if (sigmoid && __builtin_expect(__builtin_amdgcn_ballot_w64(small) != 0, 0)) {           // e^-l may overflow, and 1 + e^l is 1
      const float from = renormalize && m < -60.0f ? m : 0.0f;               // (the largest logit is chosen)
      #pragma unroll
      for (int j = 0; j < NL; ++j)
        if (x[j] < -60.0f && x[j] != none) score[j] = expf(x[j] - from);
    }
  }
  expert = 0;
  if constexpr (NL <= 4) {
    // a lane's experts in order (neighbours change places only where the later one is larger, so equal ones stay), then the best of all lanes'
    // first ones again and again
    uint32_t order = 0;
    int index[NL];
    #pragma unroll
    for (int j = 0; j < NL; ++j) index[j] = j;
    #pragma unroll
    for (int round = 0; round < NL; ++round)
      #pragma unroll
      for (int j = round & 1; j + 1 < NL; j += 2) {
        const bool swap = key[j + 1] > key[j];
        const uint32_t k = key[j], i = index[j];
        key[j] = swap ? key[j + 1] : k;
        index[j] = swap ? index[j + 1] : i;
        key[j + 1] = swap ? k : key[j + 1];
        index[j + 1] = swap ? i : index[j + 1];
      }
    #pragma unroll
    for (int j = 0; j < NL; ++j) order |= (uint32_t)index[j] << 8 * j;
    for (int s = 0; s < r.top; ++s) {
      const int from = __builtin_ctzll(__ballot(key[0] == wave_max(key[0])));                // (the lowest lane has the lowest experts)
      const int e = from * NL + (__builtin_amdgcn_readlane((int)order, from) & 255);
      if (lane == s) expert = e;
      if (lane == from) {
        #pragma unroll
        for (int j = 0; j < NL; ++j) key[j] = j + 1 < NL ? key[j + 1] : 0u;
        order >>= 8;
      }
    }
  } else {
    for (int s = 0; s < r.top; ++s) {
      uint32_t best = key[0];
      int at = 0;
      #pragma unroll
      for (int j = 1; j < NL; ++j)
        if (key[j] > best) { best = key[j]; at = j; }
      const int from = __builtin_ctzll(__ballot(best == wave_max(best)));
      const int e = from * NL + __builtin_amdgcn_readlane(at, from);
      if (lane == s) expert = e;
      #pragma unroll
      for (int j = 0; j < NL; ++j)
        if (lane == from && at == j) key[j] = 0;
    }
  }
  // what the lane's expert has of `of`
  const auto gathered = [&](const float (&of)[NL], float other) {
    float v = other;
    #pragma unroll
    for (int j = 0; j < NL; ++j) {
      const float w = u2f((uint32_t)__builtin_amdgcn_ds_bpermute(expert / NL * 4, (int)f2u(of[j])));
      if (lane < r.top && expert % NL == j) v = w;
    }
    return v;
  };
  weight = gathered(score, 0.0f);
  if (renormalize) {
    float sum = team_sum<64>(weight);
    // With a correction the chosen logits may all lie far below those that the scores are relative to (NaN: stays one).
    if (r.correction && __builtin_expect(sum < 0x1p-100f, 0)) {
      const float l = gathered(x, none), best = team_reduce<64, true>(l);
      weight = l == none ? 0.0f : expf(l - best);   // (of sigmoid too: 1 + e^l is 1)
      sum = team_sum<64>(weight);
    }
    weight = sum == 0.0f ? 0.0f : weight / sum;
  }
  weight *= r.scale;
}

// A wave per token, as much as fits a CU on its way: 64 tokens of 256 experts with a correction 5.2 us, a launch and the chain of one token; 16384 of 64 experts 8.4 us.
template <int NL>
__global__ __launch_bounds__(256) void route_kernel(RouterArgs r, int64_t T, int* __restrict__ experts, float* __restrict__ weights) {
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= T) return;
  int e;
  float w;
  route_token<NL>(r, t, e, w);
  const int lane = threadIdx.x & 63;
  if (lane < r.top) { experts[t * r.top + lane] = e; weights[t * r.top + lane] = w; }
}

// ---- what the products are told -----------------------------------------------------------------------------------
// A pass: the slots (token and choice) sorted by expert, in groups of at most `size` of one expert for gate and up.  Down takes the same groups, or, as three planes
// of 32 slots do not fit LDS, groups of at most 16, which stand behind them.
struct Group {
  int expert, first, count, pad;                    // first: slot
  uint32_t token[MOST_GROUP / 4];                   // four to a word
};
struct Plan {
  int groups, down_first, down_groups, pad[13];
  uint32_t counter[COUNTERS];                       // parts of gate and up that are done (fewer than 384 units have any)
  int slot[MOST_PASS * MOST_TOP], expert[MOST_PASS * MOST_TOP];              // of a token's choices; slot -1: none
  float weight[MOST_PASS * MOST_TOP];
  Group group[MOST_PASS * MOST_TOP];
};

struct Operand { const char* x; int64_t ldx; int dtype, planes, K, Kp; uint16_t* out; };

// Values as sums of bf16 numbers (what is infinite or NaN: in the first alone).  What the first would round to an infinity is cut off instead: 16 bits are left.
__device__ __forceinline__ void planes_of(float v, uint16_t* out) {
  #pragma unroll
  for (int p = 0; p < PLANES; ++p) {
    const uint32_t raw = f2u(v), u = p == 0 && (raw & 0x7fffffff) < 0x7f800000 && (raw & 0x7fffffff) >= 0x7f7f8000 ? raw >> 16 : bf16_bits(v);
    out[p] = (uint16_t)u;
    const float taken = u2f(u << 16);
    v = (u & 0x7f80) == 0x7f80 ? 0.0f : v - taken;
  }
}

// Workgroup 0 plans the pass; the others lay the tokens out as planes [T, planes, Kp] where they are not that already.  One workgroup, as every place depends on
// all choices: 6.5 us with the routing of 1 token of 256 experts, 10.9 of 16 tokens (their choices are a chain in each wave), 5.2 behind the router's kernel.
template <int NL>
__global__ __launch_bounds__(1024) void plan_kernel(RouterArgs r, const int* __restrict__ given, const float* __restrict__ given_weights, int T,
                                                    Operand o, int size, Plan* __restrict__ plan) {
  if (blockIdx.x) {
    const int64_t all = (int64_t)T * o.Kp;
    for (int64_t i = (int64_t)(blockIdx.x - 1) * 1024 + threadIdx.x; i < all; i += (int64_t)(gridDim.x - 1) * 1024) {
      const int64_t t = i / o.Kp;
      const int k = (int)(i - t * o.Kp);
      const float v = k < o.K ? load_any(o.x, o.dtype, t * o.ldx + k) : 0.0f;
      uint16_t p[PLANES];
      planes_of(v, p);
      if (o.dtype == LCQ_F16) p[0] = __builtin_bit_cast(uint16_t, (_Float16)v);              // (one plane)
      for (int q = 0; q < o.planes; ++q) o.out[(t * o.planes + q) * o.Kp + k] = p[q];
    }
    return;
  }
  __shared__ int expert[MOST_PASS * MOST_TOP];
  __shared__ float weight[MOST_PASS * MOST_TOP];
  __shared__ uint32_t chosen[MOST_EXPERTS][MOST_PASS / 32];                  // tokens that chose an expert
  __shared__ uint32_t place[MOST_EXPERTS], sums[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, slots = T * r.top;
  for (int t = wave; t < T; t += 16) {
    int e = -1;
    float w = 0;
    if (given) {
      if (lane < r.top) { e = given[(int64_t)t * r.top + lane]; w = given_weights[(int64_t)t * r.top + lane]; }
      // a token's choices of one expert are one, with the sum of their weights
      bool later = false;
      float sum = w;
      for (int s = 0; s < r.top && !r.logits; ++s) {                         // (a router's are different ones)
        if (s == 0) sum = 0;
        const int es = __builtin_amdgcn_readlane(e, s);
        const float ws = u2f(__builtin_amdgcn_readlane(f2u(w), s));
        if (es == e) { sum += ws; later = later || s < lane; }
      }
      w = sum;
      if (later || e < 0 || e >= r.E) e = -1;
    } else {
      route_token<NL>(r, t, e, w);
    }
    if (w == 0.0f) e = -1;                          // (an expert that weighs nothing is not asked)
    if (lane < r.top) { expert[t * r.top + lane] = e; weight[t * r.top + lane] = w; }
  }
  for (int i = tid; i < MOST_EXPERTS * (MOST_PASS / 32); i += 1024) (&chosen[0][0])[i] = 0;
  __syncthreads();
  for (int i = tid; i < slots; i += 1024) {
    const int t = i / r.top;
    if (expert[i] >= 0) atomicOr(&chosen[expert[i]][t / 32], 1u << t % 32);
  }
  __syncthreads();
  int n = 0;
  #pragma unroll
  for (int q = 0; q < MOST_PASS / 32; ++q) n += __builtin_popcount(chosen[tid][q]);
  // the sum of what the experts in front of each have, and of all
  const auto in_front = [&](uint32_t mine, uint32_t& all) {
    uint32_t sum = mine, before = 0;
    #pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const uint32_t o_ = __shfl_up(sum, d);
      if (lane >= d) sum += o_;
    }
    if (lane == 63) sums[wave] = sum;
    __syncthreads();
    all = 0;
    #pragma unroll
    for (int w = 0; w < 16; ++w) {
      before += w < wave ? sums[w] : 0;
      all += sums[w];
    }
    return before + sum - mine;
  };
  const bool split = size > MOST_DOWN;
  uint32_t all, all_down = 0, before_down = 0;
  const uint32_t before = in_front((uint32_t)n | (uint32_t)((n + size - 1) / size) << 16, all);          // slots in the low half, groups in the high half
  place[tid] = before;
  __syncthreads();
  if (split) before_down = in_front((uint32_t)((n + MOST_DOWN - 1) / MOST_DOWN), all_down);
  // (all stores behind the last barrier, which would wait for them)
  const int groups = (int)(all >> 16);
  if (tid == 0) {
    plan->groups = groups;
    plan->down_first = split ? groups : 0;
    plan->down_groups = split ? (int)all_down : groups;
  }
  for (int i = tid; i < COUNTERS; i += 1024) plan->counter[i] = 0;
  const auto list = [&](uint32_t first, int size) {
    for (int g = 0; g * size < n; ++g) {
      Group& to = plan->group[first + g];
      to.expert = tid;
      to.first = (int)(before & 0xffff) + size * g;
      to.count = n - size * g < size ? n - size * g : size;
    }
  };
  list(before >> 16, size);
  if (split) list((uint32_t)groups + before_down, MOST_DOWN);
  for (int i = tid; i < slots; i += 1024) {
    const int e = expert[i], t = i / r.top;
    int slot = -1;
    if (e >= 0) {
      int at = __builtin_popcount(chosen[e][t / 32] & ((1u << t % 32) - 1));                 // among the expert's slots
      for (int q = 0; q < t / 32; ++q) at += __builtin_popcount(chosen[e][q]);
      const uint32_t b = place[e];
      slot = (int)(b & 0xffff) + at;
      ((uint8_t*)plan->group[(b >> 16) + at / size].token)[at % size] = (uint8_t)t;
    }
    plan->slot[i] = slot;
    plan->expert[i] = e;
    plan->weight[i] = weight[i];
  }
}

// ---- the products -------------------------------------------------------------------------------------------------
struct Weights {
  const uint8_t *w, *s;
  const void* bias;
  int64_t lde, ldw, ldse, lds;                      // bytes from an expert, a row of codes, an expert's and a row's scales to the next
  int B, bias_dtype;
};

struct MoeArgs {
  const uint16_t* x;                                // planes of the tokens (bf16, or one of fp16): P of Kp, ldp apart, tokens ldx apart
  int64_t ldx, ldp;
  Weights gate_up, down;
  Plan* plan;
  uint16_t* h;                                      // [slots, PLANES, Ip]
  float *up, *out;                                  // sums of parts of K: of gate and up as the lanes hold them; of down [slots, parts, N]
  void* y;
  int T, top, N, I, Kp, Ip, activation;             // Kp, Ip: whole blocks
};

// eight codes times their scale, exactly (what is 2^128 or more: an infinity)
__device__ __forceinline__ bf16x8 decoded(int codes, float f) {
  const lcq_bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4((uint32_t)codes, f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4((uint32_t)codes, f, 1),
                   c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4((uint32_t)codes, f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4((uint32_t)codes, f, 3);
  return bf16x8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// the same to fp16: exact for scale bytes of LEAST_HALF .. MOST_HALF, as 0.5 * 2^-23 is its least number and 6 * 2^13 below its largest
constexpr uint32_t LEAST_HALF = 104, MOST_HALF = 140;
__device__ __forceinline__ f16x8 decoded_half(int codes, float f) {
  const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4((uint32_t)codes, f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4((uint32_t)codes, f, 1),
              c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4((uint32_t)codes, f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4((uint32_t)codes, f, 3);
  return f16x8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}
// eight fp16 numbers as sums of two bf16 ones, exactly (what is infinite or NaN: in the first alone)
__device__ __forceinline__ void two_of(bf16x8 raw, bf16x8 (&out)[2]) {
  const f16x8 v = __builtin_bit_cast(f16x8, raw);
  #pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float f = (float)v[e], high = u2f(bf16_bits(f) << 16);
    out[0][e] = (__bf16)high;
    out[1][e] = (__bf16)(__builtin_isfinite(f) ? f - high : 0.0f);
  }
}

__device__ __forceinline__ float act(float v, int activation) {
  return activation == LCQ_ACT_SILU ? v / (1.0f + expf(-v)) : 0.5f * v * (1.0f + erff(v * 0.70710678118654752440f));
}

// The stream of weights that both products are.  A wave has 32 rows (16 gates and their ups, or 32 channels of down), a workgroup's four waves share
// the tokens' operand.  K goes by in stages of 256 codes through LDS, all by direct loads, DEPTH - 1 stages ahead of the products:
//   codes   32 rows x 128 bytes per wave, 8 rows a load: whole lines.  (Loaded straight into the matrix pipe's layout, 16 neighbouring
//           lanes are 16 rows, and every load passes the cache 64 times for 1 KB: 3.4 TB/s.)  Piece p of row r lies at p ^ (r / 2 % 8)
//   operand rows of 512 bytes, one per slot and plane
//   scales  the word-aligned 32 bytes of a row that hold those of four stages, or of three where rows are off words: a load per wave and
//           period.  (One per stage takes as many passes of the L2 as the codes: 5.55 TB/s for 6.17 without scales.)
// One barrier per stage, in front of its products: what was read before it is loaded again.
constexpr int STAGE = 128;                          // bytes of a row's codes

// P planes of a group of GS slots are ROWS rows of the operand.  Of four slots the planes are columns of one product, four of a slot (the last one is not looked
// at), added up when a unit is done; of 16 they are blocks of 16 columns, each with a product of its own into the same sums.
template <int P, int GS>
struct Shape {
  static constexpr bool JOINED = P > 1 && GS == 4;
  static constexpr int ROWS = GS * P, CB = GS == 32 ? 2 : 1;                 // blocks of columns of the sums
  static constexpr int OB = JOINED || ROWS < 16 ? 1 : ROWS / 16;             // and of the operand
  static constexpr int X = (ROWS + 7) / 8;                                   // a wave's loads of the operand, two rows each (of the last four rows: of two waves)
  static constexpr int LOADS = 4 + X, FEWER = 4 + ROWS / 8;                  // of a stage: of the first two waves, of the others
  static constexpr int BYTES = 16384 + ROWS * 512;                           // of a stage, in LDS
  static constexpr int DEPTH = 3 * (BYTES + 4096) <= 81920 ? 3 : 163840 / (BYTES + 4096) < 5 ? 163840 / (BYTES + 4096) : 5;      // two workgroups per CU, or one
  static constexpr int LDS = DEPTH * (BYTES + 4096);
  // The row that column c of block b reads, and the slot and plane of a row.
  __device__ static constexpr int row(int b, int c) { return JOINED ? c / 4 * P + (c % 4 < P ? c % 4 : P - 1) : ROWS < 16 ? c % ROWS : b * 16 + c; }
  __device__ static constexpr int slot(int r) { return JOINED ? r / P : r % GS; }
  __device__ static constexpr int plane(int r) { return JOINED ? r % P : r / GS; }
  // 16-byte piece p of an operand's row lies at p ^ turn(c) if column c reads it.  LDS serves 16 lanes of a 16-byte read at once, of lane / 16 = 0: lanes 0 .. 3 and
  // 12 .. 15, of 1: 4 .. 11 (and the other way round, and so on), and those read pieces 4 apart: with p ^ c two of them met in a bank.
  __device__ static constexpr int turn(int r) {
    const int c = JOINED ? r / P * 4 + r % P : r & 15;
    return ROWS == 4 ? r : c ^ ((c + 4 & 8) >> 1);
  }
  static_assert(DEPTH >= 3 && (P == 1 || P == PLANES) && (GS == 4 || GS == 16 || GS == 32), "stages in LDS");
};

typedef __attribute__((address_space(3))) char* lds_ptr;
template <class T> __device__ __forceinline__ T from_lds(uint32_t at) { return *(const __attribute__((address_space(3))) T*)(lds_ptr)(size_t)at; }
// what no kernel writes while this one reads it: loaded by the scalar unit, apart from the stream of vector loads
template <class T>
__device__ __forceinline__ T fixed(const T& v) {
  struct Words { uint32_t of[sizeof(T) / 4]; } w;
  #pragma unroll
  for (int i = 0; i < (int)(sizeof(T) / 4); ++i) w.of[i] = ((const __attribute__((address_space(4))) uint32_t*)(uintptr_t)&v)[i];
  return __builtin_bit_cast(T, w);
}

// Workgroups that share a result: the last of `parts` to come here has what all of them stored.
__device__ __forceinline__ bool last_of(uint32_t* counter, int parts) {
  __shared__ uint32_t before;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) before = atomicAdd(counter, 1u);
  __syncthreads();
  if (before != (uint32_t)parts - 1) return false;
  __threadfence();
  return true;
}

// Units of work, one behind the other without a break in the stream of loads:
//   gate and up (DOWN false): (group, tile of 64 channels of h, one of `parts` parts of K), a workgroup takes every gridDim.x-th;
//   down: (group, part of K) of one tile of 128 channels, a workgroup takes one of `runs` runs of them.
// With one wave per SIMD it is bound by the instructions it issues, so what is the same for all stages of a unit, or for all but its last, is
// not looked at in every stage.
template <bool DOWN, int P, int GS, bool HALF>
__global__ __launch_bounds__(256) void experts_kernel(MoeArgs g, int tiles, int parts, int runs) {
  typedef Shape<P, GS> S;
  constexpr int CB = S::CB, OB = S::OB, DEPTH = S::DEPTH, WIDTH = DOWN ? 128 : 64;
  extern __shared__ __attribute__((aligned(1024))) char lds[];               // DEPTH stages, then as many places of scales
  const int tid = threadIdx.x, lane = tid & 63, q = lane >> 4, c = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // What a new unit asks of the arguments is loaded again there: kept all the time it would not fit the scalar registers.
  const auto args = [] {
    auto p = (const __attribute__((address_space(4))) MoeArgs*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return (const MoeArgs*)p;
  };
  const int B = DOWN ? g.down.B : g.gate_up.B, stages = (B + 7) / 8;         // blocks of a row
  const bool ragged = B % 8 != 0;                   // the last stage is not whole
  struct Who { int expert, first, count; };
  const auto who = [&](const Plan* plan, int group) {
    const Group& in = plan->group[DOWN ? fixed(plan->down_first) + group : group];
    return Who{fixed(in.expert), fixed(in.first), fixed(in.count)};
  };
  const int groups = fixed(DOWN ? g.plan->down_groups : g.plan->groups);
  int unit, end, step = 1, tile = 0;
  if constexpr (DOWN) {
    const int run = blockIdx.x / tiles, units = groups * parts;
    tile = blockIdx.x - run * tiles;
    unit = (int)((uint32_t)units * (uint32_t)run / (uint32_t)runs);          // (fewer than 2^19 units, 2^10 runs)
    end = (int)((uint32_t)units * (uint32_t)(run + 1) / (uint32_t)runs);
  } else {
    unit = blockIdx.x;
    end = groups * tiles * parts;
    step = gridDim.x;
  }
  if (unit >= end) return;

  const auto one = [](uint32_t v) { return (int)__builtin_amdgcn_readfirstlane((int)v); };
  const auto buffer = [&](const void* p, int64_t size) {
    const uint64_t at = (uint64_t)(uintptr_t)p;
    return i32x4{one((uint32_t)at), one((uint32_t)(at >> 32) & 0xffff), one((uint32_t)size), 0x00020000};
  };
  const auto load = [&](uint32_t to, uint32_t of, i32x4 buf, int at) {       // (all but `of` are the wave's)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(one(to)), "v"(of), "s"(buf), "s"(one((uint32_t)at)) : "memory");
  };
  // What is read once does not wait for places in the caches and leaves what others have there: 16 tokens of 256
  // experts 426 us so, 375 past them; 1 token 52 and 48.
  const auto weights = [&](uint32_t to, uint32_t of, i32x4 buf, int at) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen nt lds" ::"s"(one(to)), "v"(of), "s"(buf), "s"(one((uint32_t)at)) : "memory");
  };
  const uint32_t lds0 = (uint32_t)(size_t)(lds_ptr)lds;

  // ---- loads: a place in the sequence of stages, and what depends on its unit alone ----
  // the first stage of part p
  const auto first_of = [&](int p) { return (int)((uint32_t)(stages * p) / (uint32_t)parts); };
  struct Place { int unit, group, tile, part, k, end; } at;
  const auto go = [&](Place& to, int u) {
    to.unit = u;
    const int all = (uint32_t)u / (uint32_t)parts;
    to.part = u - all * parts;
    to.group = DOWN ? all : (uint32_t)all / (uint32_t)tiles;
    to.tile = DOWN ? tile : all - to.group * tiles;
    to.k = first_of(to.part);
    to.end = first_of(to.part + 1);
  };
  // a wave's channels, and rows of their two halves of 16: gates, and their ups I rows behind; down: and the next 16
  struct Rows { int n0, second, of[2]; };
  const auto rows_of = [&](const Place& p, int channels) {
    Rows r;
    r.n0 = p.tile * WIDTH + wave * (WIDTH / 4);
    r.second = DOWN ? 16 : channels;
    #pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int left = channels - r.n0 - (DOWN ? 16 * u : 0);
      r.of[u] = left < 0 ? 0 : left > 16 ? 16 : left;
    }
    return r;
  };
  // 16-byte piece of a row in a lane's place: of codes (in odd loads 4 more, as 8 rows turn it), and of the operand
  const int piece = (lane & 7) ^ (lane >> 4 & 3);
  const auto operand_piece = [&](int o) { return (lane & 31) ^ S::turn((wave + 4 * o) * 2 + (lane >> 5)); };
  const i32x4 bufX = buffer(DOWN ? g.h : g.x, 0x7fffffff);
  const int period = [&](const Weights& w) { return ((uintptr_t)w.s | (uintptr_t)w.ldse | (uintptr_t)w.lds) & 3 ? 3 : 4; }(DOWN ? g.down : g.gate_up);     // stages
  uint32_t wof[4], xof[S::X], sof;
  i32x4 bufW[2], bufS;
  const auto enter = [&]() {
    const MoeArgs* const a = args();
    const Weights w = fixed(DOWN ? a->down : a->gate_up);
    const Plan* const plan = fixed(a->plan);
    const auto [e, first, count] = who(plan, at.group);
    const Rows rows = rows_of(at, DOWN ? fixed(a->N) : fixed(a->I));
    const int64_t second = rows.second, ldx = DOWN ? 0 : fixed(a->ldx), ldp = DOWN ? fixed(a->Ip) : fixed(a->ldp);
    #pragma unroll
    for (int u = 0; u < 2; ++u)
      bufW[u] = buffer(w.w + e * w.lde + (rows.n0 + u * second) * w.ldw, rows.of[u] ? (rows.of[u] - 1) * w.ldw + B * 16 : 0);
    #pragma unroll
    for (int l = 0; l < 4; ++l) {
      const int in = (l & 1) * 8 + (lane >> 3);
      wof[l] = in < rows.of[l >> 1] ? (uint32_t)(in * w.ldw) + ((piece ^ (l & 1) * 4) << 4) : OUTSIDE;
    }
    // scales: from the first half's first row to the second half's last
    const uint8_t* const s = w.s + e * w.ldse + rows.n0 * w.lds;
    const int early = (int)((uintptr_t)s & 3);
    bufS = buffer(s - early, rows.of[0] ? (early + (rows.of[1] ? second + rows.of[1] - 1 : rows.of[0] - 1) * w.lds + w.B + 3) & ~(int64_t)3 : 0);
    const int r = lane >> 1;
    sof = (r & 15) < (r & 16 ? rows.of[1] : rows.of[0]) ? ((uint32_t)(early + ((r & 15) + (r >> 4) * second) * w.lds) & ~3u) + (lane & 1) * 16 : OUTSIDE;
    #pragma unroll
    for (int o = 0; o < S::X; ++o) {                // two rows of the operand; of a group that is not full: zeros
      uint32_t of[2];
      #pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = (wave + 4 * o) * 2 + i, slot = S::slot(r), plane = S::plane(r);
        if constexpr (DOWN) of[i] = (uint32_t)((first + slot) * PLANES + plane) * (uint32_t)(ldp * 2);
        else {
          const int token = slot < count ? (int)(fixed(plan->group[at.group].token[slot >> 2]) >> 8 * (slot & 3) & 255) : 0;
          of[i] = (uint32_t)((token * ldx + plane * ldp) * 2);
        }
        if (slot >= count) of[i] = OUTSIDE;
      }
      xof[o] = (lane & 32 ? of[1] : of[0]) + operand_piece(o) * 16;
    }
  };
  // The next stage, into a place; behind the last one: nothing, from outside.  The scales of a period come in front of its first stage.
  int lperiod = 0, lplace = DEPTH - 1;
  const auto fetch = [&](int slot) {
    const uint32_t to = lds0 + slot * S::BYTES + wave * 4096, too = lds0 + slot * S::BYTES + 16384 + wave * 1024;
    const bool over = at.unit >= end;
    if (lperiod == 0) {
      lplace = lplace == DEPTH - 1 ? 0 : lplace + 1;
      load(lds0 + DEPTH * S::BYTES + (lplace * 4 + wave) * 1024, over ? OUTSIDE : sof, bufS, at.k * 8);
      lperiod = period;
    }
    --lperiod;
    if (over || (ragged && at.k == stages - 1)) {
      const int left = over ? 0 : B - at.k * 8;   // blocks
      #pragma unroll
      for (int l = 0; l < 4; ++l) weights(to + l * 1024, (piece ^ (l & 1) * 4) < left ? wof[l] : OUTSIDE, bufW[l >> 1], at.k * STAGE);
      #pragma unroll
      for (int o = 0; o < S::X; ++o)
        if (o < S::ROWS / 8 || wave < 2) load(too + o * 4096, operand_piece(o) < left * 4 ? xof[o] : OUTSIDE, bufX, at.k * 512);
    } else {
      #pragma unroll
      for (int l = 0; l < 4; ++l) weights(to + l * 1024, wof[l], bufW[l >> 1], at.k * STAGE);
      #pragma unroll
      for (int o = 0; o < S::X; ++o)
        if (o < S::ROWS / 8 || wave < 2) load(too + o * 4096, xof[o], bufX, at.k * 512);
    }
    if (++at.k == at.end && !over) {
      go(at, at.unit + step);
      lperiod = 0;
      if (at.unit < end) enter();
    }
  };

  // ---- a unit's results: accumulator register r of lane l is channel 4 (l / 16) + r of column l % 16 ----
  const auto leave = [&](const Place& p, const Who& of, f32x4 (&acc)[2][CB]) {
    const MoeArgs* const a = args();
    const Weights w = fixed(DOWN ? a->down : a->gate_up);
    const int channels = DOWN ? fixed(a->N) : fixed(a->I), Ip = fixed(a->Ip), activation = fixed(a->activation);
    const Rows rows = rows_of(p, channels);
    if (!DOWN && parts > 1) {
      const int shared = p.group * tiles + p.tile;  // by the parts
      f32x4* const mine = (f32x4*)fixed(a->up) + ((int64_t)shared * parts * 256 + tid) * (2 * CB);
      #pragma unroll
      for (int u = 0; u < 2; ++u)
        #pragma unroll
        for (int b = 0; b < CB; ++b) mine[(int64_t)p.part * 512 * CB + u * CB + b] = acc[u][b];
      if (!last_of(&fixed(a->plan)->counter[shared], parts)) return;
      #pragma unroll
      for (int u = 0; u < 2; ++u)
        #pragma unroll
        for (int b = 0; b < CB; ++b) {
          acc[u][b] = f32x4{};
          for (int s = 0; s < parts; ++s) acc[u][b] += mine[(int64_t)s * 512 * CB + u * CB + b];
        }
    }
    #pragma unroll
    for (int b = 0; b < CB; ++b) {
      if constexpr (S::JOINED) {                    // then all lanes of a slot have its sums
        #pragma unroll
        for (int u = 0; u < 2; ++u)
          #pragma unroll
          for (int r = 0; r < 4; ++r) {
            float v = c % 4 < P ? acc[u][b][r] : 0.0f;
            v += lane_xor<1>(v);
            acc[u][b][r] = v + lane_xor<2>(v);
          }
      }
      const int s = S::JOINED ? c / 4 : b * 16 + c, mine = S::JOINED ? c % 4 : 0;
      if (s >= of.count || s >= GS) continue;
      if constexpr (DOWN) {
        #pragma unroll
        for (int u = 0; u < 2; ++u)                 // (rows of whole fours; what lies behind N is not read)
          if (mine == 0 && q * 4 < rows.of[u])
            *(f32x4*)(fixed(a->out) + ((int64_t)(of.first + s) * parts + p.part) * ((channels + 3) & ~3) + rows.n0 + u * 16 + q * 4) = acc[u][b];
      } else {
        if (rows.n0 + q * 4 >= Ip) continue;
        uint16_t h[4][PLANES];
        #pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int ch = q * 4 + r;
          float v[2] = {acc[0][b][r], acc[1][b][r]};
          if (w.bias && ch < rows.of[0]) {
            #pragma unroll
            for (int u = 0; u < 2; ++u) v[u] += load_any(w.bias, w.bias_dtype, ((int64_t)of.expert * 2 + u) * channels + rows.n0 + ch);
          }
          planes_of(ch < rows.of[0] ? act(v[0], activation) * v[1] : 0.0f, h[r]);
        }
        #pragma unroll
        for (int l = 0; l < PLANES; ++l)
          if (!S::JOINED || l == mine)
            *(u32x2*)(fixed(a->h) + ((int64_t)(of.first + s) * PLANES + l) * Ip + rows.n0 + q * 4) = u32x2{h[0][l] | (uint32_t)h[1][l] << 16, h[2][l] | (uint32_t)h[3][l] << 16};
      }
    }
  };

  // ---- products ----
  go(at, unit);
  enter();
  #pragma unroll
  for (int d = 0; d < DEPTH - 1; ++d) fetch(d);
  Place now;
  Who in;
  uint32_t scales[2];                               // this lane's: of a row whose bytes start (row's address) % 4 early
  const auto begin = [&]() {
    const MoeArgs* const a = args();
    const Weights w = fixed(DOWN ? a->down : a->gate_up);
    in = who(fixed(a->plan), now.group);
    const Rows rows = rows_of(now, DOWN ? fixed(a->N) : fixed(a->I));
    #pragma unroll
    for (int u = 0; u < 2; ++u)
      scales[u] = lds0 + DEPTH * S::BYTES + wave * 1024 + u * 512 + c * 32 + q +
                  (((uint32_t)(uintptr_t)w.s + (uint32_t)in.expert * (uint32_t)w.ldse + (uint32_t)(rows.n0 + c + u * rows.second) * (uint32_t)w.lds) & 3);
  };
  go(now, unit);
  begin();
  uint32_t codes[2], operand[4];
  #pragma unroll
  for (int i = 0; i < 2; ++i) codes[i] = lds0 + wave * 4096 + c * 128 + (((i * 4 + q) ^ (c >> 1 & 7)) << 4);
  const int row = S::row(0, c);                     // (of block b 16 b behind it)
  #pragma unroll
  for (int j = 0; j < 4; ++j) operand[j] = lds0 + 16384 + row * 512 + (((q * 4 + j) ^ S::turn(row)) << 4);
  int slot = 0, cperiod = 0, cplace = 0;
  for (;;) {
    f32x4 acc[2][CB] = {};
    do {
      // the next stage has landed, and this wave has read the last one
      constexpr int MORE = (DEPTH - 2) * S::LOADS, LESS = (DEPTH - 2) * S::FEWER;              // loads that may be on their way
      if (MORE != LESS && wave >= 2) __builtin_amdgcn_s_waitcnt(0x0070 | (LESS & 15) | LESS >> 4 << 14);
      else __builtin_amdgcn_s_waitcnt(0x0070 | (MORE & 15) | MORE >> 4 << 14);
      asm volatile("s_barrier" ::: "memory");
      fetch(slot == 0 ? DEPTH - 1 : slot - 1);
      const uint32_t here = slot * S::BYTES, scales_here = cplace * 4096 + cperiod * 8;
      // all reads of the stage, then the products: left to itself the compiler has two of them on their way, and a wave alone on its SIMD waits
      // for each
      i32x4 wv[2][2];
      uint32_t byte[2][2];
      bf16x8 x[2][4][OB];
      #pragma unroll
      for (int i = 0; i < 2; ++i) {
        #pragma unroll
        for (int u = 0; u < 2; ++u) {
          wv[u][i] = from_lds<i32x4>(codes[i] + here + u * 2048);
          byte[u][i] = from_lds<uint8_t>(scales[u] + scales_here + i * 4);
        }
        #pragma unroll
        for (int j = 0; j < 4; ++j)
          #pragma unroll
          for (int b = 0; b < OB; ++b) x[i][j][b] = from_lds<bf16x8>(operand[j] + here + i * 256 + b * 8192);
      }
      __builtin_amdgcn_sched_barrier(0);
      const int left = B - now.k * 8;
      if constexpr (HALF) {
        bool other = false;                         // (a block behind the last has zeros for codes: any scale will do)
        #pragma unroll
        for (int i = 0; i < 2; ++i)
          #pragma unroll
          for (int u = 0; u < 2; ++u) {
            byte[u][i] = i * 4 + q < left ? byte[u][i] : 127u;
            other = other || byte[u][i] < LEAST_HALF || byte[u][i] > MOST_HALF;
          }
        bool apart = false;
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(other) != 0, 0)) {  // (nor does it matter to blocks of zeros, as all are behind the last channel)
          other = false;
          #pragma unroll
          for (int i = 0; i < 2; ++i)
            #pragma unroll
            for (int u = 0; u < 2; ++u) {
              if (byte[u][i] != 255 && (wv[u][i][0] | wv[u][i][1] | wv[u][i][2] | wv[u][i][3]) == 0) byte[u][i] = 127u;
              other = other || byte[u][i] < LEAST_HALF || byte[u][i] > MOST_HALF;
            }
          apart = __builtin_amdgcn_ballot_w64(other) != 0;
        }
        if (__builtin_expect(apart, 0)) {
          #pragma unroll
          for (int i = 0; i < 2; ++i)
            #pragma unroll
            for (int j = 0; j < 4; ++j) {
              bf16x8 v[2];
              #pragma unroll
              for (int u = 0; u < 2; ++u) v[u] = decoded(wv[u][i][j], mx_factor(byte[u][i]));
              #pragma unroll
              for (int b = 0; b < CB; ++b) {
                bf16x8 two[2];
                two_of(x[i][j][b], two);
                #pragma unroll
                for (int u = 0; u < 2; ++u)
                  #pragma unroll
                  for (int l = 0; l < 2; ++l) acc[u][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v[u], two[l], acc[u][b], 0, 0, 0);
              }
            }
        } else {
          #pragma unroll
          for (int i = 0; i < 2; ++i)
            #pragma unroll
            for (int j = 0; j < 4; ++j) {
              f16x8 v[2];
              #pragma unroll
              for (int u = 0; u < 2; ++u) v[u] = decoded_half(wv[u][i][j], mx_factor(byte[u][i]));
              #pragma unroll
              for (int b = 0; b < CB; ++b)
                #pragma unroll
                for (int u = 0; u < 2; ++u) acc[u][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[u], __builtin_bit_cast(f16x8, x[i][j][b]), acc[u][b], 0, 0, 0);
            }
        }
      } else
      #pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t there = i * 4 + q < left ? 255u : 0u;                 // (behind the last block: not a NaN)
        #pragma unroll
        for (int j = 0; j < 4; ++j) {
          bf16x8 v[2];
          #pragma unroll
          for (int u = 0; u < 2; ++u) v[u] = decoded(wv[u][i][j], mx_factor(byte[u][i] & there));
          #pragma unroll
          for (int b = OB - 1; b >= 0; --b)         // (the smallest planes first)
            #pragma unroll
            for (int u = 0; u < 2; ++u) acc[u][b % CB] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v[u], x[i][j][b], acc[u][b % CB], 0, 0, 0);
        }
      }
      slot = slot == DEPTH - 1 ? 0 : slot + 1;
      cperiod = cperiod == period - 1 ? 0 : cperiod + 1;
      if (cperiod == 0) cplace = cplace == DEPTH - 1 ? 0 : cplace + 1;
    } while (++now.k < now.end);
    leave(now, in, acc);
    go(now, now.unit + step);
    if (now.unit >= end) break;
    begin();
    if (cperiod) cplace = cplace == DEPTH - 1 ? 0 : cplace + 1;                // (a unit starts a period)
    cperiod = 0;
  }
  __builtin_amdgcn_s_waitcnt(0x0f70);               // nothing may still be on its way to LDS when the workgroup leaves it
}

// y of four channels of a token per lane: the weighted sum of its choices' parts in their order, eight of them on their way at a time in each of
// four waves.
template <int BF>
__global__ __launch_bounds__(256) void sum_kernel(MoeArgs g, int parts) {
  __shared__ int slot[MOST_TOP];
  __shared__ float weight[MOST_TOP];
  __shared__ f32x4 some[4][64];
  const int t = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = (blockIdx.x * 64 + lane) * 4, Np = (g.N + 3) & ~3;
  if (threadIdx.x < g.top) {
    slot[threadIdx.x] = g.plan->slot[t * g.top + threadIdx.x];
    weight[threadIdx.x] = g.plan->weight[t * g.top + threadIdx.x];
  }
  __syncthreads();
  const int all = g.top * parts, end = all * (wave + 1) / 4;
  f32x4 y = {};
  if (n < g.N) {
    for (int i0 = all * wave / 4; i0 < end; i0 += 8) {
      f32x4 v[8];
      float w[8];
      #pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int i = i0 + j < end ? i0 + j : end - 1, s = i / parts, at = slot[s];
        w[j] = i0 + j < end && at >= 0 ? weight[s] : 0.0f;
        v[j] = f32x4{};
        if (w[j] != 0.0f) v[j] = *(const f32x4*)(g.out + ((int64_t)at * parts + (i - s * parts)) * Np + n);  // (what has no weight may be anything)
      }
      #pragma unroll
      for (int j = 0; j < 8; ++j)
        #pragma unroll
        for (int r = 0; r < 4; ++r) y[r] = __builtin_fmaf(w[j], v[j][r], y[r]);
    }
  }
  some[wave][lane] = y;
  __syncthreads();
  if (wave || n >= g.N) return;
  #pragma unroll
  for (int s = 1; s < 4; ++s) y += some[s][lane];
  const int left = g.N - n;
  if (g.down.bias) {
    for (int s = 0; s < g.top; ++s) {
      if (slot[s] < 0) continue;
      const int64_t at = (int64_t)g.plan->expert[t * g.top + s] * g.N + n;
      #pragma unroll
      for (int r = 0; r < 4; ++r) if (r < left) y[r] = __builtin_fmaf(weight[s], load_any(g.down.bias, g.down.bias_dtype, at + r), y[r]);
    }
  }
  const int64_t to = (int64_t)t * g.N + n;
  #pragma unroll
  for (int r = 0; r < 4; ++r) {
    if (r >= left) break;
    if constexpr (BF == ROW_F32) ((float*)g.y)[to + r] = y[r];
    else store_scalar<BF>(g.y, to + r, rnd<BF>(y[r]));
  }
}

bool known(int dtype) { return dtype == LCQ_F32 || dtype == LCQ_BF16 || dtype == LCQ_F16; }
int64_t on256(int64_t bytes) { return (bytes + 255) / 256 * 256; }
int64_t least(int64_t a, int64_t b) { return a < b ? a : b; }

int check_router(const RouterArgs& r, int64_t T) {
  if (T <= 0 || r.E <= 0 || r.top <= 0 || r.top > r.E || r.ldl < 0) return LCQ_EINVAL;
  if (r.E > MOST_EXPERTS || r.top > MOST_TOP || T > 1 << 25) return LCQ_ESIZE;
  return LCQ_OK;
}

// are the tokens planes as they are?
bool direct(int dtype, const void* x, int64_t ldx, int64_t K) {
  return dtype != LCQ_F32 && K % 32 == 0 && ldx % 8 == 0 && (uintptr_t)x % 16 == 0 && ldx <= 1 << 22;       // (offsets have 31 bits)
}

// tokens of a pass: as many as the offsets within h, 31 bits, have room for (85 at least)
int64_t pass_of(int64_t top, int64_t I) { return least(MOST_PASS, (1 << 30) / (top * PLANES * ((I + 31) / 32 * 32) * 2)); }

// How a pass of T tokens is cut.
struct Cut {
  int P, size, up_tiles, up_parts, down_tiles, down_parts, runs;
  int64_t groups, h, up, out;                       // bytes
  Cut(int64_t T, int64_t top, int64_t E, int64_t K, int64_t I, int64_t N, int dtype) {
    P = dtype == LCQ_F32 ? PLANES : 1;
    const int64_t slots = T * top;
    // Slots of a group: few columns cost less in every stage, a second group of an expert reads its bytes again.  The whole layer in us with 4 / 16 / 32:
    //   4 tokens, 6 of 64 experts 2048 x 1408 41 / 51 / 54    16 tokens, 8 of 256 7168 x 2048 379 / 516 / 580    64 tokens, 4 of 32 4096 x 1408 152 / 100 / 107
    //   64 tokens, 2 of 8 4096 x 4096 161 / 104 / 100    96 tokens 208 / 124 / 111
    size = T <= 4 || slots <= E ? 4 : P > 1 || T <= 16 || slots <= 18 * E ? 16 : 32;
    const auto groups_of = [&](int size) { return least(slots, least(E, slots) + slots / size); };
    groups = groups_of(size);
    const int64_t up_stages = ((K + 31) / 32 + 7) / 8, down_stages = ((I + 31) / 32 + 7) / 8, Ip = (I + 31) / 32 * 32;
    up_tiles = (int)((Ip + 63) / 64);
    // Parts of K of gate and up, where a few narrow experts leave the chip to a few long units: a stage is 0.45 us, making sums visible to the workgroup that adds
    // them up 0.15 for every workgroup.  1 token, 1 of 4 experts 14336 x 128 in 1 / 2 / 4 / 8 parts 52 / 37 / 29 / 27 us, 2 of 8 7168 x 256 34 / 29 / 28 / 32, but 4 of 16
    // 1024 x 512 20 / 30 and 8 of 256 7168 x 2048 50 / 172.
    up_parts = 1;
    while (3 * up_stages > 2 * groups * up_tiles * up_parts * up_parts && up_stages / (2 * up_parts) >= 3) up_parts *= 2;
    down_tiles = (int)((N + 127) / 128);
    // Runs of down: two workgroups per CU (64 tokens, 4 of 32 experts with 1 / 2 / 4 per CU 99 / 100 / 109, 16 tokens, 8 of 256 417 / 379 / 386); K in parts
    // where there are too few groups for them (1 token, 2 of 8 experts 4096 x 14336 in 1 / 2 / 4 / 8 parts 77 / 60 / 54 / 54; 8 of 256 53 / 53 / 55 / 61).
    int64_t want = 512 / down_tiles;
    if (want < 1) want = 1;
    down_parts = 1;
    const int64_t down_groups = groups_of(size < MOST_DOWN ? size : MOST_DOWN);
    while (down_groups * down_parts < 6 * want && down_stages / (2 * down_parts) >= 6) down_parts *= 2;
    const int64_t units = down_groups * down_parts, each = (units + want - 1) / want;
    runs = (int)((units + each - 1) / each);
    h = on256(slots * PLANES * Ip * 2);
    up = up_parts > 1 ? on256(groups * up_tiles * up_parts * 256 * 32 * (size == 32 ? 2 : 1)) : 0;
    out = on256(slots * down_parts * ((N + 3) & ~(int64_t)3) * 4);
  }
};

template <bool DOWN, int P, int GS, bool HALF>
int launch_experts(const MoeArgs& g, const Cut& c, hipStream_t st) {
  typedef Shape<P, GS> S;
  const auto kernel = experts_kernel<DOWN, P, GS, HALF>;
  // (more LDS than a launch may have without asking)
  if (hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, S::LDS) != hipSuccess) return LCQ_ELAUNCH;
  // as many as run at a time, or fewer
  const int64_t blocks = DOWN ? (int64_t)c.down_tiles * c.runs : least(c.groups * c.up_tiles * c.up_parts, 256 * (163840 / S::LDS));
  kernel<<<dim3((unsigned)blocks), dim3(256), S::LDS, st>>>(g, DOWN ? c.down_tiles : c.up_tiles, DOWN ? c.down_parts : c.up_parts, c.runs);
  return LCQ_OK;
}
template <bool DOWN, int P, bool HALF>
int launch_size(const MoeArgs& g, const Cut& c, hipStream_t st) {
  if (c.size == 4) return launch_experts<DOWN, P, 4, HALF>(g, c, st);
  if constexpr (P == 1) { if (c.size == 32) return launch_experts<DOWN, P, 32, HALF>(g, c, st); }
  return launch_experts<DOWN, P, MOST_DOWN, HALF>(g, c, st);
}
template <int BF>
void launch_sum(const MoeArgs& g, const Cut& c, hipStream_t st) {
  sum_kernel<BF><<<dim3((unsigned)((g.N + 255) / 256), (unsigned)g.T), dim3(256), 0, st>>>(g, c.down_parts);
}

}  // namespace

extern "C" {

int lcq_route(const void* logits, int dtype, int64_t T, int64_t E, int64_t ldl, int top, int flags, const float* correction, float scale, int* experts,
              float* weights, void* stream) {
  if (!logits || !experts || !weights || E > (1 << 30)) return LCQ_EINVAL;
  const RouterArgs r = {logits, correction, ldl, dtype, (int)E, top, flags, scale};
  const int bad = check_router(r, T);
  if (bad) return bad;
  if (!known(dtype)) return LCQ_EDTYPE;
  const dim3 grid((unsigned)((T + 3) / 4));
  hipStream_t st = (hipStream_t)stream;
  if (E <= 64) route_kernel<1><<<grid, dim3(256), 0, st>>>(r, T, experts, weights);
  else if (E <= 256) route_kernel<4><<<grid, dim3(256), 0, st>>>(r, T, experts, weights);
  else route_kernel<16><<<grid, dim3(256), 0, st>>>(r, T, experts, weights);
  LCQ_CHECK_LAUNCH();
  return LCQ_OK;
}

int64_t lcq_mxfp4_moe_workspace_bytes(int64_t T, int64_t top, int64_t E, int64_t K, int64_t I, int64_t N, int dtype) {
  if (T <= 0 || top <= 0 || E <= 0 || K <= 0 || I <= 0 || N <= 0 || K > 65536 || I > 65536 || N > 65536 || top > MOST_TOP || E > MOST_EXPERTS || !known(dtype)) return 0;
  const int64_t pass = pass_of(top, I), t = least(T, pass);
  int64_t most = 0;                                 // (the last pass may have fewer tokens, and be cut into more parts)
  for (const int64_t n : {t, T % pass ? T % pass : t}) {
    const Cut c(n, top, E, K, I, N, dtype);
    const int64_t size = c.h + c.up + c.out + on256(n * c.P * ((K + 31) / 32 * 32) * 2) + on256(n * top * 8);
    most = size > most ? size : most;
  }
  return on256(sizeof(Plan)) + most;
}

int lcq_mxfp4_moe(const void* x, int dtype, int64_t T, int64_t K, int64_t ldx, const void* logits, int logits_dtype, int64_t ldl, int flags,
                  const float* correction, float scale, const int* experts, const float* weights, int64_t E, int top, const uint8_t* gate_up,
                  int64_t gate_up_lde, int64_t gate_up_ld, const uint8_t* gate_up_scales, int64_t gate_up_ldse, int64_t gate_up_lds,
                  const void* gate_up_bias, const uint8_t* down, int64_t down_lde, int64_t down_ld, const uint8_t* down_scales, int64_t down_ldse,
                  int64_t down_lds, const void* down_bias, int bias_dtype, int64_t I, int64_t N, int activation, void* y, int out_dtype,
                  void* workspace, void* stream) {
  if (!x || !gate_up || !gate_up_scales || !down || !down_scales || !y || ldx < 0 || E > (1 << 30)) return LCQ_EINVAL;
  if ((logits != nullptr) == (experts != nullptr) || (experts && !weights)) return LCQ_EINVAL;
  if (K <= 0 || I <= 0 || N <= 0 || (activation != LCQ_ACT_SILU && activation != LCQ_ACT_GELU)) return LCQ_EINVAL;
  RouterArgs r = {logits, correction, ldl, logits_dtype, (int)E, top, flags, scale};
  const int bad = check_router(r, T);
  if (bad) return bad;
  if (!known(dtype) || !known(out_dtype) || (logits && !known(logits_dtype)) || ((gate_up_bias || down_bias) && !known(bias_dtype))) return LCQ_EDTYPE;
  if (K > 65536 || I > 65536 || N > 65536) return LCQ_ESIZE;
  const int64_t B = (K + 31) / 32, BI = (I + 31) / 32, Kp = 32 * B, Ip = 32 * BI;
  if (gate_up_ld < 16 * B || gate_up_lds < B || down_ld < 16 * BI || down_lds < BI) return LCQ_EINVAL;
  if (gate_up_ld > 1 << 22 || down_ld > 1 << 22 || gate_up_lds > (1 << 30) / (I + 64) || down_lds > 1 << 22) return LCQ_ESIZE;
  if ((uintptr_t)gate_up % 16 || gate_up_ld % 16 || gate_up_lde % 16 || (uintptr_t)down % 16 || down_ld % 16 || down_lde % 16) return LCQ_EALIGN;
  if (!workspace) return LCQ_EWORKSPACE;
  if ((uintptr_t)workspace % 16) return LCQ_EALIGN;
  hipStream_t st = (hipStream_t)stream;
  char* const ws = (char*)workspace;
  const bool as_is = direct(dtype, x, ldx, K);
  Plan* const plan = (Plan*)ws;
  const int64_t size = dtype == LCQ_F32 ? 4 : 2, out_size = out_dtype == LCQ_F32 ? 4 : 2, logit_size = logits_dtype == LCQ_F32 ? 4 : 2;
  const int64_t pass = pass_of(top, I);
  for (int64_t t0 = 0; t0 < T; t0 += pass) {
    const int n = (int)least(T - t0, pass);
    const Cut c(n, top, E, K, I, N, dtype);
    char* at = ws + on256(sizeof(Plan));
    uint16_t* const h = (uint16_t*)at;
    float* const up_sums = (float*)(at += c.h);
    float* const out_sums = (float*)(at += c.up);
    uint16_t* const planes = (uint16_t*)(at += c.out);
    const char* const xt = (const char*)x + t0 * ldx * size;
    RouterArgs rt = r;
    if (logits) rt.logits = (const char*)logits + t0 * ldl * logit_size;
    const Operand o = {xt, ldx, dtype, c.P, (int)K, (int)Kp, planes};
    const dim3 grid(as_is ? 1u : 1u + (unsigned)least((n * Kp + 1023) / 1024, 255));
    const int64_t slots = (int64_t)n * top;
    const int* ge = experts ? experts + t0 * top : nullptr;
    const float* gw = experts ? weights + t0 * top : nullptr;
    if (logits && n > 16) {                         // (the plan's 16 waves would take turns; up to there a kernel less is 2 us less)
      int* const e = (int*)((char*)planes + on256(n * c.P * Kp * 2));
      const int rc = lcq_route(rt.logits, logits_dtype, n, E, ldl, top, flags, correction, scale, e, (float*)(e + slots), stream);
      if (rc) return rc;
      ge = e;
      gw = (float*)(e + slots);
    }
    const MoeArgs g = {as_is ? (const uint16_t*)xt : planes, as_is ? ldx : c.P * Kp, Kp,
                       {gate_up, gate_up_scales, gate_up_bias, gate_up_lde, gate_up_ld, gate_up_ldse, gate_up_lds, (int)B, bias_dtype},
                       {down, down_scales, down_bias, down_lde, down_ld, down_ldse, down_lds, (int)BI, bias_dtype}, plan, h, up_sums, out_sums,
                       (char*)y + t0 * N * out_size, n, top, (int)N, (int)I, (int)Kp, (int)Ip, activation};
    if (E <= 64) plan_kernel<1><<<grid, dim3(1024), 0, st>>>(rt, ge, gw, n, o, c.size, plan);
    else if (E <= 256) plan_kernel<4><<<grid, dim3(1024), 0, st>>>(rt, ge, gw, n, o, c.size, plan);
    else plan_kernel<16><<<grid, dim3(1024), 0, st>>>(rt, ge, gw, n, o, c.size, plan);
    int rc = dtype == LCQ_BF16 ? launch_size<false, 1, false>(g, c, st) : dtype == LCQ_F16 ? launch_size<false, 1, true>(g, c, st) : launch_size<false, PLANES, false>(g, c, st);
    if (rc) return rc;
    rc = launch_size<true, PLANES, false>(g, c, st);
    if (rc) return rc;
    if (out_dtype == LCQ_BF16) launch_sum<ROW_BF16>(g, c, st);
    else if (out_dtype == LCQ_F16) launch_sum<ROW_F16>(g, c, st);
    else launch_sum<ROW_F32>(g, c, st);
  }
  LCQ_CHECK_LAUNCH();
  return LCQ_OK;
}

}  // extern "C"

// A mixture-of-experts layer for a few tokens, on experts of microscaled 4-bit numbers:
//   y[t] = sum_s w[t, s] (down_e h + down_bias_e),   h = act(gate_e x[t] + b) * (up_e x[t] + b),   e = experts[t, s]
// Tokens that chose the same expert share one pass over its bytes, which is what bounds the layer.
//
// The activations keep their precision.  A lane takes a block of a weight row, 16 bytes, and the conversion to bf16 applies its scale: that is
// exact, so the products are those of the stored numbers.  bf16 tokens go into the matrix pipe as they are, others as sums of bf16 planes
// (fp16: two, exactly; fp32: three, to 2^-24); h, which stays within the layer, as two planes (2^-17), or three for fp32 tokens.
#include "mxfp4.h"
#include <type_traits>

namespace {
using namespace lcq;

typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;

template <int I> using Int = std::integral_constant<int, I>;

constexpr int MOST_EXPERTS = 1024, MOST_TOP = 32, MOST_PASS = 128;           // tokens of a pass
constexpr int MOST_GROUP = 32, COUNTERS = 1024;
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
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true); }
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  const auto take = [&](uint32_t o) { v = o > v ? o : v; };
  take(dpp_u<0xB1>(v));
  take(dpp_u<0x4E>(v));
  take(dpp_u<0x141>(v));
  take(dpp_u<0x140>(v));
  take((uint32_t)__builtin_amdgcn_ds_swizzle((int)v, 0x401F));
  const uint32_t lo = __builtin_amdgcn_readlane(v, 0), hi = __builtin_amdgcn_readlane(v, 32);
  return lo > hi ? lo : hi;
}
__device__ __forceinline__ double wave_sum(double v) {
  #pragma unroll
  for (int m = 1; m < 64; m *= 2) v += __shfl_xor(v, m);
  return v;
}

// One token by one wave: lane s < top gets the s-th choice.  A lane looks at NL consecutive experts.
//  softmax: e^(l - max) / sum;  sigmoid: 1 / (1 + e^-l).  Chosen by the logits (both grow with them), or, with a correction, by
//  fp32(score) + correction, the scores from 64 bits, so that they are the numbers they should be to the last bit.
// -inf is chosen last and weighs 0.
template <int NL>
__device__ __forceinline__ void route_token(const RouterArgs& r, int64_t t, int& expert, float& weight) {
  const int lane = threadIdx.x & 63;
  float x[NL], score[NL];
  uint32_t key[NL];
  float m = -__builtin_inff();
  #pragma unroll
  for (int j = 0; j < NL; ++j) {
    const int e = lane * NL + j;
    x[j] = e < r.E ? load_any(r.logits, r.dtype, t * r.ldl + e) : -__builtin_inff();
    m = nan_max(m, x[j]);
  }
  const float none = -__builtin_inff();
  if (!(r.flags & LCQ_ROUTE_SIGMOID)) m = team_reduce<64, true>(m);
  if (r.correction) {
    double s[NL], sum = 0;
    #pragma unroll
    for (int j = 0; j < NL; ++j) {
      if (r.flags & LCQ_ROUTE_SIGMOID) s[j] = 1.0 / (1.0 + exp(-(double)x[j]));
      else { s[j] = x[j] == none ? 0.0 : exp((double)x[j] - (double)m); sum += s[j]; }
    }
    if (!(r.flags & LCQ_ROUTE_SIGMOID)) sum = wave_sum(sum);
    #pragma unroll
    for (int j = 0; j < NL; ++j) {
      const int e = lane * NL + j;
      score[j] = (float)(r.flags & LCQ_ROUTE_SIGMOID ? s[j] : sum == 0.0 ? 0.0 : s[j] / sum);
      key[j] = e >= r.E ? 0u : ordered(x[j] == none ? none : score[j] + r.correction[e]);
    }
  } else {
    float sum = 0;
    #pragma unroll
    for (int j = 0; j < NL; ++j) {
      if (r.flags & LCQ_ROUTE_SIGMOID) score[j] = 1.0f / (1.0f + expf(-x[j]));
      else { score[j] = x[j] == none ? 0.0f : expf(x[j] - m); sum += score[j]; }
      key[j] = lane * NL + j < r.E ? ordered(x[j]) : 0u;
    }
    if (!(r.flags & LCQ_ROUTE_SIGMOID)) {
      sum = team_sum<64>(sum);
      #pragma unroll
      for (int j = 0; j < NL; ++j) score[j] = sum == 0.0f ? 0.0f : score[j] / sum;
    }
  }
  expert = 0;
  weight = 0;
  for (int s = 0; s < r.top; ++s) {
    uint32_t best = key[0];
    int at = 0;
    float w = score[0];
    #pragma unroll
    for (int j = 1; j < NL; ++j)
      if (key[j] > best) { best = key[j]; at = j; w = score[j]; }
    const uint32_t most = wave_max(best);
    const int from = __builtin_ctzll(__ballot(best == most));                // (the lowest lane has the lowest experts)
    const int e = from * NL + __builtin_amdgcn_readlane(at, from);
    const float we = u2f(__builtin_amdgcn_readlane(f2u(w), from));
    if (lane == s) { expert = e; weight = we; }
    #pragma unroll
    for (int j = 0; j < NL; ++j)
      if (lane == from && at == j) key[j] = 0;
  }
  if (r.flags & LCQ_ROUTE_RENORMALIZE) {
    const float sum = team_sum<64>(weight);
    weight = sum == 0.0f ? 0.0f : weight / sum;
  }
  weight *= r.scale;
}

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
// A pass: the slots (token and choice) sorted by expert, in groups of at most `size` of one expert.
struct Group {
  int expert, first, count, pad;                    // first: slot
  uint8_t token[MOST_GROUP];
};
struct Plan {
  int groups, pad[15];
  uint32_t counter[2][COUNTERS];                    // parts that are done: of gate and up, of down
  int slot[MOST_PASS * MOST_TOP], expert[MOST_PASS * MOST_TOP];              // of a token's choices; slot -1: none
  float weight[MOST_PASS * MOST_TOP];
  Group group[MOST_PASS * MOST_TOP];
};

struct Operand { const char* x; int64_t ldx; int dtype, planes, K, Kp; uint16_t* out; };

// Values as sums of bf16 numbers (what is infinite or NaN: in the first alone).
template <int P>
__device__ __forceinline__ void planes_of(float v, uint16_t* out) {
  #pragma unroll
  for (int p = 0; p < P; ++p) {
    const uint32_t u = bf16_bits(v);
    out[p] = (uint16_t)u;
    const float taken = u2f(u << 16);
    v = (u & 0x7f80) == 0x7f80 ? 0.0f : v - taken;
  }
}

// Workgroup 0 plans the pass; the others lay the tokens out as planes [T, planes, Kp] where they are not that already.
template <int NL>
__global__ __launch_bounds__(1024) void plan_kernel(RouterArgs r, const int* __restrict__ given, const float* __restrict__ given_weights, int T,
                                                    Operand o, int size, int most_groups, Plan* __restrict__ plan) {
  if (blockIdx.x) {
    const int64_t all = (int64_t)T * o.Kp;
    for (int64_t i = (int64_t)(blockIdx.x - 1) * 1024 + threadIdx.x; i < all; i += (int64_t)(gridDim.x - 1) * 1024) {
      const int64_t t = i / o.Kp;
      const int k = (int)(i - t * o.Kp);
      const float v = k < o.K ? load_any(o.x, o.dtype, t * o.ldx + k) : 0.0f;
      uint16_t p[3] = {};
      planes_of<3>(v, p);
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
      float sum = 0;
      for (int s = 0; s < r.top; ++s) {
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
  for (int i = tid; i < 2 * COUNTERS; i += 1024) (&plan->counter[0][0])[i] = 0;
  __syncthreads();
  for (int i = tid; i < slots; i += 1024) {
    const int t = i / r.top;
    if (expert[i] >= 0) atomicOr(&chosen[expert[i]][t / 32], 1u << t % 32);
  }
  __syncthreads();
  // slots of the experts in front of each in the low half, their groups in the high half
  uint32_t mine = 0;
  #pragma unroll
  for (int q = 0; q < MOST_PASS / 32; ++q) mine += __builtin_popcount(chosen[tid][q]);
  const int n = (int)mine;
  mine |= (uint32_t)((n + size - 1) / size) << 16;
  uint32_t sum = mine;
  #pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const uint32_t o_ = __shfl_up(sum, d);
    if (lane >= d) sum += o_;
  }
  if (lane == 63) sums[wave] = sum;
  __syncthreads();
  for (int w = 0; w < wave; ++w) sum += sums[w];
  __syncthreads();
  const uint32_t before = sum - mine;
  place[tid] = before;
  for (int g = 0; g * size < n; ++g) {
    Group& to = plan->group[(before >> 16) + g];
    to.expert = tid;
    to.first = (int)(before & 0xffff) + size * g;
    to.count = n - size * g < size ? n - size * g : size;
  }
  if (tid == 1023) sums[0] = sum >> 16;
  __syncthreads();
  const int groups = (int)sums[0];
  if (tid == 0) plan->groups = groups;
  for (int g = groups + tid; g < most_groups; g += 1024) plan->group[g].count = 0;
  for (int i = tid; i < slots; i += 1024) {
    const int e = expert[i], t = i / r.top;
    int slot = -1;
    if (e >= 0) {
      int at = __builtin_popcount(chosen[e][t / 32] & ((1u << t % 32) - 1));                 // among the expert's slots
      for (int q = 0; q < t / 32; ++q) at += __builtin_popcount(chosen[e][q]);
      const uint32_t b = place[e];
      slot = (int)(b & 0xffff) + at;
      plan->group[(b >> 16) + at / size].token[at % size] = (uint8_t)t;
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
  const uint16_t* x;                                // planes of the tokens: P of Kp, ldp apart, tokens ldx apart
  int64_t ldx, ldp;
  Weights gate_up, down;
  Plan* plan;
  uint16_t* h;                                      // [slots, PH, Ip]
  float *up, *out;                                  // sums of parts of K: of gate and up as the lanes hold them; of down [slots, parts, N]
  void* y;
  int T, top, N, I, Kp, Ip, activation;             // Kp, Ip: whole blocks
};

// eight codes times their scale, exactly
__device__ __forceinline__ bf16x8 decoded(int codes, float f) {
  const lcq_bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4((uint32_t)codes, f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4((uint32_t)codes, f, 1),
                   c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4((uint32_t)codes, f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4((uint32_t)codes, f, 3);
  return bf16x8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

__device__ __forceinline__ float act(float v, int activation) {
  return activation == LCQ_ACT_SILU ? v / (1.0f + expf(-v)) : 0.5f * v * (1.0f + erff(v * 0.70710678118654752440f));
}

// The stream of weights that both products are.  A wave has 32 rows (16 gates and their ups, or 32 channels of down), a workgroup's four waves share
// the tokens' operand.  K goes by in stages of 256 codes through LDS, all by direct loads, DEPTH - 1 stages ahead of the products:
//   codes   32 rows x 128 bytes per wave, 8 rows a load: whole lines.  (Loaded straight into the matrix pipe's layout, 16 neighbouring
//           lanes are 16 rows, and every load passes the cache 64 times for 1 KB: 3.4 TB/s.)  Piece p of row r lies at p ^ (r / 2 % 8)
//   operand rows of 512 bytes, one per slot and plane; piece p of slot s lies at p ^ (s % 16)
//   scales  the word-aligned 32 bytes of a row that hold those of four stages, or of three where rows are off words: a load per wave and
//           period.  (One per stage takes as many passes of the L2 as the codes: 5.55 TB/s for 6.17 without scales.)
// so that 16 lanes of a read touch all banks once.  One barrier per stage, in front of its products: what was read before it is loaded again.
constexpr int STAGE = 128;                          // bytes of a row's codes

template <int P, int GS>
struct Shape {
  static constexpr int XOPS = GS * P / 2, X = (XOPS + 3) / 4, FULL = XOPS % 4;               // loads of the operand: of all waves, of the first FULL (0: of all)
  static constexpr int BYTES = 16384 + GS * P * 512;                         // of a stage, in LDS
  static constexpr int DEPTH = 3 * (BYTES + 4096) <= 81920 ? 3 : 163840 / (BYTES + 4096) < 5 ? 163840 / (BYTES + 4096) : 5;      // two workgroups per CU, or one
  static constexpr int LDS = DEPTH * (BYTES + 4096), TB = (GS + 15) / 16;
  static_assert(DEPTH >= 3, "stages in LDS");
};

typedef __attribute__((address_space(3))) char* lds_ptr;
// what no kernel writes while this one reads it: loaded by the scalar unit, apart from the stream of vector loads
template <class T> __device__ __forceinline__ T fixed(const T& v) { return *(const __attribute__((address_space(4))) T*)(uintptr_t)&v; }

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

// Gate and up (DOWN false): a workgroup has 64 channels of h of one group, and one of `parts` parts of K.
// Down: 128 channels, and a run of the units (group, part of K: `parts` of each); the last workgroup of a tile's `runs` sums up a token's choices.
template <bool DOWN, int P, int GS, int PH>
__global__ __launch_bounds__(256) void experts_kernel(MoeArgs g, int tiles, int parts, int runs) {
  typedef Shape<P, GS> S;
  constexpr int TB = S::TB, DEPTH = S::DEPTH;
  extern __shared__ __attribute__((aligned(1024))) char lds[];               // DEPTH stages
  const int tid = threadIdx.x, lane = tid & 63, q = lane >> 4, c = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Weights& w = DOWN ? g.down : g.gate_up;
  const int bytes = w.B * 16, stages = (bytes + STAGE - 1) / STAGE;
  int tile, unit, end;                              // units are numbered group by group
  if constexpr (DOWN) {
    const int run = blockIdx.x / tiles, units = fixed(g.plan->groups) * parts;
    tile = blockIdx.x - run * tiles;
    unit = (int)((uint32_t)units * (uint32_t)run / (uint32_t)runs);       // (fewer than 2^19 units, 2^10 runs)
    end = (int)((uint32_t)units * (uint32_t)(run + 1) / (uint32_t)runs);
  } else {
    const int all = blockIdx.x / parts, group = all / tiles;
    tile = all - group * tiles;
    unit = group * parts + (blockIdx.x - all * parts);
    end = unit + 1;
    if (fixed(g.plan->group[group].count) == 0) return;
  }
  constexpr int WIDTH = DOWN ? 128 : 64;
  const int channels = DOWN ? g.N : g.I, n0 = tile * WIDTH + wave * (WIDTH / 4);
  // rows of each half of 16: channels n0 .. (their gates, and their ups I rows behind; down: and n0 + 16 ..)
  int rows[2] = {channels - n0, channels - n0 - (DOWN ? 16 : 0)};
  #pragma unroll
  for (int u = 0; u < 2; ++u) rows[u] = rows[u] < 0 ? 0 : rows[u] > 16 ? 16 : rows[u];
  const int64_t second = DOWN ? 16 : g.I;           // rows from a first half to its second

  const auto one = [](uint32_t v) { return (int)__builtin_amdgcn_readfirstlane((int)v); };
  const auto buffer = [&](const void* p, int64_t size) {
    const uint64_t at = (uint64_t)(uintptr_t)p;
    return i32x4{one((uint32_t)at), one((uint32_t)(at >> 32) & 0xffff), one((uint32_t)size), 0x00020000};
  };
  const auto load = [&](uint32_t to, uint32_t of, i32x4 buf, int at) {       // (all but `of` are the wave's)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(one(to)), "v"(of), "s"(buf), "s"(one((uint32_t)at)) : "memory");
  };
  const uint32_t lds0 = (uint32_t)(size_t)(lds_ptr)lds;

  // ---- loads: a place in the sequence of stages, and what depends on its group alone ----
  uint32_t wof[4], xof[S::X], sof;
  #pragma unroll
  for (int l = 0; l < 4; ++l) {
    const int r = l * 8 + (lane >> 3), in = r & 15;
    wof[l] = in < rows[l >> 1] ? (uint32_t)(in * w.ldw) + (((lane & 7) ^ (r >> 1 & 7)) << 4) : OUTSIDE;
  }
  const int piece = (lane & 7) ^ (lane >> 4 & 3);   // of 16 bytes in a row of codes; in odd loads 4 more, as 8 rows turn it
  const i32x4 bufX = DOWN ? buffer(g.h, 0x7fffffff) : buffer(g.x, 0x7fffffff);
  i32x4 bufW[2], bufS;
  const int row_bytes = (DOWN ? g.Ip : g.Kp) * 2;
  // the first stage of part p of a group
  const auto first_of = [&](int p) { return (int)((uint32_t)(stages * p) / (uint32_t)parts); };
  struct Place { int unit, group, part, k, end; } at;
  const auto go = [&](Place& to, int u) {
    to.unit = u;
    to.group = (uint32_t)u / (uint32_t)parts;
    to.part = u - to.group * parts;
    to.k = first_of(to.part);
    to.end = first_of(to.part + 1);
  };
  const int period = ((uintptr_t)w.s | (uintptr_t)w.ldse | (uintptr_t)w.lds) & 3 ? 3 : 4;    // stages
  const auto enter = [&]() {
    const Group& in = g.plan->group[at.group];
    const int e = fixed(in.expert), first = fixed(in.first), count = fixed(in.count);
    #pragma unroll
    for (int u = 0; u < 2; ++u)
      bufW[u] = buffer(w.w + e * w.lde + (n0 + u * second) * w.ldw, rows[u] ? (rows[u] - 1) * w.ldw + bytes : 0);
    // scales of the wave's rows: from the first half's first row to the second half's last
    const uint8_t* const s = w.s + e * w.ldse + n0 * w.lds;
    const int early = (int)((uintptr_t)s & 3);
    bufS = buffer(s - early, rows[0] ? (early + (rows[1] ? second + rows[1] - 1 : rows[0] - 1) * w.lds + w.B + 3) & ~(int64_t)3 : 0);
    const int r = lane >> 1;
    sof = (r & 15) < rows[r >> 4] ? ((uint32_t)(early + ((r & 15) + (r >> 4) * second) * w.lds) & ~3u) + (lane & 1) * 16 : OUTSIDE;
    #pragma unroll
    for (int o = 0; o < S::X; ++o) {
      const int r = (wave + 4 * o) * 2 + (lane >> 5), slot = r / P, plane = r - slot * P;
      xof[o] = OUTSIDE;
      if (slot < count) {                           // (of a group that is not full: zeros)
        if constexpr (DOWN) xof[o] = (uint32_t)((first + slot) * P + plane) * (uint32_t)(g.Ip * 2);
        else xof[o] = (uint32_t)((in.token[slot] * g.ldx + plane * g.ldp) * 2);
      }
    }
  };
  // The next stage, into a place; behind the last one: nothing, from outside.  The scales of a period come in front of its first stage.
  int lperiod = 0, lplace = DEPTH - 1;
  const auto fetch = [&](int slot) {
    const uint32_t over = at.unit < end ? 0u : OUTSIDE, to = lds0 + slot * S::BYTES;
    if (lperiod == 0) {
      lplace = lplace == DEPTH - 1 ? 0 : lplace + 1;
      load(lds0 + DEPTH * S::BYTES + (lplace * 4 + wave) * 1024, sof | over, bufS, at.k * 8);
      lperiod = period;
    }
    --lperiod;
    #pragma unroll
    for (int l = 0; l < 4; ++l) {
      const uint32_t outside = (piece ^ (l & 1) * 4) * 16 < bytes - at.k * STAGE ? over : OUTSIDE;
      load(to + (wave * 4 + l) * 1024, wof[l] | outside, bufW[l >> 1], at.k * STAGE);
    }
    #pragma unroll
    for (int o = 0; o < S::X; ++o) {
      const int x = wave + 4 * o;
      if (S::FULL && o == S::X - 1 && wave >= S::FULL) break;
      const int p = (lane & 31) ^ ((x * 2 + (lane >> 5)) / P & 15);          // piece of an operand's row
      load(to + 16384 + x * 1024, (xof[o] + p * 16) | over | (p * 16 + at.k * 512 < row_bytes ? 0u : OUTSIDE), bufX, at.k * 512);
    }
    if (++at.k == at.end && at.unit < end) {
      go(at, at.unit + 1);
      lperiod = 0;
      if (DOWN && at.unit < end) enter();
    }
  };

  f32x4 acc[2][TB] = {};
  if (unit < end) {
    go(at, unit);
    enter();
    #pragma unroll
    for (int d = 0; d < DEPTH - 1; ++d) fetch(d);
    // ---- products ----
    Place now;
    int slot = 0, first = 0, count = 0, early[2];
    const auto begin = [&]() {
      const Group& in = g.plan->group[now.group];
      const int e = fixed(in.expert);
      first = fixed(in.first);
      count = fixed(in.count);
      #pragma unroll
      for (int u = 0; u < 2; ++u) early[u] = (int)((uint32_t)(uintptr_t)w.s + (uint32_t)e * (uint32_t)w.ldse + (uint32_t)(n0 + c + u * (int)second) * (uint32_t)w.lds) & 3;
    };
    go(now, unit);
    begin();
    const char* const codes = lds + wave * 4096 + c * 128;
    const char* const scales = lds + DEPTH * S::BYTES + wave * 1024 + c * 32 + q;
    const int turn = c >> 1 & 7;
    int cperiod = 0, cplace = DEPTH - 1;
    constexpr int MORE = (DEPTH - 2) * (4 + S::X), LESS = (DEPTH - 2) * (3 + S::X);          // loads that may be on their way
    while (now.unit < end) {
      // the next stage has landed, and this wave has read the last one
      if (S::FULL && wave >= S::FULL) __builtin_amdgcn_s_waitcnt(0x0070 | (LESS & 15) | LESS >> 4 << 14);
      else __builtin_amdgcn_s_waitcnt(0x0070 | (MORE & 15) | MORE >> 4 << 14);
      asm volatile("s_barrier" ::: "memory");
      fetch(slot == 0 ? DEPTH - 1 : slot - 1);
      if (cperiod == 0) cplace = cplace == DEPTH - 1 ? 0 : cplace + 1;
      const int here = slot * S::BYTES, scales_here = cplace * 4096 + cperiod * 8;
      cperiod = cperiod == period - 1 ? 0 : cperiod + 1;
      i32x4 wv[2][2];
      float f[2][2];
      #pragma unroll
      for (int u = 0; u < 2; ++u)
        #pragma unroll
        for (int i = 0; i < 2; ++i) {
          wv[u][i] = *(const i32x4*)(codes + here + u * 2048 + (((i * 4 + q) ^ turn) << 4));
          const uint32_t byte = *(const uint8_t*)(scales + scales_here + u * 512 + early[u] + i * 4);
          f[u][i] = mx_factor(now.k * 8 + i * 4 + q < w.B ? byte : 0u);      // (behind the last block: not a NaN)
        }
      #pragma unroll
      for (int i = 0; i < 2; ++i)
        #pragma unroll
        for (int j = 0; j < 4; ++j) {
          bf16x8 v[2];
          #pragma unroll
          for (int u = 0; u < 2; ++u) v[u] = decoded(wv[u][i][j], f[u][i]);
          #pragma unroll
          for (int b = 0; b < TB; ++b)
            #pragma unroll
            for (int l = P - 1; l >= 0; --l) {
              const int s = (b * 16 + c) & (GS - 1);
              const bf16x8 x = *(const bf16x8*)(lds + here + 16384 + (s * P + l) * 512 + (((i * 16 + q * 4 + j) ^ (s & 15)) << 4));
              #pragma unroll
              for (int u = 0; u < 2; ++u) acc[u][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v[u], x, acc[u][b], 0, 0, 0);
            }
        }
      slot = slot == DEPTH - 1 ? 0 : slot + 1;
      if (++now.k == now.end) {
        if constexpr (DOWN) {
          #pragma unroll
          for (int b = 0; b < TB; ++b) {
            const int s = b * 16 + c;
            #pragma unroll
            for (int u = 0; u < 2; ++u) {
              // (rows of whole fours; what lies behind N is not read)
              if (s < count && q * 4 < rows[u])
                *(f32x4*)(g.out + ((int64_t)(first + s) * parts + now.part) * ((g.N + 3) & ~3) + n0 + u * 16 + q * 4) = acc[u][b];
              acc[u][b] = f32x4{};
            }
          }
        }
        go(now, now.unit + 1);
        cperiod = 0;
        if (DOWN && now.unit < end) begin();
      }
    }
  }
  __builtin_amdgcn_s_waitcnt(0x0f70);               // nothing may still be on its way to LDS when the workgroup leaves it

  // ---- results: accumulator register r of lane l is channel 4 (l / 16) + r of slot l % 16 ----
  if constexpr (!DOWN) {
    const int group = unit / parts;
    const Group& in = g.plan->group[group];
    if (parts > 1) {
      f32x4* const mine = (f32x4*)g.up + ((int64_t)(blockIdx.x / parts) * parts * 256 + tid) * (2 * TB);
      #pragma unroll
      for (int u = 0; u < 2; ++u)
        #pragma unroll
        for (int b = 0; b < TB; ++b) mine[(int64_t)(unit - group * parts) * 512 * TB + u * TB + b] = acc[u][b];
      if (!last_of(&g.plan->counter[0][blockIdx.x / parts], parts)) return;
      #pragma unroll
      for (int u = 0; u < 2; ++u)
        #pragma unroll
        for (int b = 0; b < TB; ++b) {
          acc[u][b] = f32x4{};
          for (int p = 0; p < parts; ++p) acc[u][b] += mine[(int64_t)p * 512 * TB + u * TB + b];
        }
    }
    const int e = in.expert, count = in.count, first = in.first;
    if (n0 + q * 4 >= g.Ip) return;
    #pragma unroll
    for (int b = 0; b < TB; ++b) {
      const int s = b * 16 + c;
      if (s >= count) continue;
      uint16_t p[4][PH];
      #pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int ch = q * 4 + r;
        float v[2] = {acc[0][b][r], acc[1][b][r]};
        if (w.bias && ch < rows[0]) {
          #pragma unroll
          for (int u = 0; u < 2; ++u) v[u] += load_any(w.bias, w.bias_dtype, ((int64_t)e * 2 + u) * g.I + n0 + ch);
        }
        planes_of<PH>(ch < rows[0] ? act(v[0], g.activation) * v[1] : 0.0f, p[r]);
      }
      #pragma unroll
      for (int l = 0; l < PH; ++l)
        *(u32x2*)(g.h + ((int64_t)(first + s) * PH + l) * g.Ip + n0 + q * 4) = u32x2{p[0][l] | (uint32_t)p[1][l] << 16, p[2][l] | (uint32_t)p[3][l] << 16};
    }
  }
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
  return dtype == LCQ_BF16 && K % 32 == 0 && ldx % 8 == 0 && (uintptr_t)x % 16 == 0 && ldx <= 1 << 22;       // (offsets have 31 bits)
}

// How a pass of T tokens is cut.
struct Cut {
  int P, PH, size, up_tiles, up_parts, down_tiles, down_parts, runs;
  int64_t groups, h, up, out;                       // bytes
  Cut(int64_t T, int64_t top, int64_t E, int64_t K, int64_t I, int64_t N, int dtype) {
    P = dtype == LCQ_BF16 ? 1 : dtype == LCQ_F16 ? 2 : 3;
    PH = dtype == LCQ_F32 ? 3 : 2;
    const int64_t slots = T * top;
    size = T <= 4 || slots <= E ? 4 : P == 3 || T <= 16 || slots <= 14 * E ? 16 : 32;
    groups = least(slots, least(E, slots) + slots / size);
    const int64_t up_stages = ((K + 31) / 32 + 7) / 8, down_stages = ((I + 31) / 32 + 7) / 8, Ip = (I + 31) / 32 * 32;
    up_tiles = (int)((Ip + 63) / 64);
    up_parts = 1;
    while (groups * up_tiles * up_parts < 200 && up_stages / (2 * up_parts) >= 3) up_parts *= 2;
    down_tiles = (int)((N + 127) / 128);
    int64_t want = 512 / down_tiles;
    if (want < 1) want = 1;
    down_parts = 1;
    while (groups * down_parts < 8 * want && down_stages / (2 * down_parts) >= 2) down_parts *= 2;
    const int64_t units = groups * down_parts, each = (units + want - 1) / want;
    runs = (int)((units + each - 1) / each);
    h = on256(slots * PH * Ip * 2);
    up = up_parts > 1 ? on256(groups * up_tiles * up_parts * 256 * 32 * (size > 16 ? 2 : 1)) : 0;
    out = on256(slots * down_parts * ((N + 3) & ~(int64_t)3) * 4);
  }
};

template <bool DOWN, int P, int GS, int PH>
int launch_experts(const MoeArgs& g, const Cut& c, hipStream_t st) {
  typedef Shape<P, GS> S;
  const auto kernel = experts_kernel<DOWN, P, GS, PH>;
  // (more LDS than a launch may have without asking)
  if (hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, S::LDS) != hipSuccess) return LCQ_ELAUNCH;
  const int64_t blocks = DOWN ? (int64_t)c.down_tiles * c.runs : c.groups * c.up_tiles * c.up_parts;
  if (blocks > (1 << 24) - 1) return LCQ_ESIZE;
  kernel<<<dim3((unsigned)blocks), dim3(256), S::LDS, st>>>(g, DOWN ? c.down_tiles : c.up_tiles, DOWN ? c.down_parts : c.up_parts, c.runs);
  return LCQ_OK;
}
template <bool DOWN, int P, int PH>
int launch_size(const MoeArgs& g, const Cut& c, hipStream_t st) {
  if (c.size == 4) return launch_experts<DOWN, P, 4, PH>(g, c, st);
  if constexpr (P < 3) { if (c.size == 32) return launch_experts<DOWN, P, 32, PH>(g, c, st); }
  return launch_experts<DOWN, P, 16, PH>(g, c, st);
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
  const int64_t t = least(T, MOST_PASS);
  int64_t most = 0;                                 // (the last pass may have fewer tokens, and be cut into more parts)
  for (const int64_t n : {t, T % MOST_PASS ? T % MOST_PASS : t}) {
    const Cut c(n, top, E, K, I, N, dtype);
    const int64_t size = c.h + c.up + c.out + on256(n * c.P * ((K + 31) / 32 * 32) * 2);
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
  if (gate_up_ld > 1 << 22 || down_ld > 1 << 22 || gate_up_lds * (I + 64) > 1 << 30 || down_lds > 1 << 22) return LCQ_ESIZE;
  if ((uintptr_t)gate_up % 16 || gate_up_ld % 16 || gate_up_lde % 16 || (uintptr_t)down % 16 || down_ld % 16 || down_lde % 16) return LCQ_EALIGN;
  if (!workspace) return LCQ_EWORKSPACE;
  if ((uintptr_t)workspace % 16) return LCQ_EALIGN;
  hipStream_t st = (hipStream_t)stream;
  char* const ws = (char*)workspace;
  const bool as_is = direct(dtype, x, ldx, K);
  Plan* const plan = (Plan*)ws;
  const int64_t size = dtype == LCQ_F32 ? 4 : 2, out_size = out_dtype == LCQ_F32 ? 4 : 2, logit_size = logits_dtype == LCQ_F32 ? 4 : 2;
  for (int64_t t0 = 0; t0 < T; t0 += MOST_PASS) {
    const int n = (int)least(T - t0, MOST_PASS);
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
    const int* const ge = experts ? experts + t0 * top : nullptr;
    const float* const gw = experts ? weights + t0 * top : nullptr;
    if (E <= 64) plan_kernel<1><<<grid, dim3(1024), 0, st>>>(rt, ge, gw, n, o, c.size, (int)c.groups, plan);
    else if (E <= 256) plan_kernel<4><<<grid, dim3(1024), 0, st>>>(rt, ge, gw, n, o, c.size, (int)c.groups, plan);
    else plan_kernel<16><<<grid, dim3(1024), 0, st>>>(rt, ge, gw, n, o, c.size, (int)c.groups, plan);
    const MoeArgs g = {as_is ? (const uint16_t*)xt : planes, as_is ? ldx : c.P * Kp, Kp,
                       {gate_up, gate_up_scales, gate_up_bias, gate_up_lde, gate_up_ld, gate_up_ldse, gate_up_lds, (int)B, bias_dtype},
                       {down, down_scales, down_bias, down_lde, down_ld, down_ldse, down_lds, (int)BI, bias_dtype}, plan, h, up_sums, out_sums,
                       (char*)y + t0 * N * out_size, n, top, (int)N, (int)I, (int)Kp, (int)Ip, activation};
    int rc = c.P == 1 ? launch_size<false, 1, 2>(g, c, st) : c.P == 2 ? launch_size<false, 2, 2>(g, c, st) : launch_size<false, 3, 3>(g, c, st);
    if (rc) return rc;
    rc = c.PH == 2 ? launch_size<true, 2, 2>(g, c, st) : launch_size<true, 3, 3>(g, c, st);
    if (rc) return rc;
    if (out_dtype == LCQ_BF16) launch_sum<ROW_BF16>(g, c, st);
    else if (out_dtype == LCQ_F16) launch_sum<ROW_F16>(g, c, st);
    else launch_sum<ROW_F32>(g, c, st);
  }
  LCQ_CHECK_LAUNCH();
  return LCQ_OK;
}

}  // extern "C"

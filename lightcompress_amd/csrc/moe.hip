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
// A pass: the slots (token and choice) sorted by expert, in groups of at most 16 of one expert.
struct Plan {
  int groups;
  int expert[MOST_EXPERTS + MOST_PASS * MOST_TOP / 16], first[MOST_EXPERTS + MOST_PASS * MOST_TOP / 16], count[MOST_EXPERTS + MOST_PASS * MOST_TOP / 16];
  int token[MOST_PASS * MOST_TOP];
  float weight[MOST_PASS * MOST_TOP];
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
                                                    Operand o, Plan* __restrict__ plan) {
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
  mine |= (uint32_t)((n + 15) / 16) << 16;
  uint32_t sum = mine;
  #pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const uint32_t o_ = __shfl_up(sum, d);
    if (lane >= d) sum += o_;
  }
  if (lane == 63) sums[wave] = sum;
  __syncthreads();
  for (int w = 0; w < wave; ++w) sum += sums[w];
  const uint32_t before = sum - mine;
  place[tid] = before & 0xffff;
  for (int g = 0; g < (n + 15) / 16; ++g) {
    const int at = (int)(before >> 16) + g;
    plan->expert[at] = tid;
    plan->first[at] = (int)(before & 0xffff) + 16 * g;
    plan->count[at] = n - 16 * g < 16 ? n - 16 * g : 16;
  }
  if (tid == 1023) plan->groups = (int)(sum >> 16);
  __syncthreads();
  for (int i = tid; i < slots; i += 1024) {
    const int e = expert[i], t = i / r.top;
    if (e < 0) continue;
    int at = (int)place[e] + __builtin_popcount(chosen[e][t / 32] & ((1u << t % 32) - 1));
    for (int q = 0; q < t / 32; ++q) at += __builtin_popcount(chosen[e][q]);
    plan->token[at] = t;
    plan->weight[at] = weight[i];
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
  const uint16_t* x;                                // planes of the tokens: [T, P, Kp] or rows ldx apart
  int64_t ldx, ldp;                                 // elements from a token, a plane to the next
  Weights gate_up, down;
  const Plan* plan;
  uint16_t* h;                                      // [slots, PH, Ip]
  void* y;
  int T, K, N, I, Kp, Ip, activation, dtype;        // Kp, Ip: whole blocks
};

__device__ __forceinline__ i32x4 load16(__amdgpu_buffer_rsrc_t buf, uint32_t of, int at) {
  return __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(buf, of, at, 0));
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const void* p, int64_t size) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, (int)size, 0x00020000);
}
// eight codes times their scale, exactly
__device__ __forceinline__ bf16x8 decoded(int codes, int scale) {
  const float f = mx_factor((uint32_t)scale);
  const lcq_bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4((uint32_t)codes, f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4((uint32_t)codes, f, 1),
                   c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4((uint32_t)codes, f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4((uint32_t)codes, f, 3);
  return bf16x8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

__device__ __forceinline__ float act(float v, int activation) {
  return activation == LCQ_ACT_SILU ? v / (1.0f + expf(-v)) : 0.5f * v * (1.0f + erff(v * 0.70710678118654752440f));
}

// A lane's 16 bytes of a row are a block; a load of the wave is 16 rows x 64 bytes.  A piece is two of them.
constexpr int PIECE = 128;

// gate and up: 16 channels of one group per workgroup, whose waves take pieces of K in turn.
template <int P, int PH, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void up_kernel(MoeArgs g, int tiles) {
  __shared__ __attribute__((aligned(16))) float red[WAVES][2][64][4];
  const int group = blockIdx.x / tiles, n0 = (blockIdx.x - group * tiles) * 16;
  if (group >= g.plan->groups) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), q = lane >> 4, c = lane & 15;
  const int e = g.plan->expert[group], first = g.plan->first[group], count = g.plan->count[group];
  const Weights& w = g.gate_up;
  const int bytes = w.B * 16, rows = g.I - n0 < 16 ? g.I - n0 : 16;          // (0 or less: channels that only fill a block)
  __amdgpu_buffer_rsrc_t buf[2], sbuf[2];
  #pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int64_t row = n0 + (int64_t)u * g.I;
    buf[u] = buffer(w.w + e * w.lde + row * w.ldw, rows > 0 ? (rows - 1) * w.ldw + bytes : 0);
    sbuf[u] = buffer(w.s + e * w.ldse + row * w.lds, rows > 0 ? (rows - 1) * w.lds + w.B : 0);
  }
  const uint32_t of = c < rows ? (uint32_t)(c * w.ldw) + q * 16 : OUTSIDE, sof = c < rows ? (uint32_t)(c * w.lds) + q : OUTSIDE;
  const int token = g.plan->token[first + (c < count ? c : 0)];
  const uint16_t* const x = g.x + token * g.ldx + q * 32;
  constexpr int DEPTH = P == 1 ? 3 : 2, STEP = WAVES * PIECE;
  struct Piece { i32x4 w[2][2], x[2][P][4]; int s[2][2]; } ring[DEPTH];
  const auto load = [&](int k, Piece& p) {
    #pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int at = k + i * 64;
      const bool in = at + q * 16 < bytes;
      #pragma unroll
      for (int u = 0; u < 2; ++u) {
        p.w[u][i] = load16(buf[u], in ? of : OUTSIDE, at);
        p.s[u][i] = __builtin_amdgcn_raw_buffer_load_b8(sbuf[u], in ? sof : OUTSIDE, at >> 4, 0);
      }
      #pragma unroll
      for (int l = 0; l < P; ++l)
        #pragma unroll
        for (int j = 0; j < 4; ++j) {
          i32x4 v = {};
          if (in && c < count && at * 2 + q * 32 + j * 8 < g.Kp) v = *(const i32x4*)(x + l * g.ldp + at * 2 + j * 8);
          p.x[i][l][j] = v;
        }
    }
  };
  int k = wave * PIECE;
  #pragma unroll
  for (int d = 0; d < DEPTH; ++d) load(k + d * STEP, ring[d]);
  f32x4 acc[2] = {};
  while (k < bytes) {
    #pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      Piece& p = ring[d];
      #pragma unroll
      for (int i = 0; i < 2; ++i)
        #pragma unroll
        for (int j = 0; j < 4; ++j)
          #pragma unroll
          for (int u = 0; u < 2; ++u) {
            const bf16x8 v = decoded(p.w[u][i][j], p.s[u][i]);
            #pragma unroll
            for (int l = P - 1; l >= 0; --l) acc[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, __builtin_bit_cast(bf16x8, p.x[i][l][j]), acc[u], 0, 0, 0);
          }
      load(k + DEPTH * STEP, p);
      k += STEP;
    }
  }
  #pragma unroll
  for (int u = 0; u < 2; ++u) *(f32x4*)red[wave][u][lane] = acc[u];
  __syncthreads();
  // accumulator register r of lane l: channel 4 (l / 16) + r of slot l % 16
  for (int o = tid; o < 256; o += WAVES * 64) {
    const int ch = o & 15, slot = o >> 4;
    if (slot >= count || n0 + ch >= g.Ip) continue;
    float v[2] = {};
    #pragma unroll
    for (int u = 0; u < 2; ++u) {
      #pragma unroll
      for (int s = 0; s < WAVES; ++s) v[u] += red[s][u][(ch >> 2) * 16 + slot][ch & 3];
      if (w.bias && ch < rows) v[u] += load_any(w.bias, w.bias_dtype, (int64_t)e * 2 * g.I + u * g.I + n0 + ch);
    }
    uint16_t p[PH];
    planes_of<PH>(ch < rows ? act(v[0], g.activation) * v[1] : 0.0f, p);
    #pragma unroll
    for (int l = 0; l < PH; ++l) g.h[((int64_t)(first + slot) * PH + l) * g.Ip + n0 + ch] = p[l];
  }
}

// down and the weighted sum: 16 channels of all tokens per workgroup.  The pieces of all groups, one behind the other, are dealt to the waves
// in equal runs; a wave that leaves a group adds what it has of it to its own sums of the tokens, in LDS.  No atomics: the order is fixed.
template <int BF, int PH, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void down_kernel(MoeArgs g) {
  extern __shared__ __attribute__((aligned(16))) float sums[];               // [WAVES, T, 16]
  const int n0 = blockIdx.x * 16;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), q = lane >> 4, c = lane & 15;
  const Weights& w = g.down;
  const int bytes = w.B * 16, rows = g.N - n0 < 16 ? g.N - n0 : 16, pieces = (bytes + PIECE - 1) / PIECE;
  const int total = g.plan->groups * pieces;
  const int begin = (int)((int64_t)total * wave / WAVES), end = (int)((int64_t)total * (wave + 1) / WAVES);
  float* const mine = sums + wave * g.T * 16;
  for (int i = lane; i < g.T * 16; i += 64) mine[i] = 0;
  const uint32_t of = c < rows ? (uint32_t)(c * w.ldw) + q * 16 : OUTSIDE, sof = c < rows ? (uint32_t)(c * w.lds) + q : OUTSIDE;
  constexpr int DEPTH = 2;
  struct Piece { i32x4 w[2], h[2][PH][4]; int s[2]; } ring[DEPTH];
  const auto load = [&](int at_, Piece& p) {
    const int at = at_ < end ? at_ : end - 1;       // (behind the last: once more, unused)
    const int group = at / pieces, k = (at - group * pieces) * PIECE;
    const int e = g.plan->expert[group], first = g.plan->first[group], count = g.plan->count[group];
    const __amdgpu_buffer_rsrc_t buf = buffer(w.w + e * w.lde + n0 * w.ldw, (rows - 1) * w.ldw + bytes), sbuf = buffer(w.s + e * w.ldse + n0 * w.lds, (rows - 1) * w.lds + w.B);
    const uint16_t* const h = g.h + (int64_t)(first + (c < count ? c : 0)) * PH * g.Ip + q * 32 + k * 2;
    #pragma unroll
    for (int i = 0; i < 2; ++i) {
      const bool in = k + i * 64 + q * 16 < bytes;
      p.w[i] = load16(buf, in ? of : OUTSIDE, k + i * 64);
      p.s[i] = __builtin_amdgcn_raw_buffer_load_b8(sbuf, in ? sof : OUTSIDE, (k >> 4) + i * 4, 0);
      #pragma unroll
      for (int l = 0; l < PH; ++l)
        #pragma unroll
        for (int j = 0; j < 4; ++j) {
          i32x4 v = {};
          if (in && c < count) v = *(const i32x4*)(h + l * g.Ip + i * 128 + j * 8);
          p.h[i][l][j] = v;
        }
    }
  };
  int at = begin;
  if (begin < end) {
    #pragma unroll
    for (int d = 0; d < DEPTH; ++d) load(at + d, ring[d]);
    f32x4 acc = {};
    int group = begin / pieces, left = (group + 1) * pieces - begin;         // pieces of this group from here on
    bool whole = left == pieces;                    // does this wave have the group's first piece?
    while (at < end) {
      #pragma unroll
      for (int d = 0; d < DEPTH; ++d) {
        if (at < end) {
          Piece& p = ring[d];
          #pragma unroll
          for (int i = 0; i < 2; ++i)
            #pragma unroll
            for (int j = 0; j < 4; ++j) {
              const bf16x8 v = decoded(p.w[i][j], p.s[i]);
              #pragma unroll
              for (int l = PH - 1; l >= 0; --l) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, __builtin_bit_cast(bf16x8, p.h[i][l][j]), acc, 0, 0, 0);
            }
          load(at + DEPTH, p);
          ++at;
          if (--left == 0 || at == end) {
            const int e = g.plan->expert[group], first = g.plan->first[group], count = g.plan->count[group];
            if (c < count) {
              const float weight = g.plan->weight[first + c];
              f32x4* const to = (f32x4*)(mine + g.plan->token[first + c] * 16 + q * 4);
              f32x4 v = *to;
              #pragma unroll
              for (int r = 0; r < 4; ++r) {
                float b = 0;
                if (w.bias && whole && q * 4 + r < rows) b = load_any(w.bias, w.bias_dtype, (int64_t)e * g.N + n0 + q * 4 + r);
                v[r] = __builtin_fmaf(weight, acc[r] + b, v[r]);
              }
              *to = v;
            }
            acc = f32x4{};
            ++group;
            left = pieces;
            whole = true;
          }
        }
      }
    }
  }
  __syncthreads();
  for (int o = tid; o < g.T * 16; o += WAVES * 64) {
    const int ch = o & 15;
    const int64_t t = o >> 4;
    if (ch >= rows) continue;
    float y = 0;
    #pragma unroll
    for (int s = 0; s < WAVES; ++s) y += sums[s * g.T * 16 + o];
    if constexpr (BF == ROW_F32) ((float*)g.y)[t * g.N + n0 + ch] = y;
    else store_scalar<BF>(g.y, t * g.N + n0 + ch, rnd<BF>(y));
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
bool direct(int dtype, const void* x, int64_t ldx, int64_t K) { return dtype == LCQ_BF16 && K % 32 == 0 && ldx % 8 == 0 && (uintptr_t)x % 16 == 0; }

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

int64_t lcq_mxfp4_moe_workspace_bytes(int64_t T, int64_t top, int64_t K, int64_t I) {
  if (T <= 0 || top <= 0 || K <= 0 || I <= 0 || K > 65536 || I > 65536 || top > MOST_TOP) return 0;
  const int64_t t = least(T, MOST_PASS), Kp = (K + 31) / 32 * 32, Ip = (I + 31) / 32 * 32;
  return on256(sizeof(Plan)) + on256(t * top * 3 * Ip * 2) + t * 3 * Kp * 2;
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
  if (gate_up_ld > 1 << 22 || gate_up_lds > 1 << 22 || down_ld > 1 << 22 || down_lds > 1 << 22) return LCQ_ESIZE;
  if ((uintptr_t)gate_up % 16 || gate_up_ld % 16 || gate_up_lde % 16 || (uintptr_t)down % 16 || down_ld % 16 || down_lde % 16) return LCQ_EALIGN;
  if (!workspace) return LCQ_EWORKSPACE;
  if ((uintptr_t)workspace % 16) return LCQ_EALIGN;
  hipStream_t st = (hipStream_t)stream;
  const int64_t most = least(T, MOST_PASS);
  char* const ws = (char*)workspace;
  const bool as_is = direct(dtype, x, ldx, K);
  const int P = dtype == LCQ_BF16 ? 1 : dtype == LCQ_F16 ? 2 : 3, PH = dtype == LCQ_F32 ? 3 : 2;
  Plan* const plan = (Plan*)ws;
  uint16_t* const h = (uint16_t*)(ws + on256(sizeof(Plan)));
  uint16_t* const planes = (uint16_t*)((char*)h + on256(most * top * 3 * Ip * 2));
  const int64_t size = dtype == LCQ_F32 ? 4 : 2, out_size = out_dtype == LCQ_F32 ? 4 : 2, logit_size = logits_dtype == LCQ_F32 ? 4 : 2;
  for (int64_t t0 = 0; t0 < T; t0 += MOST_PASS) {
    const int n = (int)least(T - t0, MOST_PASS);
    const char* const xt = (const char*)x + t0 * ldx * size;
    RouterArgs rt = r;
    if (logits) rt.logits = (const char*)logits + t0 * ldl * logit_size;
    const Operand o = {xt, ldx, dtype, P, (int)K, (int)Kp, planes};
    const dim3 grid(as_is ? 1u : 1u + (unsigned)least((n * Kp + 1023) / 1024, 255));
    const int* const ge = experts ? experts + t0 * top : nullptr;
    const float* const gw = experts ? weights + t0 * top : nullptr;
    if (E <= 64) plan_kernel<1><<<grid, dim3(1024), 0, st>>>(rt, ge, gw, n, o, plan);
    else if (E <= 256) plan_kernel<4><<<grid, dim3(1024), 0, st>>>(rt, ge, gw, n, o, plan);
    else plan_kernel<16><<<grid, dim3(1024), 0, st>>>(rt, ge, gw, n, o, plan);
    MoeArgs g = {as_is ? (const uint16_t*)xt : planes, as_is ? ldx : P * Kp, Kp, {gate_up, gate_up_scales, gate_up_bias, gate_up_lde, gate_up_ld, gate_up_ldse, gate_up_lds, (int)B, bias_dtype},
                 {down, down_scales, down_bias, down_lde, down_ld, down_ldse, down_lds, (int)BI, bias_dtype}, plan, h, (char*)y + t0 * N * out_size, n, (int)K, (int)N, (int)I,
                 (int)Kp, (int)Ip, activation, out_dtype};
    const int64_t slots = (int64_t)n * top, groups = least(slots, least(E, slots) + slots / 16);
    const int tiles = (int)(Ip / 16);
    const dim3 up((unsigned)(groups * tiles));
    if (P == 1) up_kernel<1, 2, 4><<<up, dim3(256), 0, st>>>(g, tiles);
    else if (P == 2) up_kernel<2, 2, 4><<<up, dim3(256), 0, st>>>(g, tiles);
    else up_kernel<3, 3, 4><<<up, dim3(256), 0, st>>>(g, tiles);
    const dim3 dn((unsigned)((N + 15) / 16));
    const unsigned lds = 8 * n * 64;
    const auto run = [&](auto bf) {
      constexpr int BF = decltype(bf)::value;
      if (PH == 2) down_kernel<BF, 2, 8><<<dn, dim3(512), lds, st>>>(g);
      else down_kernel<BF, 3, 8><<<dn, dim3(512), lds, st>>>(g);
    };
    if (out_dtype == LCQ_BF16) run(Int<ROW_BF16>{});
    else if (out_dtype == LCQ_F16) run(Int<ROW_F16>{});
    else run(Int<ROW_F32>{});
  }
  LCQ_CHECK_LAUNCH();
  return LCQ_OK;
}

}  // extern "C"

// Product of int8 codes with a scale for each token and each channel:
//   y[m, n] = as[m] ws[n] (sum_k a[m, k] w[n, k] - az[m] sum_k w[n, k]) + bias[n]
// The sums are exact in 32-bit integers for K <= 65536 (-128 <= az <= 127, so |a - az| <= 255; |w| <= 128: 255 * 128 * 65536 < 2^31), so results do not
// depend on how the work is cut.
//
// Both operands are read along K, as the matrix pipe takes them: a lane of v_mfma_i32_32x32x32_i8 holds 16 codes of one row.
// The weight is the first operand, so an accumulator's four neighbouring registers are four neighbouring channels of one token.
#include "rowquant.h"
#include "token_codes.h"
#include "launch_rules.h"
#include <type_traits>

namespace {
using namespace lcq;

typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((ext_vector_type(16))) int i32x16;
typedef __attribute__((address_space(3))) char* lds_ptr;
typedef __attribute__((address_space(3))) i32x4* lds_frag;

template <int I> using Int = std::integral_constant<int, I>;

struct MatmulArgs {
  const int8_t *a, *w;
  const float* as;
  const int32_t* az;
  const void *ws, *bias;
  void* y;
  int64_t M, N, lda, ldw;
  int K, ws_dtype, bias_dtype, a_scalar, w_scalar;
};

__device__ __forceinline__ float load_any(const void* p, int dtype, int64_t i) {
  return dtype == LCQ_F32 ? load_scalar<ROW_F32>(p, i) : dtype == LCQ_BF16 ? load_scalar<ROW_BF16>(p, i) : load_scalar<ROW_F16>(p, i);
}
// the same in two steps, so that nothing waits for the load before the value is used
__device__ __forceinline__ uint32_t load_raw(const void* p, int dtype, int64_t i) { return dtype == LCQ_F32 ? ((const uint32_t*)p)[i] : (uint32_t)((const uint16_t*)p)[i]; }
__device__ __forceinline__ float from_raw(uint32_t u, int dtype) {
  return dtype == LCQ_F32 ? u2f(u) : dtype == LCQ_BF16 ? u2f(u << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)u);
}
// the four byte sums of a register added to `sum`
__device__ __forceinline__ int add_bytes(const i32x4& v, int sum) {
  #pragma unroll
  for (int q = 0; q < 4; ++q) sum = __builtin_amdgcn_sdot4(v[q], 0x01010101, sum, false);
  return sum;
}

// ---- tiles --------------------------------------------------------------------------------------------------------
// A workgroup of four waves (2 x 2) owns 64 FM tokens x 64 FN channels, a wave FM x FN accumulators of 32 x 32.
//  * K streams through LDS stages of 64 or 128 codes per row by direct loads; rows past the end of a matrix and codes past K lie outside
//    the buffer that the loads are told and read as zero;
//  * piece p of 16 bytes of row r lies at p ^ (r / 4 % 4) or p ^ (r / 2 % 8), so that 16 lanes of an operand read touch all 64 banks once;
//  * operands are buffered in registers: while the products of one 32-code step run, the reads of a later one are issued between them;
//    one barrier per stage, where every wave holds the rest of it in registers: its place is loaded again from there.
constexpr int ROW_I32 = 3;                          // an output type: the sums of a part of K as they are

template <int FM_, int FN_, int SLAB_, int STAGES_, int SETS_>
struct Tile {
  static constexpr int FM = FM_, FN = FN_, SLAB = SLAB_, STAGES = STAGES_, SETS = SETS_;     // codes of a row per stage; sets of operands
  static constexpr int TM = 64 * FM, TN = 64 * FN, STEPS = SLAB / 32;
  static constexpr int STAGE = (TM + TN) * SLAB;
};

// 16-byte piece p of row r of a stage lies at p ^ swizzle(r)
template <int SLAB>
__device__ __forceinline__ int swizzle(int r) { return SLAB == 64 ? (r >> 2) & 3 : (r >> 1) & 7; }

template <class T, int BF, bool ASYM>
__global__ __launch_bounds__(256, 1) void tile_kernel(MatmulArgs g, int tiles_m, int tiles_n, int parts) {
  constexpr int FM = T::FM, FN = T::FN, SLAB = T::SLAB, STAGES = T::STAGES, SETS = T::SETS, STEPS = T::STEPS;
  __shared__ __attribute__((aligned(1024))) char lds[STAGES * T::STAGE];
  __shared__ __attribute__((aligned(16))) float channel[2][T::TN];           // scales, biases
  __shared__ __attribute__((aligned(16))) int sums[ASYM ? T::TN : 4];        // sums of the weight's rows
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wr = wave >> 1, wc = wave & 1;          // tokens, channels

  // Workgroup b runs on XCD b % 8: every XCD takes a contiguous range of an order in which 32 consecutive tiles are 4 x 8, so the
  // tiles that share an L2 at one time share a handful of stripes.
  int ti, tj, part;
  {
    const int total = tiles_m * tiles_n * parts, each = (total + 7) >> 3;
    int v = ((int)blockIdx.x & 7) * each + ((int)blockIdx.x >> 3);
    if (((int)blockIdx.x >> 3) >= each || v >= total) return;
    part = v / (tiles_m * tiles_n);
    v -= part * tiles_m * tiles_n;
    const int group = v / (4 * tiles_n), first = group * 4, rows = tiles_m - first < 4 ? tiles_m - first : 4;
    const int in = v - group * 4 * tiles_n;
    tj = in / rows;
    ti = first + in - tj * rows;
  }
  const int64_t m0 = (int64_t)ti * T::TM, n0 = (int64_t)tj * T::TN;
  const int rows_a = (int)(g.M - m0 < T::TM ? g.M - m0 : T::TM), rows_w = (int)(g.N - n0 < T::TN ? g.N - n0 : T::TN);
  const int slabs = (g.K + SLAB - 1) / SLAB;
  const int begin = (int)((int64_t)slabs * part / parts), steps = (int)((int64_t)slabs * (part + 1) / parts) - begin;

  const auto buffer = [&](const int8_t* p, int64_t ld, int rows) {
    const uint64_t at = (uint64_t)(uintptr_t)p;
    const auto one = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
    return i32x4{one((int)(uint32_t)at), one((int)(uint32_t)(at >> 32) & 0xffff), one((int)((rows - 1) * ld + g.K)), 0x00020000};
  };
  const i32x4 bufA = buffer(g.a + m0 * g.lda, g.lda, rows_a), bufW = buffer(g.w + n0 * g.ldw, g.ldw, rows_w);
  constexpr uint32_t OUTSIDE = 0x80000000u;
  constexpr int ROWS = 1024 / SLAB, LANES = 64 / ROWS;                       // of a load
  constexpr int LA = T::TM / (4 * ROWS), LW = T::TN / (4 * ROWS);            // a wave's loads of tokens and of weights per stage
  static_assert(SLAB == 64 || (LA % 2 == 0 && LW % 2 == 0), "a wave's loads start with an even one");
  // this lane's 16 bytes of a row: of an even load, and of an odd one (the same for 64 codes)
  int piece16[2];
  #pragma unroll
  for (int e = 0; e < 2; ++e) piece16[e] = ((lane % LANES) ^ swizzle<SLAB>(e * ROWS + lane / LANES)) * 16;
  uint32_t gof[LA + LW];
  #pragma unroll
  for (int p = 0; p < LA + LW; ++p) {
    const int r = (wave * (p < LA ? LA : LW) + (p < LA ? p : p - LA)) * ROWS + lane / LANES;
    gof[p] = r < (p < LA ? rows_a : rows_w) ? (uint32_t)(r * (p < LA ? g.lda : g.ldw) + piece16[p & 1]) : OUTSIDE;
  }
  const uint32_t lds0 = (uint32_t)(size_t)(lds_ptr)lds;
  struct Outside { uint32_t of[2]; };
  // load p of the stage at LDS address dst, codes [at, at + SLAB) of K
  const auto gload = [&](uint32_t dst, int at, const Outside& outside, int p) {
    const uint32_t to = dst + (p < LA ? (wave * LA + p) * 1024 : T::TM * SLAB + (wave * LW + p - LA) * 1024);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                 ::"s"(to), "v"(gof[p] | outside.of[p & 1]), "s"(p < LA ? bufA : bufW), "s"(at) : "memory");
  };
  const auto outside_at = [&](int at) { return Outside{{piece16[0] < g.K - at ? 0u : OUTSIDE, piece16[1] < g.K - at ? 0u : OUTSIDE}}; };

  // step ks reads pieces 2 ks (lanes 0 .. 31) and 2 ks + 1 of a row
  const int slot = (lane >> 5) ^ swizzle<SLAB>(lane & 31);
  const lds_ptr readA = (lds_ptr)lds + (wr * FM * 32 + (lane & 31)) * SLAB + slot * 16;
  const lds_ptr readW = (lds_ptr)lds + T::TM * SLAB + (wc * FN * 32 + (lane & 31)) * SLAB + slot * 16;
  int step_at[STEPS];                               // from the first 32 codes of a stage to the others
  #pragma unroll
  for (int ks = 0; ks < STEPS; ++ks) step_at[ks] = ((slot ^ (2 * ks)) - slot) * 16;
  i32x16 acc[FN][FM];
  #pragma unroll
  for (int j = 0; j < FN; ++j)
    #pragma unroll
    for (int i = 0; i < FM; ++i)
      #pragma unroll
      for (int r = 0; r < 16; ++r) acc[j][i][r] = 0;
  int wsum[FN] = {};
  i32x4 fr[SETS][FN + FM];                          // operands of 32 codes: weights, tokens
  const auto rd = [&](int set, int ks, int f, uint32_t stage) {
    fr[set][f] = *(lds_frag)((f < FN ? readW + f * 32 * SLAB : readA + (f - FN) * 32 * SLAB) + stage + step_at[ks]);
  };
  // What the outputs need besides the sums, on its way during the products (used behind them, so no wait counts it).
  float as[FM];
  uint32_t chan[2] = {};
  int az[FM] = {};
  if constexpr (BF != ROW_I32) {
    if (tid < rows_w) {
      chan[0] = load_raw(g.ws, g.ws_dtype, g.w_scalar ? 0 : n0 + tid);
      if (g.bias) chan[1] = load_raw(g.bias, g.bias_dtype, n0 + tid);
    }
  }
  #pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int m = wr * FM * 32 + i * 32 + (lane & 31), at = m < rows_a ? m : rows_a - 1;       // (a token past the last one is not stored)
    as[i] = BF != ROW_I32 ? g.as[g.a_scalar ? 0 : m0 + at] : 0.0f;
    if (ASYM) az[i] = g.az[m0 + at];
  }
  __builtin_amdgcn_sched_barrier(0);

  constexpr int LOADS = LA + LW, PRODUCTS = FM * FN, READS = FN + FM;
  // The reads run SETS - 1 steps ahead of the products, so in front of step SWITCH of a stage the rest of it is in registers.  There is its
  // barrier: its place is free, and the stage STAGES ahead is loaded there during the next STEPS steps.
  constexpr int SWITCH = STEPS - (SETS - 1);
  static_assert(SWITCH >= 1 && STEPS % SETS == 0, "operand sets");
  const auto wait = [&](auto in_flight_) {          // for all loads but the youngest, and for the operands; then for the other waves
    constexpr int in_flight = decltype(in_flight_)::value;
    static_assert(in_flight < 64, "loads in flight");
    __builtin_amdgcn_s_waitcnt(0x0070 | (in_flight & 15) | ((in_flight >> 4) << 14));
    asm volatile("s_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  constexpr int AHEAD = (STAGES - 1) * LOADS + LOADS * (STEPS - SWITCH) / STEPS;             // loads in front of the first product
  #pragma unroll
  for (int l = 0; l < AHEAD; ++l) {
    const int k = (begin + l / LOADS) * SLAB;
    gload(lds0 + l / LOADS * T::STAGE, k, outside_at(k), l % LOADS);
  }
  wait(Int<AHEAD - LOADS>{});
  #pragma unroll
  for (int st = 0; st < SETS - 1; ++st)
    #pragma unroll
    for (int f = 0; f < READS; ++f) rd(st, st, f, 0);
  __builtin_amdgcn_sched_barrier(0);
  uint32_t cur = 0, dst = lds0 + (STAGES - 1) * T::STAGE;
  int at = (begin + STAGES - 1) * SLAB, s = 0;
  Outside outside = outside_at(at);
  do {                                              // (a part has at least one stage)
    const uint32_t nxt = cur == (STAGES - 1) * T::STAGE ? 0 : cur + T::STAGE;
    #pragma unroll
    for (int st = 0; st < STEPS; ++st) {
      if (st == SWITCH) {
        wait(Int<(STAGES - 2) * LOADS>{});          // the next stage has landed; the loads of those behind it may be in flight
        dst = lds0 + cur;
        at += SLAB;
        outside = outside_at(at);
      }
      const int set = st % SETS, after = (st + STEPS - SWITCH) % STEPS, l0 = LOADS * after / STEPS, l1 = LOADS * (after + 1) / STEPS;
      #pragma unroll
      for (int m = 0; m < PRODUCTS; ++m) {
        const int j = m / FM, i = m % FM;
        acc[j][i] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fr[set][j], fr[set][FN + i], acc[j][i], 0, 0, 0);
        if (ASYM && i == 0) wsum[j] = add_bytes(fr[set][j], wsum[j]);
        // the reads in the first three quarters of the products and in their order, the loads spread over all of them
        #pragma unroll
        for (int f = 0; f < READS; ++f)
          if (f * PRODUCTS * 3 / 4 / READS == m)
            rd((st + SETS - 1) % SETS, (st + SETS - 1) % STEPS, f == 0 ? 0 : f <= FM ? FN + f - 1 : f - FM, st < SWITCH ? cur : nxt);
        #pragma unroll
        for (int p = 0; p < LOADS; ++p)
          if (p >= l0 && p < l1 && (p - l0 + 1) * PRODUCTS / (l1 - l0) - 1 == m) gload(dst, at, outside, p);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    cur = nxt;
  } while (++s < steps);
  __builtin_amdgcn_s_waitcnt(0x0070);               // nothing may still be on its way to LDS when it is used again

  // ---- outputs: register r of lane l is channel 8 (r / 4) + 4 (l / 32) + r % 4 of token l % 32 ----
  if (BF != ROW_I32 && tid < T::TN) { channel[0][tid] = from_raw(chan[0], g.ws_dtype); channel[1][tid] = from_raw(chan[1], g.bias_dtype); }
  if (ASYM && wr == 0) {
    #pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int both = wsum[j] + __builtin_amdgcn_ds_bpermute((lane ^ 32) * 4, wsum[j]);
      if (lane < 32) sums[wc * FN * 32 + j * 32 + lane] = both;
    }
  }
  __syncthreads();
  // A wave's outputs leave through its own part of LDS, 16 bytes per lane along a token; the chunks of 16 bytes of token t are turned by t.
  constexpr int E = BF == ROW_F32 || BF == ROW_I32 ? 4 : 2, CH = 16 / E;     // bytes of an output, outputs of a chunk
  constexpr int ROW = FN * 32 * E, CHUNKS = ROW / 16;
  constexpr int STEP = E == 4 && FM > 1 ? FM / 2 : FM;                       // blocks of 32 tokens that leave together
  static_assert(4 * STEP * 32 * ROW <= STAGES * T::STAGE, "outputs on their way out");
  char* const mine = lds + wave * STEP * 32 * ROW;
  const auto turned = [](int chunk, int token) { return (chunk + token) % CHUNKS; };
  const int t = lane & 31, h = lane >> 5;
  #pragma unroll
  for (int i0 = 0; i0 < FM; i0 += STEP) {
    #pragma unroll
    for (int j = 0; j < FN; ++j) {
      // (the accumulators stay where they are until their turn: copied out together they would not fit the other registers)
      if constexpr (FM * FN > 8) {
        #pragma unroll
        for (int i = i0; i < i0 + STEP; ++i) asm volatile("" : "+a"(acc[j][i]));
      }
      #pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int c = j * 32 + 8 * q + 4 * h;       // first of four channels, in the wave
        f32x4 ws, b;
        i32x4 sum;
        if constexpr (BF != ROW_I32) { ws = *(const f32x4*)&channel[0][wc * FN * 32 + c]; b = *(const f32x4*)&channel[1][wc * FN * 32 + c]; }
        if constexpr (ASYM) sum = *(const i32x4*)&sums[wc * FN * 32 + c];
        #pragma unroll
        for (int i = i0; i < i0 + STEP; ++i) {
          float v[4];
          #pragma unroll
          for (int r = 0; r < 4; ++r) {
            int s = acc[j][i][4 * q + r];
            if constexpr (ASYM) s -= az[i] * sum[r];
            v[r] = BF == ROW_I32 ? __builtin_bit_cast(float, s) : __builtin_fmaf((float)s, as[i] * ws[r], b[r]);
          }
          char* const to = mine + ((i - i0) * 32 + t) * ROW + turned(c / CH, t) * 16 + (c % CH) * E;
          if constexpr (E == 4) *(f32x4*)to = f32x4{v[0], v[1], v[2], v[3]};
          else if constexpr (BF == ROW_BF16) *(u32x2*)to = u32x2{bf16_pack_rne(v[0], v[1]), bf16_pack_rne(v[2], v[3])};
          else *(u32x2*)to = u32x2{f16_pack_rne(v[0], v[1]), f16_pack_rne(v[2], v[3])};
        }
      }
    }
    asm volatile("" ::: "memory");                  // (LDS serves a wave in order)
    #pragma unroll
    for (int o = 0; o < STEP * 32 * CHUNKS / 64; ++o) {
      const int idx = o * 64 + lane, tt = idx / CHUNKS, ch = idx % CHUNKS;
      const u32x4 v = *(const u32x4*)(mine + tt * ROW + turned(ch, tt % 32) * 16);
      const int m = wr * FM * 32 + i0 * 32 + tt, n = wc * FN * 32 + ch * CH;
      if (m >= rows_a || n >= rows_w) continue;
      const int64_t cell = (m0 + m) * g.N + n0 + n + (BF == ROW_I32 ? part * g.M * g.N : 0);
      if (n + CH <= rows_w) {
        __builtin_memcpy((char*)g.y + cell * E, &v, 16);     // (rows may start anywhere)
      } else {
        #pragma unroll
        for (int e = 0; e < CH; ++e)
          if (n + e < rows_w) {
            if constexpr (E == 4) ((uint32_t*)g.y)[cell + e] = v[e];
            else ((uint16_t*)g.y)[cell + e] = (uint16_t)(v[e / 2] >> 16 * (e % 2));
          }
      }
    }
    asm volatile("" ::: "memory");
  }
}

// The parts of K added up, scaled and rounded: sums [parts, M, N], V channels of a token per lane.
template <int BF, int V>
__global__ __launch_bounds__(256) void join_kernel(MatmulArgs g, const int* __restrict__ sums, int parts) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V, all = g.M * g.N;
  if (i >= all) return;
  const int64_t m = i / g.N, n = i - m * g.N;
  int s[V] = {};
  for (int p = 0; p < parts; ++p) {
    if constexpr (V == 4) {
      const i32x4 v = *(const i32x4*)(sums + p * all + i);
      #pragma unroll
      for (int e = 0; e < V; ++e) s[e] += v[e];
    } else {
      s[0] += sums[p * all + i];
    }
  }
  const float as = g.as[g.a_scalar ? 0 : m];
  float v[V];
  #pragma unroll
  for (int e = 0; e < V; ++e)
    v[e] = __builtin_fmaf((float)s[e], as * load_any(g.ws, g.ws_dtype, g.w_scalar ? 0 : n + e), g.bias ? load_any(g.bias, g.bias_dtype, n + e) : 0.0f);
  if constexpr (V == 4) {
    if constexpr (BF == ROW_F32) *(f32x4*)((float*)g.y + i) = f32x4{v[0], v[1], v[2], v[3]};
    else if constexpr (BF == ROW_BF16) *(u32x2*)((uint16_t*)g.y + i) = u32x2{bf16_pack_rne(v[0], v[1]), bf16_pack_rne(v[2], v[3])};
    else *(u32x2*)((uint16_t*)g.y + i) = u32x2{f16_pack_rne(v[0], v[1]), f16_pack_rne(v[2], v[3])};
  } else {
    if constexpr (BF == ROW_F32) ((float*)g.y)[i] = v[0];
    else store_scalar<BF>(g.y, i, rnd<BF>(v[0]));
  }
}

// ---- few tokens ---------------------------------------------------------------------------------------------------
// The weight is read once, straight into the matrix pipe's operands: a lane of v_mfma_i32_16x16x64_i8 takes 16 codes of one of 16
// channels, so a load of the wave is 16 rows x 64 bytes in a row.  A workgroup owns 16 or 32 channels, its waves take pieces of 256
// codes of K in turn and meet in LDS; four (two) pieces, 16 KiB of weight per wave, are in flight, with the codes of the tokens beside them,
// which come from the cache.  What bounds it is the ramp of the first loads and then HBM, 3 us + the weight at 5.5 TB/s: 2 tokens take 6.1 us
// at N = K = 4096, 43 us (5.4 TB/s) at 8192 x 28672; the tokens' codes pass the L2 once per workgroup, which tells from 16 tokens on.
// One token or a few may come as values: every workgroup makes their codes itself, in LDS, while its first weights are on their way - cheaper
// than another kernel in front (6.4 us at N = K = 4096, the quantizer alone 3.4).
constexpr int PIECE = 256;
constexpr int64_t MOST_FUSED = 32768;               // codes of a token that is quantized in LDS
constexpr int MOST_TOKENS = 8;                      // that every workgroup quantizes itself

struct TokenArgs {
  const void* x;
  const float* scale;
  int64_t ldx;
  int asym;
};

// A row of x, KEEP pieces of eight values per lane of it in registers, and its int8 codes to LDS, by the whole workgroup or, WAVES = 1, by any
// wave of it; K % 16 == 0.  The loads are apart from the rest, so that the weight's can be issued behind them.
template <int XT, int WAVES, int KEEP = 4>
struct TokenRow {
  static constexpr int RAW = XT == ROW_F32 ? 2 : 1;
  u32x4 raw[KEEP][RAW];
  const char* x;
  int K;
  __device__ __forceinline__ void load8(int i, u32x4* r) const {
    if ((uintptr_t)x % 16 == 0) {
      #pragma unroll
      for (int p = 0; p < RAW; ++p) r[p] = *(const u32x4*)(x + i * (2 * RAW) + 16 * p);
    } else {
      #pragma unroll
      for (int p = 0; p < RAW; ++p) {
        float v[8];
        #pragma unroll
        for (int e = 0; e < 8 / RAW; ++e) v[e] = load_scalar<XT>(x, i + p * 4 + e);
        r[p] = pack<XT>(v);
      }
    }
  }
  __device__ __forceinline__ void load(const TokenArgs& t, int64_t row, int K_) {
    K = K_;
    x = (const char*)t.x + row * t.ldx * (2 * RAW);
    #pragma unroll
    for (int c = 0; c < KEEP; ++c) {
      const int i = (threadIdx.x % (WAVES * 64) + c * WAVES * 64) * 8;
      if (i < K) load8(i, raw[c]);
    }
  }
  template <class F>
  __device__ __forceinline__ void each(F&& f) const {
    #pragma unroll
    for (int c = 0; c < KEEP; ++c) {
      const int i = (threadIdx.x % (WAVES * 64) + c * WAVES * 64) * 8;
      float v[8];
      if (i < K) {
        #pragma unroll
        for (int p = 0; p < RAW; ++p) unpack<XT>(raw[c][p], v + 4 * p);
        f(i, v);
      }
    }
    for (int i = (threadIdx.x % (WAVES * 64) + KEEP * WAVES * 64) * 8; i < K; i += WAVES * 64 * 8) {
      u32x4 r[RAW];
      float v[8];
      load8(i, r);
      #pragma unroll
      for (int p = 0; p < RAW; ++p) unpack<XT>(r[p], v + 4 * p);
      f(i, v);
    }
  }
  // red: 2 WAVES floats (WAVES = 1: none, and the caller waits for the other waves)
  __device__ __forceinline__ void to_codes(const TokenArgs& t, int8_t* out, float* red, float* scale, int* zero) const {
    const int wave = threadIdx.x >> 6;
    float hi = t.asym ? -__builtin_inff() : 0.0f, lo = __builtin_inff();
    each([&](int, const float* e) {
      #pragma unroll
      for (int j = 0; j < 8; ++j) {
        hi = nan_max(hi, t.asym ? e[j] : fabsf(e[j]));
        lo = nan_min(lo, e[j]);
      }
    });
    hi = team_reduce<64, true>(hi);
    if (t.asym) lo = team_reduce<64, false>(lo);
    if constexpr (WAVES > 1) {
      if ((threadIdx.x & 63) == 0) { red[wave] = hi; red[WAVES + wave] = lo; }
      __syncthreads();
      #pragma unroll
      for (int w = 0; w < WAVES; ++w) { hi = nan_max(hi, red[w]); lo = nan_min(lo, red[WAVES + w]); }
    }
    const TokenCodes q = t.scale ? TokenCodes::given(t.scale[0]) : t.asym ? TokenCodes::asymmetric(lo, hi) : TokenCodes::symmetric(hi);
    each([&](int i, const float* e) {
      uint32_t w[2];
      q.codes<8>(e, w);
      *(u32x2*)(out + i) = u32x2{w[0], w[1]};
    });
    if (threadIdx.x % (WAVES * 64) == 0) {
      *scale = q.d.s;
      *zero = q.z;
    }
    if constexpr (WAVES > 1) __syncthreads();
  }
};
template <int WAVES, int KEEP> struct TokenRow<-1, WAVES, KEEP> {};


// 16 codes that were read `codes` too early: the first ones leave, zeros follow
__device__ __forceinline__ i32x4 later(i32x4 v, int codes) {
  struct Halves { uint64_t lo, hi; } h = __builtin_bit_cast(Halves, v);
  const int s = (codes & 7) * 8;
  if (codes >= 8) { h.lo = h.hi; h.hi = 0; }
  if (codes >= 16) h.lo = 0;
  h.lo = h.lo >> s | (h.hi << 1) << (63 - s);
  h.hi >>= s;
  return __builtin_bit_cast(i32x4, h);
}

// TB blocks of 16 tokens, NB blocks of 16 channels.  XT: the type of the tokens' values (one token, or MANY of up to MOST_TOKENS: a wave quantizes
// a row at a time), or -1 for codes.
// ODD: rows start on any byte (K >= 16).  16 codes are cut from the five words that hold them, which costs far less than loads off word
// alignment (K = 4097, N = 14336, 16 tokens: 25.5 us for 66; 38 by padded copies); a row's last codes are read from K - 16 and moved.
template <int TB, int NB, int BF, int XT, int WAVES, bool ODD, bool MANY>
__global__ __launch_bounds__(WAVES * 64) void stream_kernel(MatmulArgs g, TokenArgs t) {
  __shared__ __attribute__((aligned(16))) int red[WAVES][NB][TB + 1][64][4];
  __shared__ float token_scale[MANY ? MOST_TOKENS : 1];
  __shared__ int token_zero[MANY ? MOST_TOKENS : 1];
  extern __shared__ __attribute__((aligned(16))) int8_t codes[];             // XT >= 0: [M] rows, K + 16 apart (16 lanes' reads touch all banks once)
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t n0 = (int64_t)blockIdx.x * (16 * NB);
  const int rows_w = (int)(g.N - n0 < 16 * NB ? g.N - n0 : 16 * NB);
  const int at = (lane >> 4) * 16;                  // this lane's 16 codes of 64
  const bool asym = XT < 0 ? g.az != nullptr : t.asym;
  TokenRow<XT, MANY ? 1 : WAVES, MANY ? 8 : 4> row;
  if constexpr (XT >= 0) row.load(t, MANY && wave < g.M ? wave : 0, g.K);
  const int8_t* const mine = codes + (MANY && (lane & 15) < g.M ? (lane & 15) * (g.K + 16) : 0);       // (a token past the last one is not stored)

  // Loads are told where their matrix ends: codes past K and rows past the last one read as zero, without a branch.
  const __amdgpu_buffer_rsrc_t bufW = __builtin_amdgcn_make_buffer_rsrc((void*)(g.w + n0 * g.ldw), 0, (int)((rows_w - 1) * g.ldw + g.K), 0x00020000);
  const __amdgpu_buffer_rsrc_t bufA = __builtin_amdgcn_make_buffer_rsrc((void*)g.a, 0, XT < 0 ? (int)((g.M - 1) * g.lda + g.K) : 0, 0x00020000);
  constexpr uint32_t OUTSIDE = 0x80000000u;
  uint32_t ofW[NB], ofA[TB];
  #pragma unroll
  for (int c = 0; c < NB; ++c) ofW[c] = c * 16 + (lane & 15) < rows_w ? (uint32_t)((c * 16 + (lane & 15)) * g.ldw) + at : OUTSIDE;
  #pragma unroll
  for (int b = 0; b < TB; ++b) ofA[b] = b * 16 + (lane & 15) < g.M ? (uint32_t)((b * 16 + (lane & 15)) * g.lda) + at : OUTSIDE;
  // words around the first codes of the matrices and, from there, this lane's rows (what a channel or token past the last one gives is not stored)
  const int8_t *wordsW = nullptr, *wordsA = nullptr;
  if constexpr (ODD) {
    const int8_t *const w = g.w + n0 * g.ldw, *const a = g.a;
    const uint32_t inW = (uint32_t)(uintptr_t)w & 3, inA = (uint32_t)(uintptr_t)a & 3;
    wordsW = w - inW;
    wordsA = a - inA;
    #pragma unroll
    for (int c = 0; c < NB; ++c) ofW[c] = inW + (uint32_t)((c * 16 + (lane & 15) < rows_w ? c * 16 + (lane & 15) : rows_w - 1) * g.ldw);
    #pragma unroll
    for (int b = 0; b < TB; ++b) ofA[b] = inA + (uint32_t)((b * 16 + (lane & 15) < g.M ? b * 16 + (lane & 15) : g.M - 1) * g.lda);
  }
  const auto words = [](const int8_t* p, uint32_t of, i32x4& v, int& fifth) {          // (every word holds one of the codes at least)
    __builtin_memcpy(&v, __builtin_assume_aligned(p + (of & ~3u), 4), 16);
    fifth = *(const int*)(p + (of & ~3u) + (of & 3 ? 16 : 12));
  };
  const auto cut = [](i32x4 v, int fifth, uint32_t of) {
    return i32x4{(int)__builtin_amdgcn_alignbyte(v[1], v[0], of), (int)__builtin_amdgcn_alignbyte(v[2], v[1], of),
                 (int)__builtin_amdgcn_alignbyte(v[3], v[2], of), (int)__builtin_amdgcn_alignbyte(fifth, v[3], of)};
  };
  // DEPTH pieces of 256 codes in flight, each with its tokens': waiting for the oldest leaves the others on their way
  constexpr int DEPTH = ODD ? (TB + NB == 2 ? 3 : 2) : TB + NB <= 3 ? 4 : 2, STEP = WAVES * PIECE;
  struct Piece { i32x4 w[NB][4], a[TB][4]; int w5[ODD ? NB : 1][4], a5[ODD ? TB : 1][4]; } ring[DEPTH];
  const auto load = [&](int k, Piece& p) {          // codes k .. k + 255
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (ODD) {
        const uint32_t from = k + i * 64 + at < g.K - 16 ? k + i * 64 + at : g.K - 16;
        #pragma unroll
        for (int c = 0; c < NB; ++c) words(wordsW, ofW[c] + from, p.w[c][i], p.w5[c][i]);
        #pragma unroll
        for (int b = 0; b < TB; ++b) words(wordsA, ofA[b] + from, p.a[b][i], p.a5[b][i]);
        continue;
      }
      const uint32_t outside = k + i * 64 + at < g.K ? 0u : OUTSIDE;
      #pragma unroll
      for (int c = 0; c < NB; ++c)
        p.w[c][i] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(bufW, ofW[c] | outside, k + i * 64, 0));
      if constexpr (XT < 0) {
        #pragma unroll
        for (int b = 0; b < TB; ++b)
          p.a[b][i] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(bufA, ofA[b] | outside, k + i * 64, 0));
      }
    }
  };
  int k = wave * PIECE;
  #pragma unroll
  for (int d = 0; d < DEPTH; ++d) {
    load(k + d * STEP, ring[d]);
    __builtin_amdgcn_sched_barrier(0);              // (in this order: a wait counts the loads behind it)
  }
  if constexpr (MANY) {
    for (int r = wave; r < g.M; r += WAVES) {
      if (r != wave) row.load(t, r, g.K);
      row.to_codes(t, codes + r * (g.K + 16), nullptr, &token_scale[r], &token_zero[r]);
    }
    __syncthreads();
  } else if constexpr (XT >= 0) {
    row.to_codes(t, codes, (float*)red, token_scale, token_zero);
  }
  i32x4 acc[NB][TB] = {};
  int wsum[NB] = {};
  while (k < g.K) {
    #pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      Piece& p = ring[d];
      if constexpr (ODD) {
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int early = k + i * 64 + at - (g.K - 16);
          const uint32_t from = early < 0 ? 0 : g.K - 16;                    // (k + i 64 + at is whole words)
          #pragma unroll
          for (int c = 0; c < NB; ++c) p.w[c][i] = cut(p.w[c][i], p.w5[c][i], ofW[c] + from);
          #pragma unroll
          for (int b = 0; b < TB; ++b) p.a[b][i] = cut(p.a[b][i], p.a5[b][i], ofA[b] + from);
          if (k + PIECE > g.K) {
            #pragma unroll
            for (int c = 0; c < NB; ++c) p.w[c][i] = later(p.w[c][i], early > 0 ? early : 0);
            #pragma unroll
            for (int b = 0; b < TB; ++b) p.a[b][i] = later(p.a[b][i], early > 0 ? early : 0);
          }
        }
      }
      #pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (XT >= 0) p.a[0][i] = *(const i32x4*)(mine + (k + i * 64 + at < g.K ? k + i * 64 + at : 0));   // (past K the weight is 0)
        #pragma unroll
        for (int c = 0; c < NB; ++c) {
          #pragma unroll
          for (int b = 0; b < TB; ++b) acc[c][b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(p.w[c][i], p.a[b][i], acc[c][b], 0, 0, 0);
          if (asym) wsum[c] = add_bytes(p.w[c][i], wsum[c]);
        }
      }
      load(k + DEPTH * STEP, p);
      k += STEP;
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  #pragma unroll
  for (int c = 0; c < NB; ++c) {
    #pragma unroll
    for (int b = 0; b < TB; ++b) *(i32x4*)red[wave][c][b][lane] = acc[c][b];
    red[wave][c][TB][lane][0] = wsum[c];
  }
  __syncthreads();
  // accumulator register r of lane l: channel 4 (l / 16) + r of token l % 16
  for (int o = tid; o < TB * NB * 256; o += WAVES * 64) {
    const int c = o % (16 * NB), cb = c >> 4, cc = c & 15, token = o / (16 * NB), b = token >> 4, tok = token & 15;
    const int64_t nn = n0 + c;
    if (token >= g.M || nn >= g.N) continue;
    int s = 0, sum = 0;
    #pragma unroll
    for (int v = 0; v < WAVES; ++v) {
      s += red[v][cb][b][(cc >> 2) * 16 + tok][cc & 3];
      if (asym) sum += (red[v][cb][TB][cc][0] + red[v][cb][TB][cc + 16][0]) + (red[v][cb][TB][cc + 32][0] + red[v][cb][TB][cc + 48][0]);
    }
    if (asym) s -= (XT < 0 ? g.az[token] : token_zero[MANY ? token : 0]) * sum;
    const float as = XT < 0 ? g.as[g.a_scalar ? 0 : token] : token_scale[MANY ? token : 0];
    const float y = __builtin_fmaf((float)s, as * load_any(g.ws, g.ws_dtype, g.w_scalar ? 0 : nn), g.bias ? load_any(g.bias, g.bias_dtype, nn) : 0.0f);
    if constexpr (BF == ROW_F32) ((float*)g.y)[token * g.N + nn] = y;
    else store_scalar<BF>(g.y, token * g.N + nn, rnd<BF>(y));
  }
}

// Rows of K codes to rows of Kp, the next multiple of 16, with zeros behind them: operands whose rows do not start on 16 bytes.  The
// rows of a, then those of w; `out` has them one behind the other.  A wave takes a row at a time, 4096 codes with all loads on their way at
// once; the last 16 codes are read from K - 16 and moved.
__global__ __launch_bounds__(256) void pad_kernel(const int8_t* __restrict__ a, int64_t rows_a, const int8_t* __restrict__ w, int64_t rows, int K, int Kp,
                                                  int8_t* __restrict__ out) {
  const int lane = threadIdx.x & 63;
  for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < rows; r += (int64_t)gridDim.x * 4) {
    const int8_t* const x = r < rows_a ? a + r * K : w + (r - rows_a) * K;
    if (K < 16) {
      if (lane < 16) out[r * 16 + lane] = lane < K ? x[lane] : (int8_t)0;
      continue;
    }
    for (int k0 = lane * 16; k0 < Kp; k0 += 4096) {
      i32x4 v[4];
      #pragma unroll
      for (int i = 0; i < 4; ++i) __builtin_memcpy(&v[i], x + (k0 + i * 1024 < K - 16 ? k0 + i * 1024 : K - 16), 16);
      #pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int k = k0 + i * 1024;
        if (k < Kp) *(i32x4*)(out + r * Kp + k) = k > K - 16 ? later(v[i], k - (K - 16)) : v[i];
      }
    }
  }
}

int64_t padded(int64_t K) { return (K + 15) / 16 * 16; }
int64_t on256(int64_t bytes) { return (bytes + 255) / 256 * 256; }

// The large tiles run at the rate at which half lines reach LDS (64 codes of a row; 27 bytes per clock and CU), but two stages of 128 codes,
// all that fits next to each other, are too few for the latency of the cache: 256 x 256 took 0.59 us per 64 codes with them, 0.50 so.
// 128 x 128 has room for four stages of whole lines (41 bytes per clock): 0.167 us per 64 codes, with half lines 0.25, with two stages 0.37
// (and 0.20 as two workgroups per CU).
typedef Tile<4, 4, 64, 4, 2> Tile256;
typedef Tile<4, 3, 64, 4, 2> Tile192;
typedef Tile<2, 2, 128, 4, 2> Tile128;

template <class T, int BF>
void launch_tiles(const MatmulArgs& g, int parts, hipStream_t st) {
  const int64_t tm = (g.M + T::TM - 1) / T::TM, tn = (g.N + T::TN - 1) / T::TN;
  const dim3 grid((unsigned)((tm * tn * parts + 7) / 8 * 8));
  if (g.az) tile_kernel<T, BF, true><<<grid, dim3(256), 0, st>>>(g, (int)tm, (int)tn, parts);
  else tile_kernel<T, BF, false><<<grid, dim3(256), 0, st>>>(g, (int)tm, (int)tn, parts);
}
template <int BF>
void launch_join(const MatmulArgs& g, const int* sums, int parts, hipStream_t st) {
  const bool wide = g.N % 4 == 0 && (uintptr_t)g.y % 16 == 0;      // (four channels of one token)
  const int64_t all = g.M * g.N;
  if (wide) join_kernel<BF, 4><<<dim3((unsigned)((all / 4 + 255) / 256)), dim3(256), 0, st>>>(g, sums, parts);
  else join_kernel<BF, 1><<<dim3((unsigned)((all + 255) / 256)), dim3(256), 0, st>>>(g, sums, parts);
}

template <int TB, int NB, int BF, int XT, int WAVES, bool ODD = false, bool MANY = false>
void launch_stream(const MatmulArgs& g, const TokenArgs& t, hipStream_t st) {
  stream_kernel<TB, NB, BF, XT, WAVES, ODD, MANY><<<dim3((unsigned)((g.N + 16 * NB - 1) / (16 * NB))), dim3(WAVES * 64),
                                                    XT < 0 ? 0 : (unsigned)(g.M * (g.K + 16)), st>>>(g, t);
}

// Two blocks of channels per workgroup halve the passes of the tokens' codes through the L2, one block spreads better over 256 CUs: it is
// taken where the busiest CU then has at most 3/4 (beyond 16 tokens half) of the channels.  us for one / two blocks:
//   N = 4096, K = 4096    16 tokens  7.0 / 9.5   32 tokens  9.5 / 12.8      N = 10240, K = 8192   16 tokens 26.4 / 27.9   32 tokens 39.5 / 35.8
//   N = 6144, K = 4096    16 tokens 11.3 / 10.9  32 tokens 16.2 / 13.0      N = 14336, K = 4096   16 tokens 19.5 / 17.1   32 tokens 28.6 / 22.4
// Two waves share K (four: 7.5 us for 7.1 in the first of these), one where there are two blocks and more workgroups than CUs (the last of
// these takes 23.7 with two waves; 8192 x 28672 at 32 tokens 65.5 with one for 64.5).
template <int TB, int BF, bool ODD>
void launch_few(const MatmulArgs& g, hipStream_t st) {
  const int64_t one = (g.N + 4095) / 4096, two = (g.N + 8191) / 8192 * 2;    // blocks of 16 channels on the busiest CU
  if (4 * one <= (TB == 1 ? 3 : 2) * two) launch_stream<TB, 1, BF, -1, 2, ODD>(g, TokenArgs{}, st);
  else if (two == 2) launch_stream<TB, 2, BF, -1, 2, ODD>(g, TokenArgs{}, st);
  else launch_stream<TB, 2, BF, -1, 1, ODD>(g, TokenArgs{}, st);
}

template <int BF, bool ODD>
void launch_blocks(const MatmulArgs& g, hipStream_t st) {
  if (g.M <= 16) launch_few<1, BF, ODD>(g, st);
  else if (g.M <= 32) launch_few<2, BF, ODD>(g, st);
  else if (g.M <= 48) launch_stream<3, 1, BF, -1, 2, ODD>(g, TokenArgs{}, st);
  else launch_stream<4, 1, BF, -1, 2, ODD>(g, TokenArgs{}, st);
}

template <int BF>
void launch_codes(const MatmulArgs& g, bool streams, int* sums, hipStream_t st) {
  if (streams) {
    if (g.K % 16) launch_blocks<BF, true>(g, st);
    else launch_blocks<BF, false>(g, st);
  }
  else {
    const Int8Cut c = int8_cut(g.M, g.N, g.K);
    if (c.parts > 1) {
      MatmulArgs p = g;
      p.y = sums;
      launch_tiles<Tile128, ROW_I32>(p, c.parts, st);
      launch_join<BF>(g, sums, c.parts, st);
    }
    else if (c.tile == 0) launch_tiles<Tile256, BF>(g, 1, st);
    else if (c.tile == 1) launch_tiles<Tile192, BF>(g, 1, st);
    else launch_tiles<Tile128, BF>(g, 1, st);
  }
}

// Few waves share the quantization of a short token (N = K = 4096: four waves 6.4 us, two 6.9, eight 7.6; N = 28672: 25.4, 26.7, 34),
// eight keep enough of a long weight row on its way (4096 x 14336: 14.7 us, four 16.9; 8192 x 28672: 45.4, four 50.6).
template <int BF, int XT>
void launch_token(const MatmulArgs& g, const TokenArgs& t, hipStream_t st) {
  if (g.M > 1) launch_stream<1, 1, BF, XT, 4, false, true>(g, t, st);
  else if (g.K <= 8192) launch_stream<1, 1, BF, XT, 4>(g, t, st);
  else launch_stream<1, 1, BF, XT, 8>(g, t, st);
}

bool known(int dtype) { return dtype == LCQ_F32 || dtype == LCQ_BF16 || dtype == LCQ_F16; }

int check(const int8_t* w, const void* ws, int ws_dtype, const void* bias, int bias_dtype, int64_t M, int64_t N, int64_t K, const void* y, int dtype) {
  if (!w || !ws || !y || M <= 0 || N <= 0 || K <= 0) return LCQ_EINVAL;
  if (!known(dtype) || !known(ws_dtype) || (bias && !known(bias_dtype))) return LCQ_EDTYPE;
  // A launch has fewer than 2^32 lanes: tiles of 256, rounded up to eight; 16 channels of 256 lanes, of 512 where a token is long.
  if (K > 65536 || M > 1 << 28 || N > (K <= 8192 ? 1 << 28 : 1 << 27) - 16 || (M + 127) / 128 * ((N + 127) / 128) > (1 << 24) - 8) return LCQ_ESIZE;
  if (K % 16 == 0 && (uintptr_t)w % 16) return LCQ_EALIGN;
  return LCQ_OK;
}

// rows that only the padding kernel brings to where they can be read
bool pads(int64_t K, bool streams) { return K % 16 != 0 && (!streams || K < 16); }

// Tokens whose codes every workgroup of the product makes itself: one, and up to eight where a wave's rows are short and hardly more workgroups than
// CUs make them.  One launch instead of two costs the host 4 us less; on the GPU it takes, with the quantizer's launch beside it, us:
//   N = K = 4096, 4 tokens 9.6 / 9.7     K = 1024, 4 tokens 5.4 / 6.1, 8 tokens 6.9 / 6.6     K = 2048, 8 tokens 8.8 / 7.0 (by itself)
//   N = 14336, K = 4096, 4 tokens 21.1 / 17.7 and N = 1024, K = 8192, 2 tokens 13.3 / 10.5 (by itself both)
// The rule goes by a call from Python, whose host time is the longer at these sizes; in a captured graph 8 tokens at K = 1024 lose the 0.3 us of the table.
bool fused(int64_t M, int64_t N, int64_t K) {
  if (K % 16) return false;
  const int64_t rows = (M + 3) / 4;                 // of a wave
  return M == 1 ? K <= MOST_FUSED : M <= MOST_TOKENS && N <= 4096 && rows * rows * K <= 4096;
}

}  // namespace

extern "C" {

int64_t lcq_int8_matmul_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0 || K > 65536) return 0;
  const bool streams = int8_streams(M, N, K);
  const int parts = streams ? 1 : int8_cut(M, N, padded(K)).parts;
  return (parts > 1 ? on256(4 * M * N * parts) : 0) + (pads(K, streams) ? (M + N) * padded(K) : 0);
}

int lcq_int8_matmul(const int8_t* a, const float* as, int a_scalar, const int32_t* az, const int8_t* w, const void* ws, int ws_dtype,
                    int w_scalar, const void* bias, int bias_dtype, int64_t M, int64_t N, int64_t K, void* y, int dtype,
                    void* workspace, void* stream) {
  if (!a || !as) return LCQ_EINVAL;
  const int bad = check(w, ws, ws_dtype, bias, bias_dtype, M, N, K, y, dtype);
  if (bad) return bad;
  hipStream_t st = (hipStream_t)stream;
  MatmulArgs g = {a, w, as, az, ws, bias, y, M, N, K, K, (int)K, ws_dtype, bias_dtype, a_scalar, w_scalar};
  if (K % 16 == 0 && (uintptr_t)a % 16) return LCQ_EALIGN;
  const bool streams = int8_streams(M, N, K);
  const int parts = streams ? 1 : int8_cut(M, N, padded(K)).parts;
  if (pads(K, streams) || parts > 1) {
    if (!workspace) return LCQ_EWORKSPACE;
    if ((uintptr_t)workspace % 16) return LCQ_EALIGN;
  }
  if (pads(K, streams)) {
    const int Kp = (int)padded(K);
    int8_t* const pa = (int8_t*)workspace + (parts > 1 ? on256(4 * M * N * parts) : 0);
    const int64_t blocks = (M + N + 3) / 4;
    pad_kernel<<<dim3((unsigned)(blocks < 1 << 16 ? blocks : 1 << 16)), dim3(256), 0, st>>>(a, M, w, M + N, (int)K, Kp, pa);
    g.a = pa; g.w = pa + M * Kp; g.lda = g.ldw = g.K = Kp;
  }
  if (dtype == LCQ_BF16) launch_codes<ROW_BF16>(g, streams, (int*)workspace, st);
  else if (dtype == LCQ_F16) launch_codes<ROW_F16>(g, streams, (int*)workspace, st);
  else launch_codes<ROW_F32>(g, streams, (int*)workspace, st);
  LCQ_CHECK_LAUNCH();
  return LCQ_OK;
}

int64_t lcq_int8_linear_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0 || K > 65536 || fused(M, N, K)) return 0;
  return on256(M * K) + on256(8 * M) + lcq_int8_matmul_workspace_bytes(M, N, K);
}

int lcq_int8_linear(const void* x, int x_dtype, int64_t ldx, int asym, const float* scale, const int8_t* w, const void* ws, int ws_dtype,
                    int w_scalar, const void* bias, int bias_dtype, int64_t M, int64_t N, int64_t K, void* y, int dtype,
                    void* workspace, void* stream) {
  if (!x || ldx < 0 || (asym && scale)) return LCQ_EINVAL;
  const int bad = check(w, ws, ws_dtype, bias, bias_dtype, M, N, K, y, dtype);
  if (bad) return bad;
  if (!known(x_dtype)) return LCQ_EDTYPE;
  if (fused(M, N, K)) {
    hipStream_t st = (hipStream_t)stream;
    const MatmulArgs g = {nullptr, w, nullptr, nullptr, ws, bias, y, M, N, K, K, (int)K, ws_dtype, bias_dtype, 0, w_scalar};
    const TokenArgs t = {x, scale, ldx, asym};
    const auto run = [&](auto xt) {
      constexpr int XT = decltype(xt)::value;
      if (dtype == LCQ_BF16) launch_token<ROW_BF16, XT>(g, t, st);
      else if (dtype == LCQ_F16) launch_token<ROW_F16, XT>(g, t, st);
      else launch_token<ROW_F32, XT>(g, t, st);
    };
    if (x_dtype == LCQ_BF16) run(Int<ROW_BF16>{});
    else if (x_dtype == LCQ_F16) run(Int<ROW_F16>{});
    else run(Int<ROW_F32>{});
    LCQ_CHECK_LAUNCH();
    return LCQ_OK;
  }
  if (!workspace) return LCQ_EWORKSPACE;
  if ((uintptr_t)workspace % 16) return LCQ_EALIGN;
  int8_t* const codes = (int8_t*)workspace;
  float* const scales = (float*)(codes + on256(M * K));
  int32_t* const zeros = asym ? (int32_t*)(scales + M) : nullptr;
  const int rc = lcq_quant_tokens(x, x_dtype, M, K, ldx, asym, scale, codes, scales, zeros, stream);
  if (rc) return rc;
  return lcq_int8_matmul(codes, scale ? scale : scales, scale != nullptr, zeros, w, ws, ws_dtype, w_scalar, bias, bias_dtype, M, N, K, y, dtype,
                         (char*)scales + on256(8 * M), stream);
}

}  // extern "C"

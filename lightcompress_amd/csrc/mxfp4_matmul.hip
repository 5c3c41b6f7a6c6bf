// Product of microscaled 4-bit numbers, y[m, n] = sum_b 2^(sa[m, b] + sw[n, b] - 254) sum_{k in block b} a[m, k] w[n, k] + bias[n].
//
// The matrix pipe takes blocks as they are: a lane of v_mfma_scale_f32_*_f8f6f4 holds the 16 bytes of one block and its scale byte.  The
// products of codes and powers of two are exact, the sums are the pipe's 32-bit ones, bias and rounding come once at the end.
// The weight is the first operand, so an accumulator's four neighbouring registers are four neighbouring channels of one token.
#include "mxfp4.h"
#include "launch_rules.h"
#include <type_traits>

namespace {
using namespace lcq;

typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((ext_vector_type(8))) int i32x8;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((address_space(3))) char* lds_ptr;
typedef __attribute__((address_space(3))) i32x4* lds_frag;

template <int I> using Int = std::integral_constant<int, I>;

struct MxArgs {
  const uint8_t *a, *sa, *w, *sw;
  const void* bias;
  void* y;
  int64_t M, N, lda, ldw, ldsa, ldsw;               // distances in bytes
  int B, bias_dtype;                                // blocks of a row
};

__device__ __forceinline__ float load_any(const void* p, int dtype, int64_t i) {
  return dtype == LCQ_F32 ? load_scalar<ROW_F32>(p, i) : dtype == LCQ_BF16 ? load_scalar<ROW_BF16>(p, i) : load_scalar<ROW_F16>(p, i);
}
// the same in two steps, so that nothing waits for the load before the value is used
__device__ __forceinline__ uint32_t load_raw(const void* p, int dtype, int64_t i) { return dtype == LCQ_F32 ? ((const uint32_t*)p)[i] : (uint32_t)((const uint16_t*)p)[i]; }
__device__ __forceinline__ float from_raw(uint32_t u, int dtype) {
  return dtype == LCQ_F32 ? u2f(u) : dtype == LCQ_BF16 ? u2f(u << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)u);
}
// (the pipe reads four registers of a 4-bit operand)
__device__ __forceinline__ i32x8 wide(i32x4 v) { return __builtin_shufflevector(v, v, 0, 1, 2, 3, -1, -1, -1, -1); }

// ---- tiles --------------------------------------------------------------------------------------------------------
// A workgroup of four waves (2 x 2) owns 64 FM tokens x 64 FN channels, a wave FM x FN accumulators of 32 x 32.
//  * codes stream through LDS stages of SLAB bytes per row by direct loads; rows past the end of a matrix and bytes past a row's blocks
//    lie outside the buffer that the loads are told and read as zero;
//  * piece p of 16 bytes (a block) of row r lies at p ^ (r / 4 % 4) or p ^ (r / 2 % 8), so that 16 lanes of an operand read touch all 64
//    banks once;
//  * scales come 16 per row, for 512 codes (a period), loaded two periods ahead into one of two places and read by each lane into
//    registers at the end of the period before theirs: a load of four scales per row and stage would fetch a line per row and stage;
//  * operands are buffered in registers: while the products of one step of 64 codes run, the reads of the next are issued between them;
//    one barrier per stage, where every wave holds the rest of it in registers: its place is loaded again from there.
constexpr int ROW_SUM = 3;                          // an output type: the sums of a part of K as they are
constexpr int PERIOD = 256;                         // bytes of a row between scale loads

template <int FM_, int FN_, int SLAB_, int STAGES_>
struct Tile {
  static constexpr int FM = FM_, FN = FN_, SLAB = SLAB_, STAGES = STAGES_;   // bytes of a row per stage
  static constexpr int TM = 64 * FM, TN = 64 * FN, STEPS = SLAB / 32;
  static constexpr int STAGE = (TM + TN) * SLAB, PER = PERIOD / SLAB;        // stages of a period
  static constexpr int SL = (TM + TN + 255) / 256;                           // a wave's scale loads of a period, 64 rows each
};

// 16-byte piece p of row r of a stage lies at p ^ swizzle(r)
template <int SLAB>
__device__ __forceinline__ int swizzle(int r) { return SLAB == 64 ? (r >> 2) & 3 : (r >> 1) & 7; }

template <class T, int BF>
__global__ __launch_bounds__(256, 1) void tile_kernel(MxArgs g, int tiles_m, int tiles_n, int parts) {
  constexpr int FM = T::FM, FN = T::FN, SLAB = T::SLAB, STAGES = T::STAGES, STEPS = T::STEPS, PER = T::PER, SL = T::SL;
  __shared__ __attribute__((aligned(1024))) char lds[STAGES * T::STAGE + 2 * 4 * SL * 1024];
  __shared__ __attribute__((aligned(16))) float channel[T::TN];              // biases
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
  const int bytes = g.B * 16, groups = (g.B + 15) >> 4;                      // of a row's codes; 16-byte pieces of its scales
  const int begin = (int)((int64_t)groups * part / parts), periods = (int)((int64_t)groups * (part + 1) / parts) - begin;

  const auto buffer = [&](const uint8_t* p, int64_t ld, int rows, int row) {
    const uint64_t at = (uint64_t)(uintptr_t)p;
    const auto one = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
    return i32x4{one((int)(uint32_t)at), one((int)(uint32_t)(at >> 32) & 0xffff), one((int)((rows - 1) * ld + row)), 0x00020000};
  };
  const i32x4 bufA = buffer(g.a + m0 * g.lda, g.lda, rows_a, bytes), bufW = buffer(g.w + n0 * g.ldw, g.ldw, rows_w, bytes);
  const i32x4 bufSA = buffer(g.sa + m0 * g.ldsa, g.ldsa, rows_a, groups * 16), bufSW = buffer(g.sw + n0 * g.ldsw, g.ldsw, rows_w, groups * 16);
  constexpr uint32_t OUTSIDE = 0x80000000u;
  constexpr int ROWS = 1024 / SLAB, LANES = 64 / ROWS;                       // of a load
  constexpr int LA = T::TM / (4 * ROWS), LW = T::TN / (4 * ROWS);            // a wave's loads of tokens and of weights per stage
  static_assert(SLAB == 64 || (LA % 2 == 0 && LW % 2 == 0), "a wave's loads start with an even one");
  // this lane's 16 bytes of a row: of an even load, and of an odd one (the same for 64 bytes)
  int piece16[2];
  #pragma unroll
  for (int e = 0; e < 2; ++e) piece16[e] = ((lane % LANES) ^ swizzle<SLAB>(e * ROWS + lane / LANES)) * 16;
  uint32_t gof[LA + LW], sof[SL];
  #pragma unroll
  for (int p = 0; p < LA + LW; ++p) {
    const int r = (wave * (p < LA ? LA : LW) + (p < LA ? p : p - LA)) * ROWS + lane / LANES;
    gof[p] = r < (p < LA ? rows_a : rows_w) ? (uint32_t)(r * (p < LA ? g.lda : g.ldw) + piece16[p & 1]) : OUTSIDE;
  }
  // scale load i of this wave: rows 64 (wave + 4 i) .. + 63 of tokens, then weights (beyond both: a place that nothing reads)
  #pragma unroll
  for (int i = 0; i < SL; ++i) {
    const int r = (wave + 4 * i) * 64 + lane;
    sof[i] = r < T::TM ? (r < rows_a ? (uint32_t)(r * g.ldsa) : OUTSIDE) : r - T::TM < rows_w ? (uint32_t)((r - T::TM) * g.ldsw) : OUTSIDE;
  }
  const uint32_t lds0 = (uint32_t)(size_t)(lds_ptr)lds;
  struct Outside { uint32_t of[2]; };
  // load p of the stage at LDS address dst, bytes [at, at + SLAB) of a row
  const auto gload = [&](uint32_t dst, int at, const Outside& outside, int p) {
    const uint32_t to = dst + (p < LA ? (wave * LA + p) * 1024 : T::TM * SLAB + (wave * LW + p - LA) * 1024);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                 ::"s"(to), "v"(gof[p] | outside.of[p & 1]), "s"(p < LA ? bufA : bufW), "s"(at) : "memory");
  };
  const auto outside_at = [&](int at) { return Outside{{piece16[0] < bytes - at ? 0u : OUTSIDE, piece16[1] < bytes - at ? 0u : OUTSIDE}}; };
  // the scales of period p (counted from this part's first), place p % 2
  const auto sload = [&](int p) {
    const uint32_t outside = begin + p < groups ? 0u : OUTSIDE;
    #pragma unroll
    for (int i = 0; i < SL; ++i) {
      const uint32_t to = lds0 + STAGES * T::STAGE + ((p & 1) * 4 * SL + wave + 4 * i) * 1024;
      const i32x4 buf = (wave + 4 * i) * 64 < T::TM ? bufSA : bufSW;
      asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                   ::"s"(to), "v"(sof[i] | outside), "s"(buf), "s"((begin + p) * 16) : "memory");
    }
  };

  // step ks reads pieces 2 ks (lanes 0 .. 31) and 2 ks + 1 of a row
  const int slot = (lane >> 5) ^ swizzle<SLAB>(lane & 31);
  const lds_ptr readA = (lds_ptr)lds + (wr * FM * 32 + (lane & 31)) * SLAB + slot * 16;
  const lds_ptr readW = (lds_ptr)lds + T::TM * SLAB + (wc * FN * 32 + (lane & 31)) * SLAB + slot * 16;
  const lds_ptr scaleA = (lds_ptr)lds + STAGES * T::STAGE + (wr * FM * 32 + (lane & 31)) * 16;
  const lds_ptr scaleW = (lds_ptr)lds + STAGES * T::STAGE + (T::TM + wc * FN * 32 + (lane & 31)) * 16;
  int step_at[STEPS];                               // from the first step of a stage to the others
  #pragma unroll
  for (int ks = 0; ks < STEPS; ++ks) step_at[ks] = ((slot ^ (2 * ks)) - slot) * 16;
  f32x16 acc[FN][FM];
  #pragma unroll
  for (int j = 0; j < FN; ++j)
    #pragma unroll
    for (int i = 0; i < FM; ++i)
      #pragma unroll
      for (int r = 0; r < 16; ++r) acc[j][i][r] = 0;
  i32x4 fr[2][FN + FM];                             // operands of a step: weights, tokens
  i32x4 sc[FN + FM], next[FN + FM];                 // their scales of a period: byte 2 s + lane / 32 is step s's
  const auto rd = [&](int set, int ks, int f, uint32_t stage) {
    fr[set][f] = *(lds_frag)((f < FN ? readW + f * 32 * SLAB : readA + (f - FN) * 32 * SLAB) + stage + step_at[ks]);
  };
  const auto rds = [&](int f, int place) { next[f] = *(lds_frag)((f < FN ? scaleW + f * 512 : scaleA + (f - FN) * 512) + place * 4 * SL * 1024); };
  const int half = (lane >> 5) * 8;
  const auto take = [&]() {                         // after it step s's byte is 2 (s % 2) of word s / 2
    #pragma unroll
    for (int f = 0; f < FN + FM; ++f)
      #pragma unroll
      for (int q = 0; q < 4; ++q) sc[f][q] = (int)((uint32_t)next[f][q] >> half);
  };
  uint32_t chan = 0;                                // the bias, on its way during the products
  if constexpr (BF != ROW_SUM) {
    if (g.bias && tid < rows_w) chan = load_raw(g.bias, g.bias_dtype, n0 + tid);
  }
  __builtin_amdgcn_sched_barrier(0);

  constexpr int LOADS = LA + LW, PRODUCTS = FM * FN, READS = FN + FM;
  // The reads run a step ahead of the products, so in front of a stage's last step the rest of it is in registers.  There is its
  // barrier: its place is free, and the stage STAGES ahead is loaded there during the next STEPS steps.
  constexpr int SWITCH = STEPS - 1;
  static_assert(SWITCH >= 1 && STEPS % 2 == 0 && PER <= STAGES && 2 * PER - 1 > STAGES - 2, "stages and periods");
  const auto wait = [&](auto in_flight_) {          // for all loads but the youngest, and for the operands; then for the other waves
    constexpr int in_flight = decltype(in_flight_)::value;
    static_assert(in_flight < 64, "loads in flight");
    __builtin_amdgcn_s_waitcnt(0x0070 | (in_flight & 15) | ((in_flight >> 4) << 14));
    asm volatile("s_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  constexpr int AHEAD = (STAGES - 1) * LOADS + LOADS * (STEPS - SWITCH) / STEPS;             // loads in front of the first product
  // Scales of a period are loaded in front of the codes that follow the first switch two periods earlier; the second period's go where
  // that would be, in front of stage STAGES - PER.
  sload(0);
  #pragma unroll
  for (int l = 0; l < AHEAD; ++l) {
    const int k = begin * PERIOD + l / LOADS * SLAB;
    if (l == (STAGES - PER) * LOADS) sload(1);
    gload(lds0 + l / LOADS * T::STAGE, k, outside_at(k), l % LOADS);
  }
  wait(Int<AHEAD - LOADS + (STAGES > PER ? SL : 0)>{});
  #pragma unroll
  for (int f = 0; f < READS; ++f) rds(f, 0);
  #pragma unroll
  for (int f = 0; f < READS; ++f) rd(0, 0, f, 0);
  __builtin_amdgcn_sched_barrier(0);
  uint32_t cur = 0, dst = lds0 + (STAGES - 1) * T::STAGE;
  int at = begin * PERIOD + (STAGES - 1) * SLAB, s = 0;
  Outside outside = outside_at(at);
  // a stage: J of its period, so that its steps' scale bytes and the loads in flight are known
  const auto stage = [&](auto j_) {
    constexpr int J = decltype(j_)::value;
    const uint32_t nxt = cur == (STAGES - 1) * T::STAGE ? 0 : cur + T::STAGE;
    // scale loads among the youngest (STAGES - 2) stages of loads
    constexpr auto among = [](int j) { int n = 0; for (int t = j - (STAGES - 2); t < j; ++t) n += (t + 2 * PER) % PER == 0; return n; };
    #pragma unroll
    for (int st = 0; st < STEPS; ++st) {
      if (st == SWITCH) {
        wait(Int<(STAGES - 2) * LOADS + SL * among(J)>{});       // the next stage has landed; the loads of those behind it may be in flight
        dst = lds0 + cur;
        at += SLAB;
        outside = outside_at(at);
        if (J == 0) sload(s + 2);
      }
      const int set = st % 2, after = (st + STEPS - SWITCH) % STEPS, l0 = LOADS * after / STEPS, l1 = LOADS * (after + 1) / STEPS;
      const int step = J * STEPS + st;
      #pragma unroll
      for (int m = 0; m < PRODUCTS; ++m) {
        const int j = m / FM, i = m % FM;
        const i32x8 w = wide(fr[set][j]), a = wide(fr[set][FN + i]);
        if (step % 2) acc[j][i] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w, a, acc[j][i], 4, 4, 2, sc[j][step / 2], 2, sc[FN + i][step / 2]);
        else acc[j][i] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w, a, acc[j][i], 4, 4, 0, sc[j][step / 2], 0, sc[FN + i][step / 2]);
        // the reads in the first three quarters of the products and in their order, the loads spread over all of them
        #pragma unroll
        for (int f = 0; f < READS; ++f) {
          if (f * PRODUCTS * 3 / 4 / READS == m)
            rd((st + 1) % 2, (st + 1) % STEPS, f == 0 ? 0 : f <= FM ? FN + f - 1 : f - FM, st < SWITCH ? cur : nxt);
          if (J == PER - 1 && st == SWITCH && f * PRODUCTS * 3 / 4 / READS == m) rds(f, (s + 1) & 1);
        }
        #pragma unroll
        for (int p = 0; p < LOADS; ++p)
          if (p >= l0 && p < l1 && (p - l0 + 1) * PRODUCTS / (l1 - l0) - 1 == m) gload(dst, at, outside, p);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    cur = nxt;
  };
  do {                                              // (a part has at least one period)
    take();
    stage(Int<0>{});
    stage(Int<1>{});
    if constexpr (PER == 4) { stage(Int<2>{}); stage(Int<3>{}); }
  } while (++s < periods);
  __builtin_amdgcn_s_waitcnt(0x0070);               // nothing may still be on its way to LDS when it is used again

  // ---- outputs: register r of lane l is channel 8 (r / 4) + 4 (l / 32) + r % 4 of token l % 32 ----
  if (BF != ROW_SUM && tid < T::TN) channel[tid] = from_raw(chan, g.bias_dtype);
  __syncthreads();
  // A wave's outputs leave through its own part of LDS, 16 bytes per lane along a token; the chunks of 16 bytes of token t are turned by t.
  constexpr int E = BF == ROW_F32 || BF == ROW_SUM ? 4 : 2, CH = 16 / E;     // bytes of an output, outputs of a chunk
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
        f32x4 b = {};
        if constexpr (BF != ROW_SUM) b = *(const f32x4*)&channel[wc * FN * 32 + c];
        #pragma unroll
        for (int i = i0; i < i0 + STEP; ++i) {
          float v[4];
          #pragma unroll
          for (int r = 0; r < 4; ++r) v[r] = BF == ROW_SUM ? acc[j][i][4 * q + r] : acc[j][i][4 * q + r] + b[r];
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
      const int64_t cell = (m0 + m) * g.N + n0 + n + (BF == ROW_SUM ? part * g.M * g.N : 0);
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

// The parts of K added up in their order, with the bias, and rounded: sums [parts, M, N], V channels of a token per lane.
template <int BF, int V>
__global__ __launch_bounds__(256) void join_kernel(MxArgs g, const float* __restrict__ sums, int parts) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V, all = g.M * g.N;
  if (i >= all) return;
  const int64_t n = i % g.N;
  float v[V] = {};
  for (int p = 0; p < parts; ++p) {
    if constexpr (V == 4) {
      const f32x4 s = *(const f32x4*)(sums + p * all + i);
      #pragma unroll
      for (int e = 0; e < V; ++e) v[e] += s[e];
    } else {
      v[0] += sums[p * all + i];
    }
  }
  if (g.bias) {
    #pragma unroll
    for (int e = 0; e < V; ++e) v[e] += load_any(g.bias, g.bias_dtype, n + e);
  }
  if constexpr (V == 4) {
    if constexpr (BF == ROW_F32) *(f32x4*)((float*)g.y + i) = f32x4{v[0], v[1], v[2], v[3]};
    else if constexpr (BF == ROW_BF16) *(u32x2*)((uint16_t*)g.y + i) = u32x2{bf16_pack_rne(v[0], v[1]), bf16_pack_rne(v[2], v[3])};
    else *(u32x2*)((uint16_t*)g.y + i) = u32x2{f16_pack_rne(v[0], v[1]), f16_pack_rne(v[2], v[3])};
  } else {
    if constexpr (BF == ROW_F32) ((float*)g.y)[i] = v[0];
    else store_scalar<BF>(g.y, i, rnd<BF>(v[0]));
  }
}

// Scales of rows that do not hold whole 16-byte pieces, or do not start on them, to rows that do, with zeros behind them: those of a, then
// those of w.  (A tile's loads of scales take 16 of a row.)
__global__ __launch_bounds__(256) void pad_scales_kernel(MxArgs g, int Bp, uint8_t* __restrict__ out, int64_t words) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= words) return;
  const int per = Bp / 4;
  const int64_t r = i / per;
  const int b = (int)(i - r * per) * 4;
  const uint8_t* const from = r < g.M ? g.sa + r * g.ldsa : g.sw + (r - g.M) * g.ldsw;
  uint32_t v = 0;
  #pragma unroll
  for (int e = 0; e < 4; ++e) v |= (b + e < g.B ? (uint32_t)from[b + e] : 0u) << 8 * e;
  ((uint32_t*)out)[i] = v;
}

// ---- few tokens ---------------------------------------------------------------------------------------------------
// The weight is read once, straight into the matrix pipe's operands: a lane of v_mfma_scale_f32_16x16x128 takes a block of one of 16
// channels, so a load of the wave is 16 rows x 64 bytes in a row, and one more brings a scale byte per lane.  A workgroup owns 16 or 32
// channels, its waves take pieces of 512 codes of K in turn and meet in LDS; the tokens' codes come from the cache, or, where there are
// few, every workgroup makes them itself, in LDS, while its first weights are on their way.
constexpr int PIECE = 256;                          // bytes of a row

struct TokenArgs {
  const char* x;
  int64_t ldx, K;
};

// TB blocks of 16 tokens, NB blocks of 16 channels.  XT: the type of the tokens' values, or -1 for codes.
template <int TB, int NB, int BF, int XT, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void stream_kernel(MxArgs g, TokenArgs t) {
  __shared__ __attribute__((aligned(16))) float red[WAVES][NB][TB][64][4];
  extern __shared__ __attribute__((aligned(16))) uint8_t made[];             // XT >= 0: [M] rows of codes, 16 B + 16 apart (16 lanes' reads touch all banks once); then of scales
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t n0 = (int64_t)blockIdx.x * (16 * NB);
  const int rows_w = (int)(g.N - n0 < 16 * NB ? g.N - n0 : 16 * NB);
  const int bytes = g.B * 16, q = lane >> 4;        // this lane's block of four
  // Loads are told where their matrix ends: blocks past the last and rows past the end read as zero, without a branch.
  const auto buffer = [](const uint8_t* p, int64_t size) { return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, (int)size, 0x00020000); };
  const __amdgpu_buffer_rsrc_t bufW = buffer(g.w + n0 * g.ldw, (rows_w - 1) * g.ldw + bytes), bufSW = buffer(g.sw + n0 * g.ldsw, (rows_w - 1) * g.ldsw + g.B);
  const __amdgpu_buffer_rsrc_t bufA = buffer(g.a, XT < 0 ? (g.M - 1) * g.lda + bytes : 0), bufSA = buffer(g.sa, XT < 0 ? (g.M - 1) * g.ldsa + g.B : 0);
  constexpr uint32_t OUTSIDE = 0x80000000u;
  uint32_t ofW[NB], ofSW[NB], ofA[TB], ofSA[TB];
  #pragma unroll
  for (int c = 0; c < NB; ++c) {
    const int r = c * 16 + (lane & 15);
    ofW[c] = r < rows_w ? (uint32_t)(r * g.ldw) + q * 16 : OUTSIDE;
    ofSW[c] = r < rows_w ? (uint32_t)(r * g.ldsw) + q : OUTSIDE;
  }
  #pragma unroll
  for (int b = 0; b < TB; ++b) {
    const int r = b * 16 + (lane & 15);
    ofA[b] = r < g.M ? (uint32_t)(r * g.lda) + q * 16 : OUTSIDE;
    ofSA[b] = r < g.M ? (uint32_t)(r * g.ldsa) + q : OUTSIDE;
  }
  constexpr int DEPTH = TB + NB <= 3 ? 4 : 2, STEP = WAVES * PIECE;
  struct Piece { i32x4 w[NB][4], a[TB][4]; int sw[NB][4], sa[TB][4]; } ring[DEPTH];
  const auto load = [&](int k, Piece& p) {          // bytes k .. k + 255 of a row
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t outside = k + i * 64 + q * 16 < bytes ? 0u : OUTSIDE;
      #pragma unroll
      for (int c = 0; c < NB; ++c) {
        p.w[c][i] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(bufW, ofW[c] | outside, k + i * 64, 0));
        p.sw[c][i] = __builtin_amdgcn_raw_buffer_load_b8(bufSW, ofSW[c] | outside, (k >> 4) + i * 4, 0);
      }
      if constexpr (XT < 0) {
        #pragma unroll
        for (int b = 0; b < TB; ++b) {
          p.a[b][i] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(bufA, ofA[b] | outside, k + i * 64, 0));
          p.sa[b][i] = __builtin_amdgcn_raw_buffer_load_b8(bufSA, ofSA[b] | outside, (k >> 4) + i * 4, 0);
        }
      }
    }
  };
  int k = wave * PIECE;
  #pragma unroll
  for (int d = 0; d < DEPTH; ++d) {
    load(k + d * STEP, ring[d]);
    __builtin_amdgcn_sched_barrier(0);              // (in this order: a wait counts the loads behind it)
  }
  uint8_t* const made_scales = made + g.M * (bytes + 16);
  if constexpr (XT >= 0) {                          // four lanes make a block
    const int pieces = g.B * 4;
    for (int r = 0; r < g.M; ++r) {
      const char* const x = t.x + r * t.ldx * (XT == ROW_F32 ? 4 : 2);
      for (int p = tid; p < pieces; p += WAVES * 64) {
        float v[8];
        mx_load8<XT>(x, p * 8, t.K, v);
        const uint32_t s = mx_scale(mx_quad_max(mx_max_bits(v)));
        *(uint32_t*)(made + r * (bytes + 16) + p * 4) = mx_codes(v, s);
        if ((p & 3) == 0) made_scales[r * g.B + (p >> 2)] = (uint8_t)s;
      }
    }
    __syncthreads();
  }
  const int mine = (lane & 15) < g.M ? lane & 15 : 0;       // (a token past the last one is not stored)
  f32x4 acc[NB][TB] = {};
  while (k < bytes) {
    #pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      Piece& p = ring[d];
      #pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (XT >= 0) {                    // (behind the last block the weight's codes are 0)
          const int block = ((k + i * 64) >> 4) + q < g.B ? ((k + i * 64) >> 4) + q : 0;
          p.a[0][i] = *(const i32x4*)(made + mine * (bytes + 16) + block * 16);
          p.sa[0][i] = made_scales[mine * g.B + block];
          // a scale that is NaN must not meet the zeros behind the last block
          if (((k + i * 64) >> 4) + q >= g.B) p.sa[0][i] = 0;
        }
        #pragma unroll
        for (int c = 0; c < NB; ++c)
          #pragma unroll
          for (int b = 0; b < TB; ++b)
            acc[c][b] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide(p.w[c][i]), wide(p.a[b][i]), acc[c][b], 4, 4, 0, p.sw[c][i], 0, p.sa[b][i]);
      }
      load(k + DEPTH * STEP, p);
      k += STEP;
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  #pragma unroll
  for (int c = 0; c < NB; ++c)
    #pragma unroll
    for (int b = 0; b < TB; ++b) *(f32x4*)red[wave][c][b][lane] = acc[c][b];
  __syncthreads();
  // accumulator register r of lane l: channel 4 (l / 16) + r of token l % 16
  for (int o = tid; o < TB * NB * 256; o += WAVES * 64) {
    const int c = o % (16 * NB), cb = c >> 4, cc = c & 15, token = o / (16 * NB), b = token >> 4, tok = token & 15;
    const int64_t nn = n0 + c;
    if (token >= g.M || nn >= g.N) continue;
    float y = 0;
    #pragma unroll
    for (int v = 0; v < WAVES; ++v) y += red[v][cb][b][(cc >> 2) * 16 + tok][cc & 3];
    if (g.bias) y += load_any(g.bias, g.bias_dtype, nn);
    if constexpr (BF == ROW_F32) ((float*)g.y)[token * g.N + nn] = y;
    else store_scalar<BF>(g.y, token * g.N + nn, rnd<BF>(y));
  }
}

int64_t on256(int64_t bytes) { return (bytes + 255) / 256 * 256; }
int64_t on16(int64_t blocks) { return (blocks + 15) / 16 * 16; }

typedef Tile<4, 4, 64, 4> Tile256;
typedef Tile<2, 2, 128, 4> Tile128;

template <class T, int BF>
void launch_tiles(const MxArgs& g, int parts, hipStream_t st) {
  const int64_t tm = (g.M + T::TM - 1) / T::TM, tn = (g.N + T::TN - 1) / T::TN;
  tile_kernel<T, BF><<<dim3((unsigned)((tm * tn * parts + 7) / 8 * 8)), dim3(256), 0, st>>>(g, (int)tm, (int)tn, parts);
}
template <int BF>
void launch_join(const MxArgs& g, const float* sums, int parts, hipStream_t st) {
  const bool four = g.N % 4 == 0 && (uintptr_t)g.y % 16 == 0;      // (four channels of one token)
  const int64_t all = g.M * g.N;
  if (four) join_kernel<BF, 4><<<dim3((unsigned)((all / 4 + 255) / 256)), dim3(256), 0, st>>>(g, sums, parts);
  else join_kernel<BF, 1><<<dim3((unsigned)((all + 255) / 256)), dim3(256), 0, st>>>(g, sums, parts);
}

template <int TB, int NB, int BF, int XT, int WAVES>
void launch_stream(const MxArgs& g, const TokenArgs& t, hipStream_t st) {
  const unsigned lds = XT < 0 ? 0 : (unsigned)(g.M * (g.B * 16 + 16) + g.M * g.B);
  stream_kernel<TB, NB, BF, XT, WAVES><<<dim3((unsigned)((g.N + 16 * NB - 1) / (16 * NB))), dim3(WAVES * 64), lds, st>>>(g, t);
}

template <int BF>
void launch(const MxArgs& g, float* sums, hipStream_t st) {
  const Mxfp4Cut c = mxfp4_cut(g.M, g.N, g.B);
  if (c.stream) {
    if (g.M <= 16) launch_stream<1, 1, BF, -1, 2>(g, TokenArgs{}, st);
    else if (g.M <= 32) launch_stream<2, 1, BF, -1, 2>(g, TokenArgs{}, st);
    else launch_stream<4, 1, BF, -1, 2>(g, TokenArgs{}, st);
  }
  else if (c.parts > 1) {
    MxArgs p = g;
    p.y = sums;
    launch_tiles<Tile128, ROW_SUM>(p, c.parts, st);
    launch_join<BF>(g, sums, c.parts, st);
  }
  else if (c.tile == 0) launch_tiles<Tile256, BF>(g, 1, st);
  else launch_tiles<Tile128, BF>(g, 1, st);
}

bool known(int dtype) { return dtype == LCQ_F32 || dtype == LCQ_BF16 || dtype == LCQ_F16; }

int check(const uint8_t* w, int64_t ldw, const uint8_t* sw, int64_t ldsw, const void* bias, int bias_dtype, int64_t M, int64_t N, int64_t K, const void* y, int dtype) {
  if (!w || !sw || !y || M <= 0 || N <= 0 || K <= 0) return LCQ_EINVAL;
  if (!known(dtype) || (bias && !known(bias_dtype))) return LCQ_EDTYPE;
  // A launch has fewer than 2^32 lanes: tiles of 128 x 128, rounded up to eight; 16 channels of 256 lanes.  Offsets within a tile have 31 bits.
  if (K > 65536 || M > 1 << 28 || N > (1 << 28) - 16 || (M + 127) / 128 * ((N + 127) / 128) > (1 << 24) - 8) return LCQ_ESIZE;
  const int64_t B = (K + 31) / 32;
  if (ldw < 16 * B || ldsw < B) return LCQ_EINVAL;
  if (ldw > 1 << 22 || ldsw > 1 << 22) return LCQ_ESIZE;
  if ((uintptr_t)w % 16 || ldw % 16) return LCQ_EALIGN;
  return LCQ_OK;
}

// tokens whose codes every workgroup of the product makes itself
bool fused(int64_t M, int64_t K) { return M <= 2 && K <= 32768; }

bool on_pieces(const void* p, int64_t ld, int64_t B) { return (uintptr_t)p % 16 == 0 && ld % 16 == 0 && B % 16 == 0; }

}  // namespace

extern "C" {

int64_t lcq_mxfp4_matmul_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0 || K > 65536) return 0;
  const int64_t B = (K + 31) / 32;
  const Mxfp4Cut c = mxfp4_cut(M, N, B);
  return c.stream ? 0 : (c.parts > 1 ? on256(4 * M * N * c.parts) : 0) + (M + N) * on16(B);
}

int lcq_mxfp4_matmul(const uint8_t* a, int64_t lda, const uint8_t* sa, int64_t ldsa, const uint8_t* w, int64_t ldw, const uint8_t* sw, int64_t ldsw,
                     const void* bias, int bias_dtype, int64_t M, int64_t N, int64_t K, void* y, int dtype, void* workspace, void* stream) {
  if (!a || !sa) return LCQ_EINVAL;
  const int bad = check(w, ldw, sw, ldsw, bias, bias_dtype, M, N, K, y, dtype);
  if (bad) return bad;
  const int64_t B = (K + 31) / 32;
  if (lda < 16 * B || ldsa < B) return LCQ_EINVAL;
  if (lda > 1 << 22 || ldsa > 1 << 22) return LCQ_ESIZE;
  if ((uintptr_t)a % 16 || lda % 16) return LCQ_EALIGN;
  hipStream_t st = (hipStream_t)stream;
  MxArgs g = {a, sa, w, sw, bias, y, M, N, lda, ldw, ldsa, ldsw, (int)B, bias_dtype};
  const Mxfp4Cut c = mxfp4_cut(M, N, B);
  if (!c.stream) {
    const bool pads = !on_pieces(sa, ldsa, B) || !on_pieces(sw, ldsw, B);
    if (pads || c.parts > 1) {
      if (!workspace) return LCQ_EWORKSPACE;
      if ((uintptr_t)workspace % 16) return LCQ_EALIGN;
    }
    if (pads) {
      const int Bp = (int)on16(B);
      uint8_t* const to = (uint8_t*)workspace + (c.parts > 1 ? on256(4 * M * N * c.parts) : 0);
      const int64_t words = (M + N) * (Bp / 4);
      pad_scales_kernel<<<dim3((unsigned)((words + 255) / 256)), dim3(256), 0, st>>>(g, Bp, to, words);
      g.sa = to; g.sw = to + M * Bp; g.ldsa = g.ldsw = Bp;
    }
  }
  if (dtype == LCQ_BF16) launch<ROW_BF16>(g, (float*)workspace, st);
  else if (dtype == LCQ_F16) launch<ROW_F16>(g, (float*)workspace, st);
  else launch<ROW_F32>(g, (float*)workspace, st);
  LCQ_CHECK_LAUNCH();
  return LCQ_OK;
}

int64_t lcq_mxfp4_linear_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0 || K > 65536 || fused(M, K)) return 0;
  const int64_t B = (K + 31) / 32;
  return on256(M * B * 16) + on256(M * on16(B)) + lcq_mxfp4_matmul_workspace_bytes(M, N, K);
}

int lcq_mxfp4_linear(const void* x, int x_dtype, int64_t ldx, const uint8_t* w, int64_t ldw, const uint8_t* sw, int64_t ldsw, const void* bias,
                     int bias_dtype, int64_t M, int64_t N, int64_t K, void* y, int dtype, void* workspace, void* stream) {
  if (!x || ldx < 0) return LCQ_EINVAL;
  const int bad = check(w, ldw, sw, ldsw, bias, bias_dtype, M, N, K, y, dtype);
  if (bad) return bad;
  if (!known(x_dtype)) return LCQ_EDTYPE;
  const int64_t B = (K + 31) / 32;
  if (fused(M, K)) {
    const MxArgs g = {nullptr, nullptr, w, sw, bias, y, M, N, 0, ldw, 0, ldsw, (int)B, bias_dtype};
    const TokenArgs t = {(const char*)x, ldx, K};
    hipStream_t st = (hipStream_t)stream;
    const auto run = [&](auto xt) {
      constexpr int XT = decltype(xt)::value;
      if (dtype == LCQ_BF16) launch_stream<1, 1, ROW_BF16, XT, 4>(g, t, st);
      else if (dtype == LCQ_F16) launch_stream<1, 1, ROW_F16, XT, 4>(g, t, st);
      else launch_stream<1, 1, ROW_F32, XT, 4>(g, t, st);
    };
    if (x_dtype == LCQ_BF16) run(Int<ROW_BF16>{});
    else if (x_dtype == LCQ_F16) run(Int<ROW_F16>{});
    else run(Int<ROW_F32>{});
    LCQ_CHECK_LAUNCH();
    return LCQ_OK;
  }
  if (!workspace) return LCQ_EWORKSPACE;
  if ((uintptr_t)workspace % 16) return LCQ_EALIGN;
  uint8_t* const codes = (uint8_t*)workspace;
  uint8_t* const scales = codes + on256(M * B * 16);
  const int rc = lcq_mxfp4_quant(x, x_dtype, M, K, ldx, codes, scales, B, stream);
  if (rc) return rc;
  return lcq_mxfp4_matmul(codes, 16 * B, scales, B, w, ldw, sw, ldsw, bias, bias_dtype, M, N, K, y, dtype, scales + on256(M * on16(B)), stream);
}

}  // extern "C"

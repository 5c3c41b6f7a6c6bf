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
  int64_t nextsa, nextsw;                           // tiles: from 16 scales of a row to the next 16
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
template <class T> __device__ __forceinline__ T from_lds(uint32_t at) { return *(const __attribute__((address_space(3))) T*)(lds_ptr)(size_t)at; }
// (the pipe reads four registers of a 4-bit operand)
__device__ __forceinline__ i32x8 wide(i32x4 v) { return __builtin_shufflevector(v, v, 0, 1, 2, 3, -1, -1, -1, -1); }

// ---- tiles --------------------------------------------------------------------------------------------------------
// A workgroup of four waves (2 x 2) owns 64 FM tokens x 64 FN channels, a wave FM x FN accumulators of 32 x 32.  (Two of 64 x 64 share a CU.)
//  * codes stream through LDS stages of SLAB bytes per row by direct loads; rows past the end of a matrix and bytes past a row's blocks
//    lie outside the buffer that the loads are told and read as zero;
//  * piece p of 16 bytes (a block) of row r lies at p ^ (r / 4 % 4) or p ^ (r / 2 % 8), so that 16 lanes of an operand read touch all 64
//    banks once;
//  * scales come 16 per row, for 512 codes (a period), loaded two periods ahead into one of two places and read by each lane into
//    registers at the end of the period before theirs: a load of four scales per row and stage would fetch a line per row and stage;
//  * operands are buffered in registers: while the products of one step of 64 codes run, the reads of the next are issued between them;
//    one barrier per stage, where every wave holds the rest of it in registers: its place is loaded again from there.
// Tiles of 256 x 256 are bound by the chip's power: 8192 x 14336 x 4096 takes 251 us (3.8 PFLOP/s) with the products at 1.55 GHz, 192 on zeros at 2.35.  A
// round of tiles is 3.4 us of first loads, 25 of products (38 900 clocks, the pipe alone 32 800), 4.5 of outputs.  With nothing loaded behind the first stages the products
// run at 1.68 GHz, without reads of LDS either at 1.92; loading the next tile's first stages before the outputs leave, or whole lines in two stages of 128
// bytes, took as long.  The others are bound by the loads on their way (a round of 224 tiles of 128 x 128 with K = 4096 18 us, 1.7 TB/s of weights from memory, 14.7 from the caches, of 64 x 64
// 10 us, 3 TB/s).
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
    uint32_t v = (blockIdx.x & 7) * each + (blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= each || v >= (uint32_t)total) return;
    part = parts == 1 ? 0 : v / (uint32_t)(tiles_m * tiles_n);
    v -= part * tiles_m * tiles_n;
    const int group = v / (4u * tiles_n), first = group * 4, rows = tiles_m - first < 4 ? tiles_m - first : 4;
    const uint32_t in = v - group * 4 * tiles_n;
    tj = rows == 4 ? in / 4 : rows == 2 ? in / 2 : rows == 1 ? in : in / 3;
    ti = first + in - tj * rows;
  }
  const int64_t m0 = (int64_t)ti * T::TM, n0 = (int64_t)tj * T::TN;
  const int rows_a = (int)(g.M - m0 < T::TM ? g.M - m0 : T::TM), rows_w = (int)(g.N - n0 < T::TN ? g.N - n0 : T::TN);
  const int bytes = g.B * 16, groups = (g.B + 15) >> 4;                      // of a row's codes; 16-byte pieces of its scales
  const int begin = parts == 1 ? 0 : (uint32_t)(groups * part) / (uint32_t)parts, periods = (parts == 1 ? groups : (uint32_t)(groups * (part + 1)) / (uint32_t)parts) - begin;

  const auto buffer = [&](const uint8_t* p, int64_t ld, int rows, int row) {
    const uint64_t at = (uint64_t)(uintptr_t)p;
    const auto one = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
    return i32x4{one((int)(uint32_t)at), one((int)(uint32_t)(at >> 32) & 0xffff), one((int)((rows - 1) * ld + row)), 0x00020000};
  };
  const i32x4 bufA = buffer(g.a + m0 * g.lda, g.lda, rows_a, bytes), bufW = buffer(g.w + n0 * g.ldw, g.ldw, rows_w, bytes);
  const uint8_t *sa = g.sa + m0 * g.ldsa + begin * g.nextsa, *sw = g.sw + n0 * g.ldsw + begin * g.nextsw;       // of the period that is loaded next
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
    gof[p] = r < (p < LA ? rows_a : rows_w) ? (uint32_t)r * (uint32_t)(p < LA ? g.lda : g.ldw) + piece16[p & 1] : OUTSIDE;
  }
  // scale load i of this wave: rows 64 (wave + 4 i) .. + 63 of tokens, then weights (beyond both: a place that nothing reads)
  #pragma unroll
  for (int i = 0; i < SL; ++i) {
    const int r = (wave + 4 * i) * 64 + lane;
    sof[i] = r < T::TM ? (r < rows_a ? (uint32_t)r * (uint32_t)g.ldsa : OUTSIDE) : r - T::TM < rows_w ? (uint32_t)(r - T::TM) * (uint32_t)g.ldsw : OUTSIDE;
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
    const i32x4 bufSA = buffer(sa, g.ldsa, rows_a, 16), bufSW = buffer(sw, g.ldsw, rows_w, 16);
    sa += g.nextsa;
    sw += g.nextsw;
    #pragma unroll
    for (int i = 0; i < SL; ++i) {
      const uint32_t to = lds0 + STAGES * T::STAGE + ((p & 1) * 4 * SL + wave + 4 * i) * 1024;
      const i32x4 buf = (wave + 4 * i) * 64 < T::TM ? bufSA : bufSW;
      asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                   ::"s"(to), "v"(sof[i] | outside), "s"(buf) : "memory");
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
  static_assert(SWITCH >= 1 && STEPS % 2 == 0 && (PRODUCTS >= LOADS / STEPS) && PER <= STAGES && 2 * PER - 1 > STAGES - 2, "stages and periods");
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
  float zero = 0;
  asm volatile("" : "+v"(zero));                    // (not before the loads are on their way)
  #pragma unroll
  for (int j = 0; j < FN; ++j)
    #pragma unroll
    for (int i = 0; i < FM; ++i)
      #pragma unroll
      for (int r = 0; r < 16; ++r) acc[j][i][r] = zero;
  __builtin_amdgcn_sched_barrier(0);
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
  // Outputs that the caches (256 MB) would not keep until they are read go past them: 235 MB with a pass that reads them 346 us, through the caches 354, and what comes
  // next does not wait for them to drain (codes of the next 8192 x 4096 values 18.7 us, 30); 117 MB 180 past, 178 through.
  const bool past = BF != ROW_SUM && g.M * g.N * E > (int64_t)192 << 20;
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
    constexpr int AT_ONCE = Mxfp4Store<FN, E>::TOKENS, TIMES = STEP * 32 / AT_ONCE, SOME = TIMES < 8 ? TIMES : 8;          // tokens of a store, stores, those on their way together
    const int t0 = lane / CHUNKS, ch = lane % CHUNKS, n = wc * FN * 32 + ch * CH;
    char* const to = (char*)g.y + ((m0 + wr * FM * 32 + i0 * 32) * g.N + n0 + (BF == ROW_SUM ? part * g.M * g.N : 0)) * E;
    if (rows_a == T::TM && rows_w == T::TN) {       // (uniform, as most tiles of a large product are: no comparison, no address but a scalar one)
      const auto of = (typename Mxfp4Store<FN, E>::Offset)((t0 * g.N + n) * E);
      #pragma unroll
      for (int o0 = 0; o0 < TIMES; o0 += SOME) {
        u32x4 v[SOME];
        #pragma unroll
        for (int o = 0; o < SOME; ++o) v[o] = *(const u32x4*)(mine + ((o0 + o) * AT_ONCE + t0) * ROW + turned(ch, ((o0 + o) * AT_ONCE + t0) % 32) * 16);
        if (past) {
          #pragma unroll
          for (int o = 0; o < SOME; ++o) mx_store_past(to + (int64_t)(o0 + o) * AT_ONCE * g.N * E + of, v[o]);
        } else {
          #pragma unroll
          for (int o = 0; o < SOME; ++o) *(u32x4_anywhere*)(to + (int64_t)(o0 + o) * AT_ONCE * g.N * E + of) = v[o];
        }
      }
    } else {
      #pragma unroll 1
      for (int o0 = 0; o0 < TIMES; o0 += SOME) {
        u32x4 v[SOME];
        #pragma unroll
        for (int o = 0; o < SOME; ++o) v[o] = *(const u32x4*)(mine + ((o0 + o) * AT_ONCE + t0) * ROW + turned(ch, ((o0 + o) * AT_ONCE + t0) % 32) * 16);
        #pragma unroll
        for (int o = 0; o < SOME; ++o) {
          const int tt = (o0 + o) * AT_ONCE + t0, m = wr * FM * 32 + i0 * 32 + tt;
          if (m >= rows_a || n >= rows_w) continue;
          char* const cell = to + ((int64_t)tt * g.N + n) * E;
          if (n + CH <= rows_w) {
            __builtin_memcpy(cell, &v[o], 16);
          } else {
            #pragma unroll
            for (int e = 0; e < CH; ++e)
              if (n + e < rows_w) {
                if constexpr (E == 4) ((uint32_t*)cell)[e] = v[o][e];
                else ((uint16_t*)cell)[e] = (uint16_t)(v[o][e / 2] >> 16 * (e % 2));
              }
          }
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

// Scales for tiles: [16 scales of a row][row][16], with zeros behind a row's last, those of a and then those of w.  A tile's loads of them are then whole
// lines; in the rows' own order each of 64 lanes reads 16 bytes of a line of its own, again in every tile of its stripe (8192 x 14336 x 4096: 285 us, with
// this kernel's 4 276).  Tiles of 128 x 128 gain nothing by it: 1024 x 4096 x 4096 16.2 us, 18.4 with it.
__global__ __launch_bounds__(256) void order_scales_kernel(MxArgs g, int groups, uint8_t* __restrict__ out) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, of_a = g.M * groups;
  if (i >= of_a + g.N * groups) return;
  const bool a = i < of_a;
  const int64_t rows = a ? g.M : g.N, j = a ? i : i - of_a, group = j / rows, r = j - group * rows, ld = a ? g.ldsa : g.ldsw;
  const uint8_t* const from = (a ? g.sa : g.sw) + r * ld + group * 16;
  u32x4 v = {};
  if ((uintptr_t)from % 16 == 0 && group * 16 + 16 <= g.B) {
    v = *(const u32x4*)from;
  } else {
    #pragma unroll
    for (int e = 0; e < 16; ++e) v[e / 4] |= (group * 16 + e < g.B ? (uint32_t)from[e] : 0u) << 8 * (e % 4);
  }
  *(u32x4*)(out + i * 16) = v;
}

// ---- few tokens ---------------------------------------------------------------------------------------------------
// The weight streams past the tokens.  A wave has a block of 16 channels and a KS-th of K; stages of 256 codes go through its own part of LDS by
// direct loads of whole lines, DEPTH - 1 stages ahead, without a break from one block to the next, and nothing but the joining of a
// block's KS waves makes waves wait for one another.  16 tokens by 4096 x 14336 take 9.7 us (3.2 TB/s of weights; 3.4 are the launch and the first loads).
// Loaded straight into the matrix pipe's layout, 16 neighbouring lanes are 16 rows and every KB passes the cache 64 times: 16.5 us.
//   codes of the weight and of the tokens   16 rows x 128 bytes; 16-byte piece p of row r lies at p ^ (r / 2 % 8)
//   scales   the word-aligned 64 bytes of a row that hold those of eight stages, or of seven where rows are off words
// Where there are few tokens, every workgroup makes their codes itself, in LDS, while its first weights are on their way.
constexpr int STAGE_BYTES = 128;                    // of a row
constexpr int MOST_BIASES = 64;                     // blocks of channels of a workgroup whose biases are read before the stream begins

struct TokenArgs {
  const char* x;
  int64_t ldx, K;
};

template <int TB, int XT, int DEPTH_, int PLACES_>
struct Few {
  static constexpr int DEPTH = DEPTH_, PLACES = PLACES_, OWN = XT < 0 ? TB : 0;              // blocks of tokens that are loaded
  static constexpr int BYTES = 2048 * (1 + OWN), SCALES = 1024 * (1 + OWN), LOADS = 2 * (1 + OWN);           // of a stage, a period, a stage's loads
  static constexpr int WAVE = DEPTH * BYTES + PLACES * SCALES;
  static constexpr int RED = 4 * WAVE, BIAS = RED + 2 * 4 * TB * 1024, MADE = BIAS + MOST_BIASES * 64;
};

// A unit of work: 4 / KS blocks of channels and a group of 16 TB tokens, the groups of the same channels one behind the other.  Workgroup b runs on
// XCD b % 8: every XCD takes neighbouring units, and the weights that they share from its L2.  XT: the type of the tokens' values, or -1 for codes.
template <int TB, int BF, int XT, int DEPTH, int PLACES>
__global__ __launch_bounds__(256) void few_kernel(MxArgs g, TokenArgs t, int KS) {
  typedef Few<TB, XT, DEPTH, PLACES> S;
  constexpr int OWN = S::OWN;
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const int tid = threadIdx.x, lane = tid & 63, q = lane >> 4, c = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), part = wave % KS, of_group = wave / KS, groups = 4 / KS;        // blocks at a time
  const int stages = (g.B + 7) >> 3, first = stages * part / KS, last = stages * (part + 1) / KS;
  const int blocks = (int)((g.N + 15) >> 4), rounds = (blocks + groups - 1) / groups;
  const int first_unit = gridDim.x % 8 == 0 ? (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3) : blockIdx.x;          // and every gridDim.x-th from there
  const int teams = XT < 0 ? (int)((g.M + 16 * TB - 1) / (16 * TB)) : 1;     // of tokens
  struct Unit { int round, team; };
  const auto next = [&](Unit u) {
    u.team += gridDim.x % teams;
    u.round += gridDim.x / teams + (u.team >= teams);
    u.team -= u.team >= teams ? teams : 0;
    return u;
  };
  const Unit start = {first_unit / teams, first_unit % teams};
  const bool ragged = g.B % 8 != 0;
  const auto one = [](uint32_t v) { return (int)__builtin_amdgcn_readfirstlane((int)v); };
  const auto buffer = [&](const void* p, int64_t size) {
    const uint64_t at = (uint64_t)(uintptr_t)p;
    return i32x4{one((uint32_t)at), one((uint32_t)(at >> 32) & 0xffff), one((uint32_t)size), 0x00020000};
  };
  const auto load = [&](uint32_t to, uint32_t of, i32x4 buf, int at) {       // (all but `of` are the wave's)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(one(to)), "v"(of), "s"(buf), "s"(one((uint32_t)at)) : "memory");
  };
  // What is read once does not wait for places in the caches and leaves what others have there: 1 token by
  // 4096 x 14336 9.1 us so, 8.8 past them, 32000 x 4096 15.3 and 14.7.
  const auto weights = [&](uint32_t to, uint32_t of, i32x4 buf, int at) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen nt lds" ::"s"(one(to)), "v"(of), "s"(buf), "s"(one((uint32_t)at)) : "memory");
  };
  constexpr uint32_t OUTSIDE = 0x80000000u;
  const uint32_t lds0 = (uint32_t)(size_t)(lds_ptr)lds, mine = lds0 + wave * S::WAVE;

  // biases of the first blocks (loads that the compiler knows of would end the stream where they are waited for)
  float* const biases = (float*)(lds + S::BIAS);
  if (g.bias) {
    for (int i = tid; i < MOST_BIASES * 16; i += 256) {
      const int64_t n = ((first_unit + (int64_t)((i >> 4) / groups) * gridDim.x) / teams * groups + (i >> 4) % groups) * 16 + (i & 15);
      if (n < g.N) biases[i] = load_any(g.bias, g.bias_dtype, n);
    }
  }

  // ---- loads ----
  const int piece = (lane & 7) ^ (lane >> 4 & 3);   // of 16 bytes in a row of codes; in odd loads 4 more, as 8 rows turn it
  uint32_t wof[2], sof, aof[OWN ? OWN : 1][2], saof[OWN ? OWN : 1];
  i32x4 bufW, bufS, bufA, bufSA;
  const int period = ((uintptr_t)g.sw | (uintptr_t)g.ldsw | (uintptr_t)g.sa | (uintptr_t)g.ldsa) & 3 ? 7 : 8;
  Unit lunit = start;
  int lk = first, lperiod = 0, lplace = PLACES - 1;
  const auto enter = [&]() {
    const int64_t n0 = ((int64_t)lunit.round * groups + of_group) * 16;
    const int rows = n0 >= g.N ? 0 : g.N - n0 < 16 ? (int)(g.N - n0) : 16;
    bufW = buffer(g.w + n0 * g.ldw, rows ? (rows - 1) * g.ldw + g.B * 16 : 0);
    const uint8_t* const s = g.sw + n0 * g.ldsw;
    const int early = (int)((uintptr_t)s & 3);
    bufS = buffer(s - early, rows ? (early + (rows - 1) * g.ldsw + g.B + 3) & ~(int64_t)3 : 0);
    #pragma unroll
    for (int l = 0; l < 2; ++l) wof[l] = l * 8 + (lane >> 3) < rows ? (uint32_t)((l * 8 + (lane >> 3)) * g.ldw) + ((piece ^ l * 4) << 4) : OUTSIDE;
    sof = lane >> 2 < rows ? ((uint32_t)(early + (lane >> 2) * g.ldsw) & ~3u) + (lane & 3) * 16 : OUTSIDE;
    if constexpr (OWN > 0) {
      const int64_t m0 = (int64_t)lunit.team * 16 * TB;
      const int tokens = g.M - m0 < 16 * TB ? (int)(g.M - m0) : 16 * TB;
      const uint8_t* const sa = g.sa + m0 * g.ldsa;
      const int early_a = (int)((uintptr_t)sa & 3);
      bufA = buffer(g.a + m0 * g.lda, (tokens - 1) * g.lda + g.B * 16);
      bufSA = buffer(sa - early_a, (early_a + (tokens - 1) * g.ldsa + g.B + 3) & ~(int64_t)3);
      #pragma unroll
      for (int b = 0; b < OWN; ++b) {
        #pragma unroll
        for (int l = 0; l < 2; ++l) {
          const int r = b * 16 + l * 8 + (lane >> 3);
          aof[b][l] = r < tokens ? (uint32_t)r * (uint32_t)g.lda + ((piece ^ l * 4) << 4) : OUTSIDE;
        }
        const int r = b * 16 + (lane >> 2);
        saof[b] = r < tokens ? ((uint32_t)early_a + (uint32_t)r * (uint32_t)g.ldsa & ~3u) + (lane & 3) * 16 : OUTSIDE;
      }
    }
  };
  // The next stage, into a place; behind the last one: nothing, from outside.  The scales of a period come in front of its first stage.
  const auto fetch = [&](int slot) {
    const uint32_t to = mine + slot * S::BYTES;
    const bool over = lunit.round >= rounds;
    if (lperiod == 0) {
      lplace = lplace == PLACES - 1 ? 0 : lplace + 1;
      const uint32_t too = mine + DEPTH * S::BYTES + lplace * S::SCALES;
      load(too, over ? OUTSIDE : sof, bufS, lk * 8);
      #pragma unroll
      for (int b = 0; b < OWN; ++b) load(too + 1024 * (1 + b), over ? OUTSIDE : saof[b], bufSA, lk * 8);
      lperiod = period;
    }
    --lperiod;
    if (over || (ragged && lk == stages - 1)) {
      const int left = over ? 0 : g.B - lk * 8;     // blocks
      #pragma unroll
      for (int l = 0; l < 2; ++l) {
        const bool in = (piece ^ l * 4) < left;
        weights(to + l * 1024, in ? wof[l] : OUTSIDE, bufW, lk * STAGE_BYTES);
        #pragma unroll
        for (int b = 0; b < OWN; ++b) load(to + 2048 * (1 + b) + l * 1024, in ? aof[b][l] : OUTSIDE, bufA, lk * STAGE_BYTES);
      }
    } else {
      #pragma unroll
      for (int l = 0; l < 2; ++l) {
        weights(to + l * 1024, wof[l], bufW, lk * STAGE_BYTES);
        #pragma unroll
        for (int b = 0; b < OWN; ++b) load(to + 2048 * (1 + b) + l * 1024, aof[b][l], bufA, lk * STAGE_BYTES);
      }
    }
    if (++lk >= last && !over) {
      lk = first;
      lunit = next(lunit);
      lperiod = 0;
      if (lunit.round < rounds) enter();
    }
  };
  const bool works = first < last;                  // (K may have fewer stages than waves)
  if (works) {
    enter();
    #pragma unroll
    for (int d = 0; d < DEPTH - 1; ++d) fetch(d);
  }
  uint8_t* const made = (uint8_t*)lds + S::MADE;    // XT >= 0: [M] rows of codes, 16 B + 16 apart, then of scales
  const int bytes = g.B * 16;
  uint8_t* const made_scales = made + g.M * (bytes + 16);
  if constexpr (XT >= 0) {                          // four lanes make a block
    const uint32_t pieces = g.B * 4, all = (uint32_t)g.M * pieces;
    constexpr int AT_ONCE = 4;                      // (a loop of single loads waits for memory every time)
    for (uint32_t i0 = tid; i0 < all; i0 += AT_ONCE * 256) {
      float v[AT_ONCE][8];
      #pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) {
        const uint32_t i = i0 + j * 256, r = i / pieces, p = i - r * pieces;
        if (i < all) mx_load8<XT>(t.x + r * t.ldx * (XT == ROW_F32 ? 4 : 2), p * 8, t.K, v[j]);
      }
      #pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) {
        const uint32_t i = i0 + j * 256, r = i / pieces, p = i - r * pieces;
        if (i >= all) break;                        // (four neighbouring lanes together)
        const uint32_t s = mx_scale(mx_quad_max(mx_max_bits(v[j])));
        *(uint32_t*)(made + r * (bytes + 16) + p * 4) = mx_codes(v[j], s);
        if ((p & 3) == 0) made_scales[r * g.B + (p >> 2)] = (uint8_t)s;
      }
    }
  }
  __syncthreads();

  // ---- products ----
  uint32_t at[2], mat = 0, msat = 0;
  #pragma unroll
  for (int i = 0; i < 2; ++i) at[i] = mine + c * 128 + (((i * 4 + q) ^ (c >> 1 & 7)) << 4);
  if constexpr (XT >= 0) {
    const int row = c < g.M ? c : 0;                // (a token past the last one is not stored)
    mat = lds0 + S::MADE + row * (bytes + 16);
    msat = lds0 + S::MADE + (uint32_t)g.M * (bytes + 16) + row * g.B;
  }
  int slot = 0, cperiod = 0, cplace = 0, turn = 0;
  Unit unit = start;
  for (int nth = 0; unit.round < rounds; unit = next(unit), ++nth) {
    const int64_t n0 = ((int64_t)unit.round * groups + of_group) * 16, m0 = (int64_t)unit.team * 16 * TB;
    uint32_t sat[OWN ? OWN : 1];
    #pragma unroll
    for (int b = 0; b < OWN; ++b)
      sat[b] = mine + DEPTH * S::BYTES + 1024 * (1 + b) + c * 64 + q + (((uint32_t)(uintptr_t)g.sa + (uint32_t)(m0 + b * 16 + c) * (uint32_t)g.ldsa) & 3);
    const uint32_t sw = mine + DEPTH * S::BYTES + c * 64 + q + (((uint32_t)(uintptr_t)g.sw + (uint32_t)(n0 + c) * (uint32_t)g.ldsw) & 3);
    f32x4 acc[TB] = {};
    for (int k = first; k < last; ++k) {
      // the stage has landed, and what this wave reads of the last one
      __builtin_amdgcn_s_waitcnt(0x0070 | ((DEPTH - 2) * S::LOADS & 15) | (DEPTH - 2) * S::LOADS >> 4 << 14);
      asm volatile("" ::: "memory");
      fetch(slot == 0 ? DEPTH - 1 : slot - 1);
      const uint32_t here = slot * S::BYTES, scales_here = cplace * S::SCALES + cperiod * 8;
      const int left = g.B - k * 8;
      i32x4 w[2], a[TB][2];
      uint32_t s[2], sa[TB][2];
      #pragma unroll
      for (int i = 0; i < 2; ++i) {
        w[i] = from_lds<i32x4>(at[i] + here);
        s[i] = from_lds<uint8_t>(sw + scales_here + i * 4);
        if constexpr (XT >= 0) {                    // (behind the last block the weight's codes are 0, and the scales here made to be)
          const int block = k * 8 + i * 4 + q < g.B ? k * 8 + i * 4 + q : g.B - 1;
          a[0][i] = from_lds<i32x4>(mat + block * 16);
          sa[0][i] = from_lds<uint8_t>(msat + block);
        } else {
          #pragma unroll
          for (int b = 0; b < TB; ++b) {
            a[b][i] = from_lds<i32x4>(at[i] + here + 2048 * (1 + b));
            sa[b][i] = from_lds<uint8_t>(sat[b] + scales_here + i * 4);
          }
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      #pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t there = i * 4 + q < left ? 255u : 0u;                 // (behind the last block: not a NaN)
        #pragma unroll
        for (int b = 0; b < TB; ++b)
          acc[b] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide(w[i]), wide(a[b][i]), acc[b], 4, 4, 0, (int)(s[i] & there), 0, (int)(sa[b][i] & there));
      }
      slot = slot == DEPTH - 1 ? 0 : slot + 1;
      cperiod = cperiod == period - 1 ? 0 : cperiod + 1;
      if (cperiod == 0) cplace = cplace == PLACES - 1 ? 0 : cplace + 1;
    }
    if (cperiod) cplace = cplace == PLACES - 1 ? 0 : cplace + 1;             // (a block starts a period)
    cperiod = 0;
    // accumulator register r of lane l: channel 4 (l / 16) + r of token l % 16
    f32x4* const red = (f32x4*)(lds + S::RED) + turn * 4 * TB * 64;
    turn ^= 1;                                      // (what is read here is written again behind the next barrier but one)
    #pragma unroll
    for (int b = 0; b < TB; ++b) red[(wave * TB + b) * 64 + lane] = acc[b];
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    for (int o = tid; o < groups * TB * 64; o += 256) {      // four channels of a token
      const int four = o & 3, tok = o >> 2 & 15, b = (o >> 6) % TB, group = (o >> 6) / TB, block = nth * groups + group;
      const int64_t n = ((int64_t)unit.round * groups + group) * 16 + four * 4, token = m0 + b * 16 + tok;
      if (token >= g.M || n >= g.N) continue;
      const int left = g.N - n < 4 ? (int)(g.N - n) : 4;
      f32x4 y = {};
      for (int p = 0; p < KS; ++p) y += red[((group * KS + p) * TB + b) * 64 + four * 16 + tok];
      if (g.bias) {
        if (block < MOST_BIASES) y += *(const f32x4*)&biases[block * 16 + four * 4];           // (behind the last channel: anything)
        else
          #pragma unroll
          for (int r = 0; r < 4; ++r) if (r < left) y[r] += load_any(g.bias, g.bias_dtype, n + r);
      }
      const int64_t cell = token * g.N + n;         // (rows may start anywhere)
      if constexpr (BF == ROW_F32) {
        if (left == 4) __builtin_memcpy((float*)g.y + cell, &y, 16);
        else
          #pragma unroll
          for (int r = 0; r < 3; ++r) if (r < left) ((float*)g.y)[cell + r] = y[r];
      } else {
        const u32x2 v = BF == ROW_BF16 ? u32x2{bf16_pack_rne(y[0], y[1]), bf16_pack_rne(y[2], y[3])} : u32x2{f16_pack_rne(y[0], y[1]), f16_pack_rne(y[2], y[3])};
        if (left == 4) __builtin_memcpy((uint16_t*)g.y + cell, &v, 8);
        else
          #pragma unroll
          for (int r = 0; r < 3; ++r) if (r < left) ((uint16_t*)g.y)[cell + r] = (uint16_t)(v[r / 2] >> 16 * (r % 2));
      }
    }
  }
  __builtin_amdgcn_s_waitcnt(0x0f70);               // nothing may still be on its way to LDS when the workgroup leaves it
}

int64_t on256(int64_t bytes) { return (bytes + 255) / 256 * 256; }
int64_t on16(int64_t blocks) { return (blocks + 15) / 16 * 16; }

typedef Tile<4, 4, 64, 4> Tile256;
typedef Tile<2, 2, 128, 4> Tile128;
typedef Tile<1, 1, 128, 4> Tile64;

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

template <int TB, int BF, int XT, int DEPTH, int PLACES>
int launch_few(const MxArgs& g, const TokenArgs& t, int KS, hipStream_t st) {
  typedef Few<TB, XT, DEPTH, PLACES> S;
  const auto kernel = few_kernel<TB, BF, XT, DEPTH, PLACES>;
  const int lds = S::MADE + (XT < 0 ? 0 : (int)(g.M * (g.B * 16 + 16) + g.M * g.B));
  if (hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess) return LCQ_ELAUNCH;
  const int64_t units = mxfp4_units(g.M, g.N, KS), most = 256 * (163840 / lds);
  kernel<<<dim3((unsigned)(units < most ? units : most)), dim3(256), lds, st>>>(g, t, KS);
  return LCQ_OK;
}
// Scales of seven stages on their way are those of three periods at most if every period but a unit's last has seven or eight stages, and a unit four;
// with fewer, those of five stages are of five.
template <int TB, int BF, int XT>
int launch_few(const MxArgs& g, const TokenArgs& t, hipStream_t st) {
  const int KS = mxfp4_waves(g.M, g.N, g.B);
  const bool four = ((g.B + 7) / 8) / KS >= 4;
  if constexpr (TB == 2) return four ? launch_few<2, BF, XT, 4, 3>(g, t, KS, st) : launch_few<2, BF, XT, 3, 3>(g, t, KS, st);
  else return four ? launch_few<1, BF, XT, 7, 3>(g, t, KS, st) : launch_few<1, BF, XT, 5, 5>(g, t, KS, st);
}

template <int BF>
int launch(const MxArgs& g, float* sums, hipStream_t st) {
  const Mxfp4Cut c = mxfp4_cut(g.M, g.N, g.B);
  if (c.stream) return g.M <= 16 ? launch_few<1, BF, -1>(g, TokenArgs{}, st) : launch_few<2, BF, -1>(g, TokenArgs{}, st);
  if (c.parts > 1) {
    MxArgs p = g;
    p.y = sums;
    if (c.tile == 2) launch_tiles<Tile64, ROW_SUM>(p, c.parts, st);
    else launch_tiles<Tile128, ROW_SUM>(p, c.parts, st);
    launch_join<BF>(g, sums, c.parts, st);
  }
  else if (c.tile == 0) launch_tiles<Tile256, BF>(g, 1, st);
  else if (c.tile == 2) launch_tiles<Tile64, BF>(g, 1, st);
  else launch_tiles<Tile128, BF>(g, 1, st);
  return LCQ_OK;
}

bool known(int dtype) { return dtype == LCQ_F32 || dtype == LCQ_BF16 || dtype == LCQ_F16; }

int check(const uint8_t* w, int64_t ldw, const uint8_t* sw, int64_t ldsw, const void* bias, int bias_dtype, int64_t M, int64_t N, int64_t K, const void* y, int dtype) {
  if (!w || !sw || !y || M <= 0 || N <= 0 || K <= 0) return LCQ_EINVAL;
  if (!known(dtype) || (bias && !known(bias_dtype))) return LCQ_EDTYPE;
  // A launch has fewer than 2^32 lanes: tiles of 128 x 128, rounded up to eight; 16 channels of 256 lanes.  Offsets within a tile have 31 bits.
  if (K > 65536 || M > 1 << 28 || N > MXFP4_MOST_N || (M + 127) / 128 * ((N + 127) / 128) > (1 << 24) - 8) return LCQ_ESIZE;
  const int64_t B = (K + 31) / 32;
  if (ldw < 16 * B || ldsw < B) return LCQ_EINVAL;
  if (ldw > 1 << 22 || ldsw > 1 << 22) return LCQ_ESIZE;
  if ((uintptr_t)w % 16 || ldw % 16) return LCQ_EALIGN;
  return LCQ_OK;
}

// Tokens whose codes every workgroup of the product makes itself, instead of a kernel of their own in front: that is 2.2 us, and 4 of the host's; 4096 values by 256 lanes are
// 0.7 and off 16 bytes 1.0 (fused / not, us, N x K: 4096 x 4096 1 token 6.3 / 8.1, 4 tokens 8.4 / 8.3, 6 tokens 9.9 / 8.4; 1024 x 1024 16 tokens 6.7 / 6.3;
// 1001 x 2047 3 tokens 6.7 / 6.9, 4 tokens 7.6 / 6.9).
bool fused(int64_t M, int64_t K) { return M <= 16 && M * K <= (K % 8 ? 8192 : 16384); }

// Are scales put in order in front of the tiles?
bool orders(const Mxfp4Cut& c, bool aligned, int64_t B) { return c.tile == 0 || !aligned || B % 16; }

}  // namespace

extern "C" {

int64_t lcq_mxfp4_matmul_workspace_bytes(int64_t M, int64_t N, int64_t K, int aligned) {
  if (M <= 0 || N <= 0 || K <= 0 || K > 65536) return 0;
  const int64_t B = (K + 31) / 32;
  const Mxfp4Cut c = mxfp4_cut(M, N, B);
  if (c.stream) return 0;
  return (c.parts > 1 ? on256(4 * M * N * c.parts) : 0) + (orders(c, aligned, B) ? (M + N) * on16(B) : 0);
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
  MxArgs g = {a, sa, w, sw, bias, y, M, N, lda, ldw, ldsa, ldsw, 0, 0, (int)B, bias_dtype};
  const Mxfp4Cut c = mxfp4_cut(M, N, B);
  if (!c.stream) {
    const bool ordered = orders(c, ((uintptr_t)sa | (uintptr_t)sw | (uintptr_t)ldsa | (uintptr_t)ldsw) % 16 == 0, B);
    if (ordered || c.parts > 1) {
      if (!workspace) return LCQ_EWORKSPACE;
      if ((uintptr_t)workspace % 16) return LCQ_EALIGN;
    }
    g.nextsa = g.nextsw = 16;
    if (ordered) {
      const int groups = (int)((B + 15) / 16);
      uint8_t* const to = (uint8_t*)workspace + (c.parts > 1 ? on256(4 * M * N * c.parts) : 0);
      order_scales_kernel<<<dim3((unsigned)(((M + N) * groups + 255) / 256)), dim3(256), 0, st>>>(g, groups, to);
      g.sa = to; g.sw = to + M * groups * 16; g.ldsa = g.ldsw = 16; g.nextsa = M * 16; g.nextsw = N * 16;
    }
  }
  float* const sums = (float*)workspace;
  const int rc = dtype == LCQ_BF16 ? launch<ROW_BF16>(g, sums, st) : dtype == LCQ_F16 ? launch<ROW_F16>(g, sums, st) : launch<ROW_F32>(g, sums, st);
  if (rc) return rc;
  LCQ_CHECK_LAUNCH();
  return LCQ_OK;
}

int64_t lcq_mxfp4_linear_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0 || K > 65536 || fused(M, K)) return 0;
  const int64_t B = (K + 31) / 32;
  return on256(M * B * 16) + on256(M * on16(B)) + lcq_mxfp4_matmul_workspace_bytes(M, N, K, 0);
}

int lcq_mxfp4_linear(const void* x, int x_dtype, int64_t ldx, const uint8_t* w, int64_t ldw, const uint8_t* sw, int64_t ldsw, const void* bias,
                     int bias_dtype, int64_t M, int64_t N, int64_t K, void* y, int dtype, void* workspace, void* stream) {
  if (!x || ldx < 0) return LCQ_EINVAL;
  const int bad = check(w, ldw, sw, ldsw, bias, bias_dtype, M, N, K, y, dtype);
  if (bad) return bad;
  if (!known(x_dtype)) return LCQ_EDTYPE;
  const int64_t B = (K + 31) / 32;
  if (fused(M, K)) {
    const MxArgs g = {nullptr, nullptr, w, sw, bias, y, M, N, 0, ldw, 0, ldsw, 0, 0, (int)B, bias_dtype};
    const TokenArgs t = {(const char*)x, ldx, K};
    hipStream_t st = (hipStream_t)stream;
    const auto run = [&](auto xt) {
      constexpr int XT = decltype(xt)::value;
      return dtype == LCQ_BF16 ? launch_few<1, ROW_BF16, XT>(g, t, st) : dtype == LCQ_F16 ? launch_few<1, ROW_F16, XT>(g, t, st) : launch_few<1, ROW_F32, XT>(g, t, st);
    };
    const int rc = x_dtype == LCQ_BF16 ? run(Int<ROW_BF16>{}) : x_dtype == LCQ_F16 ? run(Int<ROW_F16>{}) : run(Int<ROW_F32>{});
    if (rc) return rc;
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

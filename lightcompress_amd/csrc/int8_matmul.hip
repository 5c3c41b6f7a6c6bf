// Product of int8 codes with a scale for each token and each channel:
//   y[m, n] = as[m] ws[n] (sum_k a[m, k] w[n, k] - az[m] sum_k w[n, k]) + bias[n]
// The sums are exact in 32-bit integers for K <= 65536 (|a - az| <= 255, |w| <= 128: 255 * 128 * 65536 < 2^31), so results do not
// depend on how the work is cut.
//
// Both operands are read along K, as the matrix pipe takes them: a lane of v_mfma_i32_32x32x32_i8 holds 16 codes of one row.
// The weight is the first operand, so an accumulator's four neighbouring registers are four neighbouring channels of one token.
#include "rowquant.h"
#include "token_codes.h"
#include <type_traits>

namespace {
using namespace lcq;

typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((ext_vector_type(16))) int i32x16;
typedef __attribute__((address_space(3))) char* lds_ptr;
typedef __attribute__((address_space(3))) i32x4* lds_frag;

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
// the four byte sums of a register added to `sum`
__device__ __forceinline__ int add_bytes(const i32x4& v, int sum) {
  #pragma unroll
  for (int q = 0; q < 4; ++q) sum = __builtin_amdgcn_sdot4(v[q], 0x01010101, sum, false);
  return sum;
}

// ---- tiles --------------------------------------------------------------------------------------------------------
// A workgroup of four waves (2 x 2) owns 64 FM tokens x 64 FN channels, a wave FM x FN accumulators of 32 x 32.
//  * K streams through four LDS stages of 64 codes per row by direct loads; rows past the end of a matrix and codes past K lie outside the
//    buffer that the loads are told and read as zero;
//  * a row of a stage is 64 bytes, 16 bytes per lane of a load; piece p of row r lies at p ^ (r / 4 % 4), so that the 16 lanes of an
//    operand read touch all 64 banks once;
//  * operands are double-buffered in registers: while the products of one 32-code step run, the reads of the next are issued between
//    them, and the direct loads of the stage three ahead are spread over them; one barrier per stage, at its middle, where every wave holds
//    the rest of it in registers.
constexpr int STAGES = 4, SLAB = 64;

template <int FM, int FN>
struct Tile {
  static constexpr int TM = 64 * FM, TN = 64 * FN;
  static constexpr int STAGE = (TM + TN) * SLAB;
};

template <int FM, int FN, int BF, bool ASYM>
__global__ __launch_bounds__(256, 1) void tile_kernel(MatmulArgs g, int tiles_m, int tiles_n) {
  typedef Tile<FM, FN> T;
  __shared__ __attribute__((aligned(1024))) char lds[STAGES * T::STAGE];
  __shared__ __attribute__((aligned(16))) float channel[2][T::TN];           // scales, biases
  __shared__ __attribute__((aligned(16))) int sums[ASYM ? T::TN : 4];        // sums of the weight's rows
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wr = wave >> 1, wc = wave & 1;          // tokens, channels

  // Workgroup b runs on XCD b % 8: every XCD takes a contiguous range of an order in which 32 consecutive tiles are 4 x 8, so the
  // tiles that share an L2 at one time share a handful of stripes.
  int ti, tj;
  {
    const int total = tiles_m * tiles_n, each = (total + 7) >> 3;
    const int v = ((int)blockIdx.x & 7) * each + ((int)blockIdx.x >> 3);
    if (((int)blockIdx.x >> 3) >= each || v >= total) return;
    const int group = v / (4 * tiles_n), first = group * 4, rows = tiles_m - first < 4 ? tiles_m - first : 4;
    const int in = v - group * 4 * tiles_n;
    tj = in / rows;
    ti = first + in - tj * rows;
  }
  const int64_t m0 = (int64_t)ti * T::TM, n0 = (int64_t)tj * T::TN;
  const int rows_a = (int)(g.M - m0 < T::TM ? g.M - m0 : T::TM), rows_w = (int)(g.N - n0 < T::TN ? g.N - n0 : T::TN);
  const int steps = (g.K + SLAB - 1) / SLAB;

  const auto buffer = [&](const int8_t* p, int64_t ld, int rows) {
    const uint64_t at = (uint64_t)(uintptr_t)p;
    return i32x4{(int)(uint32_t)at, (int)(uint32_t)(at >> 32) & 0xffff, (int)((rows - 1) * ld + g.K), 0x00020000};
  };
  const i32x4 bufA = buffer(g.a + m0 * g.lda, g.lda, rows_a), bufW = buffer(g.w + n0 * g.ldw, g.ldw, rows_w);
  constexpr uint32_t OUTSIDE = 0x80000000u;
  constexpr int LA = T::TM / 64, LW = T::TN / 64;   // a wave's loads of tokens and of weights per stage
  const int piece16 = ((lane & 3) ^ ((lane >> 4) & 3)) * 16;                 // this lane's 16 bytes of a row of 64
  uint32_t gof[LA + LW];
  #pragma unroll
  for (int p = 0; p < LA + LW; ++p) {
    const int r = (wave * (p < LA ? LA : LW) + (p < LA ? p : p - LA)) * 16 + (lane >> 2);
    gof[p] = r < (p < LA ? rows_a : rows_w) ? (uint32_t)(r * (p < LA ? g.lda : g.ldw) + piece16) : OUTSIDE;
  }
  const uint32_t lds0 = (uint32_t)(size_t)(lds_ptr)lds;
  // load p of the stage at LDS address dst, codes [at, at + 64) of K
  const auto gload = [&](uint32_t dst, int at, uint32_t outside, int p) {
    const uint32_t to = dst + (p < LA ? (wave * LA + p) * 1024 : T::TM * SLAB + (wave * LW + p - LA) * 1024);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                 ::"s"(to), "v"(gof[p] | outside), "s"(p < LA ? bufA : bufW), "s"(at) : "memory");
  };
  const auto outside_at = [&](int at) { return piece16 < g.K - at ? 0u : OUTSIDE; };

  const int slot = (lane >> 5) ^ ((lane >> 2) & 3);
  const lds_ptr readA = (lds_ptr)lds + (wr * FM * 32 + (lane & 31)) * SLAB + slot * 16;
  const lds_ptr readW = (lds_ptr)lds + T::TM * SLAB + (wc * FN * 32 + (lane & 31)) * SLAB + slot * 16;
  const int second = ((slot ^ 2) - slot) * 16;      // from the first 32 codes of a stage to the others
  i32x16 acc[FN][FM];
  #pragma unroll
  for (int j = 0; j < FN; ++j)
    #pragma unroll
    for (int i = 0; i < FM; ++i)
      #pragma unroll
      for (int r = 0; r < 16; ++r) acc[j][i][r] = 0;
  int wsum[FN] = {};
  i32x4 fr[2][FN + FM];                             // two sets of operands: weights, tokens
  const auto rd = [&](int set, int f, uint32_t stage, int ks) {
    fr[set][f] = *(lds_frag)((f < FN ? readW + f * 32 * SLAB : readA + (f - FN) * 32 * SLAB) + stage + (ks ? second : 0));
  };
  constexpr int PRODUCTS = FM * FN, HALF = (LA + LW) / 2;
  const auto products = [&](int set, auto&& read, auto&& load) {
    #pragma unroll
    for (int m = 0; m < PRODUCTS; ++m) {
      const int i = m % FM, j = m / FM;
      acc[j][i] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fr[set][j], fr[set][FN + i], acc[j][i], 0, 0, 0);
      if (ASYM && i == 0) wsum[j] = add_bytes(fr[set][j], wsum[j]);
      // the operand reads in the first three quarters of the products, the loads spread over all of them
      #pragma unroll
      for (int f = 0; f < FN + FM; ++f)             // in the order in which the products need them
        if (f * PRODUCTS * 3 / 4 / (FN + FM) == m) read(f == 0 ? 0 : f <= FM ? FN + f - 1 : f - FM);
      #pragma unroll
      for (int p = 0; p < HALF; ++p)
        if ((p + 1) * PRODUCTS / HALF - 1 == m) load(p);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  constexpr int LOADS = LA + LW;
  #pragma unroll
  for (int s = 0; s < STAGES; ++s) {
    const uint32_t outside = outside_at(s * SLAB);
    #pragma unroll
    for (int p = 0; p < (s == STAGES - 1 ? HALF : LOADS); ++p) gload(lds0 + s * T::STAGE, s * SLAB, outside, p);
  }
  constexpr int FIRST = (STAGES - 1) * LOADS - LOADS + HALF, LATER = (STAGES - 2) * LOADS;
  __builtin_amdgcn_s_waitcnt(0x0F70 | (FIRST & 15) | ((FIRST >> 4) << 14));
  __syncthreads();
  #pragma unroll
  for (int f = 0; f < FN + FM; ++f) rd(0, f, 0, 0);
  uint32_t cur = 0, dst = lds0 + (STAGES - 1) * T::STAGE;
  int at = (STAGES - 1) * SLAB;
  uint32_t outside = outside_at(at);
  __builtin_amdgcn_sched_barrier(0);
  for (int s = 0; s < steps; ++s) {
    // the first 32 codes of the stage; meanwhile the reads of the others, and the second half of the loads three stages ahead
    products(0, [&](int f) { rd(1, f, cur, 1); }, [&](int p) { gload(dst, at, outside, HALF + p); });
    // The next stage has landed (the loads of the two behind it may be in flight) and this one is in registers, in every wave: its place
    // takes the stage four ahead.
    __builtin_amdgcn_s_waitcnt(0x0070 | (LATER & 15) | ((LATER >> 4) << 14));
    asm volatile("s_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    const uint32_t nxt = cur == (STAGES - 1) * T::STAGE ? 0 : cur + T::STAGE;
    dst = lds0 + cur;
    at += SLAB;
    outside = outside_at(at);
    products(1, [&](int f) { rd(0, f, nxt, 0); }, [&](int p) { gload(dst, at, outside, p); });
    cur = nxt;
  }
  __builtin_amdgcn_s_waitcnt(0x0070);               // nothing may still be on its way to LDS when it is used again

  // ---- outputs: register r of lane l is channel 8 (r / 4) + 4 (l / 32) + r % 4 of token l % 32 ----
  for (int c = tid; c < T::TN; c += 256) {
    const int64_t n = n0 + c;
    channel[0][c] = c < rows_w ? load_any(g.ws, g.ws_dtype, g.w_scalar ? 0 : n) : 0.0f;
    channel[1][c] = c < rows_w && g.bias ? load_any(g.bias, g.bias_dtype, n) : 0.0f;
  }
  if (ASYM && wr == 0) {
    #pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int both = wsum[j] + __builtin_amdgcn_ds_bpermute((lane ^ 32) * 4, wsum[j]);
      if (lane < 32) sums[wc * FN * 32 + j * 32 + lane] = both;
    }
  }
  __syncthreads();
  // A wave's outputs leave through its own part of LDS, 16 bytes per lane along a token: 32 or (fp32) 64 bytes of a token's row per
  // accumulator; chunk c of 16 bytes of token t lies at c ^ t.
  constexpr int E = BF == ROW_F32 ? 4 : 2, CH = 16 / E;                      // bytes of an output, outputs of a chunk
  constexpr int ROW = FN * 32 * E, CHUNKS = ROW / 16;
  char* const mine = lds + wave * 32 * ROW;
  const int t = lane & 31, h = lane >> 5;
  const bool wide = (uintptr_t)g.y % 16 == 0 && (g.N * E) % 16 == 0;
  #pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int m = wr * FM * 32 + i * 32;            // token 0 of these 32, in the tile
    const bool in = m + t < rows_a;
    const float as = in ? g.as[g.a_scalar ? 0 : m0 + m + t] : 0.0f;
    const int az = ASYM && in ? g.az[m0 + m + t] : 0;
    #pragma unroll
    for (int j = 0; j < FN; ++j)
      #pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int c = j * 32 + 8 * q + 4 * h;       // first of four channels, in the wave
        const f32x4 ws = *(const f32x4*)&channel[0][wc * FN * 32 + c], b = *(const f32x4*)&channel[1][wc * FN * 32 + c];
        float v[4];
        #pragma unroll
        for (int r = 0; r < 4; ++r) {
          int s = acc[j][i][4 * q + r];
          if (ASYM) s -= az * sums[wc * FN * 32 + c + r];
          v[r] = (float)s * (as * ws[r]) + b[r];
        }
        char* const to = mine + t * ROW + (((c / CH) ^ t) % CHUNKS) * 16 + (c % CH) * E;
        if constexpr (BF == ROW_F32) *(f32x4*)to = f32x4{v[0], v[1], v[2], v[3]};
        else if constexpr (BF == ROW_BF16) *(u32x2*)to = u32x2{bf16_pack_rne(v[0], v[1]), bf16_pack_rne(v[2], v[3])};
        else *(u32x2*)to = u32x2{f16_pack_rne(v[0], v[1]), f16_pack_rne(v[2], v[3])};
      }
    asm volatile("" ::: "memory");                // (LDS serves a wave in order)
    #pragma unroll
    for (int o = 0; o < 32 * CHUNKS / 64; ++o) {
      const int idx = o * 64 + lane, tt = idx / CHUNKS, ch = idx % CHUNKS;
      const u32x4 v = *(const u32x4*)(mine + tt * ROW + ((ch ^ tt) % CHUNKS) * 16);
      const int n = wc * FN * 32 + ch * CH;
      if (m + tt >= rows_a || n >= rows_w) continue;
      const int64_t cell = (m0 + m + tt) * g.N + n0 + n;
      if (wide && n + CH <= rows_w) {
        *(u32x4*)((char*)g.y + cell * E) = v;
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

// ---- few tokens ---------------------------------------------------------------------------------------------------
// The weight is read once, straight into the matrix pipe's operands: a lane of v_mfma_i32_16x16x64_i8 takes 16 codes of one of 16
// channels, so a load of the wave is 16 rows x 64 bytes in a row.  A workgroup owns 16 channels, its eight waves take pieces of 256
// codes of K in turn and meet in LDS; two pieces (8 KiB of weight per wave) are in flight.  The tokens' codes come from the cache, every
// wave other ones.
// x: the tokens as values (at most MOST_FUSED of them): every workgroup makes their codes itself, in LDS, while its first weights are on
// their way - cheaper for one token than another kernel in front.
constexpr int STREAM_THREADS = 512, STREAM_WAVES = STREAM_THREADS / 64, PIECE = 256;
constexpr int MOST_FUSED = 4;
constexpr int64_t MOST_FUSED_CODES = 40960;         // in LDS

struct TokenArgs {
  const void* x;
  const float* scale;
  int64_t ldx;
  int asym;
};

// One row of x to int8 codes in LDS, by the whole workgroup; K % 16 == 0.
template <int XT>
__device__ __forceinline__ void codes_to_lds(const TokenArgs& t, int64_t row, int K, int8_t* out, float* red, float* scale, int* zero) {
  const int tid = threadIdx.x;
  const char* const x = (const char*)t.x + row * t.ldx * (XT == ROW_F32 ? 4 : 2);
  const bool wide = (uintptr_t)x % 16 == 0;
  const auto load = [&](int i, float* v) {
    if (wide) {
      if constexpr (XT == ROW_F32) { unpack<XT>(*(const u32x4*)(x + i * 4), v); unpack<XT>(*(const u32x4*)(x + i * 4 + 16), v + 4); }
      else unpack<XT>(*(const u32x4*)(x + i * 2), v);
    } else {
      #pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = load_scalar<XT>(x, i + e);
    }
  };
  constexpr int KEEP = 4;                           // pieces of eight that stay in registers: K up to 16384
  float v[KEEP][8];
  float hi = t.asym ? -__builtin_inff() : 0.0f, lo = __builtin_inff();
  const auto range = [&](const float* e) {
    #pragma unroll
    for (int j = 0; j < 8; ++j) {
      hi = nan_max(hi, t.asym ? e[j] : fabsf(e[j]));
      lo = nan_min(lo, e[j]);
    }
  };
  #pragma unroll
  for (int c = 0; c < KEEP; ++c) {
    const int i = (tid + c * STREAM_THREADS) * 8;
    if (i < K) { load(i, v[c]); range(v[c]); }
  }
  for (int i = (tid + KEEP * STREAM_THREADS) * 8; i < K; i += STREAM_THREADS * 8) {
    float e[8];
    load(i, e);
    range(e);
  }
  hi = team_reduce<64, true>(hi);
  lo = team_reduce<64, false>(lo);
  if ((tid & 63) == 0) { red[tid >> 6] = hi; red[STREAM_WAVES + (tid >> 6)] = lo; }
  __syncthreads();
  #pragma unroll
  for (int w = 0; w < STREAM_WAVES; ++w) { hi = nan_max(hi, red[w]); lo = nan_min(lo, red[STREAM_WAVES + w]); }
  const TokenCodes q = t.scale ? TokenCodes::given(t.scale[0]) : t.asym ? TokenCodes::asymmetric(lo, hi) : TokenCodes::symmetric(hi);
  #pragma unroll
  for (int c = 0; c < KEEP; ++c) {
    const int i = (tid + c * STREAM_THREADS) * 8;
    if (i < K) *(u32x2*)(out + i) = u32x2{q.codes(v[c]), q.codes(v[c] + 4)};
  }
  for (int i = (tid + KEEP * STREAM_THREADS) * 8; i < K; i += STREAM_THREADS * 8) {
    float e[8];
    load(i, e);
    *(u32x2*)(out + i) = u32x2{q.codes(e), q.codes(e + 4)};
  }
  if (tid == 0) {
    *scale = q.d.s;
    *zero = (int)q.z;
  }
  __syncthreads();
}

// XT: the type of the tokens' values, or -1 for codes
template <int TB, int BF, int XT>
__global__ __launch_bounds__(STREAM_THREADS) void stream_kernel(MatmulArgs g, TokenArgs t) {
  __shared__ __attribute__((aligned(16))) int red[STREAM_WAVES][TB + 1][64][4];
  __shared__ float token_scale[XT < 0 ? 1 : MOST_FUSED];
  __shared__ int token_zero[XT < 0 ? 1 : MOST_FUSED];
  extern __shared__ __attribute__((aligned(16))) int8_t codes[];             // [M, K], XT >= 0 only
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  const int64_t n = n0 + (lane & 15) < g.N ? n0 + (lane & 15) : g.N - 1;
  const int at = (lane >> 4) * 16;
  const int8_t* const w = g.w + n * g.ldw + at;
  const bool asym = XT < 0 ? g.az != nullptr : t.asym;

  struct Piece { i32x4 v[4]; };
  const auto weights = [&](int k, Piece& p) {       // codes k .. k + 255 of this lane's channel
    #pragma unroll
    for (int i = 0; i < 4; ++i) p.v[i] = k + i * 64 + at < g.K ? *(const i32x4*)(w + k + i * 64) : i32x4{0, 0, 0, 0};
  };
  Piece cur, nxt;
  const int step = STREAM_WAVES * PIECE;
  int k = wave * PIECE;
  weights(k, cur);
  weights(k + step, nxt);
  if constexpr (XT >= 0) {
    for (int m = 0; m < (int)g.M; ++m)
      codes_to_lds<XT>(t, m, g.K, codes + m * g.K, (float*)red, token_scale + m, token_zero + m);
  }
  const int8_t* a[TB];
  #pragma unroll
  for (int b = 0; b < TB; ++b) {
    const int64_t m = b * 16 + (lane & 15) < g.M ? b * 16 + (lane & 15) : g.M - 1;           // (a token twice: not stored)
    a[b] = XT < 0 ? g.a + m * g.lda + at : codes + m * g.K + at;
  }
  i32x4 acc[TB] = {};
  int wsum = 0;
  while (k < g.K) {
    Piece tok[TB];
    #pragma unroll
    for (int b = 0; b < TB; ++b)
      #pragma unroll
      for (int i = 0; i < 4; ++i) tok[b].v[i] = k + i * 64 + at < g.K ? *(const i32x4*)(a[b] + k + i * 64) : i32x4{0, 0, 0, 0};
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
      #pragma unroll
      for (int b = 0; b < TB; ++b) acc[b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(cur.v[i], tok[b].v[i], acc[b], 0, 0, 0);
      if (asym) wsum = add_bytes(cur.v[i], wsum);
    }
    k += step;
    cur = nxt;
    weights(k + step, nxt);
  }
  #pragma unroll
  for (int b = 0; b < TB; ++b) *(i32x4*)red[wave][b][lane] = acc[b];
  red[wave][TB][lane][0] = wsum;
  __syncthreads();
  // accumulator register r of lane l: channel 4 (l / 16) + r of token l % 16
  for (int o = tid; o < TB * 256; o += STREAM_THREADS) {
    const int c = o & 15, tok = (o >> 4) & 15, b = o >> 8;
    const int64_t m = b * 16 + tok, nn = n0 + c;
    if (m >= g.M || nn >= g.N) continue;
    int s = 0, sum = 0;
    #pragma unroll
    for (int v = 0; v < STREAM_WAVES; ++v) {
      s += red[v][b][(c >> 2) * 16 + tok][c & 3];
      if (asym) sum += (red[v][TB][c][0] + red[v][TB][c + 16][0]) + (red[v][TB][c + 32][0] + red[v][TB][c + 48][0]);
    }
    if (asym) s -= (XT < 0 ? g.az[m] : token_zero[m]) * sum;
    const float as = XT < 0 ? g.as[g.a_scalar ? 0 : m] : token_scale[m];
    const float y = (float)s * (as * load_any(g.ws, g.ws_dtype, g.w_scalar ? 0 : nn)) + (g.bias ? load_any(g.bias, g.bias_dtype, nn) : 0.0f);
    if constexpr (BF == ROW_F32) ((float*)g.y)[m * g.N + nn] = y;
    else store_scalar<BF>(g.y, m * g.N + nn, rnd<BF>(y));
  }
}

// Rows of K codes to rows of Kp, the next multiple of 16, with zeros behind them: operands whose rows do not start on 16 bytes.
__global__ __launch_bounds__(256) void pad_kernel(const int8_t* __restrict__ x, int64_t rows, int K, int Kp, int8_t* __restrict__ out) {
  const int per = Kp / 16;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * per; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / per;
    const int k = (int)(i - r * per) * 16;
    const int8_t* const p = x + r * K + k;
    union { u32x4 v; int8_t b[16]; } u;
    if (k + 16 <= K) {
      __builtin_memcpy(&u, p, 16);
    } else {
      u.v = u32x4{0, 0, 0, 0};
      #pragma unroll
      for (int e = 0; e < 16; ++e)
        if (k + e < K) u.b[e] = p[e];
    }
    *(u32x4*)(out + i * 16) = u.v;
  }
}

int64_t padded(int64_t K) { return (K + 15) / 16 * 16; }

template <int FM, int FN, int BF>
void launch_tiles(const MatmulArgs& g, hipStream_t st) {
  const int64_t tm = (g.M + Tile<FM, FN>::TM - 1) / Tile<FM, FN>::TM, tn = (g.N + Tile<FM, FN>::TN - 1) / Tile<FM, FN>::TN;
  const dim3 grid((unsigned)((tm * tn + 7) / 8 * 8));
  if (g.az) tile_kernel<FM, FN, BF, true><<<grid, dim3(256), 0, st>>>(g, (int)tm, (int)tn);
  else tile_kernel<FM, FN, BF, false><<<grid, dim3(256), 0, st>>>(g, (int)tm, (int)tn);
}

#ifndef STREAM_MOST
#define STREAM_MOST 32
#endif
constexpr int64_t MOST_STREAMED = STREAM_MOST;      // tokens

template <int BF, int XT>
void launch_stream(const MatmulArgs& g, const TokenArgs& t, hipStream_t st) {
  const dim3 grid((unsigned)((g.N + 15) / 16));
  if constexpr (XT >= 0) {
    stream_kernel<1, BF, XT><<<grid, dim3(STREAM_THREADS), (unsigned)(g.M * g.K), st>>>(g, t);
  } else {
    if (g.M <= 16) stream_kernel<1, BF, -1><<<grid, dim3(STREAM_THREADS), 0, st>>>(g, t);
    else if (g.M <= 32) stream_kernel<2, BF, -1><<<grid, dim3(STREAM_THREADS), 0, st>>>(g, t);
    else stream_kernel<4, BF, -1><<<grid, dim3(STREAM_THREADS), 0, st>>>(g, t);
  }
}

template <int BF>
void launch_codes(const MatmulArgs& g, hipStream_t st) {
  if (g.M <= MOST_STREAMED) launch_stream<BF, -1>(g, TokenArgs{}, st);
  else if ((g.M + 255) / 256 * ((g.N + 255) / 256) >= 160) launch_tiles<4, 4, BF>(g, st);
  else launch_tiles<2, 2, BF>(g, st);
}

bool known(int dtype) { return dtype == LCQ_F32 || dtype == LCQ_BF16 || dtype == LCQ_F16; }

int check(const int8_t* w, const void* ws, int ws_dtype, const void* bias, int bias_dtype, int64_t M, int64_t N, int64_t K, const void* y, int dtype) {
  if (!w || !ws || !y || M <= 0 || N <= 0 || K <= 0) return LCQ_EINVAL;
  if (!known(dtype) || !known(ws_dtype) || (bias && !known(bias_dtype))) return LCQ_EDTYPE;
  if (K > 65536 || (M + 127) / 128 * ((N + 127) / 128) > 0x7ffffff0) return LCQ_ESIZE;
  if (K % 16 == 0 && (uintptr_t)w % 16) return LCQ_EALIGN;
  return LCQ_OK;
}

// tokens whose codes the product makes itself
bool fused(int64_t M, int64_t K) { return M <= MOST_FUSED && K % 16 == 0 && M * K <= MOST_FUSED_CODES; }
int64_t on256(int64_t bytes) { return (bytes + 255) / 256 * 256; }

}  // namespace

extern "C" {

int64_t lcq_int8_matmul_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0 || K > 65536) return 0;
  return K % 16 ? (M + N) * padded(K) : 0;
}

int lcq_int8_matmul(const int8_t* a, const float* as, int a_scalar, const int32_t* az, const int8_t* w, const void* ws, int ws_dtype,
                    int w_scalar, const void* bias, int bias_dtype, int64_t M, int64_t N, int64_t K, void* y, int dtype,
                    void* workspace, void* stream) {
  if (!a || !as) return LCQ_EINVAL;
  const int bad = check(w, ws, ws_dtype, bias, bias_dtype, M, N, K, y, dtype);
  if (bad) return bad;
  hipStream_t st = (hipStream_t)stream;
  MatmulArgs g = {a, w, as, az, ws, bias, y, M, N, K, K, (int)K, ws_dtype, bias_dtype, a_scalar, w_scalar};
  if (K % 16) {
    if (!workspace) return LCQ_EWORKSPACE;
    if ((uintptr_t)workspace % 16) return LCQ_EALIGN;
    const int Kp = (int)padded(K);
    int8_t* const pa = (int8_t*)workspace;
    int8_t* const pw = pa + M * Kp;
    const auto grid = [&](int64_t rows) { const int64_t b = (rows * (Kp / 16) + 255) / 256; return dim3((unsigned)(b < 4096 ? b : 4096)); };
    pad_kernel<<<grid(M), dim3(256), 0, st>>>(a, M, (int)K, Kp, pa);
    pad_kernel<<<grid(N), dim3(256), 0, st>>>(w, N, (int)K, Kp, pw);
    g.a = pa; g.w = pw; g.lda = g.ldw = g.K = Kp;
  } else if ((uintptr_t)a % 16) {
    return LCQ_EALIGN;
  }
  if (dtype == LCQ_BF16) launch_codes<ROW_BF16>(g, st);
  else if (dtype == LCQ_F16) launch_codes<ROW_F16>(g, st);
  else launch_codes<ROW_F32>(g, st);
  LCQ_CHECK_LAUNCH();
  return LCQ_OK;
}

int64_t lcq_int8_linear_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0 || K > 65536 || fused(M, K)) return 0;
  return on256(M * K) + on256(8 * M) + lcq_int8_matmul_workspace_bytes(M, N, K);
}

int lcq_int8_linear(const void* x, int x_dtype, int64_t ldx, int asym, const float* scale, const int8_t* w, const void* ws, int ws_dtype,
                    int w_scalar, const void* bias, int bias_dtype, int64_t M, int64_t N, int64_t K, void* y, int dtype,
                    void* workspace, void* stream) {
  if (!x || ldx < 0 || (asym && scale)) return LCQ_EINVAL;
  const int bad = check(w, ws, ws_dtype, bias, bias_dtype, M, N, K, y, dtype);
  if (bad) return bad;
  if (!known(x_dtype)) return LCQ_EDTYPE;
  if (fused(M, K)) {
    hipStream_t st = (hipStream_t)stream;
    const MatmulArgs g = {nullptr, w, nullptr, nullptr, ws, bias, y, M, N, K, K, (int)K, ws_dtype, bias_dtype, 0, w_scalar};
    const TokenArgs t = {x, scale, ldx, asym};
    const auto run = [&](auto xt) {
      constexpr int XT = decltype(xt)::value;
      if (dtype == LCQ_BF16) launch_stream<ROW_BF16, XT>(g, t, st);
      else if (dtype == LCQ_F16) launch_stream<ROW_F16, XT>(g, t, st);
      else launch_stream<ROW_F32, XT>(g, t, st);
    };
    if (x_dtype == LCQ_BF16) run(std::integral_constant<int, ROW_BF16>{});
    else if (x_dtype == LCQ_F16) run(std::integral_constant<int, ROW_F16>{});
    else run(std::integral_constant<int, ROW_F32>{});
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

// Values to microscaled 4-bit codes and back.
//
// A lane takes eight values (of a bf16 row 16 bytes), four neighbouring lanes a block: its largest magnitude comes from two quad
// permutations, so nothing waits for the rest of the row.  Four pieces of a lane are on their way at a time.  Bound by memory: 2.53 bytes a value for bf16,
// either way.  4096 x 14336 to codes 29.4 us (5.0 TB/s, a copy has 5.2), back 22.9 (6.5); 16 x 4096 2.8 and 2.8, which is a launch and a load.
#include "mxfp4.h"
#include <type_traits>

namespace {
using namespace lcq;

template <int I> using Int = std::integral_constant<int, I>;
constexpr int MOST_PIECES = 4;                      // of eight values, per lane

struct Rows {
  int64_t rows, K, pieces, ldx;                     // pieces: of eight values in the whole blocks of a row
  int lanes, each;                                  // that share a row (a power of two, 4 .. 256); pieces of a lane
  uint32_t chunks;                                  // workgroups along a row
  bool past;                                        // values go past the caches
};

// a lane's row, and its first piece; its others are `step` behind one another
__device__ __forceinline__ bool place(const Rows& r, int64_t& row, int64_t& piece, int& step) {
  const uint32_t rows = blockIdx.x / r.chunks, chunk = blockIdx.x - rows * r.chunks;
  row = (int64_t)rows * (256 / r.lanes) + threadIdx.x / r.lanes;
  piece = (int64_t)chunk * (r.lanes * r.each) + (threadIdx.x & (r.lanes - 1));
  step = r.lanes;
  return row < r.rows;
}

template <int XT, int PIECES>
__global__ __launch_bounds__(256) void quant_kernel(const char* __restrict__ x, Rows r, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                                    int64_t lds) {
  int64_t row, piece;
  int step;
  if (!place(r, row, piece, step)) return;          // (quads are whole: a block's four lanes leave together)
  const char* const from = x + row * r.ldx * (XT == ROW_F32 ? 4 : 2);
  float v[PIECES][8];
  #pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    const int64_t p = piece + i * step;
    if (p < r.pieces) mx_load8<XT>(from, p * 8, r.K, v[i]);
  }
  #pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    const int64_t p = piece + i * step;
    if (p >= r.pieces) break;
    const uint32_t s = mx_scale(mx_quad_max(mx_max_bits(v[i])));
    *(uint32_t*)(codes + (row * r.pieces + p) * 4) = mx_codes(v[i], s);
    if ((p & 3) == 0) scales[row * lds + (p >> 2)] = (uint8_t)s;
  }
}

__device__ __forceinline__ void put(void* to, u32x4 v, bool past) {
  if (past) mx_store_past(to, v);
  else *(u32x4_anywhere*)to = v;
}

template <int BF, int PIECES>
__global__ __launch_bounds__(256) void dequant_kernel(const uint8_t* __restrict__ codes, int64_t ldc, const uint8_t* __restrict__ scales, int64_t lds,
                                                      Rows r, char* __restrict__ y) {
  int64_t row, piece;
  int step;
  if (!place(r, row, piece, step)) return;
  uint32_t c[PIECES], s[PIECES];
  #pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    const int64_t p = piece + i * step;
    if (p < r.pieces) {
      c[i] = *(const uint32_t*)(codes + row * ldc + p * 4);
      s[i] = scales[row * lds + (p >> 2)];
    }
  }
  #pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    const int64_t p = piece + i * step, k = p * 8;
    if (p >= r.pieces || k >= r.K) break;
    const float f = mx_factor(s[i]);
    lcq_f32x2 v[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[i], f, 0), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[i], f, 1),
                      __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[i], f, 2), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[i], f, 3)};
    if constexpr (BF == ROW_F32) {
      float* const to = (float*)y + row * r.K + k;
      if (k + 8 <= r.K) {
        const u32x4 w[2] = {{f2u(v[0].x), f2u(v[0].y), f2u(v[1].x), f2u(v[1].y)}, {f2u(v[2].x), f2u(v[2].y), f2u(v[3].x), f2u(v[3].y)}};
        put(to, w[0], r.past);
        put(to + 4, w[1], r.past);
      } else
        #pragma unroll
        for (int e = 0; e < 8; ++e) if (k + e < r.K) to[e] = v[e / 2][e % 2];
    } else {
      uint16_t* const to = (uint16_t*)y + row * r.K + k;
      u32x4 w;                                      // (bf16 holds every one of these values that fp32 holds)
      #pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = BF == ROW_BF16 ? bf16_pack_rne(v[e].x, v[e].y) : f16_pack_rne(v[e].x, v[e].y);
      if (k + 8 <= r.K) put(to, w, r.past);
      else
        #pragma unroll
        for (int e = 0; e < 8; ++e) if (k + e < r.K) to[e] = (uint16_t)(w[e / 2] >> 16 * (e % 2));
    }
  }
}

bool known(int dtype) { return dtype == LCQ_F32 || dtype == LCQ_BF16 || dtype == LCQ_F16; }

// Rows of whole blocks without gaps (`joined`) are one long row.  A launch has fewer than 2^32 lanes.
int plan(int64_t rows, int64_t K, int64_t ldx, bool joined, Rows& r, dim3& grid) {
  if (rows <= 0 || K <= 0 || ldx < 0) return LCQ_EINVAL;
  if (K > (int64_t)1 << 36 || rows > ((int64_t)1 << 36) / ((K + 31) / 32 * 32)) return LCQ_ESIZE;
  if (joined && K % 32 == 0) { K *= rows; rows = 1; }
  r = Rows{rows, K, (K + 31) / 32 * 4, ldx, 256, MOST_PIECES, 1, false};
  // Four loads of a lane run side by side; where there would be fewer workgroups than CUs a lane has one (bf16 rows of 14336 to codes, 1 / 4 pieces: 32 rows
  // 2.8 / 3.7 us, 128 rows 3.4 / 3.8, 256 rows 4.1 / 4.3; back, 32 rows 2.8 / 3.0, 512 rows 6.0 / 5.6, 1024 rows 8.6 / 7.8).
  if (rows * r.pieces < 256 * 256 * MOST_PIECES) r.each = 1;
  while (r.lanes > 4 && r.lanes / 2 * r.each >= r.pieces) r.lanes /= 2;
  r.chunks = (uint32_t)((r.pieces + r.lanes * r.each - 1) / (r.lanes * r.each));
  const int64_t blocks = (rows + 256 / r.lanes - 1) / (256 / r.lanes) * r.chunks;
  if (blocks > (1 << 24) - 1) return LCQ_ESIZE;
  grid = dim3((unsigned)blocks);
  return LCQ_OK;
}

template <class Run>
void by_size(const Rows& r, int dtype, const Run& run) {
  const auto typed = [&](auto each) {
    if (dtype == LCQ_BF16) run(Int<ROW_BF16>{}, each);
    else if (dtype == LCQ_F16) run(Int<ROW_F16>{}, each);
    else run(Int<ROW_F32>{}, each);
  };
  if (r.each == 1) typed(Int<1>{});
  else typed(Int<MOST_PIECES>{});
}

}  // namespace

extern "C" {

int lcq_mxfp4_quant(const void* x, int dtype, int64_t rows, int64_t K, int64_t ldx, uint8_t* codes, uint8_t* scales, int64_t lds, void* stream) {
  if (!x || !codes || !scales || lds < (K + 31) / 32) return LCQ_EINVAL;
  if (!known(dtype)) return LCQ_EDTYPE;
  if ((uintptr_t)codes % 4) return LCQ_EALIGN;
  Rows r;
  dim3 grid;
  const int bad = plan(rows, K, ldx, ldx == K && lds == K / 32, r, grid);
  if (bad) return bad;
  hipStream_t st = (hipStream_t)stream;
  const auto run = [&](auto xt, auto each) { quant_kernel<decltype(xt)::value, decltype(each)::value><<<grid, dim3(256), 0, st>>>((const char*)x, r, codes, scales, lds); };
  by_size(r, dtype, run);
  LCQ_CHECK_LAUNCH();
  return LCQ_OK;
}

int lcq_mxfp4_dequant(const uint8_t* codes, int64_t ldc, const uint8_t* scales, int64_t lds, int64_t rows, int64_t K, void* y, int dtype, void* stream) {
  if (!codes || !scales || !y || ldc < 0 || lds < 0) return LCQ_EINVAL;
  if (!known(dtype)) return LCQ_EDTYPE;
  if ((uintptr_t)codes % 4 || ldc % 4) return LCQ_EALIGN;
  Rows r;
  dim3 grid;
  const int bad = plan(rows, K, 0, ldc == K / 2 && lds == K / 32, r, grid);
  if (bad) return bad;
  // More than the caches keep beside what is read goes past them: 117 MB of bf16 22.2 us, through them 23.3, with the quantization of the next 48.2 and 50.4, with a pass
  // that reads it 60.0 and 60.4; but 29 MB with such a pass 23.0 and 21.7.
  r.past = rows * K * (dtype == LCQ_F32 ? 4 : 2) > (int64_t)96 << 20;
  hipStream_t st = (hipStream_t)stream;
  const auto run = [&](auto xt, auto each) { dequant_kernel<decltype(xt)::value, decltype(each)::value><<<grid, dim3(256), 0, st>>>(codes, ldc, scales, lds, r, (char*)y); };
  by_size(r, dtype, run);
  LCQ_CHECK_LAUNCH();
  return LCQ_OK;
}

}  // extern "C"

// Rules by which an entry point takes one of several kernels, as functions of sizes, types and alignment alone.  Plain C++: they can
// be checked without a GPU and without a HIP compiler.
#pragma once

namespace lcq {

// Products with a contraction of exactly 128 (gemm_f32.h): C = alpha A op(B) + beta C.
//   solve   C = A B^T of 128 columns (C may be A)
//   waves   C -= A op(B), one wave per 16 x 32 of C; leaves out the tiles above the diagonal where `lower` asks for it
//   stream  C -= A B, a wave per 64 columns streams rows; every tile
//   none    the general kernels, which leave them out too
// The line between waves and stream is 1024 tiles of 16 x 64, a stream's one tile per wave (measured beside the launches).
enum class Rank128 { none, solve, waves, stream };
inline Rank128 rank128_form(bool b_t, long long M, long long N, float alpha, float beta, bool in_place, bool lower) {
  if (b_t && alpha == 1.0f && beta == 0.0f && N == 128) return Rank128::solve;
  if (alpha != -1.0f || beta != 1.0f || in_place) return Rank128::none;
  if (b_t || ((M + 15) / 16) * ((N + 63) / 64) <= 1024) return Rank128::waves;
  return lower ? Rank128::none : Rank128::stream;
}

// Column loop (gptq_loop.hip): does a block run by panels of 64 rows?  Whole blocks of 128 columns on 16 bytes (`on16`: all pointers),
// rounded zero points, and parameters that change at the starts of 16-column panels only: searched for groups that open inside the
// block, or given for groups of whole panels or for rows.
// Codes of 9 and 10 bits (all of them within +-512, beyond that both kernels divide everywhere) stay with sixteen lanes per row where the
// panels that run again with divisions cost more than a wave of 64 rows gains.  How many do grows with the code range and with the rows
// of a wave; the gain is smaller for long groups, and sixteen lanes lose beyond one workgroup per CU (4096 rows).  us per block by panels
// / by sixteen lanes, 9 | 10 bits, symmetric:
//   rows          64                      256                     1000                    4096                    5120
//   g = 32    13.7 / 15.3 | 14.6 / 15.4   14.7 / 15.8 | 15.8 / 15.8   15.8 / 16.5 | 16.7 / 16.5   17.1 / 17.9 | 17.9 / 17.9   17.5 / 21.4 | 18.3 / 21.4
//   g = 64    13.8 / 14.8 | 14.5 / 14.8   14.7 / 15.3 | 15.9 / 15.3   15.6 / 16.1 | 16.6 / 16.0   17.0 / 17.3 | 18.0 / 17.4   17.5 / 20.5 | 18.4 / 20.5
//   g = 128   13.3 / 14.0 | 14.6 / 14.2   14.8 / 14.4 | 15.9 / 14.6   15.7 / 15.3 | 16.7 / 15.3   17.0 / 16.5 | 18.0 / 16.6   17.5 / 19.9 | 18.3 / 19.9
// (8 bits, g = 128: 13.3 / 14.1, 14.1 / 14.5, 14.9 / 15.3, 16.2 / 16.5, 16.8 / 19.8; given parameters, 10 bits, 4096 rows: 18.0 / 20.8.)
inline bool gptq_by_panels(bool is_static, bool has_gidx, bool rounded, int group, long long R, long long K, long long i1, int count, long long ldErr,
                           bool on16, float qmin, float qmax) {
  const bool whole = is_static ? !has_gidx && (group <= 0 || group % 16 == 0) : group == 16 || group == 32 || group == 64 || group == 128;
  if (!whole || !rounded || count != 128 || i1 % 128 != 0 || K % 4 != 0 || ldErr % 4 != 0 || !on16) return false;
  const float codes = qmax - qmin + 1.0f;
  const bool divides = qmin < -512.0f || qmin > 512.0f || qmax < -512.0f || qmax > 512.0f;
  return is_static || divides || codes * group < 65536.0f || codes * R <= 32768.0f || R > 4096;
}

// Int8 product in tiles (int8_matmul.hip): which tile, and into how many parts K is cut.  A tile takes
//   start + slabs (busy + crowd share) us     slabs of 128 codes of K, share of the chip's 256 CUs at work
// and the tiles of a workgroup slot follow one another; parts leave their sums (written and read once, 4 bytes per us and MB / 4) for
// another kernel (3 us).  Constants fitted to one round at K = 4096 and 14336 (us): 256 x 256 alone 42 and 125, on all CUs 60;
// 256 x 192 35 and 98, 53; 128 x 128 15.5 and 42, 20.  Measured choices, us at K = 4096 as 256 x 256 / 256 x 192 / 128 x 128:
//   N = 4096    1024 tokens 44.3 / 37.6 / 19.8    2048 tokens  45.5 / 41.6 / 38.3
//   N = 6144    1024 tokens 44.7 / 37.7 / 34.0    2048 tokens  52.6 / 52.9 / 56.8
//   N = 14336    512 tokens 45.1 / 39.5 / 35.6    1024 tokens  57.8 / 85.0 / 68.5    2048 tokens 112 / 134 / 129
struct Int8Cut { int tile, parts; double us; };     // tile 0: 256 x 256, 1: 256 x 192, 2: 128 x 128
inline Int8Cut int8_cut(long long M, long long N, long long K) {
  struct Shape { int tm, tn; double start, busy, crowd; };
  const Shape shapes[3] = {{256, 256, 9.0, 1.03, 0.56}, {256, 192, 8.0, 0.81, 0.60}, {128, 128, 5.0, 0.333, 0.14}};
  const long long slabs = (K + 127) / 128;
  Int8Cut best = {0, 1, 0.0};
  for (int i = 0; i < 3; ++i) {
    const Shape& s = shapes[i];
    const long long tiles = (M + s.tm - 1) / s.tm * ((N + s.tn - 1) / s.tn);
    for (int parts = 1; parts <= (i == 2 ? 16 : 1); ++parts) {
      if (parts > 1 && (tiles * parts > 256 || slabs / parts < 2)) break;
      const long long rounds = tiles * parts / 256, rest = tiles * parts % 256;
      const double each = (double)((slabs + parts - 1) / parts);
      double t = rounds * (s.start + each * (s.busy + s.crowd));
      if (rest) t += s.start + each * (s.busy + s.crowd * (double)rest / 256.0);
      if (parts > 1) t += 3.0 + 8.0 * parts * (double)M * (double)N / 4e6;
      if (best.us == 0.0 || t < best.us) best = {i, parts, t};
    }
  }
  return best;
}

// Whether the weight is streamed past the tokens instead: always for up to 16 of them, up to 64 where that is the faster.  A stream takes
//   3.2 + M K (0.15 + 0.85 blocks) / 25000 us     blocks of 16 channels on the busiest of 256 CUs
// and 1.6 (beyond 32 tokens 2.4) times the second term where rows do not start on 16 bytes, which tiles need copied first.  Measured as
// stream / tiles, us:
//   512 x 512     64 tokens  5.6 / 6.1     2048 x 2048   33 tokens  6.5 / 10.2    64 tokens  8.9 / 10.2
//   4096 x 4096   33 tokens 10.0 / 13.4    64 tokens 15.2 / 14.1    14336 x 4096  32 tokens 22.3 / 18.2    4096 x 14336  32 tokens 24.0 / 19.9
//   4096 x 4097   48 tokens 21.5 / 23.4    64 tokens 26.8 / 23.5    14336 x 4097  32 tokens 35.9 / 42     33 tokens 57 / 42
constexpr int INT8_STREAMED = 64;
inline bool int8_streams(long long M, long long N, long long K) {
  if (M > INT8_STREAMED) return false;
  if (M <= 16) return true;
  const bool odd = K % 16 != 0;
  const double blocks = (double)((N + 4095) / 4096);
  const double stream = 3.2 + (odd ? M <= 32 ? 1.6 : 2.4 : 1.0) * (double)M * (double)K * (0.15 + 0.85 * blocks) / 25000.0;
  const double tiles = int8_cut(M, N, (K + 15) / 16 * 16).us + (odd ? 3.0 + 2.0 * (double)(M + N) * (double)K / 4.9e6 : 0.0);
  return stream < tiles;
}

}  // namespace lcq

// Rules by which an entry point takes one of several kernels, as functions of sizes, types and alignment alone.  Plain C++: they can
// be checked without a GPU and without a HIP compiler.
#pragma once
#include <type_traits>

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

// Product of microscaled 4-bit numbers (mxfp4_matmul.hip), B blocks of 32 in a row.  Times in us on one MI355X, other weights every time.
constexpr int MXFP4_CUS = 256;
inline double mxfp4_rounds(double workgroups) { return (double)(long long)((workgroups + MXFP4_CUS - 1) / MXFP4_CUS); }
// The weight streamed past groups of 16 or 32 tokens: a unit of work is 4 / KS blocks of 16 channels with such a group, KS waves share the K of a block, and a
// workgroup per CU takes its share of the units one behind the other.  A unit costs its waves' stages of 8 blocks of K, and 1.2 or 2.5 more where its sums are
// joined; KS is what makes that least for a workgroup.  N x K with KS 1 / 2 / 4 for 16 and for 32 tokens:
//   1024 x 1024  5.1 / 4.4 / 4.2   5.5 / 4.7 / 4.4    4096 x 4096   8.4 /  6.6 /  5.9    9.5 /  7.0 /  6.1    7168 x 2048  6.6 / 5.7 / 6.2    7.2 / 5.9 / 6.8
//   6144 x 4096  8.6 / 6.9 / 7.9   9.7 / 7.2 / 8.6   14336 x 4096   9.2 / 10.2 / 11.9   10.4 / 11.6 / 13.8    2048 x 7168  11.4 / 8.1 / 6.6  13.9 / 9.5 / 7.3
inline long long mxfp4_units(long long M, long long N, int KS) {
  const long long group = M <= 16 ? 16 : 32, blocks = (N + 15) / 16, at_once = 4 / KS;
  return (blocks + at_once - 1) / at_once * ((M + group - 1) / group);
}
inline double mxfp4_stages(long long M, long long N, long long B, int KS) {            // of a workgroup
  return mxfp4_rounds((double)mxfp4_units(M, N, KS)) * ((double)(((B + 7) / 8 + KS - 1) / KS) + (M <= 16 ? 1.2 : 2.5));
}
inline int mxfp4_waves(long long M, long long N, long long B) {
  int best = 4;
  for (int KS = 2; KS >= 1; KS /= 2)
    if (mxfp4_stages(M, N, B, KS) < mxfp4_stages(M, N, B, best)) best = KS;
  return best;
}
// Or tiles: of 256 x 256, one to a CU, of 128 x 128, one to a CU, or of 64 x 64, two to a CU, the latter two also with K cut into parts of at least two periods of
// 16 blocks, whose sums are joined.  What is estimated to be fastest, measured as streamed / 64 in 1 part / in 2 / in 4 / 128 in 1 part / in 4 (and 256):
//   4096 x 4096    64 tokens  7.2 / 8.2 /  9.4 / 10.6 / 12.3 / 12.6    128   9.9 /  8.3 /  9.9 / 13.9 / 12.6 / 14.6    211  16 /  8.7 / 13 / 18 / 12.8 / 17
//                 512 tokens   29 / 12.7 / 21  /  29  / 13.3 / 26     1024  52 / 22.7 / 36 / 50 / 17.4 / 42            2048 tokens 29.8 with 128 (32.7)
//   4096 x 14336   64 tokens   16 /  26 /  19  / 14.9 /  39  /  19     128   22 /  26  / 19.3 / 22 / 44 / 22             211  48 /  23 / 25 / 29 / 41 / 22
//   14336 x 4096   64 tokens   16 / 10.2 / 17  /  21  / 14.8 /  23     128   29 / 15.2 / 26 / 35 / 15.6 / 28             211  47 /  23 / 37 / 52 / 17.8 / 45
//   7168 x 2048    64 tokens  7.3 /  6.0 / 9.3 / 12.3 /  8.7           211   19 /  8.0 / 18 / 23 /  9.4                   512  31 /  14 / 26 / 38 / 11.2
//   1001 x 2047   128 tokens  5.4 /  5.6 / 7.1 /  7.8 /  9.4           512  7.0 /  5.9 / 9.7 / 13 /  9.6                  1333  15 / 8.1 / 18 / 24 / 10.4
struct Mxfp4Cut { bool stream; int tile, parts; };  // tile 0: 256 x 256, 1: 128 x 128, 2: 64 x 64
inline Mxfp4Cut mxfp4_cut(long long M, long long N, long long B) {
  if (M <= 32) return {true, 0, 1};
  const double stages = (double)((B + 7) / 8), outputs = (double)M * (double)N, weights = (double)N * (double)B * 17 / 5.5e6;
  const auto tiles = [&](long long side) { return (double)((M + side - 1) / side) * (double)((N + side - 1) / side); };
  const auto join = [&](int parts) { return parts > 1 ? 3 + parts * outputs / 5e5 : 0.0; };
  const auto most = [](double a, double b) { return a > b ? a : b; };
  const double scales = B % 16 ? 2.5 : 0;           // put in order in front of the tiles (of 256 x 256 always)
  double least = 9.5 + mxfp4_rounds(tiles(256)) * (3 + 1.9 * stages);
  Mxfp4Cut best = {false, 0, 1};
  for (int parts = 1; parts <= 8 && (parts == 1 || (B + 15) / 16 >= 2 * parts); parts *= 2) {
    const double w128 = tiles(128) * parts, w64 = tiles(64) * parts;
    const double us128 = 4.4 + scales + mxfp4_rounds(w128) * (1 + most(0.55, 0.0032 * (w128 < MXFP4_CUS ? w128 : MXFP4_CUS)) * stages / parts) + join(parts);
    const double us64 = 3.2 + scales + most(weights, mxfp4_rounds(w64 / 2) * most(0.30, 0.0013 * (w64 < 2 * MXFP4_CUS ? w64 : 2 * MXFP4_CUS)) * stages / parts) + join(parts);
    if (us128 < least && w128 <= (1 << 24) - 8) least = us128, best = {false, 1, parts};
    if (us64 < least && w64 <= (1 << 24) - 8) least = us64, best = {false, 2, parts};        // (a launch has fewer than 2^32 lanes)
  }
  const long long teams = (M + 31) / 32;
  if (teams <= 64 && 3.4 + 0.39 * mxfp4_stages(M, N, B, mxfp4_waves(M, N, B)) < least) best = {true, 0, 1};
  return best;
}

// A wave's outputs of a tile leave 64 pieces of 16 bytes at a time, rows of 32 FN outputs of E bytes: TOKENS rows together.  A lane's place among them, N outputs to a
// row, is told apart from the store's in 32 bits where those hold it for every N that the product takes (tiles of 256 and 128), and in 64 bits elsewhere.
constexpr long long MXFP4_MOST_N = (1 << 28) - 16;
template <int FN, int E>
struct Mxfp4Store {
  static constexpr int TOKENS = 64 * 16 / (32 * FN * E);
  static constexpr long long MOST = (TOKENS - 1) * MXFP4_MOST_N * E + 64 * FN * E;       // (a tile has twice the wave's channels)
  typedef std::conditional_t<MOST <= 0xffffffffLL, unsigned, unsigned long long> Offset;
};

}  // namespace lcq

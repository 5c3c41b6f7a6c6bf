// Log probabilities of given tokens, entropy and best alternatives of logits x [T, V], in one pass over them:
//   S = sum exp(x - c),  U = sum exp(x - c) (x - c)   for any reference c
//   log sum exp x = c + log S;   logprob of a token t = (x_t - c) - log S;   entropy = log S - U / S
//
//  * A lane keeps its own c, S and U.  c is a logit that the lane has seen; it moves only where a later one is more than 8 above
//    it, so that almost no piece pays for a change of reference, S stays below V e^8 and log S and U / S do not cancel to more than a few
//    times their last bits.  References meet once, when lanes and waves are joined.
//  * The best alternatives cost the pass one comparison per piece: a lane keeps the largest logit of each 8th (12th) of the pass.  Behind it, the k-th
//    largest of all lanes' maxima is a bound that k logits reach, few more do, and only those parts of a lane's logits that reach it are read
//    again for the keys of those logits, which one wave sorts.  A key is a whole number that orders by value and then by the lowest index.  Where
//    more keys reach the bound than there is room for, every wave finds its best by itself from a third reading: ties (constant rows), and masks
//    that leave finite logits to fewer than k lanes - fewer than k of them, or neighbours (30 in a row are 4 or 5 lanes' in bf16) -, whose bound is
//    -inf.  Such a row of 128256 bf16 takes 74 us with its best 20, an ordinary one 16; 64 of either side by side 76 and 17.6.
//  * Bound by HBM where there are many rows: 2048 x 128256 bf16 with their best 5 in 112 us (4.7 TB/s); a row alone takes 16 us with its best 20, 6 of them
//    behind the pass.  333 x 50001 fp32, best 10: 18.4 us.
//  * A row is one workgroup's: of 1024 lanes where there are at most as many rows as CUs, of 512 or 256 where there are more.  A row in parts and a
//    second kernel that joins them took 11.6 us of the GPU and 19.1 a call from Python, whose host time is then the longer; one kernel takes 16 of both.
#include "rowquant.h"
#include <type_traits>

namespace {
using namespace lcq;

constexpr float LOWEST = -3.4028234663852886e38f, MOVE = 8.0f;
constexpr int FLIGHT = 2;                           // 16-byte pieces that a lane has on their way while it works on as many

struct LogprobArgs {
  const void* x;
  const int64_t* tokens;
  float *logprobs, *entropy, *top_logprobs;
  int64_t* top_tokens;
  int64_t V, ldx, lds, m, ignore;
  uint32_t rows;                                    // of a sequence: `ldx` elements apart, sequences `lds`
  int k;
  int64_t first;                                    // row of a launch

  __device__ __forceinline__ int64_t start(int64_t row) const {              // of a row's logits
    const uint32_t s = (uint32_t)row / rows;
    return s * lds + ((uint32_t)row - s * rows) * ldx;
  }
};

// A whole number that orders logits by value and, among equal ones, by the lowest index; a NaN is above everything, -0 equals +0.
// 0 is below every logit's.
__device__ __forceinline__ uint32_t rank_of(float x) {      // the upper half: equal logits, equal ranks
  const uint32_t u = x == x ? f2u(x + 0.0f) : 0x7fc00000u;
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint64_t key_of(float x, uint32_t index) { return (uint64_t)rank_of(x) << 32 | (0xffffffffu - index); }
__device__ __forceinline__ float logit_of(uint64_t key) {
  const uint32_t u = (uint32_t)(key >> 32);
  return u2f((u & 0x80000000u) ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ uint32_t index_of(uint64_t key) { return 0xffffffffu - (uint32_t)key; }

__device__ __forceinline__ uint64_t other_lane(uint64_t v, int lane) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_ds_bpermute(lane * 4, (int)(uint32_t)v), hi = (uint32_t)__builtin_amdgcn_ds_bpermute(lane * 4, (int)(v >> 32));
  return (uint64_t)hi << 32 | lo;
}
// the value that lane i ^ D holds, without LDS: mirrors of a row's 16 lanes, their halves and quads, and swaps of rows
template <int D>
__device__ __forceinline__ uint32_t across(uint32_t v) {
  const auto dpp = [](uint32_t u, auto ctrl) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u, decltype(ctrl)::value, 0xf, 0xf, true); };
  constexpr std::integral_constant<int, 0xB1> xor1; constexpr std::integral_constant<int, 0x4E> xor2; constexpr std::integral_constant<int, 0x1B> xor3;
  constexpr std::integral_constant<int, 0x141> xor7; constexpr std::integral_constant<int, 0x140> xor15;
  if constexpr (D == 1) return dpp(v, xor1);
  else if constexpr (D == 2) return dpp(v, xor2);
  else if constexpr (D == 4) return dpp(dpp(v, xor7), xor3);
  else if constexpr (D == 8) return dpp(dpp(v, xor15), xor7);
  else if constexpr (D == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);     // rows 0, 0, 2, 2 and 1, 1, 3, 3
    return threadIdx.x & 16 ? r[0] : r[1];
  } else {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);     // the lower half twice, and the upper
    return threadIdx.x & 32 ? r[0] : r[1];
  }
}
template <int D> __device__ __forceinline__ uint64_t across(uint64_t v) { return (uint64_t)across<D>((uint32_t)(v >> 32)) << 32 | across<D>((uint32_t)v); }
// lane i and lane i ^ D, in blocks of N lanes whose order turns from block to block (down first): the larger value to the lane it belongs to
template <int D, int N, class K>
__device__ __forceinline__ K exchange(K v) {
  constexpr uint64_t larger = [] {
    uint64_t m = 0;
    for (int l = 0; l < 64; ++l) m |= (uint64_t)(((l & D) == 0) == ((l & N) == 0)) << l;
    return m;
  }();
  const K o = across<D>(v);
  if constexpr (sizeof(K) == 4) return __builtin_amdgcn_inverse_ballot_w64(larger) ? (v > o ? v : o) : (v > o ? o : v);
  else return __builtin_amdgcn_inverse_ballot_w64(~(larger ^ __builtin_amdgcn_ballot_w64(v > o))) ? v : o;
}
// bitonic sequences of N lanes into order, step by step
template <int D, int N, class K>
__device__ __forceinline__ K ordered(K v) {
  if constexpr (D > 0) return ordered<D / 2, N>(exchange<D, N>(v));
  return v;
}
// the wave's 64 values in descending order
template <class K>
__device__ __forceinline__ K sorted(K v) {
  v = ordered<1, 2>(v);
  v = ordered<2, 4>(v);
  v = ordered<4, 8>(v);
  v = ordered<8, 16>(v);
  v = ordered<16, 32>(v);
  return ordered<32, 64>(v);
}
// the 64 largest of two descending lists, `turned` with its lanes in ascending order
__device__ __forceinline__ uint64_t merged(uint64_t v, uint64_t turned) { return ordered<32, 64>(v > turned ? v : turned); }

// The best 64 keys of a wave, one per lane in descending order; of them `k` are wanted.
struct Best {
  uint64_t mine = 0, bound = 0;                     // a key that is not above bound is not among the best k
  bool some = false;                                // `mine` holds something
  int lane, k;
  __device__ __forceinline__ Best(int lane_, int k_) : lane(lane_), k(k_) {}
  // one key per lane (0: none)
  __device__ __forceinline__ void take(uint64_t key) {
    if (__builtin_amdgcn_ballot_w64(key > bound) == 0) return;
    const uint64_t s = sorted(key);
    mine = some ? merged(mine, other_lane(s, 63 - lane)) : s;
    some = true;
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)mine, k - 1), hi = (uint32_t)__builtin_amdgcn_readlane((int)(mine >> 32), k - 1);
    bound = (uint64_t)hi << 32 | lo;
  }
};

struct Sums {
  float c = LOWEST, S = 0.0f, U = 0.0f;
  // to the reference `to` >= c
  __device__ __forceinline__ void refer(float to) {
    const float d = c - to, f = __builtin_amdgcn_exp2f(d * 1.44269504088896340736f);
    U = f * (U + S * nan_max(d, -150.0f));          // (f is 0 below that)
    S *= f;
    c = to;
  }
  __device__ __forceinline__ void add(const Sums& o) { S += o.S; U += o.U; }
  __device__ __forceinline__ void join_wave() {
    refer(team_reduce<64, true>(c));
    S = team_sum<64>(S);
    U = team_sum<64>(U);
  }
};

// The row's first 64 given tokens, one per lane, read early: their logits are on their way while the lists are joined.
template <int BF>
struct Given {
  int64_t token = 0;
  float x = 0.0f;
  __device__ __forceinline__ void tokens(const LogprobArgs& a, int64_t row, int lane) { if (lane < a.m) token = a.tokens[row * a.m + lane]; }
  __device__ __forceinline__ void logits(const LogprobArgs& a, int64_t start, int lane) {
    if (lane < a.m && token >= 0 && token < a.V) x = load_scalar<BF>(a.x, start + token);
  }
};

template <int BF>
__device__ __forceinline__ void answer(const LogprobArgs& a, int64_t row, int64_t start, const Sums& s, Given<BF> g, uint64_t mine, int lane) {
  const float l = logf(s.S);
  if (lane == 0 && a.entropy) a.entropy[row] = l - s.U / s.S;
  for (int64_t j = lane; j < a.m; j += 64) {
    if (j >= 64) {
      g.token = a.tokens[row * a.m + j];
      if (g.token >= 0 && g.token < a.V) g.x = load_scalar<BF>(a.x, start + g.token);
    }
    a.logprobs[row * a.m + j] = g.token == a.ignore ? 0.0f : g.token < 0 || g.token >= a.V ? __builtin_nanf("") : (g.x - s.c) - l;
  }
  if (lane < a.k) {
    a.top_logprobs[row * a.k + lane] = (logit_of(mine) - s.c) - l;
    a.top_tokens[row * a.k + lane] = index_of(mine);
  }
}

constexpr int ROOM = 512;                           // keys that find room

template <int BF, bool TOP, int THREADS>
__global__ __launch_bounds__(THREADS) void logprobs_kernel(LogprobArgs a) {
  constexpr int N = Vec<BF>::N, PASS = THREADS * FLIGHT, WAVES = THREADS / 64, PARTS = THREADS == 1024 ? 8 : 12;
  __shared__ float most[TOP ? PARTS : 1][TOP ? THREADS : 1];                 // largest logit of a lane in each part of the row
  __shared__ uint64_t keys[TOP ? ROOM : 1], lists[TOP ? WAVES : 1][64];
  __shared__ uint32_t ranks[TOP ? WAVES : 1][64];
  __shared__ float sums[WAVES][3];
  __shared__ uint32_t reach;
  __shared__ int count;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = a.first + blockIdx.x, start = a.start(row);
  const char* const x = (const char*)a.x + start * (16 / N);
  const int V = (int)a.V, pieces = (V + N - 1) / N;
  const int last = V / N;                           // (all pieces of the row but its last hold N logits)
  const int passes = (pieces + PASS - 1) / PASS, per = (passes + PARTS - 1) / PARTS;

  Given<BF> given;
  if (wave == 0) given.tokens(a, row, lane);
  Sums s;
  float top = -__builtin_inff();
  // the pieces j0 + f THREADS of this lane; -inf past the row's end
  const auto fetch = [&](u32x4 (&raw)[FLIGHT], int j0) __attribute__((always_inline)) {
    if (j0 + PASS <= last) {
      #pragma unroll
      for (int f = 0; f < FLIGHT; ++f) __builtin_memcpy(&raw[f], x + (uint32_t)(j0 + f * THREADS + (int)threadIdx.x) * 16u, 16);      // (rows may start anywhere)
    } else if (j0 < pieces) {
      #pragma unroll
      for (int f = 0; f < FLIGHT; ++f) {
        const int j = j0 + f * THREADS + (int)threadIdx.x;
        raw[f] = N == 4 ? u32x4{0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u}
                        : u32x4{0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u} & (BF == ROW_F16 ? 0xfc00fc00u : ~0u);
        if (j < last) {
          __builtin_memcpy(&raw[f], x + (uint32_t)j * 16u, 16);
        } else if (j < pieces) {
          float v[N];
          #pragma unroll
          for (int i = 0; i < N; ++i) v[i] = j * N + i < V ? load_scalar<BF>(x, j * N + i) : -__builtin_inff();
          raw[f] = pack<BF>(v);
        }
      }
    }
  };

  // A pass is on its way while the one in front of it is worked on.
  u32x4 one[FLIGHT], two[FLIGHT];
  int part = 0, left = per;
  for (int p = -1; p < passes; ++p) {
    fetch(two, (p + 1) * PASS);
    __builtin_amdgcn_sched_barrier(0);
    if (p >= 0) {
      #pragma unroll
      for (int f = 0; f < FLIGHT; ++f) {
        float v[N];
        unpack<BF>(one[f], v);
        float t = v[0];
        #pragma unroll
        for (int i = 1; i < N; ++i) t = nan_max(t, v[i]);
        if (t > s.c + MOVE) s.refer(t);
        top = nan_max(top, t);
        #pragma unroll
        for (int i = 0; i < N; ++i) {
          const float d = v[i] - s.c, e = __builtin_amdgcn_exp2f(d * 1.44269504088896340736f);
          s.S += e;
          s.U = __builtin_fmaf(e, nan_max(d, -150.0f), s.U); // (-inf: e is 0)
        }
      }
      if (TOP && --left == 0) {
        most[part++][threadIdx.x] = top;
        top = -__builtin_inff();
        left = per;
      }
    }
    #pragma unroll
    for (int f = 0; f < FLIGHT; ++f) one[f] = two[f];
  }
  if (wave == 0) given.logits(a, start, lane);
  s.join_wave();
  if (lane == 0) { sums[wave][0] = s.c; sums[wave][1] = s.S; sums[wave][2] = s.U; }
  Best best(lane, TOP ? a.k : 1);
  if constexpr (TOP) {
    if (left != per) most[part++][threadIdx.x] = top;        // (the last part, cut short)
    for (int p = 0; p < part; ++p) top = nan_max(top, most[p][threadIdx.x]);
    // the k-th largest of the lanes' maxima: sorted by waves, joined by pairs
    uint32_t r = sorted(rank_of(top));
    ranks[wave][lane] = r;
    if (threadIdx.x == 0) count = 0;
    #pragma unroll
    for (int w = 1; w < WAVES; w *= 2) {
      __syncthreads();
      if (wave % (2 * w) == 0) {
        const uint32_t o = ranks[wave + w][63 - lane];
        r = ordered<32, 64>(r > o ? r : o);
        ranks[wave][lane] = r;
      }
    }
    if (wave == 0 && lane == a.k - 1) reach = r;
    __syncthreads();
    const uint32_t bound = reach;
    const auto keep = [&](float v, int at) {
      const int c = __hip_atomic_fetch_add(&count, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
      if (c < ROOM) keys[c] = key_of(v, (uint32_t)at);
    };
    // every logit that reaches it: each lane goes through those of its parts that do, so that the few that have any go side by side
    uint32_t todo = 0;
    for (int q = 0; q < part; ++q) todo |= (uint32_t)(rank_of(most[q][threadIdx.x]) >= bound) << q;
    while (todo) {
      const int q = __builtin_ctz(todo);
      todo &= todo - 1;
      const int end = (q + 1) * per < passes ? (q + 1) * per : passes;
      constexpr int SOME = 6;                       // pieces on their way at once
      for (int p = q * per * FLIGHT; p < end * FLIGHT; p += SOME) {
        u32x4 raw[SOME];
        const auto piece = [&](int i) { return (p + i) * THREADS + (int)threadIdx.x; };
        #pragma unroll
        for (int i = 0; i < SOME; ++i)
          if (p + i < end * FLIGHT && piece(i) < last) __builtin_memcpy(&raw[i], x + (uint32_t)piece(i) * 16u, 16);
        #pragma unroll
        for (int i = 0; i < SOME; ++i) {
          if (p + i >= end * FLIGHT || piece(i) >= last) continue;
          float v[N];
          unpack<BF>(raw[i], v);
          #pragma unroll
          for (int e = 0; e < N; ++e)
            if (rank_of(v[e]) >= bound) keep(v[e], piece(i) * N + e);
        }
        #pragma unroll 1
        for (int at = last * N; at < V; ++at) {     // (the row's last piece, if it is among these)
          const int i = (last / THREADS) - p;
          if (i < 0 || i >= SOME || p + i >= end * FLIGHT || last % THREADS != (int)threadIdx.x) break;
          const float v = load_scalar<BF>(x, at);
          if (rank_of(v) >= bound) keep(v, at);
        }
      }
    }
    __syncthreads();
    if (count > ROOM) {                             // (the same in all waves)
      #pragma unroll 1
      for (int v0 = wave * 64 + lane; v0 - lane < V; v0 += THREADS * 8) {
        float v[8];
        #pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = v0 + i * THREADS < V ? load_scalar<BF>(x, v0 + i * THREADS) : 0.0f;
        #pragma unroll 1
        for (int i = 0; i < 8; ++i) {               // (one copy of the sort)
          float e = v[0];
          #pragma unroll
          for (int j = 1; j < 8; ++j) e = i == j ? v[j] : e;
          const int at = v0 + i * THREADS;
          best.take(at < V ? key_of(e, (uint32_t)at) : 0);
        }
      }
      lists[wave][lane] = best.mine;
    }
  }
  __syncthreads();
  if (wave) return;
  float c = s.c;
  #pragma unroll
  for (int w = 1; w < WAVES; ++w) c = nan_max(c, sums[w][0]);
  s.refer(c);
  #pragma unroll
  for (int w = 1; w < WAVES; ++w) {
    Sums o;
    o.c = sums[w][0]; o.S = sums[w][1]; o.U = sums[w][2];
    o.refer(c);
    s.add(o);
  }
  if constexpr (TOP) {
    if (count > ROOM) {
      #pragma unroll 1
      for (int w = 1; w < WAVES; ++w) best.mine = merged(best.mine, lists[w][63 - lane]);
    } else {
      #pragma unroll 1
      for (int i = 0; i < count; i += 64) best.take(i + lane < count ? keys[i + lane] : 0);
    }
  }
  answer<BF>(a, row, start, s, given, best.mine, lane);
}

}  // namespace

extern "C" {

int lcq_token_logprobs_of(const void* logits, int dtype, int64_t B, int64_t S, int64_t V, int64_t lds, int64_t ldx, const int64_t* tokens,
                          int64_t m, int64_t ignore, float* logprobs, float* entropy, int k, float* top_logprobs, int64_t* top_tokens,
                          void* stream) {
  if (!logits || B <= 0 || S <= 0 || V <= 0 || lds < 0 || ldx < 0 || m < 0 || k < 0 || k > 64 || k > V) return LCQ_EINVAL;
  if ((m > 0 && (!tokens || !logprobs)) || (k > 0 && (!top_logprobs || !top_tokens))) return LCQ_EINVAL;
  if (dtype != LCQ_F32 && dtype != LCQ_BF16 && dtype != LCQ_F16) return LCQ_EDTYPE;
  if (S > 0x7fffffff || B > 0x7fffffff / S || V > (1 << 28)) return LCQ_ESIZE;
  if ((uintptr_t)logits % (dtype == LCQ_F32 ? 4 : 2)) return LCQ_EALIGN;
  const int64_t T = B * S;
  const LogprobArgs a = {logits, tokens, logprobs, entropy, top_logprobs, top_tokens, V, ldx, lds, m, ignore, (uint32_t)S, k, 0};
  const auto launch = [&](auto bf, auto threads) {
    constexpr int BF = decltype(bf)::value, THREADS = decltype(threads)::value;
    constexpr int64_t rows = 1 << 21;               // (a launch has fewer than 2^32 lanes)
    LogprobArgs part = a;
    for (; part.first < T; part.first += rows) {
      const dim3 grid((unsigned)(T - part.first < rows ? T - part.first : rows)), block(THREADS);
      if (k) logprobs_kernel<BF, true, THREADS><<<grid, block, 0, (hipStream_t)stream>>>(part);
      else logprobs_kernel<BF, false, THREADS><<<grid, block, 0, (hipStream_t)stream>>>(part);
    }
  };
  const auto run = [&](auto bf) {
    if (T <= 256) launch(bf, std::integral_constant<int, 1024>{});
    else if (T <= 1024) launch(bf, std::integral_constant<int, 512>{});
    else launch(bf, std::integral_constant<int, 256>{});
  };
  if (dtype == LCQ_BF16) run(std::integral_constant<int, ROW_BF16>{});
  else if (dtype == LCQ_F16) run(std::integral_constant<int, ROW_F16>{});
  else run(std::integral_constant<int, ROW_F32>{});
  LCQ_CHECK_LAUNCH();
  return LCQ_OK;
}

int lcq_token_logprobs(const void* logits, int dtype, int64_t T, int64_t V, int64_t ldx, const int64_t* tokens, int64_t m,
                       int64_t ignore, float* logprobs, float* entropy, int k, float* top_logprobs, int64_t* top_tokens,
                       void* stream) {
  return lcq_token_logprobs_of(logits, dtype, 1, T, V, 0, ldx, tokens, m, ignore, logprobs, entropy, k, top_logprobs, top_tokens, stream);
}

}  // extern "C"

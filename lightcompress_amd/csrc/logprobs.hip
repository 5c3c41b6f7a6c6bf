// Log probabilities of given tokens, entropy and best alternatives of logits x [T, V], in one pass over them:
//   S = sum exp(x - c),  U = sum exp(x - c) (x - c)   for any reference c
//   log sum exp x = c + log S;   logprob of a token t = (x_t - c) - log S;   entropy = log S - U / S
//
//  * A lane keeps its own c, S and U.  c is a logit that the lane has seen; it moves only where a later one is more than 8 above
//    it, so that almost no piece pays for a change of reference, S stays below V e^8 and log S and U / S do not cancel to more than a few
//    times their last bits.  References meet once, when lanes, waves and parts are joined.
//  * The best alternatives: each wave keeps 64 keys, one per lane in descending order.  A key is a whole number that orders by value
//    and then by the lowest index.  A 16-byte piece whose maximum lies below the k-th best so far costs one comparison; what passes is
//    collected in LDS and taken over 64 at a time (a bitonic sort, then a merge).  Where many lanes pass at once (the first piece,
//    ascending logits) the k-th best of the lanes' maxima is a bound first.
//  * A row is one workgroup's where there are enough rows, else it is cut into parts of whole 256-lane passes for about four workgroups
//    per CU, which leave (c, S, U) and k keys each for a second, small kernel.
#include "rowquant.h"
#include <type_traits>

namespace {
using namespace lcq;

constexpr float LOWEST = -3.4028234663852886e38f, MOVE = 8.0f;
constexpr int THREADS = 256, WAVES = THREADS / 64;
constexpr int FLIGHT = 2;                           // 16-byte pieces that a lane has on their way while it works on as many

struct LogprobArgs {
  const void* x;
  const int64_t* tokens;
  float *logprobs, *entropy, *top_logprobs;
  int64_t* top_tokens;
  int64_t V, ldx, m, ignore;
  int k, parts;
  int per;                                          // 16-byte pieces of a part
  f32x4* sums;                                      // [T, parts]: c, S, U
  uint64_t* keys;                                   // [T, parts, k]
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

// The best 64 of a wave.  `bound`, `limit` and `some` are the same in all lanes.
struct Best {
  uint64_t mine = 0, bound = 0;                   
  float limit = -__builtin_inff();                  // a logit below it is not among the best k
  bool some = false;                                // `mine` holds something
  int lane, k;
  __device__ __forceinline__ Best(int lane_, int k_) : lane(lane_), k(k_) {}
  // at least k keys lie above `key`; the k-th best logit is that of `rank` or larger
  __device__ __forceinline__ void raise(uint64_t key, uint32_t rank) {
    if (key <= bound) return;
    bound = key;
    const float x = logit_of((uint64_t)rank << 32);
    limit = x == x ? x : __builtin_inff();          // (k NaNs: whatever is not one stays out; a NaN passes every limit)
  }
  // at least k logits reach `rank`; keys of that rank are still to be collected
  __device__ __forceinline__ void raise_to(uint32_t rank) { if (rank) raise(((uint64_t)rank << 32) - 1, rank); }
  // the k-th largest of 64 ranks
  __device__ __forceinline__ uint32_t kth(uint32_t rank) const { return (uint32_t)__builtin_amdgcn_readlane((int)sorted(rank), k - 1); }
  // one key per lane (0: none)
  __device__ __forceinline__ void take(uint64_t key) {
    if (__builtin_amdgcn_ballot_w64(key > bound) == 0) return;
    const uint64_t s = sorted(key);
    mine = some ? merged(mine, other_lane(s, 63 - lane)) : s;
    some = true;
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)mine, k - 1), hi = (uint32_t)__builtin_amdgcn_readlane((int)(mine >> 32), k - 1);
    if (hi) raise((uint64_t)hi << 32 | lo, hi);
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

// The waves' sums joined in wave 0 -> true there.  Its barrier is also what the waves' lists in LDS wait for.
__device__ __forceinline__ bool join_sums(Sums& s) {
  __shared__ float part[WAVES][3];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  s.join_wave();
  if (lane == 0) { part[wave][0] = s.c; part[wave][1] = s.S; part[wave][2] = s.U; }
  __syncthreads();
  if (wave) return false;
  float c = s.c;
  #pragma unroll
  for (int w = 1; w < WAVES; ++w) c = nan_max(c, part[w][0]);
  s.refer(c);
  #pragma unroll
  for (int w = 1; w < WAVES; ++w) {
    Sums o;
    o.c = part[w][0]; o.S = part[w][1]; o.U = part[w][2];
    o.refer(c);
    s.add(o);
  }
  return true;
}
// What the waves of a workgroup collect: keys that may be among the best k, in LDS until there are 64 of them.
template <int ROOM>
struct Lists {
  uint64_t found[WAVES][ROOM], best[WAVES][64];
  int count[WAVES], some[WAVES];
  uint32_t rank;                                    // at least k logits of the row reach it: the best of the waves' bounds
};
template <int ROOM>
struct Collector {
  Lists<ROOM>& l;
  Best best;
  int count = 0, wave;
  __device__ __forceinline__ Collector(Lists<ROOM>& l_, int wave_, int lane, int k) : l(l_), best(lane, k), wave(wave_) {}
  __device__ __forceinline__ void collect(bool in, uint64_t key) {
    const uint64_t lanes = __builtin_amdgcn_ballot_w64(in);
    if (in) l.found[wave][count + __builtin_amdgcn_mbcnt_hi((uint32_t)(lanes >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)lanes, 0))] = key;
    count += __builtin_popcountll(lanes);
  }
  __device__ __forceinline__ void drain() {
    #pragma unroll 1
    for (int at = 0; at < count; at += 64) best.take(at + best.lane < count ? l.found[wave][at + best.lane] : 0);
    count = 0;
  }
  __device__ __forceinline__ void share() {
    if (best.lane == 0 && best.bound) __hip_atomic_fetch_max(&l.rank, (uint32_t)((best.bound + 1) >> 32), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
  }
  __device__ __forceinline__ uint32_t shared() const { return __hip_atomic_load(&l.rank, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP); }
  __device__ __forceinline__ void leave() {         // for the wave that joins them, behind a barrier
    if (best.some) l.best[wave][best.lane] = best.mine;
    if (best.lane == 0) { l.count[wave] = count; l.some[wave] = best.some; }
  }
  // wave 0: everything that the waves have collected and not sorted, 64 at a time, then their lists
  __device__ __forceinline__ void join() {
    int end[WAVES], total = 0;
    #pragma unroll
    for (int w = 0; w < WAVES; ++w) end[w] = total += l.count[w];
    #pragma unroll 1
    for (int at = 0; at < total; at += 64) {
      const int i = at + best.lane;
      int w = 0, begin = 0;
      #pragma unroll
      for (int v = 0; v < WAVES - 1; ++v)
        if (i >= end[v]) { w = v + 1; begin = end[v]; }
      best.take(i < total ? l.found[w][i - begin] : 0);
    }
    #pragma unroll 1
    for (int w = 1; w < WAVES; ++w)
      if (l.some[w]) {
        best.mine = best.some ? merged(best.mine, l.best[w][63 - best.lane]) : l.best[w][best.lane];
        best.some = true;
      }
  }
};

// The row's first 64 given tokens, one per lane, read early: their logits are on their way while the lists are joined.
template <int BF>
struct Given {
  int64_t token = 0;
  float x = 0.0f;
  __device__ __forceinline__ void tokens(const LogprobArgs& a, int64_t row, int lane) { if (lane < a.m) token = a.tokens[row * a.m + lane]; }
  __device__ __forceinline__ void logits(const LogprobArgs& a, int64_t row, int lane) {
    if (lane < a.m && token >= 0 && token < a.V) x = load_scalar<BF>(a.x, row * a.ldx + token);
  }
};

template <int BF>
__device__ __forceinline__ void answer(const LogprobArgs& a, int64_t row, const Sums& s, Given<BF> g, uint64_t mine, int lane) {
  const float l = logf(s.S);
  if (lane == 0 && a.entropy) a.entropy[row] = l - s.U / s.S;
  for (int64_t j = lane; j < a.m; j += 64) {
    if (j >= 64) {
      g.token = a.tokens[row * a.m + j];
      if (g.token >= 0 && g.token < a.V) g.x = load_scalar<BF>(a.x, row * a.ldx + g.token);
    }
    a.logprobs[row * a.m + j] = g.token == a.ignore ? 0.0f : g.token < 0 || g.token >= a.V ? __builtin_nanf("") : (g.x - s.c) - l;
  }
  if (lane < a.k) {
    a.top_logprobs[row * a.k + lane] = (logit_of(mine) - s.c) - l;
    a.top_tokens[row * a.k + lane] = index_of(mine);
  }
}

template <int BF, bool TOP>
__global__ __launch_bounds__(THREADS) void logprobs_kernel(LogprobArgs a) {
  constexpr int N = Vec<BF>::N, PASS = THREADS * FLIGHT;
  __shared__ Lists<TOP ? 64 * N + 64 : 1> lists;
  if constexpr (TOP) {
    if (threadIdx.x == 0) lists.rank = 0;
    __syncthreads();
  }
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = blockIdx.x;
  const int part = blockIdx.y;
  const char* const x = (const char*)a.x + row * a.ldx * (16 / N);
  const int V = (int)a.V, pieces = (V + N - 1) / N;
  const int from = part * a.per, to = from + a.per < pieces ? from + a.per : pieces;

  Given<BF> given;
  if (a.parts == 1 && wave == 0) given.tokens(a, row, lane);
  Sums s;
  Collector<TOP ? 64 * N + 64 : 1> c(lists, wave, lane, TOP ? a.k : 1);
  // the pieces j0 + f THREADS of this lane
  const auto take = [&](const u32x4 (&raw)[FLIGHT], int j0) __attribute__((always_inline)) {
    float top[FLIGHT];
    float limit = c.best.limit;
    if constexpr (TOP) {
      const float theirs = logit_of((uint64_t)c.shared() << 32);
      limit = theirs > limit ? theirs : limit;
    }
    #pragma unroll
    for (int f = 0; f < FLIGHT; ++f) {
      float v[N];
      unpack<BF>(raw[f], v);
      top[f] = v[0];
      #pragma unroll
      for (int i = 1; i < N; ++i) top[f] = nan_max(top[f], v[i]);
      if (top[f] > s.c + MOVE) s.refer(top[f]);
      #pragma unroll
      for (int i = 0; i < N; ++i) {
        const float d = v[i] - s.c, e = __builtin_amdgcn_exp2f(d * 1.44269504088896340736f);
        s.S += e;
        s.U = __builtin_fmaf(e, nan_max(d, -150.0f), s.U);   // (-inf: e is 0)
      }
    }
    if constexpr (TOP) {
      float most = top[0];
      #pragma unroll
      for (int f = 1; f < FLIGHT; ++f) most = nan_max(most, top[f]);
      const uint64_t pass = __builtin_amdgcn_ballot_w64(!(most < limit));
      if (__builtin_expect(pass != 0, 0)) {
        c.best.raise_to(c.shared());
        if (__builtin_popcountll(pass) > 16) {
          c.best.raise_to(c.best.kth(rank_of(most)));
          c.share();
        }
        #pragma unroll 1
        for (int f = 0; f < FLIGHT; ++f) {          // (one copy of the code for all of them)
          u32x4 r = raw[0];
          float t = top[0];
          #pragma unroll
          for (int g = 1; g < FLIGHT; ++g) { r = f == g ? raw[g] : r; t = f == g ? top[g] : t; }
          if (__builtin_amdgcn_ballot_w64(!(t < c.best.limit)) == 0) continue;
          const int64_t v0 = (int64_t)(j0 + f * THREADS + (int)threadIdx.x) * N;             // (past the row's end: holds nothing)
          float v[N];
          unpack<BF>(r, v);
          #pragma unroll
          for (int i = 0; i < N; ++i) {
            if (__builtin_amdgcn_ballot_w64(!(v[i] < c.best.limit)) == 0) continue;
            const uint64_t key = v0 + i < V ? key_of(v[i], (uint32_t)(v0 + i)) : 0;
            c.collect(key > c.best.bound, key);
          }
          if (c.count >= 64) {
            c.drain();
            c.share();
          }
        }
      }
    }
  };

  // A pass is on its way while the one in front of it is worked on.  Rows may start anywhere.
  const int last = to < V / N ? to : V / N;         // (all pieces of the row but its last hold N logits)
  u32x4 one[FLIGHT], two[FLIGHT];
  for (int j0 = from - PASS; j0 < to; j0 += PASS) {
    const int next = j0 + PASS;
    if (next + PASS <= last) {
      #pragma unroll
      for (int f = 0; f < FLIGHT; ++f) __builtin_memcpy(&two[f], x + (uint32_t)(next + f * THREADS + (int)threadIdx.x) * 16u, 16);
    } else if (next < to) {
      #pragma unroll
      for (int f = 0; f < FLIGHT; ++f) {
        const int j = next + f * THREADS + (int)threadIdx.x;
        two[f] = N == 4 ? u32x4{0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u}          // -inf
                        : u32x4{0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u} & (BF == ROW_F16 ? 0xfc00fc00u : ~0u);
        if (j < last) {
          __builtin_memcpy(&two[f], x + (uint32_t)j * 16u, 16);
        } else if (j < to) {
          float v[N];
          #pragma unroll
          for (int i = 0; i < N; ++i) v[i] = j * N + i < V ? load_scalar<BF>(x, j * N + i) : -__builtin_inff();
          two[f] = pack<BF>(v);
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    if (j0 >= from) take(one, j0);
    #pragma unroll
    for (int f = 0; f < FLIGHT; ++f) one[f] = two[f];
  }
  if (a.parts == 1 && wave == 0) given.logits(a, row, lane);
  if constexpr (TOP) c.leave();
  if (!join_sums(s)) return;
  if constexpr (TOP) c.join();
  if (a.parts == 1) {
    answer<BF>(a, row, s, given, c.best.mine, lane);
    return;
  }
  const int64_t at = row * a.parts + part;
  if (lane == 0) a.sums[at] = f32x4{s.c, s.S, s.U, 0.0f};
  if (lane < a.k) a.keys[at * a.k + lane] = c.best.mine;
}

// The parts of a row joined: one workgroup per row.
template <int BF>
__global__ __launch_bounds__(THREADS) void join_kernel(LogprobArgs a) {
  __shared__ Lists<128> lists;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = blockIdx.x;
  Given<BF> given;
  if (wave == 0) given.tokens(a, row, lane);
  const f32x4* const sums = a.sums + row * a.parts;
  const int all = a.parts * a.k;
  const uint64_t* const keys = a.keys + row * all;
  constexpr int KEEP = 8;                           // loads that a lane has in flight
  uint64_t key[KEEP];
  const auto fetch = [&](int at) __attribute__((always_inline)) {
    #pragma unroll
    for (int i = 0; i < KEEP; ++i) key[i] = at + i * THREADS + (int)threadIdx.x < all ? keys[at + i * THREADS + threadIdx.x] : 0;
  };
  f32x4 v = {LOWEST, 0.0f, 0.0f, 0.0f};
  if ((int)threadIdx.x < a.parts) v = sums[threadIdx.x];
  fetch(0);
  Sums s;
  for (int p = threadIdx.x;;) {
    Sums o;
    o.c = v[0]; o.S = v[1]; o.U = v[2];
    const float c = nan_max(s.c, o.c);
    s.refer(c);
    o.refer(c);
    s.add(o);
    if ((p += THREADS) >= a.parts) break;
    v = sums[p];
  }
  if (wave == 0) given.logits(a, row, lane);
  Collector<128> c(lists, wave, lane, a.k > 0 ? a.k : 1);
  #pragma unroll 1
  for (int at = 0; at < all; at += KEEP * THREADS) {
    if (at) fetch(at);
    uint32_t most = 0;
    #pragma unroll
    for (int i = 0; i < KEEP; ++i) most = (uint32_t)(key[i] >> 32) > most ? (uint32_t)(key[i] >> 32) : most;
    if (__builtin_popcountll(__builtin_amdgcn_ballot_w64(most > (uint32_t)(c.best.bound >> 32))) > 16) c.best.raise_to(c.best.kth(most));
    #pragma unroll
    for (int i = 0; i < KEEP; ++i) {
      if (__builtin_amdgcn_ballot_w64(key[i] > c.best.bound) == 0) continue;
      c.collect(key[i] > c.best.bound, key[i]);
      if (c.count >= 64) c.drain();
    }
  }
  c.leave();
  if (!join_sums(s)) return;
  if (all) c.join();
  answer<BF>(a, row, s, given, c.best.mine, lane);
}

int parts_of(int64_t T, int64_t V, int dtype) {
  const int64_t passes = (V * (dtype == LCQ_F32 ? 4 : 2) + 16 * THREADS - 1) / (16 * THREADS);
  const int64_t want = 1024 / T;
  return (int)(want < 1 ? 1 : want < passes ? want : passes);
}

}  // namespace

extern "C" {

int64_t lcq_token_logprobs_workspace_bytes(int64_t T, int64_t V, int k) {
  if (T <= 0 || V <= 0 || k < 0) return 0;
  const int parts = parts_of(T, V, LCQ_F32);        // (the most there are)
  return parts == 1 ? 0 : T * parts * (16 + 8 * (int64_t)k);
}

int lcq_token_logprobs(const void* logits, int dtype, int64_t T, int64_t V, int64_t ldx, const int64_t* tokens, int64_t m,
                       int64_t ignore, float* logprobs, float* entropy, int k, float* top_logprobs, int64_t* top_tokens,
                       void* workspace, void* stream) {
  if (!logits || T <= 0 || V <= 0 || ldx < 0 || m < 0 || k < 0 || k > 64 || k > V) return LCQ_EINVAL;
  if ((m > 0 && (!tokens || !logprobs)) || (k > 0 && (!top_logprobs || !top_tokens))) return LCQ_EINVAL;
  if (dtype != LCQ_F32 && dtype != LCQ_BF16 && dtype != LCQ_F16) return LCQ_EDTYPE;
  if (T > 0x7fffffff || V > (1 << 28)) return LCQ_ESIZE;
  if ((uintptr_t)logits % (dtype == LCQ_F32 ? 4 : 2)) return LCQ_EALIGN;
  LogprobArgs a = {logits, tokens, logprobs, entropy, top_logprobs, top_tokens, V, ldx, m, ignore, k, parts_of(T, V, dtype), 0, nullptr, nullptr};
  if (a.parts > 1) {
    if (!workspace) return LCQ_EWORKSPACE;
    if ((uintptr_t)workspace % 16) return LCQ_EALIGN;
    a.sums = (f32x4*)workspace;
    a.keys = (uint64_t*)(a.sums + T * a.parts);
  }
  const int n = dtype == LCQ_F32 ? 4 : 8;
  a.per = (int)(((V + n - 1) / n + a.parts - 1) / a.parts);
  const dim3 grid((unsigned)T, (unsigned)a.parts), block(THREADS);
  hipStream_t st = (hipStream_t)stream;
  const auto run = [&](auto bf) {
    constexpr int BF = decltype(bf)::value;
    if (k) logprobs_kernel<BF, true><<<grid, block, 0, st>>>(a);
    else logprobs_kernel<BF, false><<<grid, block, 0, st>>>(a);
    if (a.parts > 1) join_kernel<BF><<<dim3((unsigned)T), block, 0, st>>>(a);
  };
  if (dtype == LCQ_BF16) run(std::integral_constant<int, ROW_BF16>{});
  else if (dtype == LCQ_F16) run(std::integral_constant<int, ROW_F16>{});
  else run(std::integral_constant<int, ROW_F32>{});
  LCQ_CHECK_LAUNCH();
  return LCQ_OK;
}

}  // extern "C"

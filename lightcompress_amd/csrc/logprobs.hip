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
__device__ __forceinline__ uint64_t key_of(float x, uint32_t index) {
  uint32_t u = x == x ? f2u(x + 0.0f) : 0x7fc00000u;
  u = (u & 0x80000000u) ? ~u : u | 0x80000000u;
  return (uint64_t)u << 32 | (0xffffffffu - index);
}
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
// lane i and lane i ^ D: the larger key to the lower lane where `down`, else the other way
template <int D>
__device__ __forceinline__ uint64_t exchange(uint64_t v, int lane, bool down) {
  const uint64_t o = (uint64_t)across<D>((uint32_t)(v >> 32)) << 32 | across<D>((uint32_t)v);
  return (((lane & D) == 0) == down) == (v > o) ? v : o;
}
// a bitonic sequence of N lanes into order
template <int N>
__device__ __forceinline__ uint64_t ordered(uint64_t v, int lane, bool down) {
  if constexpr (N > 1) return ordered<N / 2>(exchange<N / 2>(v, lane, down), lane, down);
  return v;
}
// the wave's 64 keys in descending order
__device__ __forceinline__ uint64_t sorted(uint64_t v, int lane) {
  v = ordered<2>(v, lane, (lane & 2) == 0);
  v = ordered<4>(v, lane, (lane & 4) == 0);
  v = ordered<8>(v, lane, (lane & 8) == 0);
  v = ordered<16>(v, lane, (lane & 16) == 0);
  v = ordered<32>(v, lane, (lane & 32) == 0);
  return ordered<64>(v, lane, true);
}
// the 64 largest of two descending lists, `turned` with its lanes in ascending order
__device__ __forceinline__ uint64_t merged(uint64_t v, uint64_t turned, int lane) { return ordered<64>(v > turned ? v : turned, lane, true); }

// The best 64 of a wave.  `count` and `bound` are the same in all lanes.
struct Best {
  uint64_t mine = 0, bound = 0;                     // lane i: the i-th best; the k-th best, 0 while there are fewer
  float limit = -__builtin_inff();                  // bound's logit: a logit below it is not among the best k
  int lane, k;
  __device__ __forceinline__ Best(int lane_, int k_) : lane(lane_), k(k_) {}
  __device__ __forceinline__ void raise(uint64_t key) {
    if (key > bound) { bound = key; limit = logit_of(key); }
    limit = limit == limit ? limit : __builtin_inff();       // (k NaNs: whatever is not one stays out; a NaN passes every limit)
  }
  __device__ __forceinline__ uint64_t kth(uint64_t v) const {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, k - 1), hi = (uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), k - 1);
    return (uint64_t)hi << 32 | lo;
  }
  // one key per lane (0: none)
  __device__ __forceinline__ void take(uint64_t key) {
    if (__builtin_amdgcn_ballot_w64(key > bound) == 0) return;
    mine = merged(mine, other_lane(sorted(key, lane), 63 - lane), lane);
    raise(kth(mine));
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

// What a workgroup's waves found, joined in wave 0 -> true there
template <bool TOP>
__device__ __forceinline__ bool join_waves(Sums& s, Best& best) {
  __shared__ float part[WAVES][3];
  __shared__ uint64_t keys[TOP ? WAVES : 1][64];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  s.join_wave();
  if (lane == 0) { part[wave][0] = s.c; part[wave][1] = s.S; part[wave][2] = s.U; }
  if (TOP) keys[wave][lane] = best.mine;
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
    if (TOP) best.mine = merged(best.mine, keys[w][63 - lane], lane);
  }
  return true;
}

template <int BF>
__device__ __forceinline__ void answer(const LogprobArgs& a, int64_t row, const Sums& s, uint64_t mine, int lane) {
  const float l = logf(s.S);
  if (lane == 0 && a.entropy) a.entropy[row] = l - s.U / s.S;
  for (int64_t j = lane; j < a.m; j += 64) {
    const int64_t t = a.tokens[row * a.m + j];
    a.logprobs[row * a.m + j] = t == a.ignore ? 0.0f : t < 0 || t >= a.V ? __builtin_nanf("") : (load_scalar<BF>(a.x, row * a.ldx + t) - s.c) - l;
  }
  if (lane < a.k) {
    a.top_logprobs[row * a.k + lane] = (logit_of(mine) - s.c) - l;
    a.top_tokens[row * a.k + lane] = index_of(mine);
  }
}

template <int BF, bool TOP>
__global__ __launch_bounds__(THREADS) void logprobs_kernel(LogprobArgs a) {
  constexpr int N = Vec<BF>::N, PASS = THREADS * FLIGHT;
  __shared__ uint64_t found[TOP ? WAVES : 1][TOP ? 64 * N + 64 : 1];
  __shared__ uint32_t shared;                       // the upper half of a key: the largest k-th best that a wave has
  if (threadIdx.x == 0) shared = 0;
  if constexpr (TOP) __syncthreads();
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = (int64_t)blockIdx.x / a.parts;
  const int part = (int)((int64_t)blockIdx.x - row * a.parts);
  const char* const x = (const char*)a.x + row * a.ldx * (16 / N);
  const int V = (int)a.V, pieces = (V + N - 1) / N;
  const int from = part * a.per, to = from + a.per < pieces ? from + a.per : pieces;

  Sums s;
  Best best(lane, TOP ? a.k : 1);
  int count = 0;
  const auto drain = [&]() __attribute__((always_inline)) {                          // takes over what was collected
    for (int at = 0; at < count; at += 64) best.take(at + lane < count ? found[wave][at + lane] : 0);
    count = 0;
  };
  // The waves share the best of their bounds: what lies below one wave's k-th best is not among the row's.
  const auto share = [&]() __attribute__((always_inline)) {
    if (lane == 0 && best.bound) __hip_atomic_fetch_max(&shared, (uint32_t)(best.bound >> 32), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
  };
  // piece j of the row, its largest logit `top` (one that lies past the row's end holds nothing): what of it may be among the best
  const auto consider = [&](const u32x4& raw, float top, int j) __attribute__((always_inline)) {
    float v[N];
    unpack<BF>(raw, v);
    if (__builtin_popcountll(__builtin_amdgcn_ballot_w64(!(top < best.limit))) > 16) {
      uint64_t m = 0;
      #pragma unroll
      for (int i = 0; i < N; ++i) {
        const uint64_t key = (int64_t)j * N + i < V ? key_of(v[i], (uint32_t)(j * N + i)) : 0;
        m = key > m ? key : m;
      }
      m = best.kth(sorted(m, lane));
      if (m) best.raise(m - 1);                     // (less one: the k-th itself has still to be collected)
      share();
    }
    #pragma unroll
    for (int i = 0; i < N; ++i) {
      if (__builtin_amdgcn_ballot_w64(!(v[i] < best.limit)) == 0) continue;
      const uint64_t key = (int64_t)j * N + i < V ? key_of(v[i], (uint32_t)(j * N + i)) : 0;
      const bool in = key > best.bound && !(v[i] < best.limit);
      const uint64_t lanes = __builtin_amdgcn_ballot_w64(in);
      if (in) found[wave][count + __builtin_amdgcn_mbcnt_hi((uint32_t)(lanes >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)lanes, 0))] = key;
      count += __builtin_popcountll(lanes);
    }
    if (count >= 64) {
      drain();
      share();
    }
  };
  // the pieces j0 + f THREADS of this lane
  const auto take = [&](const u32x4 (&raw)[FLIGHT], int j0) __attribute__((always_inline)) {
    float top[FLIGHT];
    uint64_t pass[FLIGHT], any = 0;
    if constexpr (TOP) {
      const float theirs = logit_of((uint64_t)__hip_atomic_load(&shared, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP) << 32);
      best.limit = theirs > best.limit ? theirs : best.limit;
    }
    #pragma unroll
    for (int f = 0; f < FLIGHT; ++f) {
      float v[N];
      unpack<BF>(raw[f], v);
      top[f] = v[0];
      #pragma unroll
      for (int i = 1; i < N; ++i) top[f] = nan_max(top[f], v[i]);
      if constexpr (TOP) any |= pass[f] = __builtin_amdgcn_ballot_w64(!(top[f] < best.limit));
      if (top[f] > s.c + MOVE) s.refer(top[f]);
      #pragma unroll
      for (int i = 0; i < N; ++i) {
        const float d = v[i] - s.c, e = __builtin_amdgcn_exp2f(d * 1.44269504088896340736f);
        s.S += e;
        s.U = __builtin_fmaf(e, nan_max(d, -150.0f), s.U);   // (-inf: e is 0)
      }
    }
    if constexpr (TOP) {
      if (__builtin_expect(any != 0, 0)) {
        #pragma unroll 1
        for (int f = 0; f < FLIGHT; ++f) {          // (one copy of the code for all of them)
          u32x4 r = raw[0];
          float t = top[0];
          uint64_t p = pass[0];
          #pragma unroll
          for (int g = 1; g < FLIGHT; ++g) { r = f == g ? raw[g] : r; t = f == g ? top[g] : t; p = f == g ? pass[g] : p; }
          if (p) consider(r, t, j0 + f * THREADS + (int)threadIdx.x);
        }
      }
    }
  };
  const auto fetch = [&](u32x4 (&raw)[FLIGHT], int j0) {    // whole pieces
    #pragma unroll
    for (int f = 0; f < FLIGHT; ++f) __builtin_memcpy(&raw[f], x + (uint32_t)(j0 + f * THREADS + (int)threadIdx.x) * 16u, 16);      // (rows may start anywhere)
  };

  // whole passes, one of them on its way while another is worked on
  const int last = to < V / N ? to : V / N;         // (all pieces of the row but its last hold N logits)
  int j0 = from;
  u32x4 one[FLIGHT], two[FLIGHT];
  if (j0 + PASS <= last) fetch(one, j0);
  while (j0 + 2 * PASS <= last) {
    fetch(two, j0 + PASS);
    __builtin_amdgcn_sched_barrier(0);
    take(one, j0);
    j0 += PASS;
    #pragma unroll
    for (int f = 0; f < FLIGHT; ++f) one[f] = two[f];
  }
  if (j0 + PASS <= last) {
    take(one, j0);
    j0 += PASS;
  }
  // what is left, less than a pass and the row's last piece
  for (; j0 < to; j0 += PASS) {
    #pragma unroll
    for (int f = 0; f < FLIGHT; ++f) {
      const int j = j0 + f * THREADS + (int)threadIdx.x;
      one[f] = N == 4 ? u32x4{0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u}            // -inf
                      : u32x4{0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u} & (BF == ROW_F16 ? 0xfc00fc00u : ~0u);
      if (j < last) {
        __builtin_memcpy(&one[f], x + (uint32_t)j * 16u, 16);
      } else if (j < to) {
        float v[N];
        #pragma unroll
        for (int i = 0; i < N; ++i) v[i] = j * N + i < V ? load_scalar<BF>(x, j * N + i) : -__builtin_inff();
        one[f] = pack<BF>(v);
      }
    }
    take(one, j0);
  }
  if constexpr (TOP) drain();
  if (!join_waves<TOP>(s, best)) return;
  if (a.parts == 1) {
    answer<BF>(a, row, s, best.mine, lane);
    return;
  }
  if (lane == 0) a.sums[blockIdx.x] = f32x4{s.c, s.S, s.U, 0.0f};
  if (lane < a.k) a.keys[(int64_t)blockIdx.x * a.k + lane] = best.mine;
}

// The parts of a row joined: one workgroup per row.
template <int BF>
__global__ __launch_bounds__(THREADS) void join_kernel(LogprobArgs a) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row = blockIdx.x;
  Sums s;
  for (int p = threadIdx.x; p < a.parts; p += THREADS) {
    const f32x4 v = a.sums[row * a.parts + p];
    Sums o;
    o.c = v[0]; o.S = v[1]; o.U = v[2];
    const float c = nan_max(s.c, o.c);
    s.refer(c);
    o.refer(c);
    s.add(o);
  }
  Best best(lane, a.k > 0 ? a.k : 1);
  const int all = a.parts * a.k;
  for (int i = wave * 64; i < all; i += THREADS) best.take(i + lane < all ? a.keys[row * all + i + lane] : 0);
  if (join_waves<true>(s, best)) answer<BF>(a, row, s, best.mine, lane);
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
  const dim3 grid((unsigned)(T * a.parts)), block(THREADS);
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

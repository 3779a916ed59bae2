// Log probabilities of given tokens, the entropy and the most probable alternatives of every
// logits row (fdllm_token_logprobs), in one pass over the logits.
//
//   m = max x,  S = sum e^(x - m),  A = sum (x - m) e^(x - m)
//   log p(t) = x_t - m - log S,     H = -sum p log p = log S - A / S
//
// Each thread holds (m, S, A) of the logits it has read, S and A in powers of two, and rescales when its
// maximum grows (2^d with d = (m - m') log2 e: S' = 2^d S, A' = 2^d (A + d S)); states of threads, and of
// workgroups that share a long row, are joined by the same rule, in an order that is always the same. All in
// fp32: the sums are short chains (32 logits a step) under trees, each addition off by at most 2^-24.
//
// Alternatives without keeping a list while reading: the pass leaves the maximum of every
// group of neighbouring logits that a wave loads at once (64 vectors of 16 bytes). The K-th of 64
// maxima, each over a 64th of the groups, is a bound that K logits reach, so the K first logits
// (larger value, then lower index) are from the bound up, and only groups whose maximum is need be
// read again: about K of them, in which hardly more than K logits are. Where that finds too many
// (many equal logits, sorted ones) the K-th largest value itself is found by halving the range of
// values, then the logits above it are ranked and its first equals fill up.
//
// What bounds it: many rows, the one read of the logits beside the vector units: 4 x 512 rows of 152064
// bf16 logits (623 MB) 112 us, 5.6 TB/s, where a plain read of the memory takes 99. 9.2 vector instructions
// a logit, one of them the exponential, are about 90 us of every SIMD (with edge checks in every step
// and (x - m) log2 e as two operations 12 a logit and 117 us). The next step's loads ahead of this one's
// arithmetic took 4 us more, as fewer waves fit. Few rows, latency: one fp32 row with 20 alternatives 8.9
// us, 16 x 8 bf16 rows with 5 15.0 us, of which the finish is 5: states and maxima 0.9 us, bound 0.9, groups 0.3, their
// logits 0.9, ranks 0.5, launch. Its code runs once a row and is loaded for it, so it is kept
// short: with loops unrolled the finish took 9 us (K = 5) to 19 (K = 20).
#include <algorithm>
#include <type_traits>

#include "fdllm_common.h"

namespace fdllm {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
// Threads of a row's finish: 256 take 0.9 us more for 20 alternatives of one fp32 row, 1024 1.3 us
// more (2 to 5 us where there are many rows).
constexpr int kFinishThreads = 512;
// Workgroups that a call aims at where rows are shared: 1024 take 1.8 us more for 16 x 8 rows of 152064, 4096
// 0.9 us more (more partials, one step each).
constexpr int kWorkgroups = 2048;
constexpr int kStep = 2048 * kWaves;      // logits of a workgroup's step
constexpr int kMaxVocab = 1 << 20;
constexpr int kCandidates = 1024;
constexpr int kMaxTop = 32;
constexpr int kMaxRows = (1 << 24) - 1;   // a launch has fewer than 2^32 threads, a row kThreads

struct ScoreArgs {
  const void* logits;
  int64_t stride_b, stride_r;
  int rows_per_batch, V;
  const int64_t* tokens;  // [rows, given]
  int given, top;
  float* logprobs;
  float* entropy;
  float* top_logprobs;
  int64_t* top_tokens;
  int splits, steps;  // workgroups per row, steps of each
  float* parts;       // splits > 1: [rows][splits][waves] of float4 (m, S, A, -), then [rows][n_groups] maxima
  int n_groups;
  int64_t rows;
};

// Elements of a 16-byte vector.
template <typename T>
struct Vec {
  static constexpr int N = 8;
  static constexpr int kGroup = 64 * N;                     // neighbouring logits under one maximum: a vector a lane
  static constexpr int kMaxGroups = kMaxVocab / kGroup;
  __device__ __forceinline__ static void get(const u32x4& w, float* f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = Elt<T>::lo(w[i]);
      f[2 * i + 1] = Elt<T>::hi(w[i]);
    }
  }
  __device__ __forceinline__ static float one(const void* p, int64_t at) {
    return Elt<T>::lo(static_cast<const uint16_t*>(p)[at]);
  }
};
template <>
struct Vec<float> {
  static constexpr int N = 4;
  static constexpr int kGroup = 64 * N;
  static constexpr int kMaxGroups = kMaxVocab / kGroup;
  __device__ __forceinline__ static void get(const u32x4& w, float* f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(w[i]);
  }
  __device__ __forceinline__ static float one(const void* p, int64_t at) { return static_cast<const float*>(p)[at]; }
};

// A row as 16-byte vectors from the aligned address at or below its start: the first `mis`
// elements of vector 0 precede the row, the last vector may run past its end. Every vector
// holds at least one logit of the row, so an aligned load of it touches no page the row does
// not.
struct RowVecs {
  const u32x4* v;
  const void* row;
  int mis, nv;
};
template <typename T>
__device__ __forceinline__ RowVecs row_of(const ScoreArgs& a, uint32_t r) {  // 32-bit division: fewer than 2^31 rows
  constexpr int N = Vec<T>::N, E = 16 / N;
  const uint32_t b = r / static_cast<uint32_t>(a.rows_per_batch), i = r - b * a.rows_per_batch;
  const char* row = static_cast<const char*>(a.logits) + (b * a.stride_b + i * a.stride_r) * E;
  const int mis = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15u) / E);
  return RowVecs{reinterpret_cast<const u32x4*>(row - mis * E), row, mis, (a.V + mis + N - 1) / N};
}
// vector v's logits, -inf where there is none
template <typename T>
__device__ __forceinline__ void unpack(const u32x4& w, int v, const RowVecs& rv, int V, float* x) {
  constexpr int N = Vec<T>::N;
  Vec<T>::get(w, x);
  const int j0 = N * v - rv.mis;
  if (j0 < 0 || j0 + N > V) {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j0 + j < 0 || j0 + j >= V) x[j] = -INFINITY;
  }
}

// Orders one wave's LDS accesses.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// The sums in powers of two: u = x log2 e - R with R = m log2 e rounded, one fused operation a logit;
// S = sum 2^u, A = sum u 2^u. That R is not m log2 e to the last bit does not matter, as long as
// every use takes the same one. Where it could overflow (a maximum near the type's largest or
// lowest value) u = (x - m) log2 e.
constexpr float kLog2e = 1.44269504f, kLn2 = 0.693147181f;
constexpr float kLargeMax = 1e37f;
__device__ __forceinline__ float powers_above(float x, float m) {  // u
  return fabsf(m) < kLargeMax ? __builtin_fmaf(x, kLog2e, -(m * kLog2e)) : (x - m) * kLog2e;
}

// S and A relative to the maximum m. While nothing above -inf was read they are 0, or NaN
// after a NaN logit, which then stays.
struct State {
  float m, s, a;
};
// the state relative to another maximum to >= m: S' = 2^d S, A' = 2^d (A + d S)
__device__ __forceinline__ void rescale(State& x, float to) {
  if (x.m == to) return;
  float d = 0.f;
  if (x.m != -INFINITY) {
    const bool small = fabsf(x.m) < kLargeMax && fabsf(to) < kLargeMax;
    d = small ? x.m * kLog2e - to * kLog2e : (x.m - to) * kLog2e;
  }
  const float e = __builtin_amdgcn_exp2f(d);
  x.a = e * __builtin_fmaf(fmaxf(d, -1e30f), x.s, x.a);  // e is 0 long before that bound: 0 times -inf is not 0
  x.s *= e;
  x.m = to;
}

// Joins a wave's states.
__device__ __forceinline__ State join_wave(State x) {
  rescale(x, wave_allreduce_max(x.m));
  x.s = wave_allreduce_sum(x.s);
  x.a = wave_allreduce_sum(x.a);
  return x;
}
// Joins the waves' states; every thread returns with the workgroup's.
template <int NW>
__device__ __forceinline__ State join(const State& x, float* s_red) {
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) {
    s_red[3 * wave] = x.m;
    s_red[3 * wave + 1] = x.s;
    s_red[3 * wave + 2] = x.a;
  }
  __syncthreads();
  float m = s_red[0];
#pragma unroll
  for (int w = 1; w < NW; ++w) m = fmaxf(m, s_red[3 * w]);
  State r{m, 0.f, 0.f};
#pragma unroll 1
  for (int w = 0; w < NW; ++w) {
    State y{s_red[3 * w], s_red[3 * w + 1], s_red[3 * w + 2]};
    rescale(y, m);
    r.s += y.s;
    r.a += y.a;
  }
  return r;
}

struct Cand {
  float v;
  int i;
};
template <typename T, int NT>
struct Shared {
  float red[3 * (NT / 64)];
  __attribute__((aligned(16))) float lane_max[64];
  float group[Vec<T>::kMaxGroups];
  uint16_t sel[Vec<T>::kMaxGroups];
  Cand cand[kCandidates];
  float bound;
  int n_sel, n_cand, n_above[33];
};

// The given token of this thread and its logit, read ahead of the row's sums.
struct Given {
  bool in;
  float x;
};
template <typename T>
__device__ __forceinline__ Given given_of(const ScoreArgs& a, int64_t r, int j, const RowVecs& rv) {
  Given g{false, 0.f};
  if (j < a.given) {
    const int64_t t = a.tokens[r * a.given + j];
    g.in = t >= 0 && t < a.V;
    if (g.in) g.x = Vec<T>::one(rv.row, t);
  }
  return g;
}

// Values in their order, as numbers without gaps: -inf is 0.
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);  // -0 is 0
  return ((b >> 31) ? ~b : b | 0x80000000u) - 0x007fffffu;
}

// Into sh.bound a bound that K logits reach, by one wave: the K-th of 64 maxima, each over the groups
// that a lane takes. Clears the counters of what follows.
template <typename T, int NT>
__device__ __forceinline__ void find_bound(const ScoreArgs& a, int lane, Shared<T, NT>& sh) {
  float mine = -INFINITY;
#pragma unroll 2
  for (int g = lane; g < a.n_groups; g += 64) mine = fmaxf(mine, sh.group[g]);
  sh.lane_max[lane] = mine;
  wave_sync();
  int above = 0;
#pragma unroll
  for (int h = 0; h < 64; h += 4) {
    const f32x4 y = *reinterpret_cast<const f32x4*>(&sh.lane_max[h]);
#pragma unroll
    for (int j = 0; j < 4; ++j) above += y[j] > mine;
  }
  const float m = -wave_allreduce_max(above < a.top ? -mine : -INFINITY);  // the least that fewer than K exceed
  if (lane < 33) sh.n_above[lane] = 0;
  if (lane == 0) {
    sh.bound = m;
    sh.n_sel = sh.n_cand = 0;
  }
}

// A row's alternatives, by NT threads; sh.group holds its groups' maxima, sh.bound the bound. The code
// runs once a row, so its own loading counts: no loop is unrolled that need not be.
template <typename T, int NT, typename Put>
__device__ __forceinline__ void alternatives(const ScoreArgs& a, const RowVecs& rv, Put put, Shared<T, NT>& sh) {
  constexpr int N = Vec<T>::N;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int K = a.top, ng = a.n_groups;
  const float bound = sh.bound;
  // the groups that hold a logit from the bound up
#pragma unroll 1
  for (int g0 = wave * 64; g0 < ng; g0 += NT) {
    const float m = g0 + lane < ng ? sh.group[g0 + lane] : -INFINITY;
    if (m >= bound && m > -INFINITY) sh.sel[atomicAdd(&sh.n_sel, 1)] = static_cast<uint16_t>(g0 + lane);
  }
  __syncthreads();
  const int ns = sh.n_sel;
  // f(a vector of those groups, its number), the next one in flight
  auto each = [&](auto f) __attribute__((always_inline)) {
    int v = 0;
    u32x4 next;
    auto fetch = [&](int i) __attribute__((always_inline)) {
      if (i < ns) {
        v = sh.sel[i] * 64 + lane;
        if (v < rv.nv) next = rv.v[v];
      }
    };
    fetch(wave);
#pragma unroll 1
    for (int i = wave; i < ns; i += NT / 64) {
      const u32x4 w = next;
      const int at = v;
      fetch(i + NT / 64);
      if (at < rv.nv) f(w, at);
    }
  };
  // those from `than` up (without its equals, if strict) into the list
  auto collect = [&](float than, bool strict) __attribute__((always_inline)) {
    each([&](const u32x4& w, int v) __attribute__((always_inline)) {
      float x[N];
      unpack<T>(w, v, rv, a.V, x);
      uint32_t in = 0;
#pragma unroll
      for (int j = 0; j < N; ++j) in |= ((x[j] > than || (x[j] == than && !strict)) && x[j] > -INFINITY ? 1u : 0u) << j;
      if (in == 0) return;
      int c = atomicAdd(&sh.n_cand, __builtin_popcount(in));
#pragma unroll
      for (int j = 0; j < N; ++j) {
        if ((in >> j & 1) && c < kCandidates) sh.cand[c++] = Cand{x[j], N * v + j - rv.mis};
      }
    });
    __syncthreads();
  };
  collect(bound, false);
  int n = sh.n_cand;
  float rest = -INFINITY;  // what is left to take is equal to this
  if (__builtin_expect(n > kCandidates, 0)) {
    // Too many (equal logits, sorted ones): the K-th largest value itself, by halving the range of
    // values that it can have; at most K - 1 logits are above it
    uint32_t lo = order_of(bound), hi = 0xff800000u;  // more than K - 1 logits reach lo, no finite one hi
    int round = 0;
#pragma unroll 1
    for (uint32_t mid = lo + 1; lo + 1 < hi; mid = lo + (hi - lo) / 2, ++round) {
      int c = 0;
      each([&](const u32x4& w, int v) __attribute__((always_inline)) {
        float x[N];
        unpack<T>(w, v, rv, a.V, x);
#pragma unroll
        for (int j = 0; j < N; ++j) c += order_of(x[j]) >= mid;
      });
      c = static_cast<int>(wave_allreduce_sum(static_cast<float>(c)));  // at most 2^20: exact
      if (lane == 0) atomicAdd(&sh.n_above[round], c);
      __syncthreads();
      if (sh.n_above[round] >= K) lo = mid;
      else hi = mid;
    }
    const uint32_t b = lo + 0x007fffffu;
    rest = __uint_as_float((b >> 31) ? b & 0x7fffffffu : ~b);
    if (tid == 0) sh.n_cand = 0;
    __syncthreads();
    collect(rest, true);
    n = sh.n_cand;
  }
  // eight threads rank one: a loop over them all by itself is a chain of LDS latencies
#pragma unroll 1
  for (int c = tid >> 3; c < n; c += NT / 8) {
    const Cand mine = sh.cand[c];
    float rank = 0.f;
#pragma unroll 2
    for (int h = tid & 7; h < n; h += 8) {
      const Cand o = sh.cand[h];
      rank += o.v > mine.v || (o.v == mine.v && o.i < mine.i) ? 1.f : 0.f;
    }
    rank += dpp_f32<0xB1>(rank);
    rank += dpp_f32<0x4E>(rank);
    rank += dpp_f32<0x141>(rank);
    if ((tid & 7) == 0 && rank < K) put(static_cast<int>(rank), mine.v, mine.i);
  }
  // fewer than K: of those equal to `rest`, the first ones
  if (__builtin_expect(n < K, 0) && wave == 0) {
#pragma unroll 1
    for (int i0 = 0; i0 < a.V && n < K; i0 += 64) {
      const bool in = i0 + lane < a.V && Vec<T>::one(rv.row, i0 + lane) == rest;
      const uint64_t all = __builtin_amdgcn_ballot_w64(in);
      const int rank = n + __builtin_popcountll(all & ((1ull << lane) - 1));
      if (in && rank < K) put(rank, rest, i0 + lane);
      n += __builtin_popcountll(all);
    }
  }
}

// A row's outputs from its state, by NT threads; g: the thread's given token.
template <typename T, int NT>
__device__ __forceinline__ void finish(const ScoreArgs& a, int64_t r, const RowVecs& rv, const State& st, Given g,
                                       Shared<T, NT>& sh) {
  const int tid = threadIdx.x;
  // a NaN or +inf logit makes the sum NaN, a row without a finite one leaves it 0
  const bool good = st.s > 0.f;
  const float log2s = __builtin_amdgcn_logf(st.s);
  const float nan = __builtin_nanf("");
  // log p = x - m - log of the sum relative to m itself, which R is off from
  const float off = fabsf(st.m) < kLargeMax ? __builtin_fmaf(st.m, kLog2e, -(st.m * kLog2e)) : 0.f;
  const float lse = (log2s - off) * kLn2;
  auto logp = [&](float x) __attribute__((always_inline)) { return x - st.m - lse; };
  if (tid == 0) a.entropy[r] = good ? (log2s - st.a / st.s) * kLn2 : nan;
#pragma unroll 1
  for (int j = tid; j < a.given; j += NT) {
    a.logprobs[r * a.given + j] = good && g.in ? logp(g.x) : nan;
    g = given_of<T>(a, r, j + NT, rv);
  }
  const int K = a.top;
  if (good && K > 0) {  // uniform
    alternatives<T, NT>(a, rv, [&](int k, float v, int i) __attribute__((always_inline)) {
      a.top_tokens[r * K + k] = i;
      a.top_logprobs[r * K + k] = logp(v);
    }, sh);
  } else if (tid < K) {
    a.top_tokens[r * K + tid] = -1;
    a.top_logprobs[r * K + tid] = nan;
  }
}

// The maximum of a value and another lane's, by a lane move within rows of 16.
template <int CTRL>
__device__ __forceinline__ float max_moved(float v) {
  return fmaxf(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, true)));
}

// The maximum over the lanes of each of the U values m[u], the u-th group's: where it is, value u of the
// wave's U / 4 to a lane. Lanes trade halves of their values for halves of the others', so that two and
// a few exchanges serve all.
template <int U>
__device__ __forceinline__ void group_maxima(float* m) {
#pragma unroll
  for (int u = 0; u < U / 2; ++u) {  // the upper 32 lanes take the second half's values
    const auto w = __builtin_amdgcn_permlane32_swap(__float_as_uint(m[u]), __float_as_uint(m[u + U / 2]), false, false);
    m[u] = fmaxf(__uint_as_float(w[0]), __uint_as_float(w[1]));
  }
#pragma unroll
  for (int u = 0; u < U / 4; ++u) {  // odd rows of 16 lanes the second half's of those
    const auto w = __builtin_amdgcn_permlane16_swap(__float_as_uint(m[u]), __float_as_uint(m[u + U / 4]), false, false);
    m[u] = fmaxf(__uint_as_float(w[0]), __uint_as_float(w[1]));
    m[u] = max_moved<0xB1>(m[u]);
    m[u] = max_moved<0x4E>(m[u]);
    m[u] = max_moved<0x141>(m[u]);
    m[u] = max_moved<0x140>(m[u]);
  }
}

// One workgroup per row, or (SPLIT) per `steps` steps of a row that several share; the latter without the
// finish's LDS and code.
template <typename T, bool SPLIT>
__global__ __launch_bounds__(kThreads) void score_kernel(const ScoreArgs a) {
  constexpr int N = Vec<T>::N, U = kStep / kWaves / Vec<T>::kGroup;  // a lane's vectors in a step
  __shared__ std::conditional_t<SPLIT, char, Shared<T, kThreads>> sh;
  const uint32_t row = SPLIT ? blockIdx.x / static_cast<uint32_t>(a.splits) : blockIdx.x;
  const int split = static_cast<int>(blockIdx.x - row * a.splits);
  const int64_t r = row;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const RowVecs rv = row_of<T>(a, row);
  float* groups = a.parts + a.rows * a.splits * (4 * kWaves) + r * a.n_groups;  // splits > 1
  State st{-INFINITY, 0.f, 0.f};
  Given given{false, 0.f};
  if constexpr (!SPLIT) given = given_of<T>(a, r, threadIdx.x, rv);
#pragma unroll 1
  for (int k = 0; k < a.steps; ++k) {
    const int g = ((split * a.steps + k) * kWaves + wave) * U;
    const int v0 = g * 64 + lane;
    if (g >= a.n_groups) break;  // uniform over the wave
    const int e0 = g * Vec<T>::kGroup - rv.mis;
    float x[U][N], mu[U];
    u32x4 w[U];
    if (e0 >= 0 && e0 + U * Vec<T>::kGroup <= a.V) {  // uniform: all of them are the row's
#pragma unroll
      for (int u = 0; u < U; ++u) w[u] = __builtin_nontemporal_load(rv.v + v0 + 64 * u);
#pragma unroll
      for (int u = 0; u < U; ++u) Vec<T>::get(w[u], x[u]);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) w[u] = rv.v[min(v0 + 64 * u, rv.nv - 1)];
#pragma unroll
      for (int u = 0; u < U; ++u) unpack<T>(w[u], v0 + 64 * u, rv, a.V, x[u]);  // -inf past the row's end
    }
    float m = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      mu[u] = x[u][0];
#pragma unroll
      for (int j = 1; j < N; ++j) mu[u] = fmaxf(mu[u], x[u][j]);
      m = fmaxf(m, mu[u]);
    }
    if (m > st.m) rescale(st, m);
    const float ref = st.m == -INFINITY ? 0.f : st.m;
    // a banned token's 0 times -inf counts as 0
    if (__builtin_amdgcn_ballot_w64(fabsf(ref) >= kLargeMax) == 0) {
      const float r2 = ref * kLog2e;
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const float t = __builtin_fmaf(x[u][j], kLog2e, -r2);
          const float e = __builtin_amdgcn_exp2f(t);
          st.s += e;
          st.a = __builtin_fmaf(e, fmaxf(t, -1e30f), st.a);
        }
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const float t = powers_above(x[u][j], ref);
          const float e = __builtin_amdgcn_exp2f(t);
          st.s += e;
          st.a = __builtin_fmaf(e, fmaxf(t, -1e30f), st.a);
        }
    }
    if (a.top > 0) {
      group_maxima<U>(mu);
      const int u0 = (lane >> 5) * (U / 2) + ((lane >> 4) & 1) * (U / 4);
      if ((lane & 15) == 0) {
#pragma unroll
        for (int u = 0; u < U / 4; ++u)
          if (g + u0 + u < a.n_groups) {
            if constexpr (SPLIT) groups[g + u0 + u] = mu[u];
            else sh.group[g + u0 + u] = mu[u];
          }
      }
    }
  }
  st = join_wave(st);
  if constexpr (!SPLIT) {
    st = join<kWaves>(st, sh.red);  // a barrier: the group maxima are in LDS after it
    if (a.top > 0) {
      if (wave == 0) find_bound<T, kThreads>(a, lane, sh);
      __syncthreads();
    }
    finish<T, kThreads>(a, r, rv, st, given, sh);
  } else if (lane == 0) {  // each wave's own: the finish folds them
    reinterpret_cast<float4*>(a.parts)[blockIdx.x * static_cast<int64_t>(kWaves) + wave] = make_float4(st.m, st.s, st.a, 0.f);
  }
}

template <typename T>
__global__ __launch_bounds__(kFinishThreads) void score_finish_kernel(const ScoreArgs a) {
  __shared__ Shared<T, kFinishThreads> sh;
  const int64_t r = blockIdx.x;
  const RowVecs rv = row_of<T>(a, blockIdx.x);
  const int tid = threadIdx.x, lane = tid & 63;
  // what is read of the row: the waves' states by the second wave, the groups' maxima by all
  const int np = a.splits * kWaves;
  const float4* parts = reinterpret_cast<const float4*>(a.parts) + r * np;
  const float* groups = a.parts + a.rows * np * 4 + r * a.n_groups;
  float4 p = make_float4(-INFINITY, 0.f, 0.f, 0.f);
  if (tid >> 6 == 1 && lane < np) p = parts[lane];
  if (a.top > 0) {
    // two in flight
#pragma unroll 1
    for (int g = tid; g < a.n_groups; g += 2 * kFinishThreads) {
      const int h = g + kFinishThreads;
      const float x = groups[g], y = h < a.n_groups ? groups[h] : -INFINITY;
      sh.group[g] = x;
      if (h < a.n_groups) sh.group[h] = y;
    }
  }
  const Given given = given_of<T>(a, r, tid, rv);
  __syncthreads();
  if (tid >> 6 == 0) {
    if (a.top > 0) find_bound<T, kFinishThreads>(a, lane, sh);
  } else if (tid >> 6 == 1) {
    State st{p.x, p.y, p.z};
#pragma unroll 1
    for (int s = lane + 64; s < np; s += 64) {
      const float4 q = parts[s];
      State y{q.x, q.y, q.z};
      const float m = fmaxf(st.m, y.m);
      rescale(st, m);
      rescale(y, m);
      st.s += y.s;
      st.a += y.a;
    }
    st = join_wave(st);
    sh.red[0] = st.m;
    sh.red[1] = st.s;
    sh.red[2] = st.a;
  }
  __syncthreads();
  finish<T, kFinishThreads>(a, r, rv, State{sh.red[0], sh.red[1], sh.red[2]}, given, sh);
}

struct Cut {
  int n_groups, steps, splits;
  size_t bytes;
};
// A workgroup takes a whole row where it has at most two steps, and where there are many rows (a finish less, and
// no partials); else several share one. us, bf16, whole rows / shared: 9000 logits, 16 rows 8.7 / 8.8, 500
// 9.2 / 10.9, 1000 11.1 / 15.2; 32000, 16 rows 9.8 / 8.6, 333 13.2 / 12.0, 500 14.1 / 15.0, 1000 19.4 / 22.7;
// 152064, 333 37.6 / 27.8, 500 39.2 / 36.5, 600 45.6 / 43.4, 850 56.6 / 59.8, 1000 60.8 / 65.
Cut cut(int vocab, int64_t rows, int dtype) {
  Cut c;
  const int slack = dtype == FDLLM_DTYPE_F32 ? 3 : 7;  // a row may start inside a vector
  const int group = dtype == FDLLM_DTYPE_F32 ? Vec<float>::kGroup : Vec<bf16_t>::kGroup;
  c.n_groups = (vocab + slack + group - 1) / group;
  const int64_t all = (static_cast<int64_t>(c.n_groups) * group + kStep - 1) / kStep;
  const bool whole = all <= 2 || rows >= (all <= 4 ? 448 : 640);
  const int64_t splits = whole ? 1 : std::min<int64_t>(kWorkgroups / rows, all);
  c.steps = static_cast<int>((all + splits - 1) / splits);
  c.splits = static_cast<int>((all + c.steps - 1) / c.steps);
  c.bytes = c.splits > 1 ? (static_cast<size_t>(rows) * c.splits * (4 * kWaves) + static_cast<size_t>(rows) * c.n_groups) * 4 : 0;
  return c;
}

template <typename T>
void launch(const ScoreArgs& a, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(a.rows * a.splits)), block(kThreads);
  if (a.splits == 1) {
    score_kernel<T, false><<<grid, block, 0, s>>>(a);
  } else {
    score_kernel<T, true><<<grid, block, 0, s>>>(a);
    score_finish_kernel<T><<<dim3(static_cast<unsigned>(a.rows)), dim3(kFinishThreads), 0, s>>>(a);
  }
}

int check_sizes(const char* what, int vocab, int64_t rows, int dtype) {
  FDLLM_CHECK_ARG(dtype == FDLLM_DTYPE_BF16 || dtype == FDLLM_DTYPE_F16 || dtype == FDLLM_DTYPE_F32,
                  "%s: dtype %d unsupported", what, dtype);
  FDLLM_CHECK_ARG(vocab > 0 && vocab <= kMaxVocab - 8, "%s: vocab %d (1 to %d)", what, vocab, kMaxVocab - 8);
  FDLLM_CHECK_ARG(rows >= 0 && rows <= kMaxRows, "%s: %lld rows (0 to %d)", what, static_cast<long long>(rows), kMaxRows);
  return FDLLM_OK;
}

}  // namespace
}  // namespace fdllm

extern "C" int fdllm_token_logprobs_workspace_size(int vocab, int64_t rows, int dtype, size_t* bytes) {
  using namespace fdllm;
  const char* what = "fdllm_token_logprobs_workspace_size";
  FDLLM_CHECK_ARG(bytes != nullptr, "%s: null pointer", what);
  if (const int rc = check_sizes(what, vocab, rows, dtype)) return rc;
  *bytes = rows > 0 ? cut(vocab, rows, dtype).bytes : 0;
  return FDLLM_OK;
}

extern "C" int fdllm_token_logprobs(const void* logits, int64_t stride_b, int64_t stride_r, int batch,
                                    int rows_per_batch, int vocab, const int64_t* tokens, int given, int top,
                                    float* logprobs, float* entropy, float* top_logprobs, int64_t* top_tokens,
                                    int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace fdllm;
  const char* what = "fdllm_token_logprobs";
  FDLLM_CHECK_ARG(batch >= 0 && rows_per_batch >= 0, "%s: bad sizes", what);
  const int64_t rows = static_cast<int64_t>(batch) * rows_per_batch;
  if (const int rc = check_sizes(what, vocab, rows, dtype)) return rc;
  FDLLM_CHECK_ARG(given >= 0 && top >= 0 && top <= kMaxTop && top <= vocab,
                  "%s: %d alternatives (at most %d, and the vocabulary's)", what, top, kMaxTop);
  if (rows == 0) return FDLLM_OK;
  FDLLM_CHECK_ARG(logits && entropy && (given == 0 || (tokens && logprobs)) && (top == 0 || (top_logprobs && top_tokens)),
                  "%s: null pointer", what);
  const Cut c = cut(vocab, rows, dtype);
  if (c.bytes > 0 && (workspace == nullptr || workspace_bytes < c.bytes || (reinterpret_cast<uintptr_t>(workspace) & 15u) != 0)) {
    set_last_error("%s: workspace of %zu bytes required (got %zu)", what, c.bytes, workspace_bytes);
    return FDLLM_ERR_WORKSPACE;
  }
  ScoreArgs a;
  a.logits = logits;
  a.stride_b = stride_b;
  a.stride_r = stride_r;
  a.rows_per_batch = rows_per_batch;
  a.V = vocab;
  a.tokens = tokens;
  a.given = given;
  a.top = top;
  a.logprobs = logprobs;
  a.entropy = entropy;
  a.top_logprobs = top_logprobs;
  a.top_tokens = top_tokens;
  a.splits = c.splits;
  a.steps = c.steps;
  a.parts = static_cast<float*>(workspace);
  a.n_groups = c.n_groups;
  a.rows = rows;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == FDLLM_DTYPE_BF16) launch<bf16_t>(a, s);
  else if (dtype == FDLLM_DTYPE_F16) launch<f16_t>(a, s);
  else launch<float>(a, s);
  FDLLM_RETURN_LAUNCH_STATUS(what);
}

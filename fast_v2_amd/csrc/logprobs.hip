// Log probabilities of given tokens, the entropy and the most probable alternatives of every
// logits row (fdllm_token_logprobs), in one pass over the logits.
//
//   m = max x,  S = sum e^(x - m),  A = sum (x - m) e^(x - m)
//   log p(t) = x_t - m - log S,     H = -sum p log p = log S - A / S
//
// Each thread holds (m, S, A) of the logits it has read and rescales when its maximum grows
// (e^d with d = m - m': S' = e^d S, A' = e^d (A + d S)); states of threads, and of workgroups
// that share a long row, are joined by the same rule. All in fp32: (x - m) is exact for 16-bit
// logits near m, and the sums are trees of at most 2^-24 relative error a level.
//
// Alternatives without keeping a list while reading: the pass leaves the maximum of every
// group of 2048 neighbouring logits, which the reduction makes anyway. The K first logits by
// (larger value, lower index) lie in the K first groups by (larger maximum, lower index): a
// logit in any other group has K logits ahead of it, those groups' maxima. Only those
// groups are read again, and of them only what is not below the K-th maximum is ranked.
//
// What bounds it: the one read of the logits.
#include <math.h>

#include "fdllm_common.h"

namespace fdllm {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kGroup = 2048;              // neighbouring logits under one maximum: a wave's share of a step
constexpr int kStep = kGroup * kWaves;    // logits of a workgroup's step
constexpr int kMaxVocab = 1 << 22;
constexpr int kMaxGroups = kMaxVocab / kGroup + 1;  // one more where a row starts off 16 bytes
constexpr int kCandidates = 1024;
constexpr int kMaxTop = 32;  // twice that many tokens are one wave's

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
  float* parts;       // splits > 1: [rows][splits] of float4 (m, S, A, -), then [rows][n_groups] maxima
  int n_groups;
  int64_t rows;
};

// Elements of a 16-byte vector.
template <typename T>
struct Vec {
  static constexpr int N = 8;
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
__device__ __forceinline__ RowVecs row_of(const ScoreArgs& a, int64_t r) {
  constexpr int N = Vec<T>::N, E = 16 / N;
  const int64_t b = r / a.rows_per_batch;
  const char* row = static_cast<const char*>(a.logits) + (b * a.stride_b + (r - b * a.rows_per_batch) * a.stride_r) * E;
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

// S and A relative to the maximum m. While nothing above -inf was read they are 0, or NaN
// after a NaN logit, which then stays.
struct State {
  float m, s, a;
};
// the state relative to another maximum to >= m
__device__ __forceinline__ void rescale(State& x, float to) {
  if (x.m == to) return;
  const float d = x.m == -INFINITY ? 0.f : x.m - to;
  const float e = expf(d);
  x.a = e * __builtin_fmaf(fmaxf(d, -1e30f), x.s, x.a);  // e is 0 long before that bound: 0 times -inf is not 0
  x.s *= e;
  x.m = to;
}

// Joins the workgroup's states; every thread returns with the row's.
__device__ __forceinline__ State join(State x, float* s_red) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const float mw = wave_allreduce_max(x.m);
  rescale(x, mw);
  x.s = wave_allreduce_sum(x.s);
  x.a = wave_allreduce_sum(x.a);
  if (lane == 0) {
    s_red[3 * wave] = x.m;
    s_red[3 * wave + 1] = x.s;
    s_red[3 * wave + 2] = x.a;
  }
  __syncthreads();
  float m = s_red[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) m = fmaxf(m, s_red[3 * w]);
  State r{m, 0.f, 0.f};
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    State y{s_red[3 * w], s_red[3 * w + 1], s_red[3 * w + 2]};
    rescale(y, m);
    r.s += y.s;
    r.a += y.a;
  }
  return r;
}

// The largest (value, lowest index) of the workgroup, to every thread.
__device__ __forceinline__ void block_first(float& v, int& i, float* s_v, int* s_i) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    const float v2 = __shfl_xor(v, o, kWave);
    const int i2 = __shfl_xor(i, o, kWave);
    if (v2 > v || (v2 == v && i2 < i)) {
      v = v2;
      i = i2;
    }
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) {
    s_v[threadIdx.x >> 6] = v;
    s_i[threadIdx.x >> 6] = i;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w)
    if (s_v[w] > v || (s_v[w] == v && s_i[w] < i)) {
      v = s_v[w];
      i = s_i[w];
    }
}

// f(i, rank) for every i < n of its thread: its place by (larger value, lower index).
template <typename F>
__device__ __forceinline__ void rank_all(const float* v, int n, F f) {
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const float x = v[i];
    int rank = 0;
    for (int h = 0; h < n; ++h) rank += v[h] > x || (v[h] == x && h < i);
    f(i, rank);
  }
}

struct Shared {
  float red[3 * kWaves];
  float group[kMaxGroups];
  float cand_v[kCandidates];
  int cand_i[kCandidates];
  int sel[kMaxTop];
  float sel_v[kMaxTop];
  int n_cand;
};

// A row's outputs from its state; sh.group holds its groups' maxima.
template <typename T>
__device__ void finish(const ScoreArgs& a, int64_t r, const State& st, Shared& sh) {
  const int tid = threadIdx.x;
  const RowVecs rv = row_of<T>(a, r);
  // a NaN or +inf logit makes the sum NaN, a row without a finite one leaves it 0
  const bool good = st.s > 0.f;
  const float lse = logf(st.s);
  const float nan = __builtin_nanf("");
  if (tid == 0) a.entropy[r] = good ? lse - st.a / st.s : nan;
  for (int j = tid; j < a.given; j += kThreads) {
    const int64_t t = a.tokens[r * a.given + j];
    a.logprobs[r * a.given + j] = good && t >= 0 && t < a.V ? Vec<T>::one(rv.row, t) - st.m - lse : nan;
  }
  const int K = a.top;
  if (K == 0) return;
  if (!good) {  // uniform
    for (int k = tid; k < K; k += kThreads) {
      a.top_tokens[r * K + k] = -1;
      a.top_logprobs[r * K + k] = nan;
    }
    return;
  }
  auto put = [&](int k, float v, int i) __attribute__((always_inline)) {
    a.top_tokens[r * K + k] = i;
    a.top_logprobs[r * K + k] = v - st.m - lse;
  };
  // the K first groups
  const int ng = a.n_groups;
  rank_all(sh.group, ng, [&](int g, int rank) __attribute__((always_inline)) {
    if (rank < K) {
      sh.sel[rank] = g;
      sh.sel_v[rank] = sh.group[g];
    }
  });
  if (tid == 0) sh.n_cand = 0;
  __syncthreads();
  const int ns = min(ng, K);
  // every logit of those groups: f(value, index)
  constexpr int N = Vec<T>::N, GV = kGroup / N;
  auto each = [&](auto f) __attribute__((always_inline)) {
    for (int q = tid; q < ns * GV; q += kThreads) {
      const int v = sh.sel[q / GV] * GV + q % GV;
      if (v >= rv.nv) continue;
      float x[N];
      unpack<T>(rv.v[v], v, rv, a.V, x);
#pragma unroll
      for (int j = 0; j < N; ++j) f(x[j], N * v + j - rv.mis);  // -inf outside of the row
    }
  };
  float least = ng < K ? -INFINITY : sh.sel_v[K - 1];
  int n = 0;
  // With fewer groups than K, or too many logits from their K-th maximum up (sorted ones), the
  // K-th of the threads' own maxima is the bound: K threads have a logit that reaches it.
  for (int round = ng < K ? 1 : 0; round < 2; ++round) {
    if (round == 1) {
      float m = -INFINITY;
      each([&](float x, int) __attribute__((always_inline)) { m = fmaxf(m, x); });
      sh.cand_v[tid] = m;
      __syncthreads();
      rank_all(sh.cand_v, kThreads, [&](int t, int rank) __attribute__((always_inline)) {
        if (rank == K - 1) sh.sel_v[0] = sh.cand_v[t];
      });
      if (tid == 0) sh.n_cand = 0;
      __syncthreads();
      least = sh.sel_v[0];
    }
    each([&](float x, int at) __attribute__((always_inline)) {
      if (x >= least && x > -INFINITY) {
        const int c = atomicAdd(&sh.n_cand, 1);
        if (c < kCandidates) {
          sh.cand_v[c] = x;
          sh.cand_i[c] = at;
        }
      }
    });
    __syncthreads();
    n = sh.n_cand;
    __syncthreads();  // read before another round clears it
    if (n <= kCandidates) break;
  }
  if (n <= kCandidates) {
    for (int c = tid; c < n; c += kThreads) {
      const float v = sh.cand_v[c];
      const int i = sh.cand_i[c];
      int rank = 0;
      for (int h = 0; h < n; ++h) rank += sh.cand_v[h] > v || (sh.cand_v[h] == v && sh.cand_i[h] < i);
      if (rank < K) put(rank, v, i);
    }
    // fewer than K above -inf: the excluded tokens of lowest index, which are among the first 2 K
    if (n < K && tid < 64) {
      const bool out = tid < a.V && Vec<T>::one(rv.row, tid) == -INFINITY;
      const uint64_t all = __builtin_amdgcn_ballot_w64(out);
      const int rank = n + __builtin_popcountll(all & ((1ull << tid) - 1));
      if (out && rank < K) put(rank, -INFINITY, tid);
    }
    return;
  }
  // many equal logits: one at a time
  float last_v = INFINITY;
  int last_i = -1;
  for (int k = 0; k < K; ++k) {
    float bv = -INFINITY;
    int bi = 0x7fffffff;
    each([&](float x, int at) __attribute__((always_inline)) {
      const bool after = x < last_v || (x == last_v && at > last_i);
      if (after && (x > bv || (x == bv && at < bi))) {
        bv = x;
        bi = at;
      }
    });
    block_first(bv, bi, sh.red, reinterpret_cast<int*>(sh.red + kWaves));
    if (tid == 0) put(k, bv, bi);
    last_v = bv;
    last_i = bi;
  }
}

// One workgroup per row, or per `steps` steps of a row that several share.
template <typename T>
__global__ __launch_bounds__(kThreads) void score_kernel(const ScoreArgs a) {
  constexpr int N = Vec<T>::N, GV = kGroup / N, U = GV / 64;  // vectors of a group, of a lane in it
  __shared__ Shared sh;
  const int64_t r = blockIdx.x / a.splits;
  const int split = static_cast<int>(blockIdx.x - r * a.splits);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const RowVecs rv = row_of<T>(a, r);
  float* groups = a.parts + a.rows * a.splits * 4 + r * a.n_groups;  // splits > 1
  State st{-INFINITY, 0.f, 0.f};
  for (int k = 0; k < a.steps; ++k) {
    const int g = (split * a.steps + k) * kWaves + wave;
    const int v0 = g * GV + lane;
    if (g >= a.n_groups) break;  // uniform over the wave
    u32x4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (v0 + 64 * u < rv.nv) w[u] = __builtin_nontemporal_load(rv.v + v0 + 64 * u);
    float x[U][N];
    float m = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (v0 + 64 * u < rv.nv) {
        unpack<T>(w[u], v0 + 64 * u, rv, a.V, x[u]);
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j) x[u][j] = -INFINITY;
      }
#pragma unroll
      for (int j = 0; j < N; ++j) m = fmaxf(m, x[u][j]);
    }
    if (m > st.m) rescale(st, m);
    const float ref = st.m == -INFINITY ? 0.f : st.m;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float t = x[u][j] - ref;
        // exp2 of the product with log2 e in two parts: with one, the constant's rounding
        // biases every term the same way
        const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(t, 1.44269502f, t * 1.92596299e-8f));
        st.s += e;
        st.a = __builtin_fmaf(e, fmaxf(t, -1e30f), st.a);  // a banned token's 0 times -inf counts as 0
      }
    if (a.top > 0) {
      m = wave_allreduce_max(m);
      if (lane == 0) {
        if (a.splits > 1) groups[g] = m;
        else sh.group[g] = m;
      }
    }
  }
  st = join(st, sh.red);  // a barrier: the group maxima are in LDS after it
  if (a.splits == 1) {
    finish<T>(a, r, st, sh);
  } else if (threadIdx.x == 0) {
    reinterpret_cast<float4*>(a.parts)[blockIdx.x] = make_float4(st.m, st.s, st.a, 0.f);
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void score_finish_kernel(const ScoreArgs a) {
  __shared__ Shared sh;
  const int64_t r = blockIdx.x;
  const float4* parts = reinterpret_cast<const float4*>(a.parts) + r * a.splits;
  State st{-INFINITY, 0.f, 0.f};
  for (int s = threadIdx.x; s < a.splits; s += kThreads) {
    const float4 p = parts[s];
    State y{p.x, p.y, p.z};
    const float m = fmaxf(st.m, y.m);
    rescale(st, m);
    rescale(y, m);
    st.s += y.s;
    st.a += y.a;
  }
  if (a.top > 0) {
    const float* groups = a.parts + a.rows * a.splits * 4 + r * a.n_groups;
    for (int g = threadIdx.x; g < a.n_groups; g += kThreads) sh.group[g] = groups[g];
  }
  st = join(st, sh.red);
  finish<T>(a, r, st, sh);
}

struct Cut {
  int n_groups, steps, splits;
  size_t bytes;
};
// Rows are shared by workgroups until there are about eight for every compute unit.
Cut cut(int vocab, int64_t rows, int dtype) {
  Cut c;
  const int slack = dtype == FDLLM_DTYPE_F32 ? 3 : 7;  // a row may start inside a vector
  c.n_groups = (vocab + slack + kGroup - 1) / kGroup;
  const int64_t all = (c.n_groups + kWaves - 1) / kWaves;
  const int64_t want = rows < 2048 ? 2048 / rows : 1;
  const int64_t splits = want < all ? want : all;
  c.steps = static_cast<int>((all + splits - 1) / splits);
  c.splits = static_cast<int>((all + c.steps - 1) / c.steps);
  c.bytes = c.splits > 1 ? (static_cast<size_t>(rows) * c.splits * 4 + static_cast<size_t>(rows) * c.n_groups) * 4 : 0;
  return c;
}

template <typename T>
void launch(const ScoreArgs& a, hipStream_t s) {
  score_kernel<T><<<dim3(static_cast<unsigned>(a.rows * a.splits)), dim3(kThreads), 0, s>>>(a);
  if (a.splits > 1) score_finish_kernel<T><<<dim3(static_cast<unsigned>(a.rows)), dim3(kThreads), 0, s>>>(a);
}

int check_sizes(const char* what, int vocab, int64_t rows, int dtype) {
  FDLLM_CHECK_ARG(dtype == FDLLM_DTYPE_BF16 || dtype == FDLLM_DTYPE_F16 || dtype == FDLLM_DTYPE_F32,
                  "%s: dtype %d unsupported", what, dtype);
  FDLLM_CHECK_ARG(vocab > 0 && vocab <= kMaxVocab - 8, "%s: vocab %d (1 to %d)", what, vocab, kMaxVocab - 8);
  FDLLM_CHECK_ARG(rows >= 0 && rows <= 0x7fffffff, "%s: bad row count", what);
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
  FDLLM_CHECK_ARG(rows * c.splits <= 0x7fffffff, "%s: too many rows", what);
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

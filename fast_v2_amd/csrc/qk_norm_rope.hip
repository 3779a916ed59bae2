// Norms of the query and key heads, the position rotation and the paged K / V write in one
// pass (fdllm_norm_rope_kv_write).
//
//   x^ = x rsqrt(mean(x^2) + eps) w            (per head; x itself without a weight)
//   y0 = x0 c - x1 s,  y1 = x1 c + x0 s        c, s = rope_scale cos, sin(position f_i)
//
// over the pairs (i, i + R/2) or (2i, 2i + 1) of a head's first R dimensions; the others pass.
// Everything is held in fp32 and rounded once, where it is stored.
//
// Angles: position f_i reaches 2^17 radians and more at far positions, where fp32 is off by
// 2^-7, so the turns are counted in 64 bits and only the part of a turn that is left goes to
// fp32. What a token's heads have in common (w cos, w sin of every dimension) is a table in LDS,
// computed once while the heads' rows are in flight.
//
// A head's row lies across 2^k lanes, 8 elements each (16-byte loads of 16-bit types); the
// mean of squares is a sum over those lanes, and the partner of a half-layout pair comes from
// another lane of the group, by a lane shuffle where R/2 is a multiple of 8 and through LDS
// elsewhere.
//
// What bounds it: many tokens, memory: 4 x 4096 tokens of 28 + 4 + 4 heads of 128 in bf16 (302 MB)
// take 61 us, 4.98 TB/s, what a large copy reaches (4.9); with stores that stay in the caches 65
// us (fp32 rows, whose 32 bytes a lane are two stores, 60 us so and 75 us past the caches, so
// they stay). Few tokens, latency: one token 3.4 us, 16 x 8 4.1 us, of which an empty kernel is
// 1.5: arguments, position and slot, rows and weights, stores. A workgroup for every token with a
// barrier before its heads took 140 us for the large call; angles per wave with weights read
// and converted one by one 66 us, and 8.2 us for 1501 packed tokens (6.5 with two waves for each).
#include <algorithm>

#include "fdllm_common.h"

namespace fdllm {
namespace {

// 8 elements of a row in registers.
template <typename T>
struct Row8 {
  u32x4 w;
  __device__ __forceinline__ void load(const void* base, int64_t at) {
    w = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(base) + at));
  }
  __device__ __forceinline__ void store(void* base, int64_t at) const {
    __builtin_nontemporal_store(w, reinterpret_cast<u32x4*>(static_cast<uint16_t*>(base) + at));
  }
  __device__ __forceinline__ void get(float* f) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = Elt<T>::lo(w[i]);
      f[2 * i + 1] = Elt<T>::hi(w[i]);
    }
  }
  __device__ __forceinline__ void set(const float* f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = Elt<T>::pack(f[2 * i], f[2 * i + 1]);
  }
  __device__ __forceinline__ Row8 of_lane(int from) const {
    Row8 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r.w[i] = __shfl(static_cast<int>(w[i]), from, kWave);
    return r;
  }
  __device__ __forceinline__ static float lo(uint32_t word) { return Elt<T>::lo(word); }
  __device__ __forceinline__ static float hi(uint32_t word) { return Elt<T>::hi(word); }
};
template <>
struct Row8<float> {
  f32x4 w[2];
  __device__ __forceinline__ void load(const void* base, int64_t at) {
    const f32x4* p = reinterpret_cast<const f32x4*>(static_cast<const float*>(base) + at);
    w[0] = __builtin_nontemporal_load(p);
    w[1] = __builtin_nontemporal_load(p + 1);
  }
  __device__ __forceinline__ void store(void* base, int64_t at) const {
    f32x4* p = reinterpret_cast<f32x4*>(static_cast<float*>(base) + at);
    p[0] = w[0];
    p[1] = w[1];
  }
  __device__ __forceinline__ void get(float* f) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = w[i >> 2][i & 3];
  }
  __device__ __forceinline__ void set(const float* f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i >> 2][i & 3] = f[i];
  }
  __device__ __forceinline__ Row8 of_lane(int from) const {
    Row8 r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r.w[i >> 2][i & 3] = __shfl(w[i >> 2][i & 3], from, kWave);
    return r;
  }
  __device__ __forceinline__ static float lo(uint32_t word) { return __uint_as_float(word); }
  __device__ __forceinline__ static float hi(uint32_t word) { return __uint_as_float(word); }
};

struct NormRopeArgs {
  fdllm_norm_rope_kv_desc d;
  int shift;  // log2(page_size)
  int q_steps, k_steps, all_steps;  // of a token: 64 / LPH query, key or value heads each
  uint32_t tokens;
  int parts;  // waves that share a token
};

constexpr int kMaxDim = 256;
constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
// Tokens from which a wave takes a whole one. Below, a workgroup's four waves share a token (its angles
// are computed once), with other workgroups while there are at most kResident waves; from kPairTokens on two
// waves share one, which is less code to issue in all and fills the machine no less. us, four / two waves / one:
//   bf16, 28 + 4 + 4 heads of 128: 1 token 3.4 / - / 7.3, 128 4.1 / - / 8.3, 1000 7.1 / 8.0 / -,
//     1501 10.3 / 9.4 / 11.6, 2048 13.8 / 10.9 / 12.8, 3000 - / 15.4 / 14.4
//   fp32, 12 + 2 + 2 heads of 128: 1000 6.6 / 6.7 / -, 1501 9.7 / 8.8 / -, 2048 - / 10.7 / 10.9, 3000 - / 15.2 / 14.6
// More waves a token, the latter (eight / four): 128 tokens 3.8 / 3.9, 314 4.7 / 4.4, 600 7.7 / 5.3.
constexpr int kTokenPerWave = 2560;
constexpr int kPairTokens = 1280;
constexpr int kResident = 2048;
constexpr int kAhead = 2;  // a wave's steps in flight
constexpr int kMaxTokens = (1 << 25) - 1;  // a launch has fewer than 2^32 threads, a token 64, and workgroups are whole

// Sum over groups of L consecutive lanes.
template <int L>
__device__ __forceinline__ float group_sum(float v) {
  v += dpp_f32<0xB1>(v);
  v += dpp_f32<0x4E>(v);
  v += dpp_f32<0x141>(v);
  if constexpr (L >= 16) v += dpp_f32<0x140>(v);
  if constexpr (L >= 32) v += __shfl_xor(v, 16, kWave);
  return v;
}

// Orders one wave's LDS accesses (a head's lanes are in one wave).
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// By value: a conditional on members of the arguments would select between their addresses, and
// a copy of the whole struct would go to scratch.
template <typename V>
__device__ __forceinline__ V pick(int kind, V q, V k, V v) {
  return kind == 0 ? q : (kind == 1 ? k : v);
}

enum Layout { kHalfLanes, kHalfLds, kInterleaved };

// LPH: lanes per head (8, 16 or 32).
template <typename T, int LPH, Layout LAY>
__global__ __launch_bounds__(kThreads) void norm_rope_kernel(const NormRopeArgs a) {
  const fdllm_norm_rope_kv_desc& d = a.d;
  constexpr int HPS = 64 / LPH;  // heads per step, all of one kind
  constexpr int W = LPH * 8;     // head_dim at most
  // y_e = r (x_e C_e + x_partner(e) S_e), C_e = w_e cos, S_e = -+ w_partner(e) sin: C and S are
  // the same for all query heads of a token and for all of its key heads
  __shared__ __attribute__((aligned(16))) float s_c[kWaves][2][W], s_s[kWaves][2][W];
  __shared__ __attribute__((aligned(16))) float s_rows[LAY == kHalfLds ? kWaves : 1][LAY == kHalfLds ? 64 * 8 : 1];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  // A wave takes a whole token (parts 1), two share one, or a workgroup's waves, and those of others, do. 32-bit
  // divisions: there are fewer than 2^31 tokens, and a token has parts only where there are few
  const uint32_t job = blockIdx.x * kWaves + wave;
  const uint32_t row = min(job / static_cast<uint32_t>(a.parts), a.tokens - 1);
  const int part = static_cast<int>(job - row * a.parts);  // a wave past the last token has part >= parts
  const int last = part < a.parts ? a.all_steps : 0;
  const int64_t token = row;
  const int b = static_cast<int>(row / static_cast<uint32_t>(d.seq_len));
  const int t = static_cast<int>(row - static_cast<uint32_t>(b) * d.seq_len);
  const int D = d.head_dim, R = d.rotary_dim, half = R / 2;
  const int g = lane & (LPH - 1), c = g * 8, sub = lane / LPH;
  const int64_t slot = d.slots ? d.slots[token] : -1;
  const bool keep = slot >= 0 && (slot >> a.shift) < d.num_pages;
  const int64_t page = slot >> a.shift, off = slot & ((1 << a.shift) - 1);

  // step s: its kind (0 query, 1 key, 2 value heads), this lane's head and whether it has one
  auto kind_of = [&](int s) __attribute__((always_inline)) {
    return s < a.q_steps ? 0 : (s < a.q_steps + a.k_steps ? 1 : 2);
  };
  auto head_of = [&](int s, int kind) __attribute__((always_inline)) {
    return (s - pick(kind, 0, a.q_steps, a.q_steps + a.k_steps)) * HPS + sub;
  };
  auto live = [&](int kind, int head) __attribute__((always_inline)) {
    return c < D && head < pick(kind, d.num_q_heads, d.num_kv_heads, d.num_kv_heads) && (kind != 2 || keep);
  };
  const int64_t q_at = b * d.q_stride_b + t * d.q_stride_s, k_at = b * d.k_stride_b + t * d.k_stride_s,
                v_at = b * d.v_stride_b + t * d.v_stride_s;
  auto fetch = [&](int s, Row8<T>& x) __attribute__((always_inline)) {
    if (s >= last) return;
    const int kind = kind_of(s), head = head_of(s, kind);
    if (live(kind, head))
      x.load(pick(kind, d.q, d.k, d.v), pick(kind, q_at, k_at, v_at) + head * pick(kind, d.q_stride_h, d.k_stride_h, d.v_stride_h) + c);
  };
  Row8<T> x[kAhead];
#pragma unroll
  for (int k = 0; k < kAhead; ++k) fetch(part + k * a.parts, x[k]);

  // the tables, while the rows are in flight. Weights are read as whole words and taken apart
  // later: a conversion beside each load would wait for them one after another
  // (parts is 1, 2 or a multiple of kWaves)
  const int by = 64 * min(a.parts, kWaves), at = threadIdx.x & (by - 1), tab = a.parts == 1 ? wave : a.parts == 2 ? wave >> 1 : 0;
  const bool wide = d.weight_dtype == FDLLM_DTYPE_F32;
  const void* const wq = d.q_weight ? d.q_weight : d.k_weight;
  const void* const wk = d.k_weight ? d.k_weight : d.q_weight;
  auto word = [&](const void* w, int e) __attribute__((always_inline)) {
    return static_cast<const uint32_t*>(w)[wide ? e : e >> 1];
  };
  auto value = [&](uint32_t w, int e, const void* given) __attribute__((always_inline)) {
    const float v = wide ? __uint_as_float(w) : (e & 1 ? Row8<T>::hi(w) : Row8<T>::lo(w));
    return given != nullptr ? v : 1.f;
  };
  for (int i = at; i < half; i += by) {
    const int e0 = LAY == kInterleaved ? 2 * i : i, e1 = LAY == kInterleaved ? e0 + 1 : i + half;
    const float f = d.inv_freq[i];
    uint32_t u[4] = {0, 0, 0, 0};
    if (wq != nullptr) {
      u[0] = word(wq, e0);
      u[1] = word(wq, e1);
      u[2] = word(wk, e0);
      u[3] = word(wk, e1);
    }
    // half turns: an even number of them is left out, so the rest is within one of zero
    const double turns = static_cast<double>(d.positions[token]) * static_cast<double>(f) * 0.318309886183790671538;
    float sn, cs;
    sincospif(static_cast<float>(turns - 2.0 * __builtin_rint(0.5 * turns)), &sn, &cs);
    cs *= d.rope_scale;
    sn *= d.rope_scale;
    const float q0 = value(u[0], e0, d.q_weight), q1 = value(u[1], e1, d.q_weight);
    const float k0 = value(u[2], e0, d.k_weight), k1 = value(u[3], e1, d.k_weight);
    s_c[tab][0][e0] = q0 * cs;
    s_c[tab][0][e1] = q1 * cs;
    s_s[tab][0][e0] = -q1 * sn;
    s_s[tab][0][e1] = q0 * sn;
    s_c[tab][1][e0] = k0 * cs;
    s_c[tab][1][e1] = k1 * cs;
    s_s[tab][1][e0] = -k1 * sn;
    s_s[tab][1][e1] = k0 * sn;
  }
  for (int e = R + at; e < D; e += by) {
    uint32_t u[2] = {0, 0};
    if (wq != nullptr) {
      u[0] = word(wq, e);
      u[1] = word(wk, e);
    }
    s_c[tab][0][e] = value(u[0], e, d.q_weight);
    s_c[tab][1][e] = value(u[1], e, d.k_weight);
  }
  __syncthreads();
  // the lane that holds the partners of this one's dimensions (itself where they have none)
  int from = lane;
  if (LAY == kHalfLanes && c < R) from = lane + (c < half ? half / 8 : -half / 8);

  float C[8], S[8];
  int now = -1;
  for (int s0 = part; s0 < last; s0 += kAhead * a.parts) {
#pragma unroll
    for (int p = 0; p < kAhead; ++p) {
      const int s = s0 + p * a.parts;
      if (s >= last) break;
      const int kind = kind_of(s), head = head_of(s, kind);
      const bool mine = live(kind, head);
      const Row8<T> here = x[p];
      fetch(s + kAhead * a.parts, x[p]);
      if (kind == 2) {
        if (mine) here.store(d.v_cache, page * d.v_stride_page + off * d.v_stride_slot + head * d.v_stride_ch + c);
        continue;
      }
      if (kind != now) {
        now = kind;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          C[j] = s_c[tab][kind][c + j];
          S[j] = s_s[tab][kind][c + j];
        }
      }
      float f[8], o[8];
      here.get(f);
      if (!mine) {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = 0.f;
      }
      float r = 1.f;
      if (pick(kind, d.q_weight, d.k_weight, d.k_weight) != nullptr) {
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = __builtin_fmaf(f[j], f[j], ss);
        r = rsqrtf(group_sum<LPH>(ss) * (1.f / D) + d.eps);
      }
      if constexpr (LAY == kInterleaved) {
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = f[j ^ 1];
      } else if constexpr (LAY == kHalfLanes) {
        here.of_lane(from).get(o);
      } else {
        float* all = s_rows[wave] + (lane & ~(LPH - 1)) * 8;
#pragma unroll
        for (int j = 0; j < 8; ++j) all[c + j] = f[j];
        wave_sync();
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int e = c + j;
          o[j] = all[e < half ? e + half : (e < R ? e - half : e)];
        }
        wave_sync();
      }
      if (!mine) continue;
      float y[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float own = f[j] * C[j];
        y[j] = r * (c + j < R ? __builtin_fmaf(o[j], S[j], own) : own);  // what is not turned has no partner
      }
      Row8<T> out;
      out.set(y);
      if (kind == 0) {
        out.store(d.q_out, (token * d.num_q_heads + head) * D + c);
      } else {
        if (keep) out.store(d.k_cache, page * d.k_stride_page + off * d.k_stride_slot + head * d.k_stride_ch + c);
        if (d.k_out) out.store(d.k_out, (token * d.num_kv_heads + head) * D + c);
      }
    }
  }
}

template <typename T, int LPH>
void launch(NormRopeArgs a, Layout lay, int64_t tokens, hipStream_t s) {
  a.tokens = static_cast<uint32_t>(tokens);
  constexpr int HPS = 64 / LPH;
  a.q_steps = (a.d.num_q_heads + HPS - 1) / HPS;
  a.k_steps = (a.d.num_kv_heads + HPS - 1) / HPS;
  const int all = a.all_steps = a.q_steps + (a.d.k_cache ? 2 : 1) * a.k_steps;  // value heads only go to the cache
  a.parts = 1;
  if (tokens < kTokenPerWave && tokens >= kPairTokens) {
    a.parts = 2;
  } else if (tokens < kTokenPerWave) {
    a.parts = (all + kWaves - 1) / kWaves * kWaves;
    while (a.parts > kWaves && tokens * a.parts > kResident) a.parts -= kWaves;
  }
  const dim3 grid(static_cast<unsigned>((tokens * a.parts + kWaves - 1) / kWaves)), block(kThreads);
  if (lay == kInterleaved) norm_rope_kernel<T, LPH, kInterleaved><<<grid, block, 0, s>>>(a);
  else if (lay == kHalfLanes) norm_rope_kernel<T, LPH, kHalfLanes><<<grid, block, 0, s>>>(a);
  else norm_rope_kernel<T, LPH, kHalfLds><<<grid, block, 0, s>>>(a);
}

template <typename T>
void launch(const NormRopeArgs& a, Layout lay, int64_t tokens, hipStream_t s) {
  if (a.d.head_dim <= 64) launch<T, 8>(a, lay, tokens, s);
  else if (a.d.head_dim <= 128) launch<T, 16>(a, lay, tokens, s);
  else launch<T, 32>(a, lay, tokens, s);
}

}  // namespace
}  // namespace fdllm

extern "C" int fdllm_norm_rope_kv_write(const fdllm_norm_rope_kv_desc* desc, void* stream) {
  using namespace fdllm;
  const char* what = "fdllm_norm_rope_kv_write";
  FDLLM_CHECK_ARG(desc != nullptr, "%s: null descriptor", what);
  const fdllm_norm_rope_kv_desc& d = *desc;
  FDLLM_CHECK_ARG(d.dtype == FDLLM_DTYPE_BF16 || d.dtype == FDLLM_DTYPE_F16 || d.dtype == FDLLM_DTYPE_F32,
                  "%s: dtype %d unsupported", what, d.dtype);
  FDLLM_CHECK_ARG(d.weight_dtype == d.dtype || d.weight_dtype == FDLLM_DTYPE_F32,
                  "%s: norm weights must have the heads' dtype or be fp32", what);
  FDLLM_CHECK_ARG(d.head_dim >= 8 && d.head_dim % 8 == 0 && d.head_dim <= kMaxDim,
                  "%s: head_dim %d must be a multiple of 8, at most %d", what, d.head_dim, kMaxDim);
  FDLLM_CHECK_ARG(d.rotary_dim >= 0 && d.rotary_dim % 2 == 0 && d.rotary_dim <= d.head_dim,
                  "%s: rotary_dim %d must be even and at most head_dim", what, d.rotary_dim);
  FDLLM_CHECK_ARG(d.batch >= 0 && d.seq_len >= 0 && d.num_q_heads > 0 && d.num_kv_heads > 0 &&
                      d.num_q_heads <= 4096 && d.num_kv_heads <= 4096,
                  "%s: bad sizes", what);
  const int64_t tokens = static_cast<int64_t>(d.batch) * d.seq_len;
  if (tokens == 0) return FDLLM_OK;
  FDLLM_CHECK_ARG(tokens <= kMaxTokens, "%s: %lld tokens (at most %d)", what, static_cast<long long>(tokens), kMaxTokens);
  FDLLM_CHECK_ARG(d.q && d.k && d.v && d.q_out && (d.rotary_dim == 0 || (d.positions && d.inv_freq)),
                  "%s: null pointer", what);
  FDLLM_CHECK_ARG((d.k_cache != nullptr) == (d.v_cache != nullptr) && (d.k_cache != nullptr) == (d.slots != nullptr),
                  "%s: give both caches with the slots", what);
  FDLLM_CHECK_ARG(d.k_cache == nullptr || (d.page_size > 0 && (d.page_size & (d.page_size - 1)) == 0 && d.num_pages >= 0),
                  "%s: page_size %d is not a power of two", what, d.page_size);
  const int64_t vec = d.dtype == FDLLM_DTYPE_F32 ? 4 : 8;  // elements of 16 bytes
  for (int64_t st : {d.q_stride_b, d.q_stride_s, d.q_stride_h, d.k_stride_b, d.k_stride_s, d.k_stride_h, d.v_stride_b,
                     d.v_stride_s, d.v_stride_h, d.k_stride_page, d.k_stride_slot, d.k_stride_ch, d.v_stride_page,
                     d.v_stride_slot, d.v_stride_ch})
    FDLLM_CHECK_ARG(st % vec == 0, "%s: strides must be multiples of 16 bytes", what);
  for (const void* p : {d.q, d.k, d.v, static_cast<const void*>(d.q_out), static_cast<const void*>(d.k_out),
                        static_cast<const void*>(d.k_cache), static_cast<const void*>(d.v_cache), d.q_weight, d.k_weight})
    FDLLM_CHECK_ARG((reinterpret_cast<uintptr_t>(p) & 15u) == 0, "%s: rows must be 16-byte aligned", what);
  NormRopeArgs a;
  a.d = d;
  a.shift = d.k_cache ? __builtin_ctz(static_cast<unsigned>(d.page_size)) : 0;
  const Layout lay = d.interleaved ? kInterleaved : ((d.rotary_dim / 2) % 8 == 0 ? kHalfLanes : kHalfLds);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (d.dtype == FDLLM_DTYPE_BF16) launch<bf16_t>(a, lay, tokens, s);
  else if (d.dtype == FDLLM_DTYPE_F16) launch<f16_t>(a, lay, tokens, s);
  else launch<float>(a, lay, tokens, s);
  FDLLM_RETURN_LAUNCH_STATUS(what);
}

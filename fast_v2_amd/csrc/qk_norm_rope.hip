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
// fp32. One workgroup takes one token, so its R/2 angles are computed once and meet its heads
// in LDS; their arithmetic runs while the heads' rows are in flight.
//
// A head's row lies across 2^k lanes, 8 elements each (16-byte loads of 16-bit types); the
// mean of squares is a sum over those lanes, and the partner of a half-layout pair comes from
// another lane of the group, by a lane shuffle where R/2 is a multiple of 8 and through LDS
// elsewhere.
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
    *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(base) + at) = w;
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
};

struct NormRopeArgs {
  fdllm_norm_rope_kv_desc d;
  int shift;  // log2(page_size)
  int units;  // heads of a token: query, key and value heads
};

constexpr int kMaxDim = 256;

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

enum Layout { kHalfLanes, kHalfLds, kInterleaved };

// LPH: lanes per head (8, 16 or 32).
template <typename T, int LPH, Layout LAY>
__global__ __launch_bounds__(1024) void norm_rope_kernel(const NormRopeArgs a) {
  const fdllm_norm_rope_kv_desc& d = a.d;
  __shared__ __attribute__((aligned(16))) float s_cos[kMaxDim / 2], s_sin[kMaxDim / 2];
  extern __shared__ __attribute__((aligned(16))) float s_row[];  // kHalfLds: 8 floats per thread
  const int64_t token = blockIdx.x;
  const int b = static_cast<int>(token / d.seq_len);
  const int t = static_cast<int>(token - static_cast<int64_t>(b) * d.seq_len);
  const int tid = threadIdx.x;
  const int D = d.head_dim, R = d.rotary_dim, half = R / 2;
  const int g = tid & (LPH - 1), c = g * 8;
  const bool in_row = c < D;
  const int step = blockDim.x / LPH;

  const int64_t slot = d.slots ? d.slots[token] : -1;
  const bool keep = slot >= 0 && (slot >> a.shift) < d.num_pages;
  const int64_t page = slot >> a.shift, off = slot & ((1 << a.shift) - 1);
  const int Hq = d.num_q_heads, Hk = d.num_kv_heads;
  auto where = [&](int u) __attribute__((always_inline)) {
    const int kind = u < Hq ? 0 : (u < Hq + Hk ? 1 : 2);
    return kind;
  };
  auto fetch = [&](int u, Row8<T>& x) __attribute__((always_inline)) {
    const int kind = where(u);
    const void* base = kind == 0 ? d.q : (kind == 1 ? d.k : d.v);
    const int h = u - (kind == 0 ? 0 : (kind == 1 ? Hq : Hq + Hk));
    const int64_t sb = kind == 0 ? d.q_stride_b : (kind == 1 ? d.k_stride_b : d.v_stride_b);
    const int64_t ss = kind == 0 ? d.q_stride_s : (kind == 1 ? d.k_stride_s : d.v_stride_s);
    const int64_t sh = kind == 0 ? d.q_stride_h : (kind == 1 ? d.k_stride_h : d.v_stride_h);
    x.load(base, b * sb + t * ss + h * sh + c);
  };
  int u = tid / LPH;
  Row8<T> x;
  if (u < a.units && in_row) fetch(u, x);
  for (int i = tid; i < half; i += blockDim.x) {
    // half turns: an even number of them is left out, so the rest is within one of zero
    const double turns = static_cast<double>(d.positions[token]) * static_cast<double>(d.inv_freq[i]) *
                         0.318309886183790671538;
    const float rest = static_cast<float>(turns - 2.0 * __builtin_rint(0.5 * turns));
    float sn, cs;
    sincospif(rest, &sn, &cs);
    s_cos[i] = cs * d.rope_scale;
    s_sin[i] = sn * d.rope_scale;
  }
  __syncthreads();
  for (; u < a.units; u += step) {  // uniform over a head's lanes
    const int kind = where(u);
    if (kind == 2) {
      if (in_row && keep) x.store(d.v_cache, page * d.v_stride_page + off * d.v_stride_slot + (u - Hq - Hk) * d.v_stride_ch + c);
    } else {
      float f[8];
      if (in_row) {
        x.get(f);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = 0.f;
      }
      const void* wp = kind == 0 ? d.q_weight : d.k_weight;
      if (wp != nullptr) {
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = __builtin_fmaf(f[j], f[j], ss);
        ss = group_sum<LPH>(ss);
        const float r = rsqrtf(ss * (1.f / D) + d.eps);
        float w[8];
        if (in_row) {
          if (d.weight_dtype == FDLLM_DTYPE_F32) {
            Row8<float> ww;
            ww.load(wp, c);
            ww.get(w);
          } else {
            Row8<T> ww;
            ww.load(wp, c);
            ww.get(w);
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) f[j] = f[j] * r * w[j];
        }
      }
      float y[8];
      if constexpr (LAY == kInterleaved) {
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          const bool turn = c + j < R;
          const int i = min((c + j) >> 1, kMaxDim / 2 - 1);
          const float cs = s_cos[i], sn = s_sin[i];
          y[j] = turn ? f[j] * cs - f[j + 1] * sn : f[j];
          y[j + 1] = turn ? f[j + 1] * cs + f[j] * sn : f[j + 1];
        }
      } else {
        float o[8];  // the partners
        if constexpr (LAY == kHalfLanes) {
          const int hop = half / 8;  // lanes
          const int from = (tid & 63 & ~(LPH - 1)) + (c < half ? g + hop : g - hop);
#pragma unroll
          for (int j = 0; j < 8; ++j) o[j] = __shfl(f[j], from, kWave);
        } else {
          float* row = s_row + (tid & ~(LPH - 1)) * 8;
#pragma unroll
          for (int j = 0; j < 8; ++j) row[c + j] = f[j];
          wave_sync();
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int e = c + j;
            o[j] = row[e < half ? e + half : (e < R ? e - half : e)];
          }
          wave_sync();
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int e = c + j;
          const int i = min(e < half ? e : e - half, kMaxDim / 2 - 1);
          const float cs = s_cos[i], sn = e < half ? -s_sin[i] : s_sin[i];
          y[j] = e < R ? f[j] * cs + o[j] * sn : f[j];
        }
      }
      if (in_row) {
        Row8<T> out;
        out.set(y);
        if (kind == 0) {
          out.store(d.q_out, (token * Hq + u) * D + c);
        } else {
          if (keep) out.store(d.k_cache, page * d.k_stride_page + off * d.k_stride_slot + (u - Hq) * d.k_stride_ch + c);
          if (d.k_out) out.store(d.k_out, (token * Hk + u - Hq) * D + c);
        }
      }
    }
    if (u + step < a.units && in_row) fetch(u + step, x);
  }
}

template <typename T, int LPH>
void launch(const NormRopeArgs& a, Layout lay, unsigned tokens, int threads, hipStream_t s) {
  if (lay == kInterleaved) norm_rope_kernel<T, LPH, kInterleaved><<<dim3(tokens), dim3(threads), 0, s>>>(a);
  else if (lay == kHalfLanes) norm_rope_kernel<T, LPH, kHalfLanes><<<dim3(tokens), dim3(threads), 0, s>>>(a);
  else norm_rope_kernel<T, LPH, kHalfLds><<<dim3(tokens), dim3(threads), threads * 8 * sizeof(float), s>>>(a);
}

template <typename T>
void launch(const NormRopeArgs& a, Layout lay, unsigned tokens, hipStream_t s) {
  const int lph = a.d.head_dim <= 64 ? 8 : (a.d.head_dim <= 128 ? 16 : 32);
  // every head of the token at once, if a workgroup holds so many lanes
  const int lanes = (a.units * lph + 63) / 64 * 64;
  const int threads = lanes < 1024 ? lanes : 1024;
  if (lph == 8) launch<T, 8>(a, lay, tokens, threads, s);
  else if (lph == 16) launch<T, 16>(a, lay, tokens, threads, s);
  else launch<T, 32>(a, lay, tokens, threads, s);
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
  FDLLM_CHECK_ARG(tokens <= 0x7fffffff, "%s: too many tokens", what);
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
  a.units = d.num_q_heads + (d.k_cache ? 2 : 1) * d.num_kv_heads;  // v rows only go to the cache
  const Layout lay = d.interleaved ? kInterleaved : ((d.rotary_dim / 2) % 8 == 0 ? kHalfLanes : kHalfLds);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (d.dtype == FDLLM_DTYPE_BF16) launch<bf16_t>(a, lay, static_cast<unsigned>(tokens), s);
  else if (d.dtype == FDLLM_DTYPE_F16) launch<f16_t>(a, lay, static_cast<unsigned>(tokens), s);
  else launch<float>(a, lay, static_cast<unsigned>(tokens), s);
  FDLLM_RETURN_LAUNCH_STATUS(what);
}

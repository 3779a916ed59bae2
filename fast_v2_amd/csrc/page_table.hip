// Pages for a step's new tokens (fdllm_assign_pages) and back (fdllm_release_pages): the page
// table, slots and positions that the paged cache's callers need, from the requests' lengths,
// without a word from the host.
//
// With page size p, request b's pages in hand h_b = ceil(len_b / p) and after the step
// t_b = ceil((len_b + n_b) / p), it needs d_b = t_b - h_b pages; with c_b the running sum of d
// it gets them when c_b is at most the free count, as new page number i = c_b - d_b + (0 ..
// d_b - 1), which is free_pages[free_count - 1 - i]. Rows of a packed token list begin at the
// running sum of n. Both sums are one scan over the requests in one workgroup (saturating
// 32-bit sums of non-negative numbers, which stay associative: what does not fit saturates
// above every capacity). A new page's first row is a granted one, so the row that it begins with
// enters it into the table, and the rows' threads take page ids from the free list by themselves. A
// packed row's request, and of a page that goes back, is found by a binary search of the running sums
// in LDS: long prompts are spread over all threads as evenly as single tokens.
//
// What bounds it: latency. The bytes of the largest call take 0.2 us; the calls are chains
// of dependent memory round trips (arguments, lengths, table or free list, stores) and the scans' barriers:
// 16 x 8 rows 2.3 us and 2.0 us to release them, 2048 x 32 rows (4096 pages) 2.8 + 3.5 and 5.4. With the
// pages searched and entered by the plan's workgroup the plan took 8.5, and with scans that exchange through
// LDS each scan 0.5 us more.
#include "fdllm_common.h"

namespace fdllm {
namespace {

constexpr int kPlanThreads = 1024;
// Threads where there are at most as many requests and, to assign, rows. us, 256 / 1024 (assign and
// release): 16 x 8 rows 4.3 / 4.6, 64 x 8 4.9 / 4.6; to release up to 256 pages 0.15 less, 512 0.2 more, 4096 4.5
// more (once a request, the others at every step).
constexpr int kSmallThreads = 256;
constexpr int kMaxRequests = 8192;
// Rows up to which the plan's workgroup makes them too. us, one kernel / two (assign and release): 16 x 8
// rows 4.3 / 5.8, 256 x 16 6.5 / 7.0, 256 x 32 8.7 / 7.0, 1024 x 16 13.5 / 7.9; packed, 300 requests and
// 4096 rows 7.4 / 8.5, 16 and 8192 10.1 / 8.0.
constexpr int kOneKernelRows = 4096;

__device__ __forceinline__ uint32_t add_sat(uint32_t a, uint32_t b) { return __builtin_elementwise_add_sat(a, b); }

// A thread's k-th request: neighbouring lanes take neighbouring ones, so that loads and stores are whole lines.
template <int ITEMS>
__device__ __forceinline__ int request_of(int k) {
  return (threadIdx.x & ~63u) * ITEMS + k * 64 + (threadIdx.x & 63u);
}

// x from another lane of the wave; 0 where there is none, or outside of the rows (of 16 lanes) in ROWS
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_up(uint32_t x) {
  return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), CTRL, ROWS, 0xf, false));
}

// Per request the sum over those before it; returns the sum over all.
template <int T, int ITEMS>
__device__ __forceinline__ uint32_t block_scan(const uint32_t (&x)[ITEMS], uint32_t (&before)[ITEMS], uint32_t* s_wave) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint32_t of_wave = 0;
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    uint32_t y = x[k];
    y = add_sat(y, dpp_up<0x111, 0xf>(y));  // from 1, 2, 4 and 8 lanes below in a row
    y = add_sat(y, dpp_up<0x112, 0xf>(y));
    y = add_sat(y, dpp_up<0x114, 0xf>(y));
    y = add_sat(y, dpp_up<0x118, 0xf>(y));
    y = add_sat(y, dpp_up<0x142, 0xa>(y));  // a row's last lane to the next row: 0 to 1, 2 to 3
    y = add_sat(y, dpp_up<0x143, 0xc>(y));  // lane 31 to rows 2 and 3
    before[k] = add_sat(of_wave, dpp_up<0x138, 0xf>(y));  // from the lane below: saturated sums do not subtract
    of_wave = add_sat(of_wave, __builtin_amdgcn_readlane(y, 63));
  }
  if ((threadIdx.x & 63) == 0) s_wave[wave] = of_wave;
  __syncthreads();
  uint32_t y = s_wave[threadIdx.x & (T / 64 - 1)];
  y = add_sat(y, dpp_up<0x111, 0xf>(y));
  y = add_sat(y, dpp_up<0x112, 0xf>(y));
  if constexpr (T > 256) {
    y = add_sat(y, dpp_up<0x114, 0xf>(y));
    y = add_sat(y, dpp_up<0x118, 0xf>(y));
  }
  const uint32_t lower = wave != 0 ? __builtin_amdgcn_readlane(y, max(wave - 1, 0)) : 0;
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) before[k] = add_sat(lower, before[k]);
  return __builtin_amdgcn_readlane(y, T / 64 - 1);
}

// First b with upto[b] > i, of N (a power of two) entries; N where there is none. Without branches, so
// that several searches run side by side.
template <int N>
__device__ __forceinline__ int first_above(const uint32_t* upto, uint32_t i) {
  int at = 0;
#pragma unroll
  for (int s = N / 2; s >= 1; s /= 2) at += upto[at + s - 1] <= i ? s : 0;
  return at + (upto[at] <= i ? 1 : 0);
}

// Pages of a thread's release at a time: many requests need them, few are quicker in little code, which is
// loaded for every call (16 requests of 8 pages 0.3 us less with one than with four).
template <int ITEMS>
constexpr int side() {
  return ITEMS == 1 ? 1 : 4;
}

struct AssignArgs {
  fdllm_page_pool pool;
  const int32_t* new_lens;
  int width, rows, shift;
  int64_t* slots;
  int32_t* positions;
  int32_t* sequences;
  int32_t* row_starts;
  int32_t* starts;
  int32_t* seqlens;
  int32_t* granted;
  int32_t* list_at;  // of the rows' kernel: a request's page j, if it is new, is the free list's entry list_at - j
};

// Row r: the request's t-th asked token (b < 0: none), from its length before the step. A page in hand
// comes from the table, a new one from the free list; its first row enters it.
__device__ __forceinline__ void put_row(const AssignArgs& a, int r, int b, int t, uint32_t len, bool ok, int32_t list_at) {
  const fdllm_page_pool& p = a.pool;
  const uint32_t mask = (1u << a.shift) - 1;
  int64_t pos = 0, slot = -1;
  if (b >= 0) {
    pos = static_cast<int64_t>(len) + t;
    if (ok) {
      const uint32_t j = static_cast<uint32_t>(pos >> a.shift), off = static_cast<uint32_t>(pos) & mask;
      int32_t* const entry = p.page_table + b * p.table_stride + j;
      int32_t page;
      if (j < (len + mask) >> a.shift) {
        page = *entry;
      } else {
        page = p.free_pages[list_at - static_cast<int32_t>(j)];
        if (off == 0) *entry = page;
      }
      slot = (static_cast<int64_t>(page) << a.shift) + off;
    }
  }
  a.slots[r] = slot;
  a.positions[r] = static_cast<int32_t>(pos);
  if (a.sequences) a.sequences[r] = b;
}

// The requests' part, and in the form of one kernel (ROWS) the rows': one workgroup, ITEMS
// requests per thread.
template <int T, int ITEMS, bool ROWS>
__global__ __launch_bounds__(T) void assign_plan_kernel(const AssignArgs a, int n_rows) {
  __shared__ uint32_t s_wave[2][T / 64];
  __shared__ int32_t s_at[ROWS ? T * ITEMS : 1];     // list_at
  __shared__ uint32_t s_end[ROWS ? T * ITEMS : 1];  // running sum of the asked tokens
  __shared__ uint32_t s_len[ROWS ? T * ITEMS : 1];  // length, the top bit: granted
  __shared__ uint32_t s_new[ROWS ? T * ITEMS : 1];
  const fdllm_page_pool& p = a.pool;
  const int tid = threadIdx.x;
  const uint32_t mask = (1u << a.shift) - 1;
  const int count = *p.free_count;
  uint32_t n[ITEMS], len[ITEMS], need[ITEMS], have[ITEMS], at[ITEMS], before[ITEMS];
  int32_t old[ITEMS];
  bool asks[ITEMS];
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    const int b = request_of<ITEMS>(k);
    n[k] = b < p.requests ? max(a.new_lens[b], 0) : 0;
    old[k] = b < p.requests ? p.lens[b] : 0;
    len[k] = max(old[k], 0);
  }
  // rows first (their sum does not depend on what is granted), then the needs of those that fit
  if (a.width == 0) block_scan<T, ITEMS>(n, at, s_wave[0]);
  const uint32_t avail = static_cast<uint32_t>(min(max(count, 0), p.num_free));
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    const int b = request_of<ITEMS>(k);
    const uint32_t end = a.width > 0 ? 0 : add_sat(at[k], n[k]);
    if (a.row_starts && b < p.requests) {
      a.row_starts[b + 1] = static_cast<int32_t>(min(end, 0x7fffffffu));
      if (b == 0) a.row_starts[0] = 0;
    }
    if (ROWS) s_end[b] = end;
    // lengths are below 2^31, so their sum fits 32 unsigned bits
    const uint32_t total = (len[k] + n[k] + mask) >> a.shift;
    have[k] = (len[k] + mask) >> a.shift;
    asks[k] = n[k] > 0 && len[k] + n[k] <= 0x7fffffffu && total <= static_cast<uint32_t>(p.max_pages) &&
              (a.width > 0 ? n[k] <= static_cast<uint32_t>(a.width) : end <= static_cast<uint32_t>(a.rows));
    need[k] = asks[k] ? total - have[k] : 0;
  }
  block_scan<T, ITEMS>(need, before, s_wave[1]);
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    const int b = request_of<ITEMS>(k);
    const int32_t list_at = static_cast<int32_t>(avail - 1 + have[k] - before[k]);
    const uint32_t c = add_sat(before[k], need[k]);
    // by the one request at which the pages run out, or the last
    if (before[k] <= avail && (c > avail || b == T * ITEMS - 1))
      *p.free_count = static_cast<int32_t>(avail - (c > avail ? before[k] : c));
    const bool ok = asks[k] && (need[k] == 0 || c <= avail);
    const uint32_t got = ok ? n[k] : 0;
    if (ROWS) {
      s_at[b] = list_at;
      s_len[b] = len[k] | (ok ? 0x80000000u : 0);
      s_new[b] = n[k];
    }
    if (b < p.requests) {
      a.starts[b] = static_cast<int32_t>(len[k]);
      a.seqlens[b] = static_cast<int32_t>(len[k] + got);
      a.granted[b] = static_cast<int32_t>(got);
      if (!ROWS) a.list_at[b] = list_at;
      if (got != 0 || old[k] < 0) p.lens[b] = static_cast<int32_t>(len[k] + got);
    }
  }
  if constexpr (ROWS) {
    __syncthreads();
#pragma unroll 1
    for (int r = tid; r < n_rows; r += T) {
      int b, t;
      if (a.width > 0) {
        b = static_cast<int>(static_cast<uint32_t>(r) / static_cast<uint32_t>(a.width));
        t = r - b * a.width;
        if (static_cast<uint32_t>(t) >= s_new[b]) b = -1;
      } else {
        b = first_above<T * ITEMS>(s_end, static_cast<uint32_t>(r));
        t = b < p.requests ? r - static_cast<int>(s_end[b] - s_new[b]) : 0;  // an end past r and a begin at most r: no saturation
        if (b >= p.requests) b = -1;
      }
      const uint32_t len = b >= 0 ? s_len[b] : 0;
      put_row(a, r, b, t, len & 0x7fffffffu, len >> 31, b >= 0 ? s_at[b] : 0);
    }
  }
}

// The rows' part by itself, after the plan: their begins in LDS where they have to be searched.
constexpr int kRowsPerWg = 256;  // with 1024 rows the searches of 16384 took 7.4 us in place of 4.2
template <int N>  // at least as many requests
__global__ __launch_bounds__(kRowsPerWg) void assign_rows_kernel(const AssignArgs a, int n_rows) {
  constexpr bool kAll = N <= kPlanThreads;  // what a request's rows need beside it: a round trip less
  __shared__ uint32_t s_end[N], s_len[kAll ? N : 1];
  __shared__ int32_t s_at[kAll ? N : 1];
  const fdllm_page_pool& p = a.pool;
  if (a.width == 0) {
#pragma unroll 4
    for (int k = 0; k < N; k += kRowsPerWg) {
      const int b = threadIdx.x + k, c = min(b, p.requests - 1);
      s_end[b] = static_cast<uint32_t>(a.row_starts[c + 1]);
      if (kAll) {
        s_len[b] = static_cast<uint32_t>(a.starts[c]) | (a.granted[c] > 0 ? 0x80000000u : 0);
        s_at[b] = a.list_at[c];
      }
    }
    __syncthreads();
  }
  const int r = blockIdx.x * kRowsPerWg + threadIdx.x;
  if (r >= n_rows) return;
  int b, t;
  if (a.width > 0) {
    b = static_cast<int>(static_cast<uint32_t>(r) / static_cast<uint32_t>(a.width));
    t = r - b * a.width;
    if (t >= a.new_lens[b]) b = -1;
  } else {
    b = first_above<N>(s_end, static_cast<uint32_t>(r));
    t = b > 0 ? r - static_cast<int>(s_end[min(b, N) - 1]) : r;  // begins are at most r: no saturation
    if (b >= p.requests) b = -1;
  }
  if (b < 0) put_row(a, r, -1, 0, 0, false, 0);
  else if (kAll && a.width == 0) put_row(a, r, b, t, s_len[b] & 0x7fffffffu, s_len[b] >> 31, s_at[b]);
  else put_row(a, r, b, t, static_cast<uint32_t>(a.starts[b]), a.granted[b] > 0, a.list_at[b]);
}

// keep_lens: pages behind the kept lengths go back, the last ones first.
struct ReleaseArgs {
  fdllm_page_pool pool;
  const int32_t* keep_lens;
  int shift;
};

template <int T, int ITEMS>
__global__ __launch_bounds__(T) void release_kernel(const ReleaseArgs a) {
  __shared__ uint32_t s_wave[T / 64];
  __shared__ uint32_t s_upto[T * ITEMS];
  __shared__ int32_t s_at[T * ITEMS];
  constexpr int kSide = side<ITEMS>();
  const fdllm_page_pool& p = a.pool;
  const int tid = threadIdx.x;
  const uint32_t count = static_cast<uint32_t>(min(max(*p.free_count, 0), p.num_free));
  const uint32_t mask = (1u << a.shift) - 1;
  uint32_t kept[ITEMS], back[ITEMS], before[ITEMS];
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    const int b = request_of<ITEMS>(k);
    kept[k] = back[k] = 0;
    if (b < p.requests) {
      const uint32_t len = max(p.lens[b], 0);
      const uint32_t keep = min(static_cast<uint32_t>(max(a.keep_lens[b], 0)), len);
      const uint32_t most = static_cast<uint32_t>(p.max_pages);
      kept[k] = min((keep + mask) >> a.shift, most);
      back[k] = min((len + mask) >> a.shift, most) - kept[k];
      p.lens[b] = static_cast<int32_t>(keep);
    }
  }
  const uint32_t n = min(block_scan<T, ITEMS>(back, before, s_wave), static_cast<uint32_t>(p.num_free) - count);
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    s_at[request_of<ITEMS>(k)] = static_cast<int32_t>(kept[k] - before[k]);
    s_upto[request_of<ITEMS>(k)] = add_sat(before[k], back[k]);
  }
  __syncthreads();
  for (uint32_t i0 = tid; i0 < n; i0 += kSide * T) {
    int page[kSide];
#pragma unroll
    for (int k = 0; k < kSide; ++k) {
      const uint32_t i = min(i0 + k * T, n - 1);  // the last one may be written twice
      const int b = first_above<T * ITEMS>(s_upto, i);
      page[k] = p.page_table[b * p.table_stride + static_cast<int32_t>(s_at[b] + i)];
    }
#pragma unroll
    for (int k = 0; k < kSide; ++k) p.free_pages[count + n - 1 - min(i0 + k * T, n - 1)] = page[k];
  }
  if (tid == 0) *p.free_count = static_cast<int32_t>(count + n);
}

int check_pool(const char* what, const fdllm_page_pool* p) {
  FDLLM_CHECK_ARG(p != nullptr, "%s: null pool", what);
  FDLLM_CHECK_ARG(p->requests >= 0 && p->requests <= kMaxRequests, "%s: %d requests (0 to %d)", what, p->requests,
                  kMaxRequests);
  FDLLM_CHECK_ARG(p->page_size > 0 && (p->page_size & (p->page_size - 1)) == 0,
                  "%s: page_size %d is not a power of two", what, p->page_size);
  FDLLM_CHECK_ARG(p->max_pages >= 0 && p->num_free >= 0 && p->table_stride >= p->max_pages,
                  "%s: bad table or free list size", what);
  if (p->requests == 0) return FDLLM_OK;
  FDLLM_CHECK_ARG((p->page_table || p->max_pages == 0) && p->lens && (p->free_pages || p->num_free == 0) && p->free_count,
                  "%s: null pointer", what);
  return FDLLM_OK;
}

}  // namespace
}  // namespace fdllm

extern "C" int fdllm_assign_pages(const fdllm_page_pool* pool, const int32_t* new_lens, int width, int rows,
                                  int64_t* slots, int32_t* positions, int32_t* sequences, int32_t* row_starts,
                                  int32_t* starts, int32_t* seqlens, int32_t* granted, int32_t* scratch, void* stream) {
  using namespace fdllm;
  const char* what = "fdllm_assign_pages";
  if (const int rc = check_pool(what, pool)) return rc;
  FDLLM_CHECK_ARG(width >= 0 && rows >= 0 && (width > 0) != (rows > 0),
                  "%s: give the padded form's width or the packed form's rows", what);
  if (pool->requests == 0 && width > 0) return FDLLM_OK;
  FDLLM_CHECK_ARG(pool->requests > 0, "%s: a packed list without requests", what);
  FDLLM_CHECK_ARG(new_lens && slots && positions && starts && seqlens && granted && scratch && (width > 0 || (sequences && row_starts)),
                  "%s: null pointer", what);
  AssignArgs a;
  a.pool = *pool;
  a.new_lens = new_lens;
  a.width = width;
  a.rows = rows;
  a.shift = __builtin_ctz(static_cast<unsigned>(pool->page_size));
  a.slots = slots;
  a.positions = positions;
  a.sequences = width > 0 ? nullptr : sequences;
  a.row_starts = width > 0 ? nullptr : row_starts;
  a.starts = starts;
  a.seqlens = seqlens;
  a.granted = granted;
  a.list_at = scratch;
  const int64_t all_rows = width > 0 ? static_cast<int64_t>(width) * pool->requests : rows;
  FDLLM_CHECK_ARG(all_rows <= 0x7fffffff - kRowsPerWg, "%s: too many rows", what);
  const int n_rows = static_cast<int>(all_rows);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int B = pool->requests;
  constexpr int T = kPlanThreads, S = kSmallThreads;
  if (B <= 2 * T && n_rows <= kOneKernelRows) {
    if (B <= S && n_rows <= S) assign_plan_kernel<S, 1, true><<<dim3(1), dim3(S), 0, s>>>(a, n_rows);
    else if (B <= T) assign_plan_kernel<T, 1, true><<<dim3(1), dim3(T), 0, s>>>(a, n_rows);
    else assign_plan_kernel<T, 2, true><<<dim3(1), dim3(T), 0, s>>>(a, n_rows);
    FDLLM_RETURN_LAUNCH_STATUS(what);
  }
  if (B <= T) assign_plan_kernel<T, 1, false><<<dim3(1), dim3(T), 0, s>>>(a, 0);
  else if (B <= 2 * T) assign_plan_kernel<T, 2, false><<<dim3(1), dim3(T), 0, s>>>(a, 0);
  else assign_plan_kernel<T, kMaxRequests / T, false><<<dim3(1), dim3(T), 0, s>>>(a, 0);
  const dim3 grid(static_cast<unsigned>((n_rows + kRowsPerWg - 1) / kRowsPerWg));
  if (width > 0 || B <= T) assign_rows_kernel<T><<<grid, dim3(kRowsPerWg), 0, s>>>(a, n_rows);
  else assign_rows_kernel<kMaxRequests><<<grid, dim3(kRowsPerWg), 0, s>>>(a, n_rows);
  FDLLM_RETURN_LAUNCH_STATUS(what);
}

extern "C" int fdllm_release_pages(const fdllm_page_pool* pool, const int32_t* keep_lens, void* stream) {
  using namespace fdllm;
  const char* what = "fdllm_release_pages";
  if (const int rc = check_pool(what, pool)) return rc;
  if (pool->requests == 0) return FDLLM_OK;
  FDLLM_CHECK_ARG(keep_lens != nullptr, "%s: null pointer", what);
  ReleaseArgs a{*pool, keep_lens, __builtin_ctz(static_cast<unsigned>(pool->page_size))};
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int B = pool->requests;
  constexpr int T = kPlanThreads, S = kSmallThreads;
  if (B <= S) release_kernel<S, 1><<<dim3(1), dim3(S), 0, s>>>(a);
  else if (B <= T) release_kernel<T, 1><<<dim3(1), dim3(T), 0, s>>>(a);
  else if (B <= 2 * T) release_kernel<T, 2><<<dim3(1), dim3(T), 0, s>>>(a);
  else release_kernel<T, kMaxRequests / T><<<dim3(1), dim3(T), 0, s>>>(a);
  FDLLM_RETURN_LAUNCH_STATUS(what);
}

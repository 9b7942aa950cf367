// Tables of a serving step, from the requests' lengths alone (fp_build_step_tables): which
// pages come back from finished requests, which ones the new tokens take, and every token's
// position and slot. Integers only, each result unique: no atomics, no order that varies.
//
// Every place follows from prefix sums over the requests: of the pages that come back
// (row r's lie behind those of the rows before it), of the new tokens (cu_seqlens), and of
// the pages needed (page x of the step is the x-th from the free pages' end). One workgroup
// makes them; what is spread over more threads than requests (pages, tokens) finds its
// request by a search in the sums.
//
// A decode step (few tokens) is one launch of that workgroup, the sums in LDS: latency, about
// ten dependent steps. Larger ones share the moves over the card: the sums in a
// workspace, then a launch that returns pages, if any request can be finished, and one that
// takes pages and writes tokens: 16 bytes for each, to be written at the memory's rate.
// 256 requests with a token each: 6.5 us. 1,000 requests with 400,000 tokens, of which half can
// be granted: 4.8 us for the sums (the requests' loads and two passes of prefix sums, one
// after the other), 4.2 to 4.4 for the pages that return, 7.0 for those taken and the tokens.
#include "fp_internal.h"

namespace fp {

constexpr int kStepThreads = 1024;
constexpr int kStepWaves = kStepThreads / 64;

// x of another lane, by DPP control C; 0 in the rows that mask M leaves out and where there is
// no such lane
template <int C, int M>
__device__ __forceinline__ int32_t lane_of(int32_t x) {
  return __builtin_amdgcn_update_dpp(0, x, C, M, 0xf, false);
}
template <int C, int M>
__device__ __forceinline__ int64_t lane_of(int64_t x) {
  return static_cast<int64_t>(
      static_cast<uint64_t>(static_cast<uint32_t>(lane_of<C, M>(static_cast<int32_t>(x >> 32))))
          << 32 |
      static_cast<uint32_t>(lane_of<C, M>(static_cast<int32_t>(x))));
}
// sums over the lanes up to this one within rows of 16 lanes
template <typename X>
__device__ __forceinline__ X row_prefix(X x) {
  x += lane_of<0x111, 0xf>(x);
  x += lane_of<0x112, 0xf>(x);
  x += lane_of<0x114, 0xf>(x);
  return x + lane_of<0x118, 0xf>(x);
}
__device__ __forceinline__ int32_t at_lane(int32_t x, int l) {
  return __builtin_amdgcn_readlane(x, l);
}
__device__ __forceinline__ int64_t at_lane(int64_t x, int l) {
  return static_cast<int64_t>(
      static_cast<uint64_t>(static_cast<uint32_t>(at_lane(static_cast<int32_t>(x >> 32), l)))
          << 32 |
      static_cast<uint32_t>(at_lane(static_cast<int32_t>(x), l)));
}
// Inclusive sums over the workgroup's threads; `total` is that of all of them. Every thread
// calls it; s is its own buffer until the next barrier. A step's sums are three of these and two
// block_max, one after the other: with the exchanges through LDS, 7.0 us instead of 4.8.
template <typename X>
__device__ __forceinline__ X block_prefix(X x, int64_t* s, X& total) {
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  x = row_prefix(x);
  x += lane_of<0x142, 0xa>(x);  // (lane 15 of the row below, then lane 31 of the lower half)
  x += lane_of<0x143, 0xc>(x);
  if (lane == 63) s[w] = x;
  __syncthreads();
  static_assert(kStepWaves == 16, "a row of lanes");
  const X y = row_prefix(static_cast<X>(s[lane & 15]));
  total = at_lane(y, 15);
  __syncthreads();
  return x + (w > 0 ? at_lane(y, max(w - 1, 0)) : X(0));
}
__device__ __forceinline__ int32_t block_max(int32_t x, int64_t* s) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x = max(x, __shfl_xor(x, o));
  if (lane == 0) s[threadIdx.x >> 6] = x;
  __syncthreads();
  x = static_cast<int32_t>(s[lane & 15]);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) x = max(x, __shfl_xor(x, o));
  __syncthreads();
  return x;
}

// (a row has room for fewer than 2^31 tokens)
__device__ __forceinline__ int32_t pages_of(int32_t tokens, int32_t block_size) {
  return static_cast<int32_t>((static_cast<uint32_t>(tokens) + block_size - 1) /
                              static_cast<uint32_t>(block_size));
}

// What the moves need of the requests: inclusive sums of the pages that come back and of
// those needed, the length before the step's tokens, the offsets, and the grants
struct StepSums {
  int32_t* back;
  int32_t* need;
  int32_t* len;
  const int32_t* cu;
  const int32_t* granted;
};
struct StepTotals {
  int32_t free, all, taken;  // free pages before the step, with those that came back, taken
};

// the first r in [lo, hi] with sum[r] > x (hi if none before it has)
__device__ __forceinline__ int find_row(const int32_t* sum, int lo, int hi, int x) {
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (sum[mid] > x) hi = mid; else lo = mid + 1;
  }
  return lo;
}

// The same by a whole wave, of one x for all lanes: 64 places are looked at together, so that
// 1,000 requests take two loads one after the other, not ten.
__device__ __forceinline__ int find_row64(const int32_t* sum, int lo, int hi, int x) {
  const int lane = threadIdx.x & 63;
  while (lo < hi) {
    const int step = (hi - lo + 63) / 64;
    const uint64_t past = __ballot(sum[min(lo + (lane + 1) * step, hi) - 1] > x);
    if (past == 0) return hi;
    const int f = __ffsll(static_cast<long long>(past)) - 1;
    hi = min(lo + (f + 1) * step, hi) - 1;
    lo += f * step;
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

// The sums of a.R requests, by one workgroup. The host has checked that all rows together
// have fewer than 2^31 pages, and one room for fewer than 2^31 tokens.
__device__ __forceinline__ StepTotals step_sums(const StepArgs& a, const StepSums& m, int32_t* cu,
                                                int32_t* granted, int64_t* s) {
  const int t = threadIdx.x, bs = a.block_size;
  const int64_t room = static_cast<int64_t>(a.W) * bs;
  const int32_t free = min(max(a.num_free[0], 0), a.P);
  int32_t returned = 0, came = 0;
  int64_t tokens = 0;
  if (t == 0) {
    cu[0] = 0;
    if (cu != a.cu_seqlens) a.cu_seqlens[0] = 0;
  }
  // pages that come back, tokens, and the pages that a request needs if it is granted
  for (int base = 0; base < a.R; base += kStepThreads) {
    const int r = base + t;
    const bool in = r < a.R;
    const int32_t len = in ? a.seq_lens[r] : 0, add = in ? a.new_lens[r] : 0;
    const bool done = in && a.finished && a.finished[r] != 0;
    const bool held = len >= 0 && len <= room;
    const int32_t back = done && held ? pages_of(len, bs) : 0;
    const int32_t n = max(add, 0);
    int32_t total;
    const int32_t behind = returned + block_prefix(back, s, total);
    returned += total;
    int64_t total_n;
    const int64_t end = tokens + block_prefix(static_cast<int64_t>(n), s, total_n);
    tokens += total_n;
    const bool ends = done && held && (back == 0 || behind <= a.P - free);
    if (ends && back > 0) came = max(came, behind);
    const int32_t now = ends ? 0 : len;
    const bool fits = in && held && add >= 0 && done == ends && end <= a.N &&
                      static_cast<int64_t>(now) + n <= room;
    if (in) {
      m.back[r] = behind;
      m.len[r] = now;
      m.need[r] = fits ? pages_of(now + n, bs) - pages_of(now, bs) : -1;
      const int32_t c = static_cast<int32_t>(min(end, a.N));
      cu[r + 1] = c;
      if (cu != a.cu_seqlens) a.cu_seqlens[r + 1] = c;
    }
  }
  came = block_max(came, s);
  const int32_t all = free + came;
  // which requests get their pages: those that need none, and of the others, in the order of
  // the rows, as many as the free pages serve
  int32_t wanted = 0, taken = 0;
  for (int base = 0; base < a.R; base += kStepThreads) {
    const int r = base + t;
    const bool in = r < a.R;
    const int32_t need = in ? m.need[r] : -1;
    int32_t total;
    const int32_t upto = wanted + block_prefix(max(need, 0), s, total);
    wanted += total;
    const bool ok = need == 0 || (need > 0 && upto <= all);
    if (need > 0 && ok) taken = max(taken, upto);
    if (in) {
      m.need[r] = upto;
      granted[r] = ok;
      if (granted != a.granted) a.granted[r] = ok;
      a.seq_lens_out[r] = m.len[r] + (ok ? a.new_lens[r] : 0);
    }
  }
  taken = block_max(taken, s);
  if (t == 0) a.num_free_out[0] = all - taken;
  return StepTotals{free, all, taken};
}

// finished rows' pages behind the free ones: page x of them, in a row from lo to hi
__device__ __forceinline__ void return_page(const StepArgs& a, const StepSums& m,
                                            const StepTotals& k, int x, int lo, int hi) {
  const int r = find_row(m.back, lo, hi, x);
  const int j = x - (r > 0 ? m.back[r - 1] : 0);
  a.free_pages[k.free + x] = a.block_table[r * a.table_stride + j];
}
// The same for all n of them, by a workgroup whose waves take 1,024 neighbours at a time: the whole
// wave searches for their rows, and of one row's a lane's sixteen loads are on their way together.
__device__ __forceinline__ void return_pages(const StepArgs& a, const StepSums& m,
                                             const StepTotals& k, int n) {
  constexpr int U = 16;
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  for (int64_t x0 = w * 64 * U; x0 < n; x0 += kStepThreads * U) {
    const int first = static_cast<int>(x0), last = static_cast<int>(min(x0 + 64 * U, int64_t(n))) - 1;
    const int lo = find_row64(m.back, 0, a.R - 1, first);
    const int hi = find_row64(m.back, lo, a.R - 1, last);
    if (lo < hi) {
      for (int x = first + lane; x <= last; x += 64) return_page(a, m, k, x, lo, hi);
      continue;
    }
    const int32_t* row = a.block_table + lo * a.table_stride - (lo > 0 ? m.back[lo - 1] : 0);
    int32_t page[U];
#pragma unroll
    for (int u = 0; u < U; ++u) page[u] = row[min(first + 64 * u + lane, last)];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (first + 64 * u + lane <= last) a.free_pages[k.free + first + 64 * u + lane] = page[u];
  }
}
// page x of the step's, from the free ones' end
__device__ __forceinline__ void take_page(const StepArgs& a, const StepSums& m,
                                          const StepTotals& k, int x, int lo, int hi) {
  const int r = find_row(m.need, lo, hi, x);
  const int64_t at = pages_of(m.len[r], a.block_size) + x - (r > 0 ? m.need[r - 1] : 0);
  a.block_table[r * a.table_stride + at] = a.free_pages[k.all - 1 - x];
}
// one(x, lo, hi) for x < n by the waves first, first + step .., 64 at a time, whose rows lie
// from lo to hi
template <typename F>
__device__ __forceinline__ void by_waves(const int32_t* sum, int R, int n, int first, int step,
                                         F&& one) {
  const int lane = threadIdx.x & 63;
  for (int64_t x0 = static_cast<int64_t>(first) * 64; x0 < n; x0 += static_cast<int64_t>(step) * 64) {
    const int last = static_cast<int>(min(x0 + 63, static_cast<int64_t>(n - 1)));
    const int lo = find_row64(sum, 0, R - 1, static_cast<int>(x0));
    const int hi = find_row64(sum, lo, R - 1, last);
    if (x0 + lane < n) one(static_cast<int>(x0) + lane, lo, hi);
  }
}
// a token's position and slot; lo, hi: rows among which its request lies
__device__ __forceinline__ void place_token(const StepArgs& a, const StepSums& m,
                                            const StepTotals& k, int64_t x, int lo, int hi) {
  int64_t position = 0, slot = -1;
  if (x < m.cu[a.R]) {
    const int r = find_row(m.cu + 1, lo, hi, static_cast<int>(x));
    position = static_cast<int64_t>(m.len[r]) + x - m.cu[r];
    if (m.granted[r]) {
      const int bs = a.block_size, at = static_cast<int>(position);
      const int col = static_cast<int>(static_cast<uint32_t>(at) / static_cast<uint32_t>(bs));
      const int held = pages_of(m.len[r], bs);
      // (a page of this step's from where it comes: its entry may not be written yet)
      const int64_t page = col < held
                               ? a.block_table[r * a.table_stride + col]
                               : a.free_pages[k.all - 1 - (r > 0 ? m.need[r - 1] : 0) - (col - held)];
      slot = page * bs + (at - col * bs);
    }
  }
  a.positions[x] = position;
  a.slots[x] = slot;
}

// Pages that come back up to here go by return_page, a thread each, past it by return_pages (256
// requests, 4,000, 16,000, 24,576, 65,536 and 491,520 pages of rows of 250 .. 8,192: 9.0, 17, 23.5,
// 53 and 356 us the first way, 17, 16, 9.5, 14.5 and 68 the second, whose waves move rows of few
// pages no faster). How many come back the host cannot know, and three launches would cost
// every step that ends none 3 us.
constexpr int kStepFew = 16384;
// A whole step by one workgroup, of at most kStepThreads requests
__global__ __launch_bounds__(kStepThreads) void k_step_one(StepArgs a) {
  __shared__ int64_t s[kStepWaves];
  __shared__ int32_t back[kStepThreads], need[kStepThreads], len[kStepThreads];
  __shared__ int32_t cu[kStepThreads + 1], granted[kStepThreads];
  const StepSums m{back, need, len, cu, granted};
  const StepTotals k = step_sums(a, m, cu, granted, s);
  __syncthreads();
  const int t = static_cast<int>(threadIdx.x);
  const int back_n = k.all - k.free;
  if (back_n > kStepFew) {
    return_pages(a, m, k, back_n);
  } else {
    for (int x = t; x < back_n; x += kStepThreads) return_page(a, m, k, x, 0, a.R - 1);
  }
  __syncthreads();  // (pages taken may have just come back, rows that gave them be written)
  for (int x = t; x < k.taken; x += kStepThreads) take_page(a, m, k, x, 0, a.R - 1);
  for (int64_t x = t; x < a.N; x += kStepThreads) place_token(a, m, k, x, 0, a.R - 1);
}

__device__ __forceinline__ StepSums ws_sums(const StepArgs& a) {
  int32_t* p = a.ws + 4;
  return StepSums{p, p + a.R, p + 2 * static_cast<int64_t>(a.R), a.cu_seqlens, a.granted};
}
__device__ __forceinline__ StepTotals ws_totals(const StepArgs& a) {
  return StepTotals{a.ws[0], a.ws[1], a.ws[2]};
}

__global__ __launch_bounds__(kStepThreads) void k_step_sums(StepArgs a) {
  __shared__ int64_t s[kStepWaves];
  const StepTotals k = step_sums(a, ws_sums(a), a.cu_seqlens, a.granted, s);
  if (threadIdx.x == 0) {
    a.ws[0] = k.free;
    a.ws[1] = k.all;
    a.ws[2] = k.taken;
  }
}
constexpr int kStepMovers = 128;  // workgroups that move pages
__global__ __launch_bounds__(256) void k_step_return(StepArgs a) {
  const StepSums m = ws_sums(a);
  const StepTotals k = ws_totals(a);
  by_waves(m.back, a.R, k.all - k.free, static_cast<int>(blockIdx.x * 4 + (threadIdx.x >> 6)),
           static_cast<int>(gridDim.x) * 4,
           [&](int x, int lo, int hi) { return_page(a, m, k, x, lo, hi); });
}
// The first kStepMovers workgroups take pages, the others place tokens, kStepTokens each: one
// for each thread (400,000: with two, one after the other, 0.1 us more, with four 2.5).
constexpr int kStepTokens = 256;
__global__ __launch_bounds__(256) void k_step_place(StepArgs a) {
  const StepSums m = ws_sums(a);
  const StepTotals k = ws_totals(a);
  if (blockIdx.x < kStepMovers) {
    by_waves(m.need, a.R, k.taken, static_cast<int>(blockIdx.x * 4 + (threadIdx.x >> 6)),
             kStepMovers * 4, [&](int x, int lo, int hi) { take_page(a, m, k, x, lo, hi); });
    return;
  }
  const int64_t x0 = static_cast<int64_t>(blockIdx.x - kStepMovers) * kStepTokens;
  const int64_t x1 = min(x0 + kStepTokens, a.N);
  // (the requests of the workgroup's first and last token)
  const int lo = find_row64(m.cu + 1, 0, a.R - 1, static_cast<int>(x0));
  const int hi = find_row64(m.cu + 1, lo, a.R - 1, static_cast<int>(x1 - 1));
  if (x0 + threadIdx.x < x1) place_token(a, m, k, x0 + threadIdx.x, lo, hi);
}

hipError_t launch_steps(const StepArgs& a, bool one, hipStream_t s) {
  if (one) {
    hipLaunchKernelGGL(k_step_one, dim3(1), dim3(kStepThreads), 0, s, a);
    return hipGetLastError();
  }
  hipLaunchKernelGGL(k_step_sums, dim3(1), dim3(kStepThreads), 0, s, a);
  if (a.finished) hipLaunchKernelGGL(k_step_return, dim3(kStepMovers), dim3(256), 0, s, a);
  const int64_t wgs = (a.N + kStepTokens - 1) / kStepTokens;
  hipLaunchKernelGGL(k_step_place, dim3(static_cast<unsigned>(kStepMovers + wgs)), dim3(256), 0, s,
                     a);
  return hipGetLastError();
}

}  // namespace fp

// What the kernels that move rows into and out of a paged cache share (fp_kvcache.hip:
// 16- and 8-bit caches, fp_kvcache4.hip: 4-bit ones).
#pragma once

#include "fp_paged_common.h"

namespace fp {

// Rows and codes pass once: nontemporal moves (131072 tokens of 8 heads of 128 written:
// 177 us without them, 169 with them; 218,000 tokens read back 344 and 325). Addresses
// are of global memory, also where the compiler cannot see it.
template <typename X>
__device__ __forceinline__ __attribute__((address_space(1))) X* global_ptr(const void* p) {
  return (__attribute__((address_space(1))) X*)(p);
}
__device__ __forceinline__ uint4 ld16_once(const void* p) {
  const u32x4 v = __builtin_nontemporal_load(global_ptr<const u32x4>(p));
  return make_uint4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ uint2 ld8_once(const void* p) {
  const uint64_t v = __builtin_nontemporal_load(global_ptr<const uint64_t>(p));
  return make_uint2(static_cast<uint32_t>(v), static_cast<uint32_t>(v >> 32));
}
__device__ __forceinline__ void st16_once(void* p, uint4 v) {
  __builtin_nontemporal_store(u32x4{v.x, v.y, v.z, v.w}, global_ptr<u32x4>(p));
}
__device__ __forceinline__ void st8_once(void* p, uint2 v) {
  __builtin_nontemporal_store(static_cast<uint64_t>(v.y) << 32 | v.x, global_ptr<uint64_t>(p));
}

// Block and place in it of a slot: a 64-bit division only where the slot needs one
__device__ __forceinline__ void split_slot(int64_t slot, int32_t block_size, int64_t& blk,
                                           int64_t& off) {
  if (slot >> 32) {
    blk = slot / block_size;
    off = slot % block_size;
  } else {
    const uint32_t q = static_cast<uint32_t>(slot) / static_cast<uint32_t>(block_size);
    blk = q;
    off = static_cast<uint32_t>(slot) - q * static_cast<uint32_t>(block_size);
  }
}

// The cached token that a row of the read-back stands for, by one wave with a row per
// lane, 64 sequences at a time: a row belongs to the last sequence b with cu[b] <= row, if
// row < cu[b + 1].
constexpr int64_t kSkip = -1, kNaN = -2;  // rows of no sequence; rows that cannot be read
struct CachedToken {
  int64_t page, in;  // page and slot in it, or page one of the above
};
__device__ __forceinline__ CachedToken find_cached_token(const GatherArgs& a, int64_t tok) {
  const KvCacheArgs& c = a.g.c;
  const int lane = threadIdx.x & 63;
  int64_t b = -1, seq0 = 0;
  bool off = false;
  for (int base = 0; base < a.B; base += 64) {
    int64_t c0 = INT64_MAX, c1 = 0;
    const bool in = base + lane < a.B;
    if (in) {
      c0 = ld_int(a.cu, a.cu64, base + lane);
      c1 = ld_int(a.cu, a.cu64, base + lane + 1);
    }
    off = off || __ballot(in && (c0 < 0 || c1 > c.num_tokens || c1 < c0)) != 0;
    int last = 0;  // the last of these that begins at or before the token
#pragma unroll
    for (int step = 32; step > 0; step >>= 1)
      if (shfl64(c0, last + step) <= tok) last += step;
    const int64_t f = shfl64(c0, last), e = shfl64(c1, last);
    if (f <= tok && tok < e) {
      b = base + last;
      seq0 = f;
    }
  }
  CachedToken r{kSkip, 0};
  if (off) {
    r.page = kNaN;
  } else if (b >= 0) {
    int64_t pos = tok - seq0;
    const int64_t start = a.starts ? ld_int(a.starts, a.starts64, b) : 0;
    const int64_t room = static_cast<int64_t>(a.width) * c.block_size;
    r.page = kNaN;
    if (start >= 0 && start < room && pos + start < room) {
      pos += start;
      int64_t blk;
      split_slot(pos, c.block_size, blk, r.in);
      int64_t page = ld_int(a.table, a.table64, b * a.table_stride + blk);
      if (page < 0) page += a.num_blocks;
      if (page >= 0 && page < a.num_blocks) r.page = page;
    }
  }
  return r;
}

}  // namespace fp

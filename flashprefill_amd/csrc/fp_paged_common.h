// What the kernels over a paged cache share (fp_paged.hip: 16-bit caches,
// fp_paged8.hip: 8-bit ones): which sequence and rows a workgroup serves, the page
// lookup, sums over the lanes of a query row, and the V^T operand of a tile in LDS.
#pragma once

#include "fp_attn_common.h"

namespace fp {

__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// entry x of a 32- or 64-bit (is64 1) integer array. Loads under no branch: several of
// them are in flight together, where a branch makes the compiler wait for each.
__device__ __forceinline__ int64_t ld_int(const void* p, int is64, int64_t x) {
  const int32_t* q = static_cast<const int32_t*>(p) + (x << is64);
  const int32_t lo = q[0], hi = q[is64];
  return is64 ? static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(hi)) << 32 |
                                     static_cast<uint32_t>(lo))
              : static_cast<int64_t>(lo);
}

// One sequence as the workgroups see it. `bad`: more tokens than the block
// table has room for; its rows are written as NaN. `off`: its query offsets
// descend or lie outside the call's rows.
struct PagedSeq {
  int64_t q0;  // first query row
  int nq;      // query rows
  int64_t nk;  // cached tokens
  bool bad, off;
};

__device__ __forceinline__ PagedSeq paged_seq(const PagedArgs& a, int b) {
  PagedSeq s;
  s.q0 = ld_int(a.cu, a.cu64, b);
  const int64_t q1 = ld_int(a.cu, a.cu64, b + 1);
  s.off = s.q0 < 0 || q1 > a.T || q1 < s.q0;
  s.nq = s.off ? 0 : static_cast<int>(q1 - s.q0);
  s.nk = ld_int(a.used, a.used64, b);
  s.bad = s.nk > static_cast<int64_t>(a.width) * a.bs;
  if (s.bad || s.nk < 0) s.nk = 0;
  return s;
}

__device__ __forceinline__ int64_t shfl64(int64_t x, int lane) {
  return static_cast<int64_t>(
      (static_cast<uint64_t>(static_cast<uint32_t>(__shfl(static_cast<int>(x >> 32), lane))) << 32) |
      static_cast<uint32_t>(__shfl(static_cast<int>(x), lane)));
}

// The sequence that owns row tile `x` (tiles of `rt` rows of nq * G, numbered
// over the sequences) and the tile's index in it, or with tok >= 0 the one
// that owns query row `tok`; and the chunk length all workgroups use. By one
// wave (64 sequences at a time); b < 0 when there is none. Where some sequence's
// offsets do not fit, which rows are whose is unknown: all rows of the call are
// one sequence's then, and bad.
struct PagedTile {
  PagedSeq s;
  int b, tl, chunk;
};
__device__ __forceinline__ PagedTile paged_find(const PagedArgs& a, int rt, int64_t x,
                                                int64_t tok) {
  const int lane = threadIdx.x & 63;
  PagedTile r;
  r.b = -1;
  r.tl = 0;
  r.s = PagedSeq{0, 0, 0, false, false};
  int64_t carry = 0;
  int maxlen = 0;
  bool off = false;
  for (int base = 0; base < a.B; base += 64) {
    PagedSeq s{0, 0, 0, false, false};
    if (base + lane < a.B) s = paged_seq(a, base + lane);
    off = off || __ballot(s.off) != 0;
    const int tiles =
        static_cast<int>((static_cast<int64_t>(s.nq) * a.G + rt - 1) / rt);
    if (s.nq > 0) maxlen = max(maxlen, static_cast<int>(s.nk));
    int incl = tiles;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(incl, o);
      if (lane >= o) incl += y;
    }
    const bool mine = tok >= 0 ? tok >= s.q0 && tok < s.q0 + s.nq
                               : tiles > 0 && x >= carry + incl - tiles && x < carry + incl;
    const uint64_t hit = __ballot(mine);
    if (r.b < 0 && hit) {
      const int l = __ffsll(static_cast<long long>(hit)) - 1;
      r.b = base + l;
      r.tl = static_cast<int>(x - carry) - __shfl(incl - tiles, l);
      r.s.q0 = shfl64(s.q0, l);
      r.s.nq = __shfl(s.nq, l);
      r.s.nk = shfl64(s.nk, l);
      r.s.bad = __shfl(static_cast<int>(s.bad), l) != 0;
    }
    carry += __shfl(incl, 63);
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) maxlen = max(maxlen, __shfl_xor(maxlen, o));
  const int per = (maxlen + a.nc - 1) / a.nc;
  r.chunk = (max(per, kPagedMinChunk) + 127) / 128 * 128;
  if (off) {
    r.b = tok >= 0 || x < (a.T * a.G + rt - 1) / rt ? 0 : -1;
    r.tl = static_cast<int>(x);
    r.s = PagedSeq{0, static_cast<int>(a.T), 0, true, true};
  }
  // wave-uniform values in scalar registers
  r.b = __builtin_amdgcn_readfirstlane(r.b);
  r.tl = __builtin_amdgcn_readfirstlane(r.tl);
  r.chunk = __builtin_amdgcn_readfirstlane(r.chunk);
  r.s.nq = __builtin_amdgcn_readfirstlane(r.s.nq);
  r.s.nk = __builtin_amdgcn_readfirstlane(static_cast<int>(r.s.nk));
  r.s.q0 = __builtin_amdgcn_readfirstlane(static_cast<int>(r.s.q0));
  return r;
}

// Page of cached token `key` of a sequence whose table row is `row`. A page
// number below 0 counts from the end (as the index of a torch gather); one
// outside the cache sets `bad` and reads page 0.
// UNI: `key` is wave-uniform and the lookup goes through the scalar cache (a
// vector load would wait for every K / V load issued before it).
template <bool UNI>
__device__ __forceinline__ int64_t paged_page(const PagedArgs& a, int64_t row, int key, bool& bad) {
  int idx = a.bs_shift >= 0 ? key >> a.bs_shift : key / a.bs;
  int64_t p;
  if constexpr (UNI) {
    idx = __builtin_amdgcn_readfirstlane(idx);
    p = a.table64 ? sld(static_cast<const int64_t*>(a.table) + row + idx)
                  : static_cast<int64_t>(sld(static_cast<const int32_t*>(a.table) + row + idx));
  } else {
    p = ld_int(a.table, a.table64, row + idx);
  }
  if (p < 0) p += a.nblocks;
  if (p < 0 || p >= a.nblocks) {
    bad = true;
    p = 0;
  }
  return p;
}

// max / sum over the lanes l, l ^ 16, l ^ 32, l ^ 48 (one query row), in every lane
__device__ __forceinline__ float row4_max(float x) {
  x = fmaxf(x, __uint_as_float(xchg_xor<16>(__float_as_uint(x))));
  return pair32_max(x);
}
__device__ __forceinline__ float row4_sum(float x) {
  x += __uint_as_float(xchg_xor<16>(__float_as_uint(x)));
  return pair32_sum(x);
}

// V^T operand of a 16-key step: keys r .. r + 3 and r + 8 .. r + 11, dim xx of a
// key-major tile
template <typename T, int D>
__device__ __forceinline__ typename T::vec8 read_vt(const uint16_t* sv16, int r, int xx) {
  const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (__attribute__((address_space(3))) i16x4*)(sv16 + tile_elem<D>(r, xx)));
  const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (__attribute__((address_space(3))) i16x4*)(sv16 + tile_elem<D>(r + 8, xx)));
  const uint2 lo2 = __builtin_bit_cast(uint2, lo), hi2 = __builtin_bit_cast(uint2, hi);
  return as_vec8<T>(make_uint4(lo2.x, lo2.y, hi2.x, hi2.y));
}

}  // namespace fp

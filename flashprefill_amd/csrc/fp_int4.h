// The 4-bit values of a KV cache: s (c + z) for the codes c = 0 .. 15 of a group of 32
// elements, s and z in the group's 16-bit word (fp_kv_groups). s has 4 significant bits and
// c + z, between -64 and 78, at most 7, so that their product is exactly an fp16 number
// (11 bits) and the fp16 matrix instructions take the values as they are.
//
// Codes become values two at a time. Codes moved to the top mantissa bits of a pair of fp16
// numbers whose other bits are those of 16 read as 16 + c (one shift, one and-or), and
//   s (c + z) = (16 + c) s + (z - 16) s
// is one packed fma, in which nothing is rounded: (z - 16) s has 7 + 4 bits, and magnitudes
// up to 16384 with steps up to 2304 (a 15th of 32768, rounded) keep it to 52,992.
//
// Byte m (d / 32) + j of a row holds dims 32 j + 2 m and 32 j + 2 m + 1: what a lane of 16
// loads (d / 32 bytes of each key) are two dims of every group, so that a matrix
// instruction over one dim of each lane's stays in one group, and four lanes' worth (the
// pieces of a key below) are 8 consecutive dims of every group.
#pragma once

#include "fp_attn_common.h"

namespace fp {

// Constants of the conversions, held in vector registers: an instruction takes one scalar
// operand, and the masks are that.
struct Int4Consts {
  uint32_t sixteen, zero;
  __device__ __forceinline__ Int4Consts() : sixteen(0x4c004c00u), zero(0x64006400u) {
    asm volatile("" : "+v"(sixteen), "+v"(zero));
  }
};

// (16 + c) of nibble N of each 16-bit half
template <int N>
__device__ __forceinline__ f16x2 nibbles(uint32_t h, const Int4Consts& k) {
  constexpr int kShift[4] = {6, 2, -2, -6};
  const uint32_t x = kShift[N] > 0 ? h << (kShift[N] & 31) : h >> (-kShift[N] & 31);
  return __builtin_bit_cast(f16x2, (x & 0x03c003c0u) | k.sixteen);
}

// s and (z - 16) s of a pair of group words
struct Step2 {
  f16x2 s, off;
};
__device__ __forceinline__ Step2 steps(uint32_t words, const Int4Consts& k) {
  Step2 r;
  r.s = __builtin_bit_cast(f16x2, words & 0x7f807f80u);
  const f16x2 z = __builtin_bit_cast(f16x2, (words & 0x007f007fu) | k.zero);  // 1024 + 64 + z
  r.off = (z - f16x2{1104.0f16, 1104.0f16}) * r.s;
  return r;
}
template <int N>
__device__ __forceinline__ uint32_t values2(uint32_t h, const Step2& s, const Int4Consts& k) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(nibbles<N>(h, k), s.s, s.off));
}

// 16-bit halves I of two words, as one
template <int I>
__device__ __forceinline__ uint32_t halves(uint32_t a, uint32_t b) {
  return __builtin_amdgcn_perm(b, a, I ? 0x07060302u : 0x05040100u);
}

// Pointers of global memory, also where the compiler cannot see that they are (a load of
// an unknown space waits with LDS)
typedef const __attribute__((address_space(1))) uint8_t* gbytes;
typedef const __attribute__((address_space(1))) uint16_t* gwords;
__device__ __forceinline__ gbytes in_global(const uint8_t* p) { return (gbytes)(p); }
__device__ __forceinline__ gwords in_global(const uint16_t* p) { return (gwords)(p); }
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
// N words of 32 bits (1, 2 or a multiple of 4) from P, in one load for each four
template <int N, typename P>
__device__ __forceinline__ void load32(P p, uint32_t (&w)[N]) {
  if constexpr (N == 1) {
    w[0] = *(const __attribute__((address_space(1))) uint32_t*)(p);
  } else if constexpr (N == 2) {
    const u32x2 x = *(const __attribute__((address_space(1))) u32x2*)(p);
    w[0] = x[0]; w[1] = x[1];
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const u32x4 x = *((const __attribute__((address_space(1))) u32x4*)(p) + i / 4);
      w[i] = x[0]; w[i + 1] = x[1]; w[i + 2] = x[2]; w[i + 3] = x[3];
    }
  }
}
// A piece of a key, NB = d / 32 words: bytes 4 NB p .. 4 NB (p + 1) - 1, dims
// 32 j + 8 p .. + 7 of every group j.
template <int NB, typename P>
__device__ __forceinline__ void load_piece(P p, uint32_t (&w)[NB]) {
  load32<NB>(p, w);
}
// N group words (a multiple of 2)
template <int N, typename P>
__device__ __forceinline__ void load_words(P p, uint32_t (&w)[N / 2]) {
  load32<N / 2>(p, w);
}
// Group j of a piece as 8 fp16 numbers, dims 32 j + 8 p + {0, 2, 1, 3, 4, 6, 5, 7}, by the
// group's step (in both halves)
template <int NB>
__device__ __forceinline__ uint4 piece_group(const uint32_t (&w)[NB], const Step2& s, int j,
                                             const Int4Consts& k) {
  uint32_t h[2];  // groups j & ~1 and j | 1 of dim pairs 0, 1 and of 2, 3
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (NB == 2) {
      h[i] = w[i];
    } else {
      const uint32_t a = w[2 * i * (NB / 4) + (j >> 2)], b = w[(2 * i + 1) * (NB / 4) + (j >> 2)];
      h[i] = j & 2 ? halves<1>(a, b) : halves<0>(a, b);
    }
  }
  return j & 1 ? make_uint4(values2<2>(h[0], s, k), values2<3>(h[0], s, k), values2<2>(h[1], s, k),
                            values2<3>(h[1], s, k))
               : make_uint4(values2<0>(h[0], s, k), values2<1>(h[0], s, k), values2<0>(h[1], s, k),
                            values2<1>(h[1], s, k));
}
// the same from all of the key's group words
template <int NB>
__device__ __forceinline__ uint4 piece_group(const uint32_t (&w)[NB], const uint32_t (&g)[NB / 2],
                                             int j, const Int4Consts& k) {
  return piece_group<NB>(
      w, steps(j & 1 ? halves<1>(g[j >> 1], g[j >> 1]) : halves<0>(g[j >> 1], g[j >> 1]), k), j, k);
}

}  // namespace fp

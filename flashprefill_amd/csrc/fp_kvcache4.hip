// Write and read-back of a paged KV cache of 4-bit integers (fp_int4.h, fp_kv_groups).
//
// Both move rows of head_dim elements, four lanes to a row: lane p takes dims
// 32 j + 8 p .. + 7 of every group j, 16 bytes of the 16-bit row at a time, whose codes are
// 4 (d / 32) contiguous bytes of the cached row. A workgroup serves K or V, so that strides
// and bases are scalars.
//
// The write finds each group's smallest and largest element over the four lanes and
// quantises by the rule of fp_kv_cache_write_int4. A group's step is one lane's work, passed
// to the other three. Its quotients are rounded as a division rounds them: y = x r, r about
// 1 / s, then y - r (y s - x), whose error before its own rounding is below 2^-43 of it, and
// x / s (s has 4 significant bits) is either an fp32 number or at least 2^-29 of itself
// away from a midpoint of two.
#include "fp_int4.h"
#include "fp_kvcache_common.h"

namespace fp {

// x / y for a y of few significant bits (15, 56, a step), r about 1 / y
__device__ __forceinline__ float quotient(float x, float y, float r) {
  const float q = x * r;
  return fmaf(-fmaf(q, y, -x), r, q);
}

// x / t, rounded as a division rounds it, up to magnitudes of 2^15 (larger ones stay that): two
// steps of the above make it so where no product comes near the ends of fp32's range (Markstein,
// Computation of elementary functions on the IBM RISC System/6000, 1990; of an |x| below 2^-102
// the quotient, below 2^-42, is nothing beside any step), other scales divide.
__device__ __forceinline__ void divide8(float (&x)[8], float t, float r) {
  if (fabsf(t) >= 0x1p-60f && fabsf(t) <= 0x1p60f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float y = x[e] * r;
      const float q = fmaf(-fmaf(y, t, -x[e]), r, y);
      x[e] = fabsf(y) < 0x1p15f ? fmaf(-fmaf(q, t, -x[e]), r, q) : y;  // (a NaN stays)
    }
  } else {
#pragma unroll 1
    for (int e = 0; e < 8; ++e) {
      const float y = x[0] / t;
#pragma unroll
      for (int i = 0; i < 7; ++i) x[i] = x[i + 1];
      x[7] = y;
    }
  }
}

// The larger of two numbers, as the median of them and infinity: fmaxf would first quiet
// each, since they might be signalling NaN.
__device__ __forceinline__ float larger(float a, float b) {
  return __builtin_amdgcn_fmed3f(a, b, INFINITY);
}
// max over the four lanes of a row
__device__ __forceinline__ float quad_max(float x) {
  const auto other = [](float v, auto ctrl) {
    return __uint_as_float(static_cast<uint32_t>(__builtin_amdgcn_update_dpp(
        0, static_cast<int>(__float_as_uint(v)), decltype(ctrl)::value, 0xf, 0xf, true)));
  };
  x = larger(x, other(x, IntC<0xb1>{}));  // lanes 1 0 3 2
  return larger(x, other(x, IntC<0x4e>{}));  // lanes 2 3 0 1
}

// lane L of the four, in all of them
template <int L>
__device__ __forceinline__ float quad_from(float x) {
  return __uint_as_float(static_cast<uint32_t>(__builtin_amdgcn_update_dpp(
      0, static_cast<int>(__float_as_uint(x)), 0x55 * L, 0xf, 0xf, true)));
}

constexpr float kInt4Most = 16384.0f;  // the largest magnitude that a group holds

// A group's step: x becomes the code rint(x / s) - z, within 0 .. 15. Where all codes are 0
// (s = 0, or NaN), r, s and z are 0.
struct GroupStep {
  float s, r, z;
  uint16_t word;
};
// from its largest and smallest element (the largest infinite: some element is NaN)
__device__ __forceinline__ GroupStep group_step(float hi, float lo) {
  const bool nan = hi == INFINITY;
  const float want = larger(quotient(hi - lo, 15.0f, 1.0f / 15.0f),
                            quotient(larger(hi, -lo), 56.0f, 1.0f / 56.0f));
  uint32_t m = __float_as_uint(want);  // (-0 for a group of -0: s takes the magnitude)
  m = (m + 0x7ffffu + ((m >> 20) & 1u)) & ~0xfffffu;
  const float s = fabsf(want < 0x1p-14f ? rintf(want * 0x1p17f) * 0x1p-17f : __uint_as_float(m));
  const bool none = s == 0.0f || nan;
  const float r = __builtin_amdgcn_rcpf(s);
  const float z = none ? 0.0f : __builtin_amdgcn_fmed3f(rintf(quotient(lo, s, r)), -64.0f, 63.0f);
  const uint32_t bits = __builtin_bit_cast(uint16_t, static_cast<_Float16>(s));
  return GroupStep{none ? 0.0f : s, none ? 0.0f : r, z,
                   static_cast<uint16_t>(nan ? 0x7f80u
                                             : bits | static_cast<uint32_t>(static_cast<int>(z) + 64))};
}

// 131,072 tokens of 8 heads of 128 with scales, 688 MB: 169 us, 4.1 TB/s (a copy's rate
// 5.15); without the group words' 8 bytes a row, scattered over the heads' pages, 157.
template <typename T, int NB>
__global__ __launch_bounds__(256) void k_cache_write4(Cache4Args a) {
  constexpr int K = NB == 8 ? 2 : 1;  // groups whose steps a lane makes: K p .. (p modulo NB)
  const Cache4Side& sd = a.side[blockIdx.y];
  const int p = threadIdx.x & 3;
  const uint32_t row = blockIdx.x * 64u + (threadIdx.x >> 2);
  const uint32_t H = static_cast<uint32_t>(a.num_kv_heads);
  const uint32_t tok = a.heads_shift >= 0 ? row >> a.heads_shift : row / H, h = row - tok * H;
  if (tok >= static_cast<uint32_t>(a.num_tokens)) return;  // (all four lanes of a row)
  const int64_t slot = a.slot_mapping[tok];
  const uint16_t* src = sd.rows + tok * sd.row_tok + h * sd.row_head + 8 * p;
  uint4 u[NB];
#pragma unroll
  for (int j = 0; j < NB; ++j) u[j] = ld16_once(src + 32 * j);
  if (slot < 0 || slot >= a.num_slots) return;
  int64_t blk, off;
  if (a.block_shift >= 0) {
    blk = slot >> a.block_shift;
    off = slot & (a.block_size - 1);
  } else {
    split_slot(slot, a.block_size, blk, off);
  }
  const float t = sd.t ? sd.t[h * sd.t_head] : 1.0f, rt = 1.0f / t;
  float x[NB][8], hi[NB], lo[NB], most = 0.0f;
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const uint32_t uw[4] = {u[j].x, u[j].y, u[j].z, u[j].w};
    bool nan = false;
    hi[j] = -INFINITY;
    lo[j] = INFINITY;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[j][2 * e] = T::to_f32(static_cast<uint16_t>(uw[e]));
      x[j][2 * e + 1] = T::to_f32(static_cast<uint16_t>(uw[e] >> 16));
    }
    if (sd.t) divide8(x[j], t, rt);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float* y = &x[j][2 * e];
      nan = nan || __builtin_isunordered(y[0], y[1]);
      hi[j] = fmaxf(hi[j], fmaxf(y[0], y[1]));
      lo[j] = fminf(lo[j], fminf(y[0], y[1]));
    }
    most = larger(most, larger(hi[j], -lo[j]));
    hi[j] = __builtin_amdgcn_fmed3f(hi[j], -kInt4Most, kInt4Most);
    lo[j] = __builtin_amdgcn_fmed3f(lo[j], -kInt4Most, kInt4Most);
    hi[j] = quad_max(nan ? INFINITY : hi[j]);
    lo[j] = -quad_max(-lo[j]);
  }
  // (seldom: elements past what a group holds, whose quotients may be infinite)
  if (__ballot(most > kInt4Most) != 0) {
    asm volatile("");
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        x[j][e] = __builtin_amdgcn_fmed3f(x[j][e], -kInt4Most, kInt4Most);
  }
  GroupStep mine[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    float gh = hi[k], gl = lo[k];
#pragma unroll
    for (int j = 1; j < NB / K; ++j) {
      const bool is = (p & (NB / K - 1)) == j;
      gh = is ? hi[K * j + k] : gh;
      gl = is ? lo[K * j + k] : gl;
    }
    mine[k] = group_step(gh, gl);
  }
  uint32_t w[NB] = {};  // the piece's bytes: dim pair e of group j at e NB + j
  const auto codes = [&](auto jc) {
    constexpr int j = decltype(jc)::value;
    const GroupStep& m = mine[j % K];
    const float s = quad_from<j / K>(m.s), r = quad_from<j / K>(m.r), z = quad_from<j / K>(m.z);
    const float z15 = z + 15.0f, z17 = 17.0f * z;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float n[2];  // codes + z
#pragma unroll
      for (int i = 0; i < 2; ++i)
        n[i] = rintf(__builtin_amdgcn_fmed3f(quotient(x[j][2 * e + i], s, r), z, z15));
      const int at = e * NB + j;
      w[at >> 2] = __builtin_amdgcn_cvt_pk_u8_f32(fmaf(16.0f, n[1], n[0] - z17), at & 3, w[at >> 2]);
    }
  };
  codes(IntC<0>{});
  codes(IntC<1>{});
  if constexpr (NB >= 4) {
    codes(IntC<2>{});
    codes(IntC<3>{});
  }
  if constexpr (NB == 8) {
    codes(IntC<4>{});
    codes(IntC<5>{});
    codes(IntC<6>{});
    codes(IntC<7>{});
  }
  uint8_t* dst = sd.cache + blk * sd.block + off * sd.slot + h * sd.head + 4 * NB * p;
  if constexpr (NB == 2) {
    st8_once(dst, make_uint2(w[0], w[1]));
  } else {
#pragma unroll
    for (int i = 0; i < NB / 4; ++i)
      st16_once(dst + 16 * i, make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]));
  }
  uint16_t* g = sd.g.p + blk * sd.g.sb + h * sd.g.sh + off * NB + K * p;
  if constexpr (K == 2)
    *reinterpret_cast<uint32_t*>(g) = mine[0].word | static_cast<uint32_t>(mine[1].word) << 16;
  else if (p < NB)
    *g = mine[0].word;
}

hipError_t launch_kv_cache_write4(Cache4Args a, int dtype, hipStream_t s) {
  const int64_t rows = static_cast<int64_t>(a.num_tokens) * a.num_kv_heads;
  if (rows <= 0) return hipSuccess;
  const auto shift = [](int n) { return (n & (n - 1)) == 0 ? 31 - __builtin_clz(n) : -1; };
  a.heads_shift = shift(a.num_kv_heads);
  a.block_shift = shift(a.block_size);
  const dim3 g(static_cast<unsigned>((rows + 63) / 64), 2), b(256);
  with_head_dim(a.head_dim, [&](auto d) {
    constexpr int NB = decltype(d)::value / 32;
    if (dtype == FP_DTYPE_BF16) hipLaunchKernelGGL((k_cache_write4<BF16, NB>), g, b, 0, s, a);
    else hipLaunchKernelGGL((k_cache_write4<F16, NB>), g, b, 0, s, a);
    return 0;
  });
  return hipGetLastError();
}

// A workgroup takes the tokens that make up a pass of its 64 rows (131,072 tokens of 8 heads
// of 128: 141 us; with two passes, the second's rows loaded before the first's are used, 154,
// with four 177), and stores through L2, since a store covers half a cache line of each of 16
// rows (past it: 169 us). 688 MB in 141 us are 4.9 TB/s, a copy's rate 5.15.
// di, dh: tokens and heads from a thread's row to its next one, 64 rows on.
constexpr int kGatherTokens = 64;
template <typename T, int NB>
__global__ __launch_bounds__(256) void k_cache_gather4(Cache4Args a, GatherArgs find, int tokens,
                                                       int di, int dh) {
  __shared__ CachedToken s_at[kGatherTokens];
  const Cache4Side& sd = a.side[blockIdx.y];
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * tokens;
  const int n = static_cast<int>(min(static_cast<int64_t>(tokens), a.num_tokens - t0));
  if (threadIdx.x < 64) {
    const CachedToken f = find_cached_token(find, t0 + threadIdx.x);
    if (static_cast<int>(threadIdx.x) < n) s_at[threadIdx.x] = f;
  }
  __syncthreads();
  const int p = threadIdx.x & 3, H = a.num_kv_heads;
  int i = static_cast<int>(threadIdx.x >> 2) / H, h = static_cast<int>(threadIdx.x >> 2) % H;
  while (i < n) {
    const CachedToken f = s_at[i];
    if (f.page != kSkip) {
      uint16_t* dst = sd.rows + (t0 + i) * sd.row_tok + h * sd.row_head + 8 * p;
      const int64_t page = max(f.page, int64_t(0)), in = f.page < 0 ? 0 : f.in;
      uint32_t w[NB], g[NB / 2];
      load_piece<NB>(sd.cache + page * sd.block + in * sd.slot + h * sd.head + 4 * NB * p, w);
      load_words<NB>(sd.g.p + page * sd.g.sb + h * sd.g.sh + in * NB, g);
      const float t = sd.t ? sd.t[h * sd.t_head] : 1.0f;
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        const uint32_t word = g[j >> 1] >> (16 * (j & 1));
        float s = static_cast<float>(
            __builtin_bit_cast(_Float16, static_cast<uint16_t>(word & 0x7f80u)));
        if (f.page == kNaN) s = __uint_as_float(0x7fc00000u);
        const float off = static_cast<float>(static_cast<int>(word & 0x7fu) - 64) * s;
        uint32_t y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int at = e * NB + j;
          const uint32_t b = w[at >> 2] >> (8 * (at & 3));
          const float lo = static_cast<float>(b & 15u), hi = static_cast<float>((b >> 4) & 15u);
          y[e] = pack2<T>(fmaf(lo, s, off) * t, fmaf(hi, s, off) * t);
        }
        st16(dst + 32 * j, make_uint4(y[0], y[1], y[2], y[3]));
      }
    }
    i += di;
    h += dh;
    if (h >= H) {
      h -= H;
      ++i;
    }
  }
}

hipError_t launch_kv_cache_gather4(const Cache4Args& a, const GatherArgs& find, int dtype,
                                   hipStream_t s) {
  if (a.num_tokens <= 0) return hipSuccess;
  const int tokens = a.num_kv_heads < kGatherTokens ? kGatherTokens / a.num_kv_heads : 1;
  const dim3 g(static_cast<unsigned>((a.num_tokens + tokens - 1) / tokens), 2), b(256);
  const int di = 64 / a.num_kv_heads, dh = 64 % a.num_kv_heads;
  with_head_dim(a.head_dim, [&](auto d) {
    constexpr int NB = decltype(d)::value / 32;
    if (dtype == FP_DTYPE_BF16)
      hipLaunchKernelGGL((k_cache_gather4<BF16, NB>), g, b, 0, s, a, find, tokens, di, dh);
    else
      hipLaunchKernelGGL((k_cache_gather4<F16, NB>), g, b, 0, s, a, find, tokens, di, dh);
    return 0;
  });
  return hipGetLastError();
}

}  // namespace fp

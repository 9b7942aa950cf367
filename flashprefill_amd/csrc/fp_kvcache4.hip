// Write and read-back of a paged KV cache of 4-bit integers (fp_int4.h, fp_kv_groups).
//
// Both move rows of head_dim elements, four lanes to a row: lane p takes dims
// 32 j + 8 p .. + 7 of every group j, 16 bytes of the 16-bit row at a time, whose codes are
// 4 (d / 32) contiguous bytes of the cached row. A workgroup serves K or V, so that strides
// and bases are scalars.
//
// The write finds each group's smallest and largest element over the four lanes and
// quantises by the rule of fp_kv_cache_write_int4. Its quotients are rounded as a division
// rounds them: y = x r, r about 1 / s, then y - r (y s - x), whose error before its own
// rounding is below 2^-43 of it, and x / s (s has 4 significant bits) is either an fp32
// number or at least 2^-29 of itself away from a midpoint of two.
#include "fp_int4.h"
#include "fp_kvcache_common.h"

namespace fp {

// x / y for a y of few significant bits (15, 56, a step), r about 1 / y
__device__ __forceinline__ float quotient(float x, float y, float r) {
  const float q = x * r;
  return fmaf(-fmaf(q, y, -x), r, q);
}

// max over the four lanes of a row
__device__ __forceinline__ float quad_max(float x) {
  const auto other = [](float v, auto ctrl) {
    return __uint_as_float(static_cast<uint32_t>(__builtin_amdgcn_update_dpp(
        0, static_cast<int>(__float_as_uint(v)), decltype(ctrl)::value, 0xf, 0xf, true)));
  };
  x = fmaxf(x, other(x, IntC<0xb1>{}));  // lanes 1 0 3 2
  return fmaxf(x, other(x, IntC<0x4e>{}));  // lanes 2 3 0 1
}

// x / t rounded once, clamped to the largest magnitude that a group holds. t from 2^-60 to
// 2^60: as above, with a second step, since t may have any bits (Markstein, Computation of
// elementary functions on the IBM RISC System/6000, 1990); others divide.
constexpr float kInt4Most = 16384.0f;
struct FixedScale {
  float t, r, most;
  bool easy;
  __device__ __forceinline__ explicit FixedScale(float t_) : t(t_) {
    easy = t >= 0x1p-60f && t <= 0x1p60f;
    r = 1.0f / t;
    most = t * (kInt4Most * 1.001f);  // (the infinite ones, whose remainder is NaN, among them)
  }
  __device__ __forceinline__ float divide(float x) const {
    if (!easy) return x / t;
    float y = x * r;
    y = fmaf(-fmaf(y, t, -x), r, y);
    y = fmaf(-fmaf(y, t, -x), r, y);
    return fabsf(x) > most ? copysignf(kInt4Most, x) : y;
  }
};

// One group's eight elements of a lane: codes as small floats, and the group's word
__device__ __forceinline__ uint16_t quantise_group(float (&x)[8]) {
  float hi = -INFINITY, low = -INFINITY, nan = 0.0f;  // low: the largest -x
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    nan = x[e] != x[e] ? 1.0f : nan;
    x[e] = __builtin_amdgcn_fmed3f(x[e], -kInt4Most, kInt4Most);
    hi = fmaxf(hi, x[e]);
    low = fmaxf(low, -x[e]);
  }
  hi = quad_max(hi);
  low = quad_max(low);
  nan = quad_max(nan);
  const float want = fmaxf(quotient(hi + low, 15.0f, 1.0f / 15.0f),
                           quotient(fmaxf(hi, low), 56.0f, 1.0f / 56.0f));
  uint32_t m = __float_as_uint(want);  // (-0 for a group of -0: s takes the magnitude)
  m = (m + 0x7ffffu + ((m >> 20) & 1u)) & ~0xfffffu;
  const float s = fabsf(want < 0x1p-14f ? rintf(want * 0x1p17f) * 0x1p-17f : __uint_as_float(m));
  const float some = s == 0.0f ? 1.0f : s;
  const float r = __builtin_amdgcn_rcpf(some);
  const float z = s == 0.0f ? 0.0f
                            : fminf(fmaxf(rintf(quotient(-low, some, r)), -64.0f), 63.0f);
  const bool none = s == 0.0f || nan != 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float c = __builtin_amdgcn_fmed3f(rintf(quotient(x[e], some, r)) - z, 0.0f, 15.0f);
    x[e] = none ? 0.0f : c;
  }
  if (nan != 0.0f) return 0x7f80u;
  const uint16_t bits = __builtin_bit_cast(uint16_t, static_cast<_Float16>(s));
  return static_cast<uint16_t>(bits | static_cast<uint32_t>(static_cast<int>(z) + 64));
}

template <typename T, int NB>
__global__ __launch_bounds__(256) void k_cache_write4(Cache4Args a) {
  const Cache4Side& sd = a.side[blockIdx.y];
  const int p = threadIdx.x & 3;
  const uint32_t row = blockIdx.x * 64u + (threadIdx.x >> 2);
  const uint32_t H = static_cast<uint32_t>(a.num_kv_heads);
  const uint32_t tok = row / H, h = row - tok * H;
  if (tok >= static_cast<uint32_t>(a.num_tokens)) return;  // (all four lanes of a row)
  const int64_t slot = a.slot_mapping[tok];
  const uint16_t* src = sd.rows + tok * sd.row_tok + h * sd.row_head + 8 * p;
  uint4 u[NB];
#pragma unroll
  for (int j = 0; j < NB; ++j) u[j] = ld16_once(src + 32 * j);
  if (slot < 0 || slot >= a.num_slots) return;
  int64_t blk, off;
  split_slot(slot, a.block_size, blk, off);
  const FixedScale fixed(sd.t ? sd.t[h * sd.t_head] : 1.0f);
  uint32_t word[NB];
  uint32_t b[4][NB];  // bytes (dim pair, group)
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const uint32_t uw[4] = {u[j].x, u[j].y, u[j].z, u[j].w};
    float x[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[2 * e] = T::to_f32(static_cast<uint16_t>(uw[e]));
      x[2 * e + 1] = T::to_f32(static_cast<uint16_t>(uw[e] >> 16));
    }
    if (sd.t) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = fixed.divide(x[e]);
    }
    word[j] = quantise_group(x);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      b[e][j] = static_cast<uint32_t>(fmaf(16.0f, x[2 * e + 1], x[2 * e]));
  }
  uint32_t w[NB];
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    const int at = 4 * i;  // the piece's bytes at .. at + 3
    w[i] = b[at / NB][at % NB] | b[(at + 1) / NB][(at + 1) % NB] << 8 |
           b[(at + 2) / NB][(at + 2) % NB] << 16 | b[(at + 3) / NB][(at + 3) % NB] << 24;
  }
  uint8_t* dst = sd.cache + blk * sd.block + off * sd.slot + h * sd.head + 4 * NB * p;
  if constexpr (NB == 2) {
    st8_once(dst, make_uint2(w[0], w[1]));
  } else {
#pragma unroll
    for (int i = 0; i < NB / 4; ++i)
      st16_once(dst + 16 * i, make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]));
  }
  // lane p stores the words of groups p (NB / 4) ..; with two groups lanes 0 and 1 one each
  uint16_t* g = sd.g.p + blk * sd.g.sb + h * sd.g.sh + off * NB;
  if constexpr (NB == 8) {
    const uint32_t x01 = word[0] | word[1] << 16, x23 = word[2] | word[3] << 16;
    const uint32_t x45 = word[4] | word[5] << 16, x67 = word[6] | word[7] << 16;
    *reinterpret_cast<uint32_t*>(g + 2 * p) = p < 2 ? (p ? x23 : x01) : p == 2 ? x45 : x67;
  } else if constexpr (NB == 4) {
    g[p] = static_cast<uint16_t>(p < 2 ? (p ? word[1] : word[0]) : p == 2 ? word[2] : word[3]);
  } else if (p < 2) {
    g[p] = static_cast<uint16_t>(p ? word[1] : word[0]);
  }
}

hipError_t launch_kv_cache_write4(const Cache4Args& a, int dtype, hipStream_t s) {
  const int64_t rows = static_cast<int64_t>(a.num_tokens) * a.num_kv_heads;
  if (rows <= 0) return hipSuccess;
  const dim3 g(static_cast<unsigned>((rows + 63) / 64), 2), b(256);
  with_head_dim(a.head_dim, [&](auto d) {
    constexpr int NB = decltype(d)::value / 32;
    if (dtype == FP_DTYPE_BF16) hipLaunchKernelGGL((k_cache_write4<BF16, NB>), g, b, 0, s, a);
    else hipLaunchKernelGGL((k_cache_write4<F16, NB>), g, b, 0, s, a);
    return 0;
  });
  return hipGetLastError();
}

// tokens: of a workgroup; di, dh: tokens and heads from a thread's row to its next one,
// 64 rows on
template <typename T, int NB>
__global__ __launch_bounds__(256) void k_cache_gather4(Cache4Args a, GatherArgs find, int tokens,
                                                       int di, int dh) {
  __shared__ CachedToken s_at[kRowTokens];
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
  for (; i < n; i += di) {
    const CachedToken f = s_at[i];
    if (f.page != kSkip) {
      uint16_t* dst = sd.rows + (t0 + i) * sd.row_tok + h * sd.row_head + 8 * p;
      const int64_t page = max(f.page, int64_t(0));
      const int64_t in = f.page < 0 ? 0 : f.in;
      const uint8_t* src = sd.cache + page * sd.block + in * sd.slot + h * sd.head + 4 * NB * p;
      uint32_t w[NB], g[NB / 2];
      load_piece<NB>(src, w);
      load_words<NB>(sd.g.p + page * sd.g.sb + h * sd.g.sh + in * NB, g);
      const float t = sd.t ? sd.t[h * sd.t_head] : 1.0f;
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        const uint32_t word = g[j >> 1] >> (16 * (j & 1));
        float s = static_cast<float>(
            __builtin_bit_cast(_Float16, static_cast<uint16_t>(word & 0x7f80u)));
        if (f.page < 0) s = __uint_as_float(0x7fc00000u);
        const float off = static_cast<float>(static_cast<int>(word & 0x7fu) - 64) * s;
        uint32_t y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int at = e * NB + j;
          const uint32_t b = w[at >> 2] >> (8 * (at & 3));
          const float lo = static_cast<float>(b & 15u), hi = static_cast<float>((b >> 4) & 15u);
          y[e] = pack2<T>(fmaf(lo, s, off) * t, fmaf(hi, s, off) * t);
        }
        st16_once(dst + 32 * j, make_uint4(y[0], y[1], y[2], y[3]));
      }
    }
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
  int tokens = kRowTokens;  // (as row_walk has them)
  while (tokens > 1 && a.num_tokens / tokens < 1024) tokens /= 2;
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

// Paged KV-cache write for the vLLM-style backend hook: the key and value row
// of every token go to the cache slot slot_mapping[t], i.e. block
// slot / block_size, offset slot % block_size (the write the reference's
// vLLM patch makes with reshape_and_cache_flash before each attention call,
// patches/patch_loader_vllm_0_12_0.py:140-149). Slots < 0 are padding tokens
// and are skipped, as are slots past the cache.
//
// HBM-bound byte copy: one workgroup per token moves its K and V rows
// (num_kv_heads x head_dim elements each) in 16-byte chunks; algorithmic
// bytes per token = 2 (K, V) x num_kv_heads x head_dim x elem_bytes, read
// once and written once.
//
// 8-bit caches (k_kv_cache_write8): element x of a row becomes
// F(clamp(x / s, -M, M)), F the rounding to e4m3 or e5m2 (nearest, ties to even)
// and M its largest finite value; infinities saturate as well, NaN stays NaN. s is
// the cache's fixed scale or, one per slot, max |x| / M over the row's finite
// values (1 where that is 0), written beside the row. x / s is the correctly
// rounded fp32 quotient, so a code differs from that of the exact quotient only
// where both lie within 2^-24 of a tie. 2 bytes read and 1 written per element:
// HBM-bound like the copy (131,072 tokens of 8 heads of 128, 798 MB: 159 us in a row of
// calls, 5.0 TB/s, where a plain stream of two reads to a write reaches 6.4). 14,500 tokens
// of 4 heads, 45 MB: 16 us (7 at that rate). There a workgroup makes one pass, its four
// loads per thread in flight together, but only once the slots' lookup has passed the
// barrier, and with 104 registers 1,024 of the 1,821 workgroups run at a time.
//
// Read-back (k_kv_cache_gather): row cu[b] + i of key / value is cached token
// starts[b] + i of sequence b, c * s in fp32 rounded once (a 16-bit cache: its
// bits). 218,000 tokens of 8 heads of 128, 1.34 GB: 239 us, 5.6 TB/s (a plain stream of
// one read to two writes: 6.0); from a 16-bit cache, 1.78 GB, 326 us, 5.5 TB/s.
#include "fp_float8.h"
#include "fp_paged_common.h"

namespace fp {

__global__ __launch_bounds__(256) void k_kv_cache_write(KvCacheArgs a) {
  const int64_t t = blockIdx.x;
  if (t >= a.num_tokens) return;
  const int64_t slot = a.slot_mapping[t];
  if (slot < 0 || slot >= a.num_slots) return;
  const int64_t blk = slot / a.block_size, off = slot % a.block_size;
  const int cpr = a.row_bytes / 16;  // 16-byte chunks per head row
  const int per = a.num_kv_heads * cpr;
  for (int c = threadIdx.x; c < 2 * per; c += blockDim.x) {
    const bool is_v = c >= per;
    const int cc = is_v ? c - per : c;
    const int h = cc / cpr, x = cc % cpr;
    const char* src = static_cast<const char*>(is_v ? a.value : a.key) +
                      (t * (is_v ? a.v_stride_tok : a.k_stride_tok) +
                       h * (is_v ? a.v_stride_head : a.k_stride_head)) * a.elem_bytes;
    char* dst = static_cast<char*>(is_v ? a.value_cache : a.key_cache) +
                (blk * (is_v ? a.vc_stride_block : a.kc_stride_block) +
                 off * (is_v ? a.vc_stride_slot : a.kc_stride_slot) +
                 h * (is_v ? a.vc_stride_head : a.kc_stride_head)) * a.elem_bytes;
    st16(dst + 16 * x, ld16(src + 16 * x));
  }
}

hipError_t launch_kv_cache_write(const KvCacheArgs& a, hipStream_t s) {
  if (a.num_tokens <= 0) return hipSuccess;
  hipLaunchKernelGGL(k_kv_cache_write, dim3(static_cast<unsigned>(a.num_tokens)), dim3(256), 0, s,
                     a);
  return hipGetLastError();
}

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

// A row's quotient x / s, rounded once, without a division per element: with r the
// rounded 1 / s, a quotient y within an ulp or two becomes one within half an ulp and
// a little by y - r (y s - x), and the same step again gives the correctly rounded one
// (Markstein, Computation of elementary functions on the IBM RISC System/6000, 1990;
// the remainders are exact). That needs no product near the ends of fp32's range: s
// from 2^-60 to 2^60 (a smaller |x| than 2^-102 has a quotient of code 0 whatever its
// last bits), other scales divide.
template <int F>
__device__ __forceinline__ void divide_row(float (&x)[8], float s) {
  constexpr float kMax = Float8<F>::kMax;
  if (s >= 0x1p-60f && s <= 0x1p60f) {
    const float r = 1.0f / s;
    // inputs past this one saturate; quotients up to it, half way from the largest
    // finite value to where one would round to more, still round to it
    const float most = s * (kMax * (1.0f + 1.0f / 56.0f));
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float y = x[e] * r;
      y = fmaf(-fmaf(y, s, -x[e]), r, y);  // (with these signs a zero keeps its own)
      y = fmaf(-fmaf(y, s, -x[e]), r, y);
      x[e] = fabsf(x[e]) > most ? copysignf(kMax, x[e]) : y;  // (a NaN stays)
    }
  } else {
#pragma unroll 1
    for (int e = 0; e < 8; ++e) {
      const float y = x[0] / s;
#pragma unroll
      for (int i = 0; i < 7; ++i) x[i] = x[i + 1];
      x[7] = fabsf(y) > kMax ? copysignf(kMax, y) : y;
    }
  }
}

__device__ __forceinline__ int64_t scale_place(const CacheScales& s, int64_t blk, int64_t off) {
  return s.slot ? blk * s.sb + off : 0;
}

// What the rows of K or of V need. A scale is at scale[place + head * scale_head], place
// 0 for a fixed one, so that it is one load without a branch; without one (`one`),
// `scale` is some other memory.
struct Side {
  int64_t tok, head;   // strides of the 16-bit rows
  char* cache;
  int64_t cache_head;
  float* scale;
  int64_t scale_head;
  int32_t per_slot, one;
};
struct Sides {
  Side k, v;
};
inline Sides sides(const Cache8Args& a, const void* other) {
  const auto side = [&](const CacheScales& s, int64_t tok, int64_t head, void* cache, int64_t ch) {
    float* p = s.p ? s.p : static_cast<float*>(const_cast<void*>(other));
    return Side{tok, head, static_cast<char*>(cache), ch, p, s.sh, s.slot, s.p == nullptr};
  };
  return Sides{
      side(a.ks, a.c.k_stride_tok, a.c.k_stride_head, a.c.key_cache, a.c.kc_stride_head),
      side(a.vs, a.c.v_stride_tok, a.c.v_stride_head, a.c.value_cache, a.c.vc_stride_head)};
}
// A kernel argument held in scalar registers: a choice between two of them by a lane's
// row would otherwise be made between their addresses and cost a load (the 131072-token
// write took 307 us so).
template <typename X>
__device__ __forceinline__ X in_sgpr(X x) {
  asm volatile("" : "+s"(x));
  return x;
}
__device__ __forceinline__ Side in_sgprs(const Side& s) {
  return Side{in_sgpr(s.tok),   in_sgpr(s.head),       in_sgpr(s.cache),    in_sgpr(s.cache_head),
              in_sgpr(s.scale), in_sgpr(s.scale_head), in_sgpr(s.per_slot), in_sgpr(s.one)};
}
__device__ __forceinline__ Side choose(bool v, const Side& a, const Side& b) {
  return Side{v ? b.tok : a.tok,
              v ? b.head : a.head,
              v ? b.cache : a.cache,
              v ? b.cache_head : a.cache_head,
              v ? b.scale : a.scale,
              v ? b.scale_head : a.scale_head,
              v ? b.per_slot : a.per_slot,
              v ? b.one : a.one};
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

// U rows of a thread are loaded before the first is used. Their loads have no branch
// around them (rows past the last and rows of no place read another's memory and are
// not stored): where a load's result meets another value behind a branch the compiler
// waits for every load before the next, and 218,000 tokens of 8 heads of 128 took 325 us
// to read back.
template <typename T, int F, int U>
__global__ __launch_bounds__(256) void k_kv_cache_write8(Cache8Args a, Sides sides, RowWalk w) {
  // a token's place in the caches and in the scales of a slot (first < 0: none)
  __shared__ int64_t s_at[kRowTokens][2], s_sc[kRowTokens][2];
  const KvCacheArgs& c = a.c;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * w.tokens;
  const int n = static_cast<int>(min(static_cast<int64_t>(w.tokens), c.num_tokens - t0));
  const int Hkv = c.num_kv_heads, per = 2 * Hkv;
  const int l = threadIdx.x & ((1 << w.lg) - 1);
  const bool on = 8 * l < c.row_bytes;  // (row_bytes: head_dim)
  const int first = static_cast<int>(threadIdx.x >> w.lg);
  int i = first / per, h = first % per;
  const int lx = on ? 8 * l : 0;
  const uint16_t* kp = static_cast<const uint16_t*>(c.key) + t0 * c.k_stride_tok + lx;
  const uint16_t* vp = static_cast<const uint16_t*>(c.value) + t0 * c.v_stride_tok + lx;
  const Side ks = in_sgprs(sides.k), vs = in_sgprs(sides.v);
  if (static_cast<int>(threadIdx.x) < n) {
    const int64_t slot = c.slot_mapping[t0 + threadIdx.x];
    int64_t at[2] = {-1, -1}, sc[2] = {0, 0};
    if (slot >= 0 && slot < c.num_slots) {
      int64_t blk, off;
      split_slot(slot, c.block_size, blk, off);
      at[0] = blk * c.kc_stride_block + off * c.kc_stride_slot;
      at[1] = blk * c.vc_stride_block + off * c.vc_stride_slot;
      sc[0] = scale_place(a.ks, blk, off);
      sc[1] = scale_place(a.vs, blk, off);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      s_at[threadIdx.x][k] = at[k];
      s_sc[threadIdx.x][k] = sc[k];
    }
  }
  __syncthreads();
  while (i < n) {
    uint4 u[U];
    float sk[U];
    int ui[U], uh[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      ui[k] = i;
      uh[k] = h;
      const int ii = min(i, n - 1);
      const bool is_v = h >= Hkv;
      const int hh = is_v ? h - Hkv : h;
      const Side sd = choose(is_v, ks, vs);
      u[k] = ld16_once((is_v ? vp : kp) + ii * sd.tok + hh * sd.head);
      sk[k] = *global_ptr<const float>(sd.scale + (sd.per_slot ? 0 : hh * sd.scale_head));
      if (sd.one) sk[k] = 1.0f;
      i += w.di;
      h += w.dh;
      if (h >= per) {
        h -= per;
        ++i;
      }
    }
    uint2 y[U];
    char* dst[U];
    bool put[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int ii = min(ui[k], n - 1);
      const bool is_v = uh[k] >= Hkv;
      const int hh = is_v ? uh[k] - Hkv : uh[k];
      const int64_t at = s_at[ii][is_v];
      put[k] = on && ui[k] < n && at >= 0;
      const Side sd = choose(is_v, ks, vs);
      dst[k] = sd.cache + at + hh * sd.cache_head + 8 * l;
      const uint32_t uw[4] = {u[k].x, u[k].y, u[k].z, u[k].w};
      float x[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[2 * e] = T::to_f32(static_cast<uint16_t>(uw[e]));
        x[2 * e + 1] = T::to_f32(static_cast<uint16_t>(uw[e] >> 16));
      }
      if (sd.per_slot) {  // (lanes past the row hold its first elements again)
        float m = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float z = fabsf(x[e]);
          m = fmaxf(m, z < INFINITY ? z : 0.0f);
        }
        for (int o = 1 << w.lg >> 1; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
        const float q = m / Float8<F>::kMax;
        sk[k] = q > 0.0f ? q : 1.0f;
        if (l == 0 && put[k])
          *global_ptr<float>(sd.scale + s_sc[ii][is_v] + hh * sd.scale_head) = sk[k];
      }
      divide_row<F>(x, sk[k]);
      y[k].x = Float8<F>::template from_f32<false>(x[0], x[1], 0u);
      y[k].x = Float8<F>::template from_f32<true>(x[2], x[3], y[k].x);
      y[k].y = Float8<F>::template from_f32<false>(x[4], x[5], 0u);
      y[k].y = Float8<F>::template from_f32<true>(x[6], x[7], y[k].y);
    }
#pragma unroll
    for (int k = 0; k < U; ++k)
      if (put[k]) st8_once(dst[k], y[k]);
  }
}

// f(T, U) of the row type and the rows in flight per thread: the most, up to MAX, that
// a workgroup's rows fill (with 4, the new tokens of 32 requests take 4.7 us instead of
// 3.9; with 8, reading back 218,000 tokens takes 236 instead of 243 and the write gains
// nothing).
template <int MAX, typename Fn>
void with_rows(const RowWalk& w, int num_kv_heads, int dtype, Fn&& f) {
  const auto run = [&](auto t) {
    const int fill = w.tokens * 2 * num_kv_heads / (256 >> w.lg);
    if constexpr (MAX >= 8) {
      if (fill >= 8) return f(t, IntC<8>{});
    }
    if (fill >= 4) f(t, IntC<4>{});
    else if (fill >= 2) f(t, IntC<2>{});
    else f(t, IntC<1>{});
  };
  if (dtype == FP_DTYPE_BF16) run(BF16{});
  else run(F16{});
}

hipError_t launch_kv_cache_write8(const Cache8Args& a, int dtype, int format, hipStream_t s) {
  if (a.c.num_tokens <= 0) return hipSuccess;
  const RowWalk w = row_walk(a.c.row_bytes, a.c.num_kv_heads, a.c.num_tokens);
  const dim3 g(static_cast<unsigned>((a.c.num_tokens + w.tokens - 1) / w.tokens)), b(256);
  const Sides sd = sides(a, a.c.slot_mapping);
  with_rows<4>(w, a.c.num_kv_heads, dtype, [&](auto t, auto u) {
    using T = decltype(t);
    constexpr int U = decltype(u)::value;
    if (format == FP_CACHE_E4M3)
      hipLaunchKernelGGL((k_kv_cache_write8<T, FP_CACHE_E4M3, U>), g, b, 0, s, a, sd, w);
    else
      hipLaunchKernelGGL((k_kv_cache_write8<T, FP_CACHE_E5M2, U>), g, b, 0, s, a, sd, w);
  });
  return hipGetLastError();
}

// F: the cache's format (FP_CACHE_16BIT: T itself). The first wave of a workgroup finds
// its tokens' sequences (64 at a time, a search over the lanes: a token belongs to the
// last sequence b with cu[b] <= token, if token < cu[b + 1]) and places, then all
// waves move their heads.
template <typename T, int F, int U>
__global__ __launch_bounds__(256) void k_kv_cache_gather(GatherArgs a, Sides sides, RowWalk w) {
  constexpr int64_t kSkip = -1, kNaN = -2;  // rows of no sequence; rows that cannot be read
  __shared__ int64_t s_at[kRowTokens][2], s_sc[kRowTokens][2];
  const KvCacheArgs& c = a.g.c;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * w.tokens;
  const int n = static_cast<int>(min(static_cast<int64_t>(w.tokens), c.num_tokens - t0));
  if (threadIdx.x < 64) {
    const int lane = threadIdx.x;
    const int64_t tok = t0 + lane;
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
    int64_t at[2] = {kSkip, kSkip}, sc[2] = {0, 0};
    if (off) {
      at[0] = at[1] = kNaN;
    } else if (b >= 0) {
      int64_t pos = tok - seq0;
      const int64_t start = a.starts ? ld_int(a.starts, a.starts64, b) : 0;
      const int64_t room = static_cast<int64_t>(a.width) * c.block_size;
      at[0] = at[1] = kNaN;
      if (start >= 0 && start < room && pos + start < room) {
        pos += start;
        int64_t blk, in;
        split_slot(pos, c.block_size, blk, in);
        int64_t page = ld_int(a.table, a.table64, b * a.table_stride + blk);
        if (page < 0) page += a.num_blocks;
        if (page >= 0 && page < a.num_blocks) {
          at[0] = page * c.kc_stride_block + in * c.kc_stride_slot;
          at[1] = page * c.vc_stride_block + in * c.vc_stride_slot;
          sc[0] = scale_place(a.g.ks, page, in);
          sc[1] = scale_place(a.g.vs, page, in);
        }
      }
    }
    if (lane < n) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        s_at[lane][i] = at[i];
        s_sc[lane][i] = sc[i];
      }
    }
  }
  __syncthreads();
  const int Hkv = c.num_kv_heads, per = 2 * Hkv;
  const int l = threadIdx.x & ((1 << w.lg) - 1);
  if (8 * l >= c.row_bytes) return;  // (row_bytes: head_dim)
  const int first = static_cast<int>(threadIdx.x >> w.lg);
  int i = first / per, h = first % per;
  uint16_t* kp = static_cast<uint16_t*>(const_cast<void*>(c.key)) + t0 * c.k_stride_tok + 8 * l;
  uint16_t* vp = static_cast<uint16_t*>(const_cast<void*>(c.value)) + t0 * c.v_stride_tok + 8 * l;
  const Side ks = in_sgprs(sides.k), vs = in_sgprs(sides.v);
  while (i < n) {
    typename std::conditional<F == FP_CACHE_16BIT, uint4, uint2>::type u[U];
    float s[U];
    int64_t at[U];
    uint16_t* dst[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int ii = min(i, n - 1);
      const bool is_v = h >= Hkv;
      const int hh = is_v ? h - Hkv : h;
      at[k] = s_at[ii][is_v];
      const Side sd = choose(is_v, ks, vs);
      dst[k] = (is_v ? vp : kp) + ii * sd.tok + hh * sd.head;
      const int64_t x = max(at[k], int64_t(0)) + hh * sd.cache_head + 8 * l;
      if constexpr (F == FP_CACHE_16BIT) {
        u[k] = ld16_once(sd.cache + 2 * x);
      } else {
        u[k] = ld8_once(sd.cache + x);
        s[k] = *global_ptr<const float>(sd.scale + s_sc[ii][is_v] + hh * sd.scale_head);
        if (sd.one) s[k] = 1.0f;
      }
      if (i >= n) at[k] = kSkip;
      i += w.di;
      h += w.dh;
      if (h >= per) {
        h -= per;
        ++i;
      }
    }
    uint4 y[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      if constexpr (F == FP_CACHE_16BIT) {
        y[k] = u[k];
      } else {
        const f32x2 x[4] = {
            Float8<F>::template to_f32<false>(u[k].x), Float8<F>::template to_f32<true>(u[k].x),
            Float8<F>::template to_f32<false>(u[k].y), Float8<F>::template to_f32<true>(u[k].y)};
        y[k] = make_uint4(pack2<T>(x[0][0] * s[k], x[0][1] * s[k]),
                          pack2<T>(x[1][0] * s[k], x[1][1] * s[k]),
                          pack2<T>(x[2][0] * s[k], x[2][1] * s[k]),
                          pack2<T>(x[3][0] * s[k], x[3][1] * s[k]));
      }
      const uint32_t nan = pack2<T>(__uint_as_float(0x7fc00000u), __uint_as_float(0x7fc00000u));
      if (at[k] == kNaN) y[k] = make_uint4(nan, nan, nan, nan);
    }
#pragma unroll
    for (int k = 0; k < U; ++k)
      if (at[k] != kSkip) st16_once(dst[k], y[k]);
  }
}

hipError_t launch_kv_cache_gather(const GatherArgs& a, int dtype, int format, hipStream_t s) {
  if (a.g.c.num_tokens <= 0) return hipSuccess;
  const RowWalk w = row_walk(a.g.c.row_bytes, a.g.c.num_kv_heads, a.g.c.num_tokens);
  const dim3 g(static_cast<unsigned>((a.g.c.num_tokens + w.tokens - 1) / w.tokens)), b(256);
  const Sides sd = sides(a.g, a.cu);
  with_rows<8>(w, a.g.c.num_kv_heads, dtype, [&](auto t, auto u) {
    using T = decltype(t);
    constexpr int U = decltype(u)::value;
    if (format == FP_CACHE_16BIT)
      hipLaunchKernelGGL((k_kv_cache_gather<T, FP_CACHE_16BIT, U>), g, b, 0, s, a, sd, w);
    else if (format == FP_CACHE_E4M3)
      hipLaunchKernelGGL((k_kv_cache_gather<T, FP_CACHE_E4M3, U>), g, b, 0, s, a, sd, w);
    else
      hipLaunchKernelGGL((k_kv_cache_gather<T, FP_CACHE_E5M2, U>), g, b, 0, s, a, sd, w);
  });
  return hipGetLastError();
}

}  // namespace fp

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
// HBM-bound like the copy.
//
// Read-back (k_kv_cache_gather): row cu[b] + i of key / value is cached token
// starts[b] + i of sequence b, c * s in fp32 rounded once (a 16-bit cache: its
// bits).
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

template <typename T, int F>
__global__ __launch_bounds__(256) void k_kv_cache_write8(Cache8Args a, int lanes) {
  constexpr float kMax = Float8<F>::kMax;
  const int l = threadIdx.x & (lanes - 1);
  const int64_t row = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) / lanes;
  const int per = 2 * a.c.num_kv_heads;  // rows of a token: its K heads, then its V heads
  const int64_t t = row / per;
  if (t >= a.c.num_tokens) return;
  const int64_t slot = a.c.slot_mapping[t];
  if (slot < 0 || slot >= a.c.num_slots) return;
  int h = static_cast<int>(row % per);
  const bool is_v = h >= a.c.num_kv_heads;
  if (is_v) h -= a.c.num_kv_heads;
  const int64_t blk = slot / a.c.block_size, off = slot % a.c.block_size;
  const bool on = 8 * l < a.c.row_bytes;  // (row_bytes: head_dim bytes)
  const uint16_t* src = static_cast<const uint16_t*>(is_v ? a.c.value : a.c.key) +
                        t * (is_v ? a.c.v_stride_tok : a.c.k_stride_tok) +
                        h * (is_v ? a.c.v_stride_head : a.c.k_stride_head) + 8 * l;
  const uint4 u = on ? ld16(src) : zero4();
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  float x[8];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    x[2 * e] = T::to_f32(static_cast<uint16_t>(w[e]));
    x[2 * e + 1] = T::to_f32(static_cast<uint16_t>(w[e] >> 16));
  }
  const CacheScales& cs = is_v ? a.vs : a.ks;
  float s;
  if (cs.slot) {
    float m = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float y = fabsf(x[e]);
      m = fmaxf(m, y < INFINITY ? y : 0.0f);
    }
    for (int o = lanes >> 1; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    s = m / kMax;
    if (!(s > 0.0f)) s = 1.0f;
    if (l == 0) cs.p[blk * cs.sb + h * cs.sh + off] = s;
  } else {
    s = fixed_scale(cs, h);
  }
  if (!on) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float y = x[e] / s;
    x[e] = fabsf(y) > kMax ? copysignf(kMax, y) : y;  // (a NaN compares false and stays)
  }
  uint2 o;
  o.x = Float8<F>::template from_f32<false>(x[0], x[1], 0u);
  o.x = Float8<F>::template from_f32<true>(x[2], x[3], o.x);
  o.y = Float8<F>::template from_f32<false>(x[4], x[5], 0u);
  o.y = Float8<F>::template from_f32<true>(x[6], x[7], o.y);
  uint8_t* dst = static_cast<uint8_t*>(is_v ? a.c.value_cache : a.c.key_cache) +
                 blk * (is_v ? a.c.vc_stride_block : a.c.kc_stride_block) +
                 off * (is_v ? a.c.vc_stride_slot : a.c.kc_stride_slot) +
                 h * (is_v ? a.c.vc_stride_head : a.c.kc_stride_head) + 8 * l;
  *reinterpret_cast<uint2*>(dst) = o;
}

hipError_t launch_kv_cache_write8(const Cache8Args& a, int dtype, int format, hipStream_t s) {
  const int lanes = row_lanes(a.c.row_bytes);
  const int64_t rows = a.c.num_tokens * 2 * a.c.num_kv_heads;
  if (rows <= 0) return hipSuccess;
  const dim3 g(static_cast<unsigned>((rows * lanes + 255) / 256)), b(256);
  const bool bf = dtype == FP_DTYPE_BF16;
  if (format == FP_CACHE_E4M3) {
    if (bf) hipLaunchKernelGGL((k_kv_cache_write8<BF16, FP_CACHE_E4M3>), g, b, 0, s, a, lanes);
    else hipLaunchKernelGGL((k_kv_cache_write8<F16, FP_CACHE_E4M3>), g, b, 0, s, a, lanes);
  } else {
    if (bf) hipLaunchKernelGGL((k_kv_cache_write8<BF16, FP_CACHE_E5M2>), g, b, 0, s, a, lanes);
    else hipLaunchKernelGGL((k_kv_cache_write8<F16, FP_CACHE_E5M2>), g, b, 0, s, a, lanes);
  }
  return hipGetLastError();
}

// F: the cache's format (FP_CACHE_16BIT: T itself). A workgroup takes kGatherTokens
// rows of key and value: its first wave finds their sequences (64 at a time: a token
// belongs to sequence b where cu[b] <= token < cu[b + 1]) and slots, then all waves
// move their heads, 8 elements per lane.
template <typename T, int F>
__global__ __launch_bounds__(256) void k_kv_cache_gather(GatherArgs a, int lanes) {
  constexpr int64_t kSkip = -1, kNaN = -2;  // rows of no sequence; rows that cannot be read
  __shared__ int64_t s_slot[kGatherTokens];
  const Cache8Args& g = a.g;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * kGatherTokens;
  const int n = static_cast<int>(min(static_cast<int64_t>(kGatherTokens), g.c.num_tokens - t0));
  if (threadIdx.x < 64) {
    const int lane = threadIdx.x;
    const int64_t tok = t0 + lane;
    int64_t b = -1, first = 0;
    bool off = false;
    for (int base = 0; base < a.B; base += 64) {
      int64_t c0 = 0, c1 = 0;
      if (base + lane < a.B) {
        c0 = ld_int(a.cu, a.cu64, base + lane);
        c1 = ld_int(a.cu, a.cu64, base + lane + 1);
      }
      off = off || __ballot(c0 < 0 || c1 > g.c.num_tokens || c1 < c0) != 0;
      for (int i = 0; i < n; ++i) {
        const uint64_t hit = __ballot(c0 <= t0 + i && t0 + i < c1);
        if (hit == 0) continue;
        const int src = __ffsll(static_cast<long long>(hit)) - 1;
        const int64_t f = shfl64(c0, src);
        if (lane == i) {
          b = base + src;
          first = f;
        }
      }
    }
    int64_t slot = kSkip;
    if (off) {
      slot = kNaN;
    } else if (b >= 0) {
      int64_t pos = tok - first;
      const int64_t start = a.starts ? ld_int(a.starts, a.starts64, b) : 0;
      slot = kNaN;
      const int64_t room = static_cast<int64_t>(a.width) * g.c.block_size;
      if (start >= 0 && start < room && pos + start < room) {
        pos += start;
        int64_t page = ld_int(a.table, a.table64, b * a.table_stride + pos / g.c.block_size);
        if (page < 0) page += a.num_blocks;
        if (page >= 0 && page < a.num_blocks)
          slot = page * g.c.block_size + pos % g.c.block_size;
      }
    }
    if (lane < n) s_slot[lane] = slot;
  }
  __syncthreads();
  const int per = 2 * g.c.num_kv_heads;
  const int l = threadIdx.x & (lanes - 1);
  if (8 * l >= g.c.row_bytes) return;  // (row_bytes: head_dim)
  for (int r = threadIdx.x / lanes; r < n * per; r += 256 / lanes) {
    const int i = r / per;
    const int64_t slot = s_slot[i];
    if (slot == kSkip) continue;
    int h = r % per;
    const bool is_v = h >= g.c.num_kv_heads;
    if (is_v) h -= g.c.num_kv_heads;
    uint16_t* dst = static_cast<uint16_t*>(const_cast<void*>(is_v ? g.c.value : g.c.key)) +
                    (t0 + i) * (is_v ? g.c.v_stride_tok : g.c.k_stride_tok) +
                    h * (is_v ? g.c.v_stride_head : g.c.k_stride_head) + 8 * l;
    if (slot == kNaN) {
      const uint32_t nan = pack2<T>(__uint_as_float(0x7fc00000u), __uint_as_float(0x7fc00000u));
      st16(dst, make_uint4(nan, nan, nan, nan));
      continue;
    }
    const int64_t blk = slot / g.c.block_size, in = slot % g.c.block_size;
    const int64_t at = blk * (is_v ? g.c.vc_stride_block : g.c.kc_stride_block) +
                       in * (is_v ? g.c.vc_stride_slot : g.c.kc_stride_slot) +
                       h * (is_v ? g.c.vc_stride_head : g.c.kc_stride_head) + 8 * l;
    const char* cache = static_cast<const char*>(is_v ? g.c.value_cache : g.c.key_cache);
    if constexpr (F == FP_CACHE_16BIT) {
      st16(dst, ld16(cache + 2 * at));
    } else {
      const CacheScales& cs = is_v ? g.vs : g.ks;
      const float s = cs.slot ? cs.p[blk * cs.sb + h * cs.sh + in] : fixed_scale(cs, h);
      const uint2 u = *reinterpret_cast<const uint2*>(cache + at);
      const f32x2 x[4] = {
          Float8<F>::template to_f32<false>(u.x), Float8<F>::template to_f32<true>(u.x),
          Float8<F>::template to_f32<false>(u.y), Float8<F>::template to_f32<true>(u.y)};
      st16(dst, make_uint4(pack2<T>(x[0][0] * s, x[0][1] * s), pack2<T>(x[1][0] * s, x[1][1] * s),
                           pack2<T>(x[2][0] * s, x[2][1] * s), pack2<T>(x[3][0] * s, x[3][1] * s)));
    }
  }
}

hipError_t launch_kv_cache_gather(const GatherArgs& a, int dtype, int format, hipStream_t s) {
  if (a.g.c.num_tokens <= 0) return hipSuccess;
  const int lanes = row_lanes(a.g.c.row_bytes);
  const dim3 g(static_cast<unsigned>((a.g.c.num_tokens + kGatherTokens - 1) / kGatherTokens));
  const dim3 b(256);
  const auto run = [&](auto t) {
    using T = decltype(t);
    if (format == FP_CACHE_16BIT)
      hipLaunchKernelGGL((k_kv_cache_gather<T, FP_CACHE_16BIT>), g, b, 0, s, a, lanes);
    else if (format == FP_CACHE_E4M3)
      hipLaunchKernelGGL((k_kv_cache_gather<T, FP_CACHE_E4M3>), g, b, 0, s, a, lanes);
    else
      hipLaunchKernelGGL((k_kv_cache_gather<T, FP_CACHE_E5M2>), g, b, 0, s, a, lanes);
  };
  if (dtype == FP_DTYPE_BF16) run(BF16{});
  else run(F16{});
  return hipGetLastError();
}

}  // namespace fp

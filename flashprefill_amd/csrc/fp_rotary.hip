// Rotary positions of any layout: the first 2 n of a head's dims are n pairs, dims i and
// n + i or, interleaved, 2 i and 2 i + 1, and pair (x, y) of a token at position p becomes
//   (x c - y s, y c + x s),  c = A cos(p f_i),  s = A sin(p f_i),
// the other dims stay. f_i are 64-bit frequencies in device memory, scaled for a long context
// by whoever made them; the inverse rotation has -s.
//
// Memory-bound: 2 bytes read and written per element. A workgroup takes a few tokens with all
// heads: it finds their n cosines and sines once, in LDS, then rotates the heads' rows, a
// thread V pairs at a time. An angle of position 131,071 needs 17 bits before the point:
// p f is a 64-bit product, reduced in 64 bits to |r| <= pi / 4 (two parts of pi / 2, so that
// the second product's rounding is below 2^-50 for angles to 2^30), and cosine and sine of r, of
// the series of Taylor in 64 bits, times A are rounded to fp32 once. 65,536 tokens of 32 heads of 128, the pairs of half of each
// rotated: 220 us, 4.9 TB/s (a copy reaches 5.15).
#include <algorithm>

#include "fp_attn_common.h"

namespace fp {

constexpr int kRotaryLds = 2048;  // (cos, sin) pairs of a workgroup's tokens

__device__ __forceinline__ float2 turn(int64_t p, double f, float amplitude, bool inverse) {
  const double t = static_cast<double>(p) * f;
  const double k = rint(t * 0x1.45f306dc9c883p-1);      // 2 / pi
  double r = fma(-k, 0x1.921fb54442d18p+0, t);          // pi / 2, its first 53 bits
  r = fma(-k, 0x1.1a62633145c07p-54, r);                // and the next
  // (the terms left out are below 2^-54 of the sine and 2^-49 of the cosine)
  const double z = r * r;
  double s = -1.0 / 1307674368000.0, c = 1.0 / 20922789888000.0;  // 15!, 16!
  constexpr double kSin[6] = {1.0 / 6227020800.0, -1.0 / 39916800.0, 1.0 / 362880.0,
                              -1.0 / 5040.0,      1.0 / 120.0,       -1.0 / 6.0};
  constexpr double kCos[7] = {-1.0 / 87178291200.0, 1.0 / 479001600.0, -1.0 / 3628800.0,
                              1.0 / 40320.0,        -1.0 / 720.0,      1.0 / 24.0, -0.5};
#pragma unroll
  for (int i = 0; i < 6; ++i) s = fma(s, z, kSin[i]);
#pragma unroll
  for (int i = 0; i < 7; ++i) c = fma(c, z, kCos[i]);
  s = fma(s * z, r, r);
  c = fma(c, z, 1.0);
  const int q = static_cast<int>(static_cast<int64_t>(k) & 3);
  const double sn = q & 1 ? c : s, cs = q & 1 ? s : c, a = amplitude;
  const double sign_s = (q & 2) != 0 ? -a : a, sign_c = q == 1 || q == 2 ? -a : a;
  return make_float2(static_cast<float>(sign_c * cs),
                     static_cast<float>((inverse ? -sign_s : sign_s) * sn));
}

// x / d for x, d < 2^16 and m = ceil(2^32 / d): m d is less than d above 2^32, so that the
// product is off by less than x d / 2^32 < 1 / d of a quotient
__device__ __forceinline__ uint32_t div16(uint32_t x, uint32_t m) { return __umulhi(x, m); }

template <int V>
struct alignas(2 * V) RotaryUnit {
  uint16_t e[V];
};

template <typename T, int V, bool INTER>
__global__ __launch_bounds__(256) void k_rotary(RotaryArgs a) {
  typedef RotaryUnit<V> unit;
  static_assert(sizeof(unit) == 2 * V, "V elements");
  __shared__ float2 turns[kRotaryLds];
  const int n = a.pairs, H = a.num_q_heads + a.num_kv_heads;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * a.tokens;
  const int nt = static_cast<int>(min(static_cast<int64_t>(a.tokens), a.num_tokens - t0));
  for (int x = threadIdx.x; x < nt * n; x += 256) {
    const int tok = x / n, i = x - tok * n;
    const int64_t at = t0 + tok;
    const int64_t p = a.pos64 ? static_cast<const int64_t*>(a.positions)[at]
                              : static_cast<const int32_t*>(a.positions)[at];
    turns[x] = turn(p, a.frequencies[i], a.amplitude, a.inverse != 0);
  }
  __syncthreads();
  const uint32_t S = static_cast<uint32_t>(a.row_tasks), R = static_cast<uint32_t>(n / V);
  const uint32_t tasks = static_cast<uint32_t>(nt * H) * S;
  for (uint32_t x = blockIdx.y * 256u + threadIdx.x; x < tasks; x += 256u * gridDim.y) {
    const uint32_t row = S == 1 ? x : div16(x, a.div_tasks), c = x - row * S;
    const uint32_t tok = H == 1 ? row : div16(row, a.div_heads);
    const int h = static_cast<int>(row - tok * H);
    const bool is_q = h < a.num_q_heads;
    const int hh = is_q ? h : h - a.num_q_heads;
    const uint16_t* in = static_cast<const uint16_t*>(is_q ? a.q : a.k) +
                         (t0 + tok) * (is_q ? a.q_stride_tok : a.k_stride_tok) +
                         hh * (is_q ? a.q_stride_head : a.k_stride_head);
    uint16_t* out = static_cast<uint16_t*>(is_q ? a.q_out : a.k_out) +
                    (t0 + tok) * (is_q ? a.qo_stride_tok : a.ko_stride_tok) +
                    hh * (is_q ? a.qo_stride_head : a.ko_stride_head);
    const bool rotated = c < R;
    if (!rotated && in == out) continue;
    // (tasks past the pairs move 2 V of the other dims)
    const uint32_t lo = !rotated ? 2 * n + (c - R) * 2 * V : INTER ? 2 * V * c : V * c;
    const uint32_t hi = rotated && !INTER ? lo + n : lo + V;
    unit u = *reinterpret_cast<const unit*>(in + lo), v = *reinterpret_cast<const unit*>(in + hi);
    if (rotated) {
      const float2* tr = turns + tok * n + V * c;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        uint16_t& ux = !INTER ? u.e[e] : 2 * e < V ? u.e[(2 * e) % V] : v.e[(2 * e) % V];
        uint16_t& uy = !INTER ? v.e[e] : 2 * e + 1 < V ? u.e[(2 * e + 1) % V] : v.e[(2 * e + 1) % V];
        const float px = T::to_f32(ux), py = T::to_f32(uy);
        const float cs = tr[e].x, sn = tr[e].y;
        // (as written, and rounded to fp32 first, so that the bits do not depend on V)
        float rx = fmaf(px, cs, -(py * sn)), ry = fmaf(py, cs, px * sn);
        asm volatile("" : "+v"(rx), "+v"(ry));
        ux = T::from_f32(rx);
        uy = T::from_f32(ry);
      }
    }
    *reinterpret_cast<unit*>(out + lo) = u;
    *reinterpret_cast<unit*>(out + hi) = v;
  }
}

hipError_t launch_rotary(RotaryArgs a, int dtype, int v, hipStream_t s) {
  const int H = a.num_q_heads + a.num_kv_heads;
  if (a.num_tokens <= 0 || H <= 0) return hipSuccess;
  a.row_tasks = a.head_dim / (2 * v);
  // tokens of a workgroup: as many as give each thread a cosine, within 2^16 tasks
  int64_t tokens = std::max(1, 256 / std::max(1, a.pairs));
  tokens = std::min<int64_t>(tokens, std::max(1, 65535 / (H * a.row_tasks)));
  while (tokens > 1 && a.num_tokens / tokens < 1024) tokens /= 2;
  a.tokens = static_cast<int32_t>(tokens);
  const auto magic = [](int d) {
    return static_cast<uint32_t>(((uint64_t(1) << 32) + static_cast<uint32_t>(d) - 1) /
                                 static_cast<uint32_t>(d));
  };
  a.div_tasks = a.row_tasks > 1 ? magic(a.row_tasks) : 0;
  a.div_heads = H > 1 ? magic(H) : 0;
  const int64_t wgs = (a.num_tokens + tokens - 1) / tokens;
  // few tokens: workgroups share a token's heads, so that each makes one pass
  const int64_t passes = (tokens * H * a.row_tasks + 255) / 256;
  const dim3 g(static_cast<unsigned>(wgs), static_cast<unsigned>(wgs < 512 ? passes : 1)), b(256);
  const auto run = [&](auto t, auto vc) {
    using T = decltype(t);
    constexpr int V = decltype(vc)::value;
    if (a.interleaved) hipLaunchKernelGGL((k_rotary<T, V, true>), g, b, 0, s, a);
    else hipLaunchKernelGGL((k_rotary<T, V, false>), g, b, 0, s, a);
  };
  const auto typed = [&](auto vc) {
    if (dtype == FP_DTYPE_BF16) run(BF16{}, vc);
    else run(F16{}, vc);
  };
  if (v == 8) typed(IntC<8>{});
  else if (v == 4) typed(IntC<4>{});
  else if (v == 2) typed(IntC<2>{});
  else typed(IntC<1>{});
  return hipGetLastError();
}

}  // namespace fp

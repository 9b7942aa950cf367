// Attention over a paged KV cache of 8-bit floats: the 8-bit form of fp_paged.hip
// (the same rows, chunks, partials and merge; cached token k of sequence b holds
// c_k, c_v and stands for k = s_k c_k, v = s_v c_v, with scales s that are fixed
// for a KV head or kept for every (slot, head)).
//
//   S = scale s_k (q . c_k),  P = exp2(S - m),  O = sum P s_v c_v / sum P
//
// No cached value is rounded on the way: c converts exactly to the MFMA's 16-bit
// types, s_k multiplies the fp32 score, a fixed s_v the fp32 row at the end and one
// per slot the fp32 P of its key. P s_v enters P.V as bf16 parts (fp32's exponents,
// so nothing underflows) beside c_v as bf16, whatever the type of q.
#include "fp_float8.h"
#include "fp_paged_common.h"

namespace fp {

// x0, x1 as N bf16 parts that add up to them to 2^-(8 N + 1) (N = 3: exactly)
template <int N>
__device__ __forceinline__ void bf16_parts(float x0, float x1, uint32_t (&u)[N]) {
#pragma unroll
  for (int p = 0; p < N; ++p) {
    u[p] = pack2<BF16>(x0, x1);
    x0 -= __uint_as_float(u[p] << 16);
    x1 -= __uint_as_float(u[p] & 0xffff0000u);
  }
}

// Few rows: a workgroup takes (16 rows of a KV head's queries, KV head, chunk of
// keys), its four waves 32 keys in turn, straight from the pages into registers.
//
//   S^T (keys x rows) = K . Q^T on v_mfma_f32_16x16x32: a lane (r = l % 16,
//     g = l / 16) loads 16-byte pieces of key r, whose two halves are the operands
//     of two k-steps (dims 64 i + 16 g + 8 e .. of step 2 i + e, in Q as in K)
//   O^T (dims x rows) += V^T . P^T on the same: k index 8 g + 4 t + v is key
//     16 t + 4 g + v, so P stays in the lanes that hold it, and row m of MFMA e is
//     dim E m + e, byte e of the E = D / 16 bytes that lane m loads of each of its
//     8 keys: whole rows are loaded and nothing crosses lanes. v_perm pairs the
//     bytes of two keys, one conversion each makes them an operand word.
template <typename T, int F, int D, bool P16>
__global__ __launch_bounds__(256, D > 128 || !P16 ? 2 : 3) void k_paged8(Paged8Args pa) {
  constexpr int KS = D / 32;  // MFMA k-steps over the head dim
  constexpr int KP = D / 64;  // 16-byte pieces of a key per lane
  constexpr int E = D / 16;   // V bytes per lane and key
  constexpr int VW = E / 4;   // the same in words
  constexpr int OS = D + 4;   // padded row of the merge buffer (floats)
  constexpr int NP = 3;       // parts of P
  __shared__ float sm[4][16][OS];
  __shared__ float sml[4][16][2];
  const PagedArgs& a = pa.a;
  const int h = static_cast<int>(blockIdx.x % a.Hkv);
  const int64_t x = blockIdx.x / a.Hkv;
  const int c = static_cast<int>(blockIdx.y);
  const PagedTile tile = paged_find(a, 16, x, -1);
  if (tile.b < 0) return;
  const PagedSeq& sq = tile.s;
  const int nk = static_cast<int>(sq.nk), nq = sq.nq;
  const int k0 = c * tile.chunk;
  if (k0 >= nk && c > 0) return;
  const bool single = nk <= tile.chunk;
  const int k1 = min(k0 + tile.chunk, nk);
  const int t = threadIdx.x, lane = t & 63;
  const int w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int r16 = lane & 15, g = lane >> 4;

  // this lane's query row (B operand column) and its last visible key
  const int rr = tile.tl * 16 + r16;
  const bool rvalid = rr < nq * a.G;
  const int qi = rvalid ? rr / a.G : 0;
  const int lim = rvalid ? nk - nq + qi : nk - 1;
  typename T::vec8 qb[KS];
  {
    const uint16_t* qp = static_cast<const uint16_t*>(a.q) + (sq.q0 + qi) * a.qst +
                         static_cast<int64_t>(h * a.G + (rvalid ? rr % a.G : 0)) * a.qhs + 16 * g;
#pragma unroll
    for (int s = 0; s < KS; ++s)
      qb[s] = as_vec8<T>(rvalid ? ld16(qp + 64 * (s >> 1) + 8 * (s & 1)) : zero4());
  }

  f32x4 acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = f32x4{};
  float m_run = -INFINITY, l_part = 0.0f;
  bool bad = false;
  const int64_t row = static_cast<int64_t>(tile.b) * a.table_stride;
  const uint8_t* kc = static_cast<const uint8_t*>(a.kc) + static_cast<int64_t>(h) * a.kch;
  const uint8_t* vc = static_cast<const uint8_t*>(a.vc) + static_cast<int64_t>(h) * a.vch;
  const float* kss = pa.ks.p + h * pa.ks.sh;  // read when there is one per slot
  const float* vss = pa.vs.p + h * pa.vs.sh;
  const float scale = a.scale_log2 * fixed_scale(pa.ks, h);

  uint4 kf[2][KP];
  uint32_t vf[2][4][VW];
  float ksc[2][4], vsc[2][4];
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int v = 0; v < 4; ++v) ksc[j][v] = vsc[j][v] = 1.0f;
  // pages and in-page offsets of the two 16-key tiles from `base` (P16); a
  // tile past the sequence repeats the last one (its scores are masked)
  const int last16 = (nk - 1) & ~15;
  int64_t page[2] = {0, 0};
  int inpage[2] = {0, 0};
  auto lookup = [&](int base) {
    if constexpr (P16) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int tb = min(base + 16 * j, last16);
        page[j] = paged_page<true>(a, row, tb, bad);
        inpage[j] = a.bs_shift >= 0 ? tb & (a.bs - 1) : tb % a.bs;
      }
    }
  };
  auto load_scales = [&](float (&dst)[2][4], const CacheScales& cs, const float* sp, int base) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if constexpr (P16) {
        const float4 u = *reinterpret_cast<const float4*>(sp + page[j] * cs.sb + inpage[j] + 4 * g);
        dst[j][0] = u.x; dst[j][1] = u.y; dst[j][2] = u.z; dst[j][3] = u.w;
      } else {
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const int key = min(base + 16 * j + 4 * g + v, nk - 1);
          dst[j][v] = sp[paged_page<false>(a, row, key, bad) * cs.sb + key % a.bs];
        }
      }
    }
  };
  auto load_k = [&](int base) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint8_t* p;
      if constexpr (P16) {
        p = kc + page[j] * a.kcb + static_cast<int64_t>(inpage[j]) * a.kcs;
        p += static_cast<uint32_t>(r16 * static_cast<int>(a.kcs) + 16 * g);
      } else {
        const int key = min(base + 16 * j + r16, nk - 1);
        const int64_t pg = paged_page<false>(a, row, key, bad);
        p = kc + pg * a.kcb + static_cast<int64_t>(key % a.bs) * a.kcs + 16 * g;
      }
#pragma unroll
      for (int s = 0; s < KP; ++s) kf[j][s] = ld16(p + 64 * s);
    }
    if (pa.ks.slot) load_scales(ksc, pa.ks, kss, base);
  };
  auto load_v = [&](int base) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const uint8_t* p;
        if constexpr (P16) {
          p = vc + page[j] * a.vcb + static_cast<int64_t>(inpage[j] + v) * a.vcs;
          p += static_cast<uint32_t>(4 * g * static_cast<int>(a.vcs));
        } else {
          const int key = min(base + 16 * j + 4 * g + v, nk - 1);
          const int64_t pg = paged_page<false>(a, row, key, bad);
          p = vc + pg * a.vcb + static_cast<int64_t>(key % a.bs) * a.vcs;
        }
        p += E * r16;
        if constexpr (VW == 1) {
          vf[j][v][0] = *reinterpret_cast<const uint32_t*>(p);
        } else if constexpr (VW == 2) {
          const uint2 u = *reinterpret_cast<const uint2*>(p);
          vf[j][v][0] = u.x; vf[j][v][1] = u.y;
        } else {
          const uint4 u = ld16(p);
          vf[j][v][0] = u.x; vf[j][v][1] = u.y; vf[j][v][2] = u.z; vf[j][v][3] = u.w;
        }
      }
    if (pa.vs.slot) load_scales(vsc, pa.vs, vss, base);
  };

  int base = k0 + 32 * w;
  if (base < k1) {
    lookup(base);
    load_k(base);
    load_v(base);
  }
  for (; base < k1; base += 128) {
    const int next = base + 128;
    const bool more = next < k1;
    f32x4 s[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      s[j] = f32x4{};
#pragma unroll
      for (int i = 0; i < KP; ++i) {
        s[j] = mfma16(as_vec8<T>(widen8<T, F>(kf[j][i].x, kf[j][i].y)), qb[2 * i], s[j]);
        s[j] = mfma16(as_vec8<T>(widen8<T, F>(kf[j][i].z, kf[j][i].w)), qb[2 * i + 1], s[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int v = 0; v < 4; ++v) s[j][v] *= scale * ksc[j][v];
    // the next round's keys fly during this round's softmax and P.V
    if (more) {
      lookup(next);
      load_k(next);
    }
    if (base + 31 > nk - nq) {  // some row's causal limit or the end lies in this round
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const int key = base + 16 * j + 4 * g + v;
          if (key > lim) s[j][v] = -INFINITY;
          if (key >= nk) {  // slots past the end may hold anything
            vsc[j][v] = 0.0f;
#pragma unroll
            for (int q = 0; q < VW; ++q) vf[j][v][q] = 0u;
          }
        }
    }
    float mx = -INFINITY;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int v = 0; v < 4; ++v) mx = fmaxf(mx, s[j][v]);
    const float m_new = fmaxf(m_run, row4_max(mx));
    if (__ballot(m_new > m_run) != 0) {
      // rows with no visible key yet keep m = -inf: their factors are 0
      const float ms = m_new == -INFINITY ? 0.0f : m_new;
      const float alpha = __builtin_amdgcn_exp2f(m_run - ms);
      m_run = m_new;
      l_part *= alpha;
#pragma unroll
      for (int e = 0; e < E; ++e)
#pragma unroll
        for (int v = 0; v < 4; ++v) acc[e][v] *= alpha;
    }
    const float ms = m_run == -INFINITY ? 0.0f : m_run;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        s[j][v] = __builtin_amdgcn_exp2f(s[j][v] - ms);
        l_part += s[j][v];
        s[j][v] *= vsc[j][v];
      }
    uint32_t pw[4][NP];  // [keys 2 i, 2 i + 1 of this lane][part]
#pragma unroll
    for (int i = 0; i < 4; ++i)
      bf16_parts<NP>(s[i >> 1][2 * (i & 1)], s[i >> 1][2 * (i & 1) + 1], pw[i]);
    typename BF16::vec8 pb[NP];
#pragma unroll
    for (int p = 0; p < NP; ++p)
      pb[p] = as_vec8<BF16>(make_uint4(pw[0][p], pw[1][p], pw[2][p], pw[3][p]));
#pragma unroll
    for (int q = 0; q < VW; ++q) {
      uint32_t pr[4][2];  // bytes (a0 b0 a1 b1) and (a2 b2 a3 b3) of a pair of keys a, b
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t ka = vf[i >> 1][2 * (i & 1)][q], kb = vf[i >> 1][2 * (i & 1) + 1][q];
        pr[i][0] = __builtin_amdgcn_perm(kb, ka, 0x05010400u);
        pr[i][1] = __builtin_amdgcn_perm(kb, ka, 0x07030602u);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          u[i] = e & 1 ? widen2<BF16, F, true>(pr[i][e >> 1])
                       : widen2<BF16, F, false>(pr[i][e >> 1]);
        const auto va = as_vec8<BF16>(make_uint4(u[0], u[1], u[2], u[3]));
#pragma unroll
        for (int p = NP - 1; p >= 0; --p) acc[4 * q + e] = mfma16(va, pb[p], acc[4 * q + e]);
      }
    }
    if (more) load_v(next);
  }

  // O not finite: P.V again over the keys that each row sees (a masked key's infinite
  // or NaN value times P = 0 is NaN, and so is an infinite one times the parts of P),
  // with P and l 2^off times smaller (m larger), so that values near the largest do
  // not overflow before the division by l
  {
    float nf = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
      for (int v = 0; v < 4; ++v) nf = fmaf(acc[e][v], 0.0f, nf);
    if (__ballot(nf != 0.0f) != 0) {
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = f32x4{};
      const float off = static_cast<float>(32 - __clz(k1 - k0));
      m_run += off;
      l_part *= __builtin_amdgcn_exp2f(-off);
      const float ms = m_run == -INFINITY ? 0.0f : m_run;
      int lane2 = static_cast<int>(threadIdx.x);  // (formed here, not kept across the loop)
      asm volatile("" : "+v"(lane2));
      const int g2 = (lane2 >> 4) & 3;
#pragma unroll 1
      for (int i = 0; i < 32 * ((k1 - k0 + 127) / 128); ++i) {
        const int key = k0 + 32 * w + 128 * (i >> 5) + (i & 31);
        if (key >= k1) break;
        const int64_t pg = paged_page<true>(a, row, key, bad);
        const int in = key % a.bs;
        const uint8_t* kp = kc + pg * a.kcb + static_cast<int64_t>(in) * a.kcs + 16 * g2;
        const uint8_t* vp = vc + pg * a.vcb + static_cast<int64_t>(in) * a.vcs;
        float d = 0.0f;  // the lane's dims of q . c_k
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const uint2 u = *reinterpret_cast<const uint2*>(kp + 64 * (ks >> 1) + 8 * (ks & 1));
          const uint4 qu = __builtin_bit_cast(uint4, qb[ks]);
          const uint32_t qw[4] = {qu.x, qu.y, qu.z, qu.w};
          const f32x2 kv[4] = {
              Float8<F>::template to_f32<false>(u.x), Float8<F>::template to_f32<true>(u.x),
              Float8<F>::template to_f32<false>(u.y), Float8<F>::template to_f32<true>(u.y)};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            d = fmaf(T::to_f32(static_cast<uint16_t>(qw[e])), kv[e][0], d);
            d = fmaf(T::to_f32(static_cast<uint16_t>(qw[e] >> 16)), kv[e][1], d);
          }
        }
        d = row4_sum(d) * (pa.ks.slot ? scale * kss[pg * pa.ks.sb + in] : scale);
        if (key > lim) continue;
        float p = __builtin_amdgcn_exp2f(d - ms);
        if (pa.vs.slot) p *= vss[pg * pa.vs.sb + in];
#pragma unroll
        for (int v = 0; v < 4; ++v)
#pragma unroll
          for (int q = 0; q < VW; ++q) {
            const uint32_t u = *reinterpret_cast<const uint32_t*>(vp + E * (4 * g2 + v) + 4 * q);
            const f32x2 lo = Float8<F>::template to_f32<false>(u);
            const f32x2 hi = Float8<F>::template to_f32<true>(u);
            acc[4 * q][v] = fmaf(p, lo[0], acc[4 * q][v]);
            acc[4 * q + 1][v] = fmaf(p, lo[1], acc[4 * q + 1][v]);
            acc[4 * q + 2][v] = fmaf(p, hi[0], acc[4 * q + 2][v]);
            acc[4 * q + 3][v] = fmaf(p, hi[1], acc[4 * q + 3][v]);
          }
      }
    }
  }

  // acc[e][v] is dim E (4 g + v) + e of row r16
  float l = row4_sum(l_part);
  if (__ballot(bad) != 0) l = __uint_as_float(0x7fc00000u);
#pragma unroll
  for (int v = 0; v < 4; ++v)
#pragma unroll
    for (int e = 0; e < E; e += 4)
      *reinterpret_cast<float4*>(&sm[w][r16][E * (4 * g + v) + e]) =
          make_float4(acc[e][v], acc[e + 1][v], acc[e + 2][v], acc[e + 3][v]);
  if (g == 0) {
    sml[w][r16][0] = m_run;
    sml[w][r16][1] = l;
  }
  __syncthreads();
  const int orow = t >> 4, od = E * (t & 15);
  const int orr = tile.tl * 16 + orow;
  if (orr >= nq * a.G) return;
  const int64_t tok = sq.q0 + orr / a.G;
  const int hq = h * a.G + orr % a.G;
  float M = -INFINITY;
#pragma unroll
  for (int k = 0; k < 4; ++k) M = fmaxf(M, sml[k][orow][0]);
  float L = 0.0f, o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.0f;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float mk = sml[k][orow][0];
    // (a quarter each: four finite sums add up to a finite one)
    const float f = mk == -INFINITY ? 0.0f : 0.25f * __builtin_amdgcn_exp2f(mk - M);
    // (a wave without keys has m = -inf and l = 0; NaN scores leave m = -inf
    // with l = NaN, which the sum keeps)
    L += mk == -INFINITY ? sml[k][orow][1] : f * sml[k][orow][1];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] += f * sm[k][orow][od + e];
  }
  if (single) {
    uint16_t* op = static_cast<uint16_t*>(a.o) + tok * a.ost + static_cast<int64_t>(hq) * a.ohs + od;
    const float rcp = 1.0f / L, vs = fixed_scale(pa.vs, h);
    uint32_t pk[E / 2];
#pragma unroll
    for (int q = 0; q < E / 2; ++q) {
      float lo = o[2 * q] * rcp * vs, hi = o[2 * q + 1] * rcp * vs;
      if (nk == 0) lo = hi = sq.bad ? __uint_as_float(0x7fc00000u) : 0.0f;
      pk[q] = pack2<T>(lo, hi);
    }
#pragma unroll
    for (int q = 0; q < E / 2; q += 2)
      *reinterpret_cast<uint2*>(op + 2 * q) = make_uint2(pk[q], pk[q + 1]);
  } else {
    const int64_t slot = (tok * a.Hq + hq) * a.nc + c;
    float* pp = a.part + slot * D + od;
#pragma unroll
    for (int e = 0; e < E; e += 4)
      *reinterpret_cast<float4*>(pp + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
    if ((t & 15) == 0) {
      a.ml[2 * slot] = M;
      a.ml[2 * slot + 1] = L;
    }
  }
}

// Many rows (prefill over a cached prefix): k_paged_rows with tiles that are
// widened on their way into LDS. The 64 keys of a tile are loaded into registers
// (16 keys by each wave, a tile ahead), widened once per workgroup and written as
// 16-bit tiles, K in q's type and V in bf16; P s_v takes two bf16 parts: 2^-17 of
// each product, an eighth of what rounding the output to fp16 may lose and a 256th
// of its cached value's own step, where a third part would add half as many MFMAs
// to P.V again.
template <typename T, int F, int D, bool P16>
__global__ __launch_bounds__(256, 2) void k_paged8_rows(Paged8Args pa) {
  constexpr int KT = 64, TT = KT / 32;
  constexpr int KS = D / 16, DT = D / 32, CH = D / 8;
  constexpr int LPR = D / 16;        // lanes per key (16 bytes each)
  constexpr int NL = 16 * LPR / 64;  // load instructions per wave and tile
  constexpr int NP = 2;
  __shared__ uint4 sk[2][KT * CH];
  __shared__ uint4 sv[2][KT * CH];
  __shared__ float ssk[2][KT];  // scale * log2 e * s_k, and s_v (one per slot) or 1
  __shared__ float ssv[2][KT];
  __shared__ int s_bad;  // some wave looked up a page outside the cache
  const PagedArgs& a = pa.a;
  const int h = static_cast<int>(blockIdx.x % a.Hkv);
  const int64_t x = blockIdx.x / a.Hkv;
  const int c = static_cast<int>(blockIdx.y);
  const PagedTile tile = paged_find(a, 128, x, -1);
  if (tile.b < 0) return;
  const PagedSeq& sq = tile.s;
  const int nk = static_cast<int>(sq.nk), nq = sq.nq;
  const int k0 = c * tile.chunk;
  if (k0 >= nk && c > 0) return;
  const bool single = nk <= tile.chunk;
  const int t = threadIdx.x, lane = t & 63;
  const int w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int half = lane >> 5, l32 = lane & 31;
  const int rows = nq * a.G;

  // this lane's query row and its last visible key
  const int rr = tile.tl * 128 + 32 * w + l32;
  const bool rvalid = rr < rows;
  const int qi = (rvalid ? rr : rows - 1) / a.G;
  const int64_t tok = sq.q0 + qi;
  const int hq = h * a.G + (rvalid ? rr : rows - 1) % a.G;
  const int lim = nk - nq + qi;
  // the wave's first and last visible keys' bounds (wave-uniform)
  const int r0 = min(tile.tl * 128 + 32 * w, rows - 1);
  const int r1 = min(tile.tl * 128 + 32 * w + 31, rows - 1);
  const int lim_lo = __builtin_amdgcn_readfirstlane(nk - nq + r0 / a.G);
  const int lim_hi = __builtin_amdgcn_readfirstlane(nk - nq + r1 / a.G);
  // keys past the last row of the tile are visible to none of its rows
  const int last_row = min(tile.tl * 128 + 127, rows - 1);
  const int k1 = __builtin_amdgcn_readfirstlane(
      min(min(k0 + tile.chunk, nk), max(nk - nq + last_row / a.G + 1, 0)));

  typename T::vec8 qb[KS];
  {
    const uint16_t* qp = static_cast<const uint16_t*>(a.q) + tok * a.qst +
                         static_cast<int64_t>(hq) * a.qhs + 8 * half;
#pragma unroll
    for (int s = 0; s < KS; ++s) qb[s] = as_vec8<T>(rvalid ? ld16(qp + 16 * s) : zero4());
  }
  f32x16 o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) o[dt] = f32x16{};
  float m_run = -INFINITY, l_part = 0.0f;
  bool bad = false;

  const int64_t row = static_cast<int64_t>(tile.b) * a.table_stride;
  const uint8_t* kc = static_cast<const uint8_t*>(a.kc) + static_cast<int64_t>(h) * a.kch;
  const uint8_t* vc = static_cast<const uint8_t*>(a.vc) + static_cast<int64_t>(h) * a.vch;
  const float* kss = pa.ks.p + h * pa.ks.sh;  // read when there is one per slot
  const float* vss = pa.vs.p + h * pa.vs.sh;
  const float scale = a.scale_log2 * fixed_scale(pa.ks, h);

  // 16 bytes per lane of the wave's 16 keys, and lane 4 i's (P16: lane i's) scales
  uint4 kr[NL], vr[NL];
  float kscr = scale, vscr = 1.0f;
  const int last16 = (nk - 1) & ~15;
  // tile of keys base .. base + 63; keys past the sequence read its last 16-key
  // group (P16) or its last key
  auto load = [&](int base) {
    if constexpr (P16) {
      const int tb = min(base + 16 * w, last16);
      const int64_t pg = paged_page<true>(a, row, tb, bad);
      const int in = a.bs_shift >= 0 ? tb & (a.bs - 1) : tb % a.bs;
      const uint8_t* kp = kc + pg * a.kcb + static_cast<int64_t>(in) * a.kcs;
      const uint8_t* vp = vc + pg * a.vcb + static_cast<int64_t>(in) * a.vcs;
#pragma unroll
      for (int q = 0; q < NL; ++q) {
        const int r = q * (64 / LPR) + lane / LPR;
        kr[q] = ld16(kp + static_cast<uint32_t>(r * static_cast<int>(a.kcs) + 16 * (lane % LPR)));
        vr[q] = ld16(vp + static_cast<uint32_t>(r * static_cast<int>(a.vcs) + 16 * (lane % LPR)));
      }
      if (pa.ks.slot) kscr = scale * kss[pg * pa.ks.sb + in + (lane & 15)];
      if (pa.vs.slot) vscr = vss[pg * pa.vs.sb + in + (lane & 15)];
    } else {
#pragma unroll
      for (int q = 0; q < NL; ++q) {
        const int key = min(base + 16 * w + q * (64 / LPR) + lane / LPR, nk - 1);
        const int64_t pg = paged_page<false>(a, row, key, bad);
        const int64_t in = key % a.bs;
        kr[q] = ld16(kc + pg * a.kcb + in * a.kcs + 16 * (lane % LPR));
        vr[q] = ld16(vc + pg * a.vcb + in * a.vcs + 16 * (lane % LPR));
      }
      if (pa.ks.slot || pa.vs.slot) {
        const int key = min(base + 16 * w + (lane & 15), nk - 1);
        const int64_t pg = paged_page<false>(a, row, key, bad);
        if (pa.ks.slot) kscr = scale * kss[pg * pa.ks.sb + key % a.bs];
        if (pa.vs.slot) vscr = vss[pg * pa.vs.sb + key % a.bs];
      }
    }
  };
  // widened into buffer `buf`; V and its scales of slots past the sequence are 0
  // (they may hold anything)
  auto store = [&](int base, int buf) {
#pragma unroll
    for (int q = 0; q < NL; ++q) {
      const int r = 16 * w + q * (64 / LPR) + lane / LPR, ch = 2 * (lane % LPR);
      const uint4 u = kr[q], v = base + r < nk ? vr[q] : zero4();
      sk[buf][r * CH + (ch ^ swz<D>(r))] = widen8<T, F>(u.x, u.y);
      sk[buf][r * CH + ((ch + 1) ^ swz<D>(r))] = widen8<T, F>(u.z, u.w);
      sv[buf][r * CH + (ch ^ swz<D>(r))] = widen8<BF16, F>(v.x, v.y);
      sv[buf][r * CH + ((ch + 1) ^ swz<D>(r))] = widen8<BF16, F>(v.z, v.w);
    }
    if (lane < 16) {
      ssk[buf][16 * w + lane] = kscr;
      ssv[buf][16 * w + lane] = base + 16 * w + lane < nk ? vscr : 0.0f;
    }
  };
  const int g16 = lane >> 4, i16 = lane & 15;
  const int tr_row = 4 * (g16 >> 1) + (i16 >> 2);
  const int tr_col = 16 * (g16 & 1) + 4 * (i16 & 3);

  // (ordered before the flag by the barrier after the loop)
  if (t == 0) s_bad = 0;
  if (k0 < k1) {
    load(k0);
    store(k0, 0);
  }
  int buf = 0;
  for (int base = k0; base < k1; base += KT, buf ^= 1) {
    // this tile is in LDS for every wave, and every wave is done with the other buffer
    lds_barrier();
    const bool more = base + KT < k1;
    if (more) load(base + KT);
    if (base <= lim_hi) {  // (else no key of this tile is visible to the wave)
      f32x16 s[TT];
#pragma unroll
      for (int t4 = 0; t4 < TT; ++t4) s[t4] = f32x16{};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int t4 = 0; t4 < TT; ++t4) {
          const int r = 32 * t4 + l32;
          const uint4 kop = sk[buf][r * CH + ((2 * ks + half) ^ swz<D>(r))];
          s[t4] = T::mfma32(as_vec8<T>(kop), qb[ks], s[t4]);
        }
      const bool edge = base + KT - 1 > lim_lo;
      float mx = -INFINITY;
#pragma unroll
      for (int t4 = 0; t4 < TT; ++t4)
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4) {
          const float4 f = *reinterpret_cast<const float4*>(&ssk[buf][32 * t4 + 8 * g4 + 4 * half]);
          const float fe[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float y = s[t4][4 * g4 + e] * fe[e];
            if (edge && base + 32 * t4 + 8 * g4 + 4 * half + e > lim) y = -INFINITY;
            s[t4][4 * g4 + e] = y;
            mx = fmaxf(mx, y);
          }
        }
      const float m_new = fmaxf(m_run, pair32_max(mx));
      if (__ballot(m_new > m_run) != 0) {
        const float ms = m_new == -INFINITY ? 0.0f : m_new;
        const float alpha = __builtin_amdgcn_exp2f(m_run - ms);
        m_run = m_new;
        l_part *= alpha;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int v = 0; v < 16; ++v) o[dt][v] *= alpha;
      }
      // rows with no visible key yet keep m = -inf: their P is 0
      const float ms = m_run == -INFINITY ? 0.0f : m_run;
#pragma unroll
      for (int t4 = 0; t4 < TT; ++t4) {
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          s[t4][v] = __builtin_amdgcn_exp2f(s[t4][v] - ms);
          l_part += s[t4][v];
        }
        if (pa.vs.slot) {
#pragma unroll
          for (int g4 = 0; g4 < 4; ++g4) {
            const float4 f =
                *reinterpret_cast<const float4*>(&ssv[buf][32 * t4 + 8 * g4 + 4 * half]);
            s[t4][4 * g4] *= f.x;
            s[t4][4 * g4 + 1] *= f.y;
            s[t4][4 * g4 + 2] *= f.z;
            s[t4][4 * g4 + 3] *= f.w;
          }
        }
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          uint32_t u[4][NP];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            bf16_parts<NP>(s[t4][8 * hh + 2 * e], s[t4][8 * hh + 2 * e + 1], u[e]);
          typename BF16::vec8 pb[NP];
#pragma unroll
          for (int p = 0; p < NP; ++p)
            pb[p] = as_vec8<BF16>(make_uint4(u[0][p], u[1][p], u[2][p], u[3][p]));
          const uint16_t* sv16 = reinterpret_cast<const uint16_t*>(sv[buf]);
          const int r = 32 * t4 + 16 * hh + tr_row;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) {
            const auto va = read_vt<BF16, D>(sv16, r, 32 * dt + tr_col);
#pragma unroll
            for (int p = NP - 1; p >= 0; --p) o[dt] = BF16::mfma32(va, pb[p], o[dt]);
          }
        }
      }
    }
    if (more) store(base + KT, buf ^ 1);
  }

  // Rows whose O is not finite take P.V again in fp32 with P whole, over the keys that
  // each row sees: an infinite or NaN value times the parts of P is NaN where its
  // product with P is not, and sums of values near the largest overflow before they
  // are divided by l.
  float nf = 0.0f;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int v = 0; v < 16; ++v) nf = fmaf(o[dt][v], 0.0f, nf);
  if (__ballot(nf != 0.0f) != 0) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] = f32x16{};
    // P and l 2^off times smaller (m larger): the sum of P V then stays below the
    // largest value, as that of normalised weights does
    const float off = static_cast<float>(32 - __clz(k1 - k0));
    m_run += off;
    l_part *= __builtin_amdgcn_exp2f(-off);
    const float ms = m_run == -INFINITY ? 0.0f : m_run;
    int half2 = static_cast<int>(threadIdx.x);  // (formed here, not kept across the loop)
    asm volatile("" : "+v"(half2));
    half2 = (half2 >> 5) & 1;
#pragma unroll 1
    for (int key = k0; key < k1; ++key) {
      const int64_t pg = paged_page<true>(a, row, key, bad);
      const int in = key % a.bs;
      const uint8_t* kp = kc + pg * a.kcb + static_cast<int64_t>(in) * a.kcs + 8 * half2;
      const uint8_t* vp = vc + pg * a.vcb + static_cast<int64_t>(in) * a.vcs + 4 * half2;
      float d = 0.0f;  // the lane's dims of q . c_k
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const uint2 u = *reinterpret_cast<const uint2*>(kp + 16 * s);
        const uint4 qu = __builtin_bit_cast(uint4, qb[s]);
        const uint32_t qw[4] = {qu.x, qu.y, qu.z, qu.w};
        const f32x2 kv[4] = {
            Float8<F>::template to_f32<false>(u.x), Float8<F>::template to_f32<true>(u.x),
            Float8<F>::template to_f32<false>(u.y), Float8<F>::template to_f32<true>(u.y)};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          d = fmaf(T::to_f32(static_cast<uint16_t>(qw[e])), kv[e][0], d);
          d = fmaf(T::to_f32(static_cast<uint16_t>(qw[e] >> 16)), kv[e][1], d);
        }
      }
      d = pair32_sum(d) * (pa.ks.slot ? scale * kss[pg * pa.ks.sb + in] : scale);
      if (key > lim) continue;
      float p = __builtin_amdgcn_exp2f(d - ms);
      if (pa.vs.slot) p *= vss[pg * pa.vs.sb + in];
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4) {
          const uint32_t u = *reinterpret_cast<const uint32_t*>(vp + 32 * dt + 8 * g4);
          const f32x2 lo = Float8<F>::template to_f32<false>(u);
          const f32x2 hi = Float8<F>::template to_f32<true>(u);
          o[dt][4 * g4] = fmaf(p, lo[0], o[dt][4 * g4]);
          o[dt][4 * g4 + 1] = fmaf(p, lo[1], o[dt][4 * g4 + 1]);
          o[dt][4 * g4 + 2] = fmaf(p, hi[0], o[dt][4 * g4 + 2]);
          o[dt][4 * g4 + 3] = fmaf(p, hi[1], o[dt][4 * g4 + 3]);
        }
    }
  }

  // A wave looks up the pages of its 16 keys of a tile only, and all four use the
  // tile: a bad page found by one makes the rows of all four NaN.
  float l = pair32_sum(l_part);
  lds_barrier();
  if (bad) s_bad = 1;
  lds_barrier();
  if (s_bad != 0) l = __uint_as_float(0x7fc00000u);
  if (!rvalid) return;
  if (single) {
    const float rcp = 1.0f / l, vs = fixed_scale(pa.vs, h);
    uint16_t* op = static_cast<uint16_t*>(a.o) + tok * a.ost + static_cast<int64_t>(hq) * a.ohs;
    const float nan = __uint_as_float(0x7fc00000u);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int g4 = 0; g4 < 4; ++g4) {
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          y[e] = o[dt][4 * g4 + e] * rcp * vs;
          if (nk == 0) y[e] = sq.bad ? nan : 0.0f;
        }
        *reinterpret_cast<uint2*>(op + 32 * dt + 8 * g4 + 4 * half) =
            make_uint2(pack2<T>(y[0], y[1]), pack2<T>(y[2], y[3]));
      }
  } else {
    const int64_t slot = (tok * a.Hq + hq) * a.nc + c;
    float* pp = a.part + slot * D;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int g4 = 0; g4 < 4; ++g4)
        *reinterpret_cast<float4*>(pp + 32 * dt + 8 * g4 + 4 * half) =
            make_float4(o[dt][4 * g4], o[dt][4 * g4 + 1], o[dt][4 * g4 + 2], o[dt][4 * g4 + 3]);
    if (half == 0) {
      a.ml[2 * slot] = m_run;
      a.ml[2 * slot + 1] = l;
    }
  }
}

template <typename T, int F, int D>
hipError_t launch_paged8_t(const Paged8Args& p, bool rows, int64_t tiles, hipStream_t s) {
  const PagedArgs& a = p.a;
  const dim3 grid(static_cast<unsigned>(tiles * a.Hkv), static_cast<unsigned>(a.nc));
  const bool p16 = a.bs % 16 == 0;
  if constexpr (D <= 128) {
    if (rows) {
      if (p16) hipLaunchKernelGGL((k_paged8_rows<T, F, D, true>), grid, dim3(256), 0, s, p);
      else hipLaunchKernelGGL((k_paged8_rows<T, F, D, false>), grid, dim3(256), 0, s, p);
      return hipGetLastError();
    }
  }
  if (p16) hipLaunchKernelGGL((k_paged8<T, F, D, true>), grid, dim3(256), 0, s, p);
  else hipLaunchKernelGGL((k_paged8<T, F, D, false>), grid, dim3(256), 0, s, p);
  return hipGetLastError();
}

template <typename T, int F>
hipError_t launch_paged8_d(const Paged8Args& p, int head_dim, bool rows, int64_t tiles,
                           hipStream_t s) {
  return with_head_dim(head_dim, [&](auto dc) {
    return launch_paged8_t<T, F, decltype(dc)::value>(p, rows, tiles, s);
  });
}

hipError_t launch_paged8(const Paged8Args& p, int dtype, int format, int head_dim, bool rows,
                         int64_t tiles, hipStream_t s) {
  const bool bf = dtype == FP_DTYPE_BF16;
  hipError_t e;
  if (format == FP_CACHE_E4M3)
    e = bf ? launch_paged8_d<BF16, FP_CACHE_E4M3>(p, head_dim, rows, tiles, s)
           : launch_paged8_d<F16, FP_CACHE_E4M3>(p, head_dim, rows, tiles, s);
  else
    e = bf ? launch_paged8_d<BF16, FP_CACHE_E5M2>(p, head_dim, rows, tiles, s)
           : launch_paged8_d<F16, FP_CACHE_E5M2>(p, head_dim, rows, tiles, s);
  if (e != hipSuccess || p.a.nc <= 1) return e;
  return launch_paged_merge(p.a, dtype, head_dim, rows, s);
}

}  // namespace fp

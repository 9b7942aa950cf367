// Attention over a paged KV cache of 4-bit integers: the 4-bit form of fp_paged8.hip (the
// same rows, shares, partials and merges). Cached element x of a key or value is
// s (c + z) t: exactly an fp16 number u = s (c + z) (fp_int4.h) times the KV head's scale.
//
//   S = scale t_k (q . u_k),  P = exp2(S - m),  O = t_v sum P u_v / sum P
//
// No cached value is rounded on the way: u enters v_mfma_f32_*_f16 as it is, whatever the
// type of q. bf16 queries become fp16 ones times a power of two f that takes their row's
// largest finite element to 2^13 .. 2^14: exactly, but for elements below 2^-39 of it,
// whose last bits fp16's subnormals lose. P enters as P 2^15 (many rows: up to P 2^15) in two
// fp16 parts, the second of what the first lost: all but 2^-22 of it, and 2^-25 of the
// factored P where the parts are subnormal. (One part would be off by up to 2^-11, as much as
// an fp16 output's rounding.)
#include "fp_int4.h"
#include "fp_paged_segments.h"

namespace fp {

constexpr float kPScale = 15.0f;  // few rows: log2 of the factor of P

// 8 elements of a query row, dims 0 .. 7 as fp16 numbers in the order {0, 2, 1, 3, 4, 6, 5,
// 7} of a key's piece (piece_group), times f
__device__ __forceinline__ uint4 query8(uint4 x, bool bf, float f) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  if (!bf && f > 0.0f) {
    return make_uint4(halves<0>(w[0], w[1]), halves<1>(w[0], w[1]), halves<0>(w[2], w[3]),
                      halves<1>(w[2], w[3]));
  }
  float y[8];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    y[2 * e] = f * (bf ? __uint_as_float(w[e] << 16) : F16::to_f32(static_cast<uint16_t>(w[e])));
    y[2 * e + 1] = f * (bf ? __uint_as_float(w[e] & 0xffff0000u)
                           : F16::to_f32(static_cast<uint16_t>(w[e] >> 16)));
  }
  return make_uint4(pack2<F16>(y[0], y[2]), pack2<F16>(y[1], y[3]), pack2<F16>(y[4], y[6]),
                    pack2<F16>(y[5], y[7]));
}
// Exponent fields of 8 bf16 elements, in both halves: one more than the largest that is not
// infinite or NaN (those wrap to the smallest 16-bit integer), and than m's
typedef short i16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ i16x2 exponents8(uint4 x, i16x2 m) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const i16x2 f = __builtin_bit_cast(i16x2, w[e] & 0x7f807f80u) + i16x2{0x80, 0x80};
    m = __builtin_elementwise_max(m, f);
  }
  return m;
}
// log2 of a bf16 row's factor, from its lanes' exponents; rows below 2^-106 keep that of
// 2^-106
__device__ __forceinline__ int row_exponent(i16x2 m) { return (max(m.x, m.y) >> 7) - 1; }
__device__ __forceinline__ int factor_exponent(int biased) { return 13 - max(biased - 127, -106); }
__device__ __forceinline__ uint32_t round2(float a, float b, bool bf) {
  return bf ? pack2<BF16>(a, b) : pack2<F16>(a, b);
}

// Two numbers as fp16 ones, hi, and what those lost, lo. minus_one: -1 that the compiler does
// not see, so that x - hi is one instruction that converts.
struct F16Parts {
  uint32_t hi, lo;
};
__device__ __forceinline__ F16Parts f16_parts(float x0, float x1, float minus_one) {
  const uint32_t hi = pack2<F16>(x0, x1);
  const f16x2 h = __builtin_bit_cast(f16x2, hi);
  return F16Parts{hi, pack2<F16>(fmaf(static_cast<float>(h[0]), minus_one, x0),
                                 fmaf(static_cast<float>(h[1]), minus_one, x1))};
}
__device__ __forceinline__ float opaque(float x) {
  asm volatile("" : "+s"(x));
  return x;
}

// a key's dot product with a lane's share of a query row: groups of a piece, in fp32
template <int NB>
__device__ __forceinline__ float piece_dot(const uint32_t (&w)[NB], const uint32_t (&gw)[NB / 2],
                                           const f16x8 (&q)[NB], const Int4Consts& k) {
  float d = 0.0f;
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const f16x8 u = as_vec8<F16>(piece_group<NB>(w, gw, j, k));
#pragma unroll
    for (int e = 0; e < 8; ++e)
      d = fmaf(static_cast<float>(q[j][e]), static_cast<float>(u[e]), d);
  }
  return d;
}

// ---------------------------------------------------------------------------
// Few rows
// ---------------------------------------------------------------------------
// What a wave's lanes pass each other through LDS: its LDS operations are carried out in
// their order, so that only the compiler has to keep it.
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}
__device__ __forceinline__ void put(uint2* p, const Step2& s) {
  *p = make_uint2(__builtin_bit_cast(uint32_t, s.s), __builtin_bit_cast(uint32_t, s.off));
}
__device__ __forceinline__ void get2(const uint2* p, Step2& a, Step2& b) {
  const uint4 x = *reinterpret_cast<const uint4*>(p);
  a = Step2{__builtin_bit_cast(f16x2, x.x), __builtin_bit_cast(f16x2, x.y)};
  b = Step2{__builtin_bit_cast(f16x2, x.z), __builtin_bit_cast(f16x2, x.w)};
}

// As k_paged8: four waves take 32 keys in turn, a round ahead of their use, straight from
// the pages into registers.
//
//   S^T (keys x rows) = K . Q^T on v_mfma_f32_16x16x32_f16: lane (r = l % 16, g = l / 16)
//     loads piece g of key r, whose group j is the operand of k-step j
//   O^T (dims x rows) += V^T . P^T: k index 8 g + 4 t + v is key 16 t + 4 g + v, row m of
//     MFMA 2 j + p is dim 32 j + 2 m + p, nibble p of byte j of the D / 32 that lane m
//     loads of each of its 8 keys
//
// HP: KV heads of a segment, each served by 4 / HP waves, so that whole cache lines are
// one segment's.
//
// Latency and bytes in flight bound it: 32 sequences of 300 .. 15,000 tokens, 8 KV heads of 128
// (252 MB), take 63 us, 4.0 TB/s, and the merge 6. 16 of the 63 pass without any keys (the
// search, the first page and key, the partials), the loads alone take 43 .. 50 beyond them
// and the arithmetic alone 33 .. 36 with P in one part; its second part is 1 to 2 us of the 63
// (5 in kernels that run apart from each other, at lower clocks).
//
// P16: the page size is a multiple of 16, so a 16-key tile lies in one page: a wave looks
// up 64 of them at a time, one per lane, and reads a tile's place from its lane. Other
// pages look up every key's.
template <int D, bool P16, int HP>
__global__ __launch_bounds__(256, D == 256 ? 2 : 3) void k_paged4(Paged4Args pa4) {
  constexpr int NB = D / 32;  // groups, MFMA k-steps over the head dim
  constexpr int GW = NB / 2;  // words of 32 bits of a key's groups
  constexpr int KG = NB == 8 ? 2 : 1;  // groups of a key that a lane makes steps of
  constexpr int TR = 2;                // 16-key tiles of a wave's round
  constexpr int VG = TR * NB >= 8 ? TR * NB / 8 : 1;  // groups of a pair of keys that a lane makes steps of
  constexpr int VL = NB / VG;          // lanes for a pair
  constexpr int E = D / 16;
  constexpr int VW = NB < 4 ? 1 : NB / 4;  // words of 32 bits of V's bytes per lane and key
  constexpr int OS = D + 4;   // padded row of the merge buffer (floats)
  constexpr int NW = 4 / HP;  // waves of a head
  constexpr int RK = 16 * TR * NW;  // keys of a round, all waves of a head
  __shared__ float sm[4][16][OS];
  __shared__ float sml[4][16][2];
  // a round's steps: of key r of tile j, of the keys 2 i, 2 i + 1 that a row of 16 lanes
  // multiplies (s of both, (z - 16) s of both)
  __shared__ __align__(16) uint2 ksteps[4][TR][16][NB];
  __shared__ __align__(16) uint2 vsteps[4][4][2 * TR][NB];
  const Paged8Args& pa = pa4.p;
  const PagedArgs& a = pa.a;
  const Work work = find_work(pa, static_cast<int>(blockIdx.x), -1);
  if (work.b < 0) return;
  const Int4Consts k4;
  const float minus_one = opaque(-1.0f);
  const bool bf = pa4.dtype == FP_DTYPE_BF16;
  const int t = threadIdx.x, lane = t & 63;
  const int w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int hw = w / NW, kw = w % NW;  // the wave's head of the segment, and its turn
  const int r16 = lane & 15, g = lane >> 4;
  int b = work.b;
  PagedSeq sq = work.s;
  const int start = static_cast<int>(blockIdx.x) * work.share;
  int left = min(work.share, work.total - start);
  int tiles = seq_tiles(a, sq), units = seq_units(pa.unit, sq);
  int seg = __builtin_amdgcn_readfirstlane((start - work.units) / units);
  int u = start - work.units - seg * units;
  for (bool first = true;; first = false) {
    const int hg = __builtin_amdgcn_readfirstlane(seg / tiles), tl = seg - hg * tiles;
    const int h = hg * HP + hw;
    const int take = min(units - u, left);
    const bool single = take == units;
    const int nk = static_cast<int>(sq.nk), nq = sq.nq;
    const int k0 = u * pa.unit;
    const int k1 = single ? nk : min(k0 + take * pa.unit, nk);

    // this lane's query row (B operand column), its factor and its last visible key
    const int rr = tl * 16 + r16;
    const bool rvalid = rr < nq * a.G;
    const int qi = rvalid ? rr / a.G : 0;
    const int lim = rvalid ? nk - nq + qi : nk - 1;
    uint4 qx[NB];  // (made fp16 numbers once the first keys are on their way)
    {
      const uint16_t* qp = static_cast<const uint16_t*>(a.q) + (sq.q0 + qi) * a.qst +
                           static_cast<int64_t>(h * a.G + (rvalid ? rr % a.G : 0)) * a.qhs + 8 * g;
#pragma unroll
      for (int j = 0; j < NB; ++j) qx[j] = ld16(qp + 32 * j);
    }

    f16x8 qb[NB];
    float scale = a.scale_log2 * fixed_scale(pa.ks, h);
    auto make_q = [&]() {
#pragma unroll
      for (int j = 0; j < NB; ++j) qx[j] = rvalid ? qx[j] : zero4();
      float f = 1.0f;
      if (scale < 0.0f) {  // (the sign goes into q, so that the largest score is the largest S)
        f = -1.0f;
        scale = -scale;
      }
      if (bf) {
        i16x2 most{};
#pragma unroll
        for (int j = 0; j < NB; ++j) most = exponents8(qx[j], most);
        // (as floats: small integers)
        const int e = factor_exponent(
            static_cast<int>(row4_max(static_cast<float>(row_exponent(most)))));
        f = __builtin_amdgcn_ldexpf(f, e);
        scale *= __builtin_amdgcn_ldexpf(1.0f, -e);
      }
      // (not 0, by which a masked score would be NaN: by 2^-149 no score reaches 2^-100)
      if (scale == 0.0f) scale = 0x1p-149f;
#pragma unroll
      for (int j = 0; j < NB; ++j) qb[j] = as_vec8<F16>(query8(qx[j], bf, f));
    };
    if constexpr (D == 256) make_q();  // (no registers to hold them in)
    f32x4 acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = f32x4{};
    float m_run = -INFINITY, l_part = 0.0f;
    bool bad = false;
    const int64_t row = static_cast<int64_t>(b) * a.table_stride;
    const uint8_t* kc = static_cast<const uint8_t*>(a.kc) + static_cast<int64_t>(h) * a.kch;
    const uint8_t* vc = static_cast<const uint8_t*>(a.vc) + static_cast<int64_t>(h) * a.vch;
    const uint16_t* kg = pa4.kg.p + h * pa4.kg.sh;
    const uint16_t* vg = pa4.vg.p + h * pa4.vg.sh;

    // what a round loads: 32 keys, lanes as above. A lane takes the words of its share of
    // the groups only (kj .. of key r, vj .. of the pair of keys vi of its row of 16 lanes)
    // and passes their steps to the others through LDS: each for itself needs five
    // instructions for every group of every key, a quarter of the loop's.
    struct {
      uint32_t k[TR][NB], kg[TR];
      uint32_t v[TR][4][VW], vg[2];  // (vg: of a key and the next, combined when they are used)
    } r;
    const int kj = KG * g & (NB - 1);
    const int vi = r16 / VL % (2 * TR), vj = VG * (r16 % VL);
    const int vkey = 16 * (vi >> 1) + 4 * g + 2 * (vi & 1);  // of the round
    // places of the 64 16-key tiles from key `win`, one per lane (P16; tiles past the
    // sequence repeat the last one, their scores are masked)
    int win = k0;
    int64_t kat = 0, vat = 0, kgat = 0, vgat = 0;
    const int last16 = (nk - 1) & ~15;
    auto look = [&](int from) {
      win = from;
      const int key = min(from + 16 * lane, last16);
      const int64_t pg = paged_page<false>(a, row, key, bad);
      const int in = a.bs_shift >= 0 ? key & (a.bs - 1) : key % a.bs;
      kat = pg * a.kcb + in * a.kcs;
      vat = pg * a.vcb + in * a.vcs;
      kgat = pg * pa4.kg.sb + in * NB;
      vgat = pg * pa4.vg.sb + in * NB;
    };
    auto place = [&](int64_t x, int tile) {
      return static_cast<int64_t>(
          static_cast<uint64_t>(static_cast<uint32_t>(
              __builtin_amdgcn_readlane(static_cast<int>(x >> 32), tile))) << 32 |
          static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(x), tile)));
    };
    // A scalar base that the compiler does not take apart: with it a load takes a 32-bit offset
    // of the lane's; else the loop holds 64-bit sums of the heads' bases and the offsets, and
    // adds tiles' places to them (11 instructions and 20 registers).
    auto at_tile = [&](const auto* head, int64_t x, int tile) {
      auto p = in_global(head + place(x, tile));
      asm volatile("" : "+s"(p));
      return p;
    };
    // a lane's offsets in a tile
    const uint32_t koff = static_cast<uint32_t>(r16 * static_cast<int>(a.kcs) + 4 * NB * g);
    const uint32_t kgoff = static_cast<uint32_t>(r16 * NB + kj);
    uint32_t voff[4];
#pragma unroll
    for (int v = 0; v < 4; ++v)
      voff[v] = static_cast<uint32_t>((4 * g + v) * static_cast<int>(a.vcs) + NB * r16);
    auto load_group = [&](auto p, uint32_t& x, auto n) {
      if constexpr (decltype(n)::value == 2) {
        uint32_t y[1];
        load32<1>(p, y);
        x = y[0];
      } else {
        x = *(gwords)(p);
      }
    };
    auto load_k = [&](int base) {
      if constexpr (P16) {
        if (base >= win + 1024) look(k0 + ((base - k0) & ~1023));
      }
#pragma unroll
      for (int j = 0; j < TR; ++j) {
        if constexpr (P16) {
          const int tile = ((base - win) >> 4) + j;
          load_piece<NB>(at_tile(kc, kat, tile) + koff, r.k[j]);
          load_group(at_tile(kg, kgat, tile) + kgoff, r.kg[j], IntC<KG>{});
        } else {
          const int key = min(base + 16 * j + r16, nk - 1);
          const int64_t pg = paged_page<false>(a, row, key, bad);
          const int in = key % a.bs;
          load_piece<NB>(kc + pg * a.kcb + static_cast<int64_t>(in) * a.kcs + 4 * NB * g, r.k[j]);
          load_group(kg + pg * pa4.kg.sb + static_cast<int64_t>(in) * NB + kj, r.kg[j], IntC<KG>{});
        }
      }
    };
    auto load_v = [&](int base) {
#pragma unroll
      for (int j = 0; j < TR; ++j) {
        const int tile = ((base - win) >> 4) + j;
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          gbytes p;
          if constexpr (P16) {
            p = at_tile(vc, vat, tile) + voff[v];
          } else {
            const int key = min(base + 16 * j + 4 * g + v, nk - 1);
            const int64_t pg = paged_page<false>(a, row, key, bad);
            const int in = key % a.bs;
            p = in_global(vc + pg * a.vcb + static_cast<int64_t>(in) * a.vcs + NB * r16);
          }
          if constexpr (NB == 2) r.v[j][v][0] = *(gwords)(p);
          else load32<VW>(p, r.v[j][v]);
        }
      }
      // (two keys, vkey and the next, in the halves of a word for each group)
      const uint16_t* w0;
      const uint16_t* w1;
      if constexpr (P16) {
        const int64_t at = shfl64(vgat, ((base - win) >> 4) + (vi >> 1));
        w0 = vg + at + ((vkey & 15) * NB + vj);
        w1 = w0 + NB;
      } else {
        const int key0 = min(base + vkey, nk - 1), key1 = min(base + vkey + 1, nk - 1);
        w0 = vg + paged_page<false>(a, row, key0, bad) * pa4.vg.sb +
             static_cast<int64_t>(key0 % a.bs) * NB + vj;
        w1 = vg + paged_page<false>(a, row, key1, bad) * pa4.vg.sb +
             static_cast<int64_t>(key1 % a.bs) * NB + vj;
      }
      load_group(w0, r.vg[0], IntC<VG>{});
      load_group(w1, r.vg[1], IntC<VG>{});
    };
    int base = k0 + 16 * TR * kw;
    if (base < k1) {
      if constexpr (P16) look(k0);
      load_k(base);
      load_v(base);
    }
    // what comes behind this sequence, on its way too
    const bool on = left > take, last_seg = seg + 1 == tiles * pa.groups;
    PagedSeq next = sq;
    if constexpr (D < 256) {
      if (on && last_seg) next = paged_seq(a, b + 1);
    }
    if constexpr (D < 256) make_q();
    f32x4 s[TR];
    auto scores = [&]() {
#pragma unroll
      for (int j = 0; j < TR; ++j) {
        put(&ksteps[w][j][r16][kj], steps(halves<0>(r.kg[j], r.kg[j]), k4));
        if constexpr (KG == 2)
          put(&ksteps[w][j][r16][kj + 1], steps(halves<1>(r.kg[j], r.kg[j]), k4));
      }
      wave_fence();
#pragma unroll
      for (int j = 0; j < TR; ++j) {
        Step2 st[NB];
#pragma unroll
        for (int i = 0; i < NB; i += 2) get2(&ksteps[w][j][r16][i], st[i], st[i + 1]);
        s[j] = f32x4{};
#pragma unroll
        for (int i = 0; i < NB; ++i)
          s[j] = mfma16(as_vec8<F16>(piece_group<NB>(r.k[j], st[i], i, k4)), qb[i], s[j]);
      }
      wave_fence();
    };
    auto softmax_pv = [&](int base) {
      if (base + 16 * TR - 1 > nk - nq) {  // some row's causal limit or the end lies in this round
        asm volatile("");  // (a branch: as selects they would be in every round)
#pragma unroll
        for (int j = 0; j < TR; ++j)
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const int key = base + 16 * j + 4 * g + v;
            if (key > lim) s[j][v] = -INFINITY;
          }
        // slots past the end may hold anything: a step of 0
        if (base + vkey >= nk) r.vg[0] = 0u;
        if (base + vkey + 1 >= nk) r.vg[1] = 0u;
      }
      put(&vsteps[w][g][vi][vj], steps(halves<0>(r.vg[0], r.vg[1]), k4));
      if constexpr (VG == 2)
        put(&vsteps[w][g][vi][vj + 1], steps(halves<1>(r.vg[0], r.vg[1]), k4));
      wave_fence();
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < TR; ++j)
#pragma unroll
        for (int v = 0; v < 4; ++v) mx = fmaxf(mx, s[j][v]);
      const float m_new = fmaxf(m_run, row4_max(mx) * scale);
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
      const float ms = m_run == -INFINITY ? 0.0f : m_run - kPScale;
#pragma unroll
      for (int j = 0; j < TR; ++j)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          s[j][v] = __builtin_amdgcn_exp2f(fmaf(s[j][v], scale, -ms));
          l_part += s[j][v];
        }
#pragma unroll
      for (int jj = 0; jj < TR; jj += 2) {  // 32 keys
        F16Parts pw[4];  // keys 2 i, 2 i + 1 of this lane
#pragma unroll
        for (int i = 0; i < 4; ++i)
          pw[i] = f16_parts(s[jj + (i >> 1)][2 * (i & 1)], s[jj + (i >> 1)][2 * (i & 1) + 1],
                            minus_one);
        const f16x8 ph = as_vec8<F16>(make_uint4(pw[0].hi, pw[1].hi, pw[2].hi, pw[3].hi));
        const f16x8 pl = as_vec8<F16>(make_uint4(pw[0].lo, pw[1].lo, pw[2].lo, pw[3].lo));
#pragma unroll
        for (int q = 0; q < GW; ++q) {  // groups 2 q and 2 q + 1
          uint32_t hv[4];
          Step2 st[2][4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {  // a pair of keys
            const int jt = jj + (i >> 1), va = 2 * (i & 1);
            const uint32_t xa = r.v[jt][va][q >> 1], xb = r.v[jt][va + 1][q >> 1];
            hv[i] = q & 1 ? halves<1>(xa, xb) : halves<0>(xa, xb);
            get2(&vsteps[w][g][2 * jj + i][2 * q], st[0][i], st[1][i]);
          }
          auto pv = [&](auto nc) {
            constexpr int N = decltype(nc)::value;
            uint32_t x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = values2<N>(hv[i], st[N >> 1][i], k4);
            const f16x8 va = as_vec8<F16>(make_uint4(x[0], x[1], x[2], x[3]));
            acc[4 * q + N] = mfma16(va, pl, acc[4 * q + N]);
            acc[4 * q + N] = mfma16(va, ph, acc[4 * q + N]);
          };
          pv(IntC<0>{});
          pv(IntC<1>{});
          pv(IntC<2>{});
          pv(IntC<3>{});
        }
      }
      wave_fence();
    };

    // A round's keys are loaded while the one before is used, its values after that: the
    // last round, which loads nothing, stands apart, since with the loads under a branch
    // the compiler waits for all of them at the next use. The steps are kept in order.
    if (base < k1) {
      for (; base + RK < k1; base += RK) {
        scores();
        __builtin_amdgcn_sched_barrier(0);
        load_k(base + RK);
        __builtin_amdgcn_sched_barrier(0);
        softmax_pv(base);
        __builtin_amdgcn_sched_barrier(0);
        load_v(base + RK);
        __builtin_amdgcn_sched_barrier(0);
      }
      scores();
      softmax_pv(base);
    }

    // O not finite (a group of NaN; finite values cannot overflow: P 2^15 times 2^15 times
    // 2^30 keys): P.V again over the keys that each row sees, since a masked key's NaN
    // times P = 0 is NaN
    {
      float nf = 0.0f;
#pragma unroll
      for (int e = 0; e < E; ++e)
#pragma unroll
        for (int v = 0; v < 4; ++v) nf = fmaf(acc[e][v], 0.0f, nf);
      if (__ballot(nf != 0.0f) != 0) {
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = f32x4{};
        const float ms = m_run == -INFINITY ? 0.0f : m_run - kPScale;
        int lane2 = static_cast<int>(threadIdx.x);  // (formed here, not kept across the loop)
        asm volatile("" : "+v"(lane2));
        const int g2 = (lane2 >> 4) & 3;
#pragma unroll 1
        for (int i = 0; i < 16 * TR * ((k1 - k0 + RK - 1) / RK); ++i) {
          const int key = k0 + 16 * TR * kw + RK * (i / (16 * TR)) + i % (16 * TR);
          if (key >= k1) break;
          const int64_t pg = paged_page<true>(a, row, key, bad);
          const int64_t in = key % a.bs;
          uint32_t x[NB], gw[GW];
          load_piece<NB>(kc + pg * a.kcb + in * a.kcs + 4 * NB * g2, x);
          load_words<NB>(kg + pg * pa4.kg.sb + in * NB, gw);
          const float d = row4_sum(piece_dot<NB>(x, gw, qb, k4)) * scale;
          if (key > lim) continue;
          const float p = __builtin_amdgcn_exp2f(d - ms);
          load_piece<NB>(vc + pg * a.vcb + in * a.vcs + 4 * NB * g2, x);
          load_words<NB>(vg + pg * pa4.vg.sb + in * NB, gw);
#pragma unroll
          for (int j = 0; j < NB; ++j) {
            // dims 32 j + 8 g + {0, 2, 1, 3, 4, 6, 5, 7}: dim 2 v + p of the eight is
            // acc[2 j + p][v]
            const f16x8 y = as_vec8<F16>(piece_group<NB>(x, gw, j, k4));
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const int v = 2 * (e >> 2) + (e & 1), pp = (e >> 1) & 1;
              acc[2 * j + pp][v] = fmaf(p, static_cast<float>(y[e]), acc[2 * j + pp][v]);
            }
          }
        }
      }
    }

    // acc[2 j + p][v] is dim 32 j + 8 g + 2 v + p of row r16
    float l = row4_sum(l_part);
    if (__ballot(bad) != 0) l = __uint_as_float(0x7fc00000u);
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int v = 0; v < 4; v += 2)
        *reinterpret_cast<float4*>(&sm[w][r16][32 * j + 8 * g + 2 * v]) =
            make_float4(acc[2 * j][v], acc[2 * j + 1][v], acc[2 * j][v + 1], acc[2 * j + 1][v + 1]);
    if (g == 0) {
      sml[w][r16][0] = m_run;
      sml[w][r16][1] = l;
    }
    __syncthreads();
    int t2 = t;  // (places formed here, not kept across the loop)
    asm volatile("" : "+v"(t2));
    const int orow = t2 >> 4, od = E * (t2 & 15);
    const int orr = tl * 16 + orow;
    if (orr < nq * a.G) {
#pragma unroll
      for (int x = 0; x < HP; ++x) {
        float M = -INFINITY;
#pragma unroll
        for (int k = 0; k < NW; ++k) M = fmaxf(M, sml[x * NW + k][orow][0]);
        float L = 0.0f, o[E];
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = 0.0f;
#pragma unroll
        for (int k = 0; k < NW; ++k) {
          const float mk = sml[x * NW + k][orow][0], lk = sml[x * NW + k][orow][1];
          // (a quarter each: as k_paged8 leaves them to the merge)
          const float f = mk == -INFINITY ? 0.0f : 0.25f * __builtin_amdgcn_exp2f(mk - M);
          // (a wave without keys has m = -inf and l = 0; NaN scores leave m = -inf
          // with l = NaN, which the sum keeps)
          L += mk == -INFINITY ? lk : f * lk;
#pragma unroll
          for (int e = 0; e < E; ++e) o[e] += f * sm[x * NW + k][orow][od + e];
        }
        if (single) {
          const int ho = hg * HP + x;
          const int64_t tok = sq.q0 + orr / a.G;
          const int hq = ho * a.G + orr % a.G;
          uint16_t* op =
              static_cast<uint16_t*>(a.o) + tok * a.ost + static_cast<int64_t>(hq) * a.ohs + od;
          const float rcp = 1.0f / L, vs = fixed_scale(pa.vs, ho);
          uint32_t pk[E / 2];
#pragma unroll
          for (int q = 0; q < E / 2; ++q) {
            float lo = o[2 * q] * rcp * vs, hi = o[2 * q + 1] * rcp * vs;
            if (nk == 0) lo = hi = sq.bad ? __uint_as_float(0x7fc00000u) : 0.0f;
            pk[q] = round2(lo, hi, bf);
          }
#pragma unroll
          for (int q = 0; q < E / 2; q += 2)
            *reinterpret_cast<uint2*>(op + 2 * q) = make_uint2(pk[q], pk[q + 1]);
        } else {
          const int64_t part =
              ((2 * static_cast<int64_t>(blockIdx.x) + !first) * HP + x) * 16 + orow;
          float* pp = a.part + part * D + od;
#pragma unroll
          for (int e = 0; e < E; e += 4)
            *reinterpret_cast<float4*>(pp + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
          if (od == 0) {
            a.ml[2 * part] = M;
            a.ml[2 * part + 1] = L;
          }
        }
      }
    }
    if (!on) return;
    left -= take;
    u = 0;
    ++seg;
    if (last_seg) {  // the next sequence with rows (there are units left)
      seg = 0;
      ++b;
      if constexpr (D == 256) next = paged_seq(a, b);
      sq = uniform_seq(next);
      while (sq.nq == 0) sq = uniform_seq(paged_seq(a, ++b));
      tiles = seq_tiles(a, sq);
      units = seq_units(pa.unit, sq);
    }
    __syncthreads();  // (the merge buffer)
  }
}

template <typename T, int D, int HP>
__global__ __launch_bounds__(1024) void k_paged4_merge(Paged8Args pa) {
  merge_segments<T, D, HP, true>(pa);
}

// Many rows (prefill over a cached prefix): tiles of 32 rows of each of W waves as in
// k_paged8_rows. The 64 keys of a tile are loaded into registers (four lanes to a key, a tile
// ahead), made fp16 numbers once per workgroup and written to LDS, in which the dims of
// every eight lie in the order of a piece ({0, 2, 1, 3, 4, 6, 5, 7}); so do the queries',
// and O's come out in it. P enters as P 2^7, at most 2^15 (see kStep).
//
// The matrix instructions (busy 45 % of the cycles, a third of it P's second part) and the vector
// ones (issuing 48 %) bound it, one after the other in waves that a barrier keeps in step: 2,048
// new tokens of each of 4 sequences of 4,096 .. 6,144, 32 q / 8 kv heads of 128, take 737 us, 704
// TFLOP/s, 1,056 counting both parts (an 8192^3 fp16 product reaches 1,159). Without the second
// part 604 us. The softmax of the next 16 keys between the products of these, in the compiler's
// order or alternating with them: no gain (742).
template <int D, bool P16, int W>
__global__ __launch_bounds__(64 * W, D == 256 ? 1 : 2) void k_paged4_rows(Paged4Args pa4) {
  constexpr int KT = 64, TT = KT / 32;
  constexpr int KS = D / 16, DT = D / 32, CH = D / 8;
  constexpr int NB = D / 32, GW = NB / 2;
  constexpr int RT = 32 * W;  // rows of a tile
  constexpr float kStep = 8.0f, kPScaleRows = 7.0f;
  __shared__ uint4 sk[2][KT * CH];
  __shared__ uint4 sv[2][KT * CH];
  __shared__ int s_bad;  // some wave looked up a page outside the cache
  const Paged8Args& pa = pa4.p;
  const PagedArgs& a = pa.a;
  const int h = static_cast<int>(blockIdx.x % a.Hkv);
  const int64_t x = blockIdx.x / a.Hkv;
  const int c = static_cast<int>(blockIdx.y);
  const PagedTile tile = paged_find(a, RT, x, -1);
  if (tile.b < 0) return;
  const PagedSeq& sq = tile.s;
  const int nk = static_cast<int>(sq.nk), nq = sq.nq;
  const int k0 = c * tile.chunk;
  if (k0 >= nk && c > 0) return;
  const Int4Consts k4;
  const float minus_one = opaque(-1.0f);
  const bool bf = pa4.dtype == FP_DTYPE_BF16;
  const bool single = nk <= tile.chunk;
  const int t = threadIdx.x, lane = t & 63;
  const int w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int half = lane >> 5, l32 = lane & 31;
  const int rows = nq * a.G;
  // (a sequence's last rows see most keys and start first)
  const int tl = (rows + RT - 1) / RT - 1 - tile.tl;

  // this lane's query row and its last visible key
  const int rr = tl * RT + 32 * w + l32;
  const bool rvalid = rr < rows;
  const int qi = (rvalid ? rr : rows - 1) / a.G;
  const int64_t tok = sq.q0 + qi;
  const int hq = h * a.G + (rvalid ? rr : rows - 1) % a.G;
  const int lim = nk - nq + qi;
  // the wave's first and last visible keys' bounds (wave-uniform)
  const int r0 = min(tl * RT + 32 * w, rows - 1);
  const int r1 = min(tl * RT + 32 * w + 31, rows - 1);
  const int lim_lo = __builtin_amdgcn_readfirstlane(nk - nq + r0 / a.G);
  const int lim_hi = __builtin_amdgcn_readfirstlane(nk - nq + r1 / a.G);
  // keys past the last row of the tile are visible to none of its rows
  const int last_row = min(tl * RT + RT - 1, rows - 1);
  const int k1 = __builtin_amdgcn_readfirstlane(
      min(min(k0 + tile.chunk, nk), max(nk - nq + last_row / a.G + 1, 0)));

  // (the factor of a row's scores: its sign in q, so that the largest score is that of the
  // largest product)
  const float signed_scale = a.scale_log2 * fixed_scale(pa.ks, h);
  float scale = fabsf(signed_scale), f = signed_scale < 0.0f ? -1.0f : 1.0f;
  f16x8 qb[KS];
  {
    const uint16_t* qp = static_cast<const uint16_t*>(a.q) + tok * a.qst +
                         static_cast<int64_t>(hq) * a.qhs + 8 * half;
    uint4 y[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) y[s] = rvalid ? ld16(qp + 16 * s) : zero4();
    if (bf) {
      i16x2 most{};
#pragma unroll
      for (int s = 0; s < KS; ++s) most = exponents8(y[s], most);
      const int e = factor_exponent(
          static_cast<int>(pair32_max(static_cast<float>(row_exponent(most)))));
      f = __builtin_amdgcn_ldexpf(f, e);
      scale *= __builtin_amdgcn_ldexpf(1.0f, -e);
    }
#pragma unroll
    for (int s = 0; s < KS; ++s) qb[s] = as_vec8<F16>(query8(y[s], bf, f));
  }
  // (not 0, by which a masked score would be NaN: by 2^-149 no score reaches 2^-100)
  if (scale == 0.0f) scale = 0x1p-149f;
  f32x16 o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) o[dt] = f32x16{};
  float m_run = -INFINITY, l_part = 0.0f;
  bool bad = false;

  const int64_t row = static_cast<int64_t>(tile.b) * a.table_stride;
  const uint8_t* kc = static_cast<const uint8_t*>(a.kc) + static_cast<int64_t>(h) * a.kch;
  const uint8_t* vc = static_cast<const uint8_t*>(a.vc) + static_cast<int64_t>(h) * a.vch;
  const uint16_t* kg = pa4.kg.p + h * pa4.kg.sh;
  const uint16_t* vg = pa4.vg.p + h * pa4.vg.sh;

  // the lane's key of a load, and its piece: of K and V, or of eight waves the first four of
  // K and the others of V
  const int lkey = 16 * (w & 3) + (lane >> 2), lp = lane & 3;
  const bool takes_k = W == 4 || w < 4, takes_v = W == 4 || w >= 4;
  constexpr int SIDES = W == 4 ? 2 : 1;
  uint32_t cr[SIDES][NB], gr[SIDES][GW];
  const int last16 = (nk - 1) & ~15;
  // tile of keys base .. base + 63; keys past the sequence read its last 16-key
  // group (P16) or its last key
  auto load = [&](int base) {
    int64_t pg, in;
    if constexpr (P16) {
      const int tb = min(base + 16 * (w & 3), last16);
      pg = paged_page<true>(a, row, tb, bad);
      in = (a.bs_shift >= 0 ? tb & (a.bs - 1) : tb % a.bs) + (lane >> 2);
    } else {
      const int key = min(base + lkey, nk - 1);
      pg = paged_page<false>(a, row, key, bad);
      in = key % a.bs;
    }
    if (takes_k) {
      load_piece<NB>(kc + pg * a.kcb + in * a.kcs + 4 * NB * lp, cr[0]);
      load_words<NB>(kg + pg * pa4.kg.sb + in * NB, gr[0]);
    }
    if (takes_v) {
      load_piece<NB>(vc + pg * a.vcb + in * a.vcs + 4 * NB * lp, cr[SIDES - 1]);
      load_words<NB>(vg + pg * pa4.vg.sb + in * NB, gr[SIDES - 1]);
    }
  };
  // as fp16 numbers into buffer `buf`; V of slots past the sequence is 0 (they may hold
  // anything)
  auto store = [&](int base, int buf) {
    if (takes_v && base + lkey >= nk) {
#pragma unroll
      for (int q = 0; q < GW; ++q) gr[SIDES - 1][q] = 0u;
    }
    uint4* to = takes_k ? sk[buf] : sv[buf];
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const int at = lkey * CH + ((4 * j + lp) ^ swz<D>(lkey));
      to[at] = piece_group<NB>(cr[0], gr[0], j, k4);
      if constexpr (SIDES == 2) sv[buf][at] = piece_group<NB>(cr[1], gr[1], j, k4);
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
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int t4 = 0; t4 < TT; ++t4) {
          const int r = 32 * t4 + l32;
          const uint4 kop = sk[buf][r * CH + ((2 * ks + half) ^ swz<D>(r))];
          s[t4] = F16::mfma32(as_vec8<F16>(kop), qb[ks], ks == 0 ? f32x16{} : s[t4]);
        }
      if (base + KT - 1 > lim_lo) {
        asm volatile("");  // (a branch: as selects they would be in every tile)
#pragma unroll
        for (int t4 = 0; t4 < TT; ++t4)
#pragma unroll
          for (int v = 0; v < 16; ++v)
            if (base + 32 * t4 + 8 * (v >> 2) + 4 * half + (v & 3) > lim) s[t4][v] = -INFINITY;
      }
      float mx = -INFINITY;
#pragma unroll
      for (int t4 = 0; t4 < TT; ++t4)
#pragma unroll
        for (int v = 0; v < 16; ++v) mx = fmaxf(mx, s[t4][v]);
      mx = pair32_max(mx) * scale;
      // m moves only where it must, so that P stays below 2^kStep: not in every tile that
      // has a new largest score for one of the wave's rows
      if (__ballot(mx > m_run + kStep) != 0) {
        const float m_new = fmaxf(m_run, mx);
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
      const float ms = m_run == -INFINITY ? 0.0f : m_run - kPScaleRows;
      // (a tile's sum apart from l: in one chain over thousands of keys fp32's roundings would be
      // most of what outputs are off by)
      float l_tile[4] = {};
#pragma unroll
      for (int t4 = 0; t4 < TT; ++t4) {
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          s[t4][v] = __builtin_amdgcn_exp2f(fmaf(s[t4][v], scale, -ms));
          l_tile[v & 3] += s[t4][v];
        }
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          F16Parts u[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            u[e] = f16_parts(s[t4][8 * hh + 2 * e], s[t4][8 * hh + 2 * e + 1], minus_one);
          const f16x8 ph = as_vec8<F16>(make_uint4(u[0].hi, u[1].hi, u[2].hi, u[3].hi));
          const f16x8 pl = as_vec8<F16>(make_uint4(u[0].lo, u[1].lo, u[2].lo, u[3].lo));
          const uint16_t* sv16 = reinterpret_cast<const uint16_t*>(sv[buf]);
          const int r = 32 * t4 + 16 * hh + tr_row;
          __builtin_amdgcn_sched_barrier(0);
          f16x8 va[DT];
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) va[dt] = read_vt<F16, D>(sv16, r, 32 * dt + tr_col);
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) o[dt] = F16::mfma32(va[dt], pl, o[dt]);
          // (a dim tile's two products apart: the second would wait for the first)
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) o[dt] = F16::mfma32(va[dt], ph, o[dt]);
        }
      }
      l_part += (l_tile[0] + l_tile[1]) + (l_tile[2] + l_tile[3]);
    }
    if (more) store(base + KT, buf ^ 1);
  }

  // Rows whose O is not finite (a group of NaN) take P.V again over the keys that each row
  // sees: a masked key's NaN times P = 0 is NaN.
  float nf = 0.0f;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int v = 0; v < 16; ++v) nf = fmaf(o[dt][v], 0.0f, nf);
  if (__ballot(nf != 0.0f) != 0) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] = f32x16{};
    const float ms = m_run == -INFINITY ? 0.0f : m_run - kPScaleRows;
    int half2 = static_cast<int>(threadIdx.x);  // (formed here, not kept across the loop)
    asm volatile("" : "+v"(half2));
    half2 = (half2 >> 5) & 1;
#pragma unroll 1
    for (int key = k0; key < k1; ++key) {
      const int64_t pg = paged_page<true>(a, row, key, bad);
      const int64_t in = key % a.bs;
      float d = 0.0f;  // the lane's eight of every 16 dims of q . u_k: pieces half, 2 + half
      uint32_t y[2][NB], gw[GW];
      load_words<NB>(kg + pg * pa4.kg.sb + in * NB, gw);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        load_piece<NB>(kc + pg * a.kcb + in * a.kcs + 4 * NB * (2 * i + half2), y[i]);
        f16x8 q[NB];
#pragma unroll
        for (int j = 0; j < NB; ++j) q[j] = qb[2 * j + i];
        d += piece_dot<NB>(y[i], gw, q, k4);
      }
      d = pair32_sum(d) * scale;
      if (key > lim) continue;
      const float p = __builtin_amdgcn_exp2f(d - ms);
      load_words<NB>(vg + pg * pa4.vg.sb + in * NB, gw);
#pragma unroll
      for (int pc = 0; pc < 4; ++pc) {  // o[dt][4 pc + e]: place 4 half + e of piece pc
        load_piece<NB>(vc + pg * a.vcb + in * a.vcs + 4 * NB * pc, y[0]);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          const uint4 g8 = piece_group<NB>(y[0], gw, dt, k4);
          const uint32_t g2[2] = {half2 ? g8.z : g8.x, half2 ? g8.w : g8.y};
#pragma unroll
          for (int e = 0; e < 4; ++e)
            o[dt][4 * pc + e] =
                fmaf(p, F16::to_f32(static_cast<uint16_t>(g2[e >> 1] >> (16 * (e & 1)))),
                     o[dt][4 * pc + e]);
        }
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
  // (dims 0, 2, 1, 3 of four)
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
            make_uint2(round2(y[0], y[2], bf), round2(y[1], y[3], bf));
      }
  } else {
    const int64_t slot = (tok * a.Hq + hq) * a.nc + c;
    float* pp = a.part + slot * D;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int g4 = 0; g4 < 4; ++g4)
        *reinterpret_cast<float4*>(pp + 32 * dt + 8 * g4 + 4 * half) =
            make_float4(o[dt][4 * g4], o[dt][4 * g4 + 2], o[dt][4 * g4 + 1], o[dt][4 * g4 + 3]);
    if (half == 0) {
      a.ml[2 * slot] = m_run;
      a.ml[2 * slot + 1] = l;
    }
  }
}

template <int D, int HP>
hipError_t launch_few4(const Paged4Args& p, hipStream_t s) {
  const PagedArgs& a = p.p.a;
  const dim3 grid(static_cast<unsigned>(a.nc)), b(256);
  if (a.bs % 16 != 0) hipLaunchKernelGGL((k_paged4<D, false, HP>), grid, b, 0, s, p);
  else hipLaunchKernelGGL((k_paged4<D, true, HP>), grid, b, 0, s, p);
  if (a.part != nullptr) {
    // few heads and rows: as many workgroups for each as make up 256 (one sequence of 131,000,
    // 16 rows of 2 KV heads of 64: 65 us with one workgroup for each head)
    unsigned split = 16;
    while (split > 1 && p.p.segs * HP * split > 256) split /= 2;
    const dim3 mg(static_cast<unsigned>(p.p.segs * HP), split), mb(1024);
    if (p.dtype == FP_DTYPE_BF16)
      hipLaunchKernelGGL((k_paged4_merge<BF16, D, HP>), mg, mb, 0, s, p.p);
    else
      hipLaunchKernelGGL((k_paged4_merge<F16, D, HP>), mg, mb, 0, s, p.p);
  }
  return hipGetLastError();
}

hipError_t launch_paged4(const Paged4Args& p, int head_dim, int hp, bool rows, int64_t tiles,
                         hipStream_t s) {
  const PagedArgs& a = p.p.a;
  return with_head_dim(head_dim, [&](auto dc) -> hipError_t {
    constexpr int D = decltype(dc)::value;
    if (!rows) {
      if constexpr (D == 64) {
        if (hp == 4) return launch_few4<D, 4>(p, s);
      }
      if constexpr (D <= 128) {
        if (hp == 2) return launch_few4<D, 2>(p, s);
      }
      return launch_few4<D, 1>(p, s);
    }
    const dim3 grid(static_cast<unsigned>(tiles * a.Hkv), static_cast<unsigned>(a.nc));
    const auto run = [&](auto wc) {
      constexpr int W = decltype(wc)::value;
      if (a.bs % 16 != 0)
        hipLaunchKernelGGL((k_paged4_rows<D, false, W>), grid, dim3(64 * W), 0, s, p);
      else
        hipLaunchKernelGGL((k_paged4_rows<D, true, W>), grid, dim3(64 * W), 0, s, p);
    };
    if constexpr (D < 256) {
      if (p.row_tile == 256) run(IntC<8>{});
      else run(IntC<4>{});
    } else {
      run(IntC<4>{});
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.nc <= 1) return e;
    return launch_paged_merge8(a, p.dtype, D, s);
  });
}

}  // namespace fp

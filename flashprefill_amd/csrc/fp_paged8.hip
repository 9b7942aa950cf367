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
//
// Few rows (k_paged8) are bound by the loads that eight waves per CU have in flight where
// there are many bytes: 32 sequences of 300 .. 15,000 tokens, 32 q / 8 kv heads of 128,
// 447 MB of codes in 96 us (4.7 TB/s, where a stream that only reads reaches 7.2) and 7 for
// the merge; one sequence of 65,000, 137 MB with its scales, 31 and 7; one of 333, 8 us,
// of which 1.7 are the launch, 1.5 the search for the place of the workgroup and 3.3 the
// first loads and the end of a segment. Many rows (k_paged8_rows) are bound by MFMA and
// VALU and by how little the two waves of a SIMD overlap them: 2,048 new tokens of each of
// 4 sequences of 4,096 .. 6,144 in 730 .. 760 us in a row of calls, about 700 TFLOP/s
// (1,050 counting both parts of P); of the kernel's cycles MFMA is busy in 49 %, vector
// instructions issue in 53 % and LDS is busy in 33 %, a quarter of them bank conflicts.
// Raised wave priorities around the MFMAs are 0 to 3 % slower.
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

// ---------------------------------------------------------------------------
// Few rows
// ---------------------------------------------------------------------------
// A segment is 16 rows of the queries of one (sequence, KV head or pair of them) with all
// its keys, in units of `unit` keys; the segments of a call lie behind each other
// (sequence, heads, row tile) and every workgroup takes an equal share of the units, whatever segments
// they belong to: a decode step reads each cached byte once, so equal bytes take equal
// times, and no workgroup starts for keys that are not there (the host cannot see the
// lengths without a synchronisation). A share is a whole number of units, so that a call of
// few leaves workgroups without any: 1,620 units are four for each of 405 workgroups of 512,
// 2,152 five for each of 431, 13,728 twenty-seven for each of 509. A segment that is one workgroup's is written out,
// the others as partials (O, m, l), the first and the last of a workgroup at most, which
// k_paged8_merge combines. Where the table has room for few keys, a unit is a whole
// sequence and a segment a workgroup's: no merge.
struct Work {
  int total, share;  // units of the call, and of a workgroup
  PagedSeq s;        // the sequence at the place asked for
  int b;             // (below 0: no such place)
  int units, segs;   // units and segments of the sequences before it
};

__device__ __forceinline__ int seq_tiles(const PagedArgs& a, const PagedSeq& s) {
  return static_cast<int>((static_cast<int64_t>(s.nq) * a.G + 15) / 16);
}
// (unit: a power of two)
__device__ __forceinline__ int seq_units(int unit, const PagedSeq& s) {
  return max(static_cast<int>((s.nk + unit - 1) >> (31 - __clz(unit))), 1);
}
__device__ __forceinline__ int64_t uniform64(int64_t x) {
  return static_cast<int64_t>(
      static_cast<uint64_t>(static_cast<uint32_t>(
          __builtin_amdgcn_readfirstlane(static_cast<int>(x >> 32)))) << 32 |
      static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(x))));
}
__device__ __forceinline__ PagedSeq uniform_seq(const PagedSeq& s) {
  return PagedSeq{uniform64(s.q0), __builtin_amdgcn_readfirstlane(s.nq), uniform64(s.nk),
                  __builtin_amdgcn_readfirstlane(static_cast<int>(s.bad)) != 0, false};
}
// sums over the lanes up to this one: within rows of 16 lanes, then across them
__device__ __forceinline__ int lane_prefix(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);
  return x;
}

// By one wave, 64 sequences at a time: the place of workgroup wg's first unit, or with
// seg >= 0 that of a segment. Where some sequence's offsets do not fit, which rows are
// whose is unknown: all rows of the call are one sequence's then, and bad.
__device__ __forceinline__ Work find_work(const Paged8Args& pa, int wg, int64_t seg) {
  const PagedArgs& a = pa.a;
  const int lane = threadIdx.x & 63;
  Work r;
  r.b = -1;
  r.units = r.segs = r.total = 0;
  r.s = PagedSeq{0, 0, 0, false, false};
  bool off = false;
  PagedSeq s = r.s;
  int ns = 0, nu = 0, is = 0, iu = 0;  // the lane's segments and units; with the lanes below
  const auto load = [&](int base) {
    s = paged_seq(a, min(base + lane, a.B - 1));
    if (base + lane >= a.B) s = PagedSeq{0, 0, 0, false, false};
    ns = seq_tiles(a, s) * pa.groups;
    nu = ns * seq_units(pa.unit, s);
    is = lane_prefix(ns);
    iu = lane_prefix(nu);
  };
  for (int base = 0; base < a.B; base += 64) {
    load(base);
    off = off || __ballot(s.off) != 0;
    r.total += __builtin_amdgcn_readlane(iu, 63);
  }
  if (off) {
    r.s = PagedSeq{0, static_cast<int>(a.T), 0, true, true};
    r.total = seq_tiles(a, r.s) * pa.groups;
  }
  r.share = max((r.total + a.nc - 1) / a.nc, pa.min_share);
  const int64_t x = static_cast<int64_t>(wg) * r.share;
  if (seg < 0 && x >= r.total) return r;
  if (off) {
    r.b = seg < r.total ? 0 : -1;
    return r;
  }
  for (int base = 0; base < a.B; base += 64) {
    if (a.B > 64) load(base);
    const int64_t y = seg >= 0 ? seg - r.segs : x - r.units;
    const bool mine = seg >= 0 ? y >= is - ns && y < is : y >= iu - nu && y < iu;
    const uint64_t hit = __ballot(mine);
    if (hit != 0) {
      const int l = __builtin_amdgcn_readfirstlane(__ffsll(static_cast<long long>(hit)) - 1);
      r.b = base + l;
      r.s = uniform_seq(PagedSeq{shfl64(s.q0, l), __shfl(s.nq, l), shfl64(s.nk, l),
                                 __shfl(static_cast<int>(s.bad), l) != 0, false});
      r.units += __builtin_amdgcn_readlane(iu - nu, l);
      r.segs += __builtin_amdgcn_readlane(is - ns, l);
      return r;
    }
    r.units += __builtin_amdgcn_readlane(iu, 63);
    r.segs += __builtin_amdgcn_readlane(is, 63);
  }
  return r;
}

// The four waves of a workgroup take 32 keys in turn, straight from the pages into
// registers, a round ahead of their use:
//
//   S^T (keys x rows) = K . Q^T on v_mfma_f32_16x16x32: a lane (r = l % 16,
//     g = l / 16) loads 16-byte pieces of key r, whose two halves are the operands
//     of two k-steps (dims 64 i + 16 g + 8 e .. of step 2 i + e, in Q as in K)
//   O^T (dims x rows) += V^T . P^T on the same: k index 8 g + 4 t + v is key
//     16 t + 4 g + v, so P stays in the lanes that hold it, and row m of MFMA e is
//     dim E m + e, byte e of the E = D / 16 bytes that lane m loads of each of its
//     8 keys: whole rows are loaded and nothing crosses lanes. v_perm pairs the
//     bytes of two keys, one conversion each makes them an operand word.
//
// HP: KV heads of a segment, each served by 4 / HP of the waves. A key of 64 bytes is half
// a cache line, and the other half its neighbour head's: served apart they are fetched
// twice (16 sequences of 40 .. 9,000 tokens, 8 KV heads, d = 64, 4 queries each: 35 us with
// one head per segment).
//
// P16: the page size is a multiple of 16, so a 16-key tile lies in one page: a wave
// looks up 64 of them at a time, one per lane, and reads a tile's place from its lane.
// PS: all scales are per slot. Other pages, and scales of which only K's or only V's are
// per slot, take the general form (neither), which looks up every key's page and scale for
// itself: the 32 sequences above in pages of 24 take 237 us (354 with scales per slot), in
// pages of 16 with K's scales per slot and V's fixed 336, where the other forms take 100 to
// 102 (whole calls).
//
// Registers: 119 to 139 at head_dim 64, 161 to 177 at 128, 229 to 256 at 256; 65 to 101
// scalar ones are kept in lanes of vector registers.
template <typename T, int F, int D, bool P16, bool PS, int HP>
__global__ __launch_bounds__(256, 2) void k_paged8(Paged8Args pa) {
  constexpr int KS = D / 32;  // MFMA k-steps over the head dim
  constexpr int KP = D / 64;  // 16-byte pieces of a key per lane
  constexpr int E = D / 16;   // V bytes per lane and key
  constexpr int VW = E / 4;   // the same in words
  constexpr int OS = D + 4;   // padded row of the merge buffer (floats)
  constexpr int NP = 3;       // parts of P
  constexpr bool kScaled = PS || !P16;
  constexpr int NW = 4 / HP;  // waves of a head
  constexpr int RK = 32 * NW;  // keys of a round, all waves of a head
  __shared__ float sm[4][16][OS];
  __shared__ float sml[4][16][2];
  const PagedArgs& a = pa.a;
  const Work work = find_work(pa, static_cast<int>(blockIdx.x), -1);
  if (work.b < 0) return;
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

    // this lane's query row (B operand column) and its last visible key
    const int rr = tl * 16 + r16;
    const bool rvalid = rr < nq * a.G;
    const int qi = rvalid ? rr / a.G : 0;
    const int lim = rvalid ? nk - nq + qi : nk - 1;
    typename T::vec8 qb[KS];
    {
      const uint16_t* qp = static_cast<const uint16_t*>(a.q) + (sq.q0 + qi) * a.qst +
                           static_cast<int64_t>(h * a.G + (rvalid ? rr % a.G : 0)) * a.qhs + 16 * g;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const uint4 x = ld16(qp + 64 * (s >> 1) + 8 * (s & 1));
        qb[s] = as_vec8<T>(rvalid ? x : zero4());
      }
    }

    f32x4 acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = f32x4{};
    float m_run = -INFINITY, l_part = 0.0f;
    bool bad = false;
    const int64_t row = static_cast<int64_t>(b) * a.table_stride;
    const uint8_t* kc = static_cast<const uint8_t*>(a.kc) + static_cast<int64_t>(h) * a.kch;
    const uint8_t* vc = static_cast<const uint8_t*>(a.vc) + static_cast<int64_t>(h) * a.vch;
    const float* kss = pa.ks.p + h * pa.ks.sh;  // read where there is one per slot
    const float* vss = pa.vs.p + h * pa.vs.sh;
    const float scale = a.scale_log2 * fixed_scale(pa.ks, h);

    // what a round loads: 32 keys, lanes as above
    struct {
      uint4 k[2][KP];
      uint32_t v[2][4][VW];
      f32x4 ks[2], vs[2];
    } r;
    // places of the 64 16-key tiles from key `win`, one per lane (P16; tiles past the
    // sequence repeat the last one, their scores are masked)
    int win = k0;
    int64_t kat = 0, vat = 0, ksat = 0, vsat = 0;
    const int last16 = (nk - 1) & ~15;
    auto look = [&](int from) {
      win = from;
      const int key = min(from + 16 * lane, last16);
      const int64_t pg = paged_page<false>(a, row, key, bad);
      const int in = a.bs_shift >= 0 ? key & (a.bs - 1) : key % a.bs;
      kat = pg * a.kcb + in * a.kcs;
      vat = pg * a.vcb + in * a.vcs;
      if constexpr (PS) {
        ksat = pg * pa.ks.sb + in;
        vsat = pg * pa.vs.sb + in;
      }
    };
    auto place = [&](int64_t x, int tile) {
      return static_cast<int64_t>(
          static_cast<uint64_t>(static_cast<uint32_t>(
              __builtin_amdgcn_readlane(static_cast<int>(x >> 32), tile))) << 32 |
          static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(x), tile)));
    };
    // a lane's offsets in a tile
    const uint32_t koff = static_cast<uint32_t>(r16 * static_cast<int>(a.kcs) + 16 * g);
    uint32_t voff[4];
#pragma unroll
    for (int v = 0; v < 4; ++v)
      voff[v] = static_cast<uint32_t>((4 * g + v) * static_cast<int>(a.vcs) + E * r16);
    auto load_k = [&](int base) {
      if constexpr (P16) {
        if (base >= win + 1024) look(k0 + ((base - k0) & ~1023));
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int tile = ((base - win) >> 4) + j;
          const uint8_t* p = kc + place(kat, tile);
#pragma unroll
          for (int s = 0; s < KP; ++s) r.k[j][s] = ld16(p + koff + 64 * s);
          if constexpr (PS)
            r.ks[j] = *reinterpret_cast<const f32x4*>(kss + place(ksat, tile) + 4 * g);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int key = min(base + 16 * j + r16, nk - 1);
          const int64_t pg = paged_page<false>(a, row, key, bad);
          const uint8_t* p = kc + pg * a.kcb + static_cast<int64_t>(key % a.bs) * a.kcs + 16 * g;
#pragma unroll
          for (int s = 0; s < KP; ++s) r.k[j][s] = ld16(p + 64 * s);
          float f[4] = {1.0f, 1.0f, 1.0f, 1.0f};
          if (pa.ks.slot)
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              const int kv = min(base + 16 * j + 4 * g + v, nk - 1);
              f[v] = kss[paged_page<false>(a, row, kv, bad) * pa.ks.sb + kv % a.bs];
            }
          r.ks[j] = f32x4{f[0], f[1], f[2], f[3]};
        }
      }
    };
    auto load_v = [&](int base) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int tile = ((base - win) >> 4) + j;
        float f[4] = {1.0f, 1.0f, 1.0f, 1.0f};
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const uint8_t* p;
          if constexpr (P16) {
            p = vc + place(vat, tile) + voff[v];
          } else {
            const int key = min(base + 16 * j + 4 * g + v, nk - 1);
            const int64_t pg = paged_page<false>(a, row, key, bad);
            const int in = key % a.bs;
            p = vc + pg * a.vcb + static_cast<int64_t>(in) * a.vcs + E * r16;
            if (pa.vs.slot) f[v] = vss[pg * pa.vs.sb + in];
          }
          if constexpr (VW == 1) {
            r.v[j][v][0] = *reinterpret_cast<const uint32_t*>(p);
          } else if constexpr (VW == 2) {
            const uint2 x = *reinterpret_cast<const uint2*>(p);
            r.v[j][v][0] = x.x; r.v[j][v][1] = x.y;
          } else {
            const uint4 x = ld16(p);
            r.v[j][v][0] = x.x; r.v[j][v][1] = x.y; r.v[j][v][2] = x.z; r.v[j][v][3] = x.w;
          }
        }
        if constexpr (P16 && PS)
          r.vs[j] = *reinterpret_cast<const f32x4*>(vss + place(vsat, tile) + 4 * g);
        else if constexpr (!P16)
          r.vs[j] = f32x4{f[0], f[1], f[2], f[3]};
      }
    };
    f32x4 s[2];
    auto scores = [&]() {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        s[j] = f32x4{};
#pragma unroll
        for (int i = 0; i < KP; ++i) {
          s[j] = mfma16(as_vec8<T>(widen8<T, F>(r.k[j][i].x, r.k[j][i].y)), qb[2 * i], s[j]);
          s[j] = mfma16(as_vec8<T>(widen8<T, F>(r.k[j][i].z, r.k[j][i].w)), qb[2 * i + 1], s[j]);
        }
        if constexpr (kScaled) {
#pragma unroll
          for (int v = 0; v < 4; ++v) s[j][v] *= scale * r.ks[j][v];
        } else {
#pragma unroll
          for (int v = 0; v < 4; ++v) s[j][v] *= scale;
        }
      }
    };
    auto softmax_pv = [&](int base) {
      if (base + 31 > nk - nq) {  // some row's causal limit or the end lies in this round
        asm volatile("");  // (a branch: as selects they would be in every round)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const int key = base + 16 * j + 4 * g + v;
            if (key > lim) s[j][v] = -INFINITY;
            if (key >= nk) {  // slots past the end may hold anything
              if constexpr (kScaled) r.vs[j][v] = 0.0f;
#pragma unroll
              for (int q = 0; q < VW; ++q) r.v[j][v][q] = 0u;
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
          if constexpr (kScaled) s[j][v] *= r.vs[j][v];
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
          const uint32_t ka = r.v[i >> 1][2 * (i & 1)][q], kb = r.v[i >> 1][2 * (i & 1) + 1][q];
          pr[i][0] = __builtin_amdgcn_perm(kb, ka, 0x05010400u);
          pr[i][1] = __builtin_amdgcn_perm(kb, ka, 0x07030602u);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t x[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            x[i] = e & 1 ? widen2<BF16, F, true>(pr[i][e >> 1])
                         : widen2<BF16, F, false>(pr[i][e >> 1]);
          const auto va = as_vec8<BF16>(make_uint4(x[0], x[1], x[2], x[3]));
#pragma unroll
          for (int p = NP - 1; p >= 0; --p) acc[4 * q + e] = mfma16(va, pb[p], acc[4 * q + e]);
        }
      }
    };

    // A round's keys are loaded while the one before is used, its values after that: the
    // last round, which loads nothing, stands apart, since with the loads under a branch
    // the compiler waits for all of them at the next use. The steps are kept in order: as
    // one block they were interleaved into more registers than a wave has.
    int base = k0 + 32 * kw;
    if (base < k1) {
      if constexpr (P16) look(k0);
      load_k(base);
      load_v(base);
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
        for (int i = 0; i < 32 * ((k1 - k0 + RK - 1) / RK); ++i) {
          const int key = k0 + 32 * kw + RK * ((i >> 5)) + (i & 31);
          if (key >= k1) break;
          const int64_t pg = paged_page<true>(a, row, key, bad);
          const int in = key % a.bs;
          const uint8_t* kp = kc + pg * a.kcb + static_cast<int64_t>(in) * a.kcs + 16 * g2;
          const uint8_t* vp = vc + pg * a.vcb + static_cast<int64_t>(in) * a.vcs;
          float d = 0.0f;  // the lane's dims of q . c_k
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) {
            const uint2 x = *reinterpret_cast<const uint2*>(kp + 64 * (ks >> 1) + 8 * (ks & 1));
            const uint4 qu = __builtin_bit_cast(uint4, qb[ks]);
            const uint32_t qw[4] = {qu.x, qu.y, qu.z, qu.w};
            const f32x2 kv[4] = {
                Float8<F>::template to_f32<false>(x.x), Float8<F>::template to_f32<true>(x.x),
                Float8<F>::template to_f32<false>(x.y), Float8<F>::template to_f32<true>(x.y)};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              d = fmaf(T::to_f32(static_cast<uint16_t>(qw[e])), kv[e][0], d);
              d = fmaf(T::to_f32(static_cast<uint16_t>(qw[e] >> 16)), kv[e][1], d);
            }
          }
          d = row4_sum(d) * (kScaled && pa.ks.slot ? scale * kss[pg * pa.ks.sb + in] : scale);
          if (key > lim) continue;
          float p = __builtin_amdgcn_exp2f(d - ms);
          if (kScaled && pa.vs.slot) p *= vss[pg * pa.vs.sb + in];
#pragma unroll
          for (int v = 0; v < 4; ++v)
#pragma unroll
            for (int q = 0; q < VW; ++q) {
              const uint32_t x = *reinterpret_cast<const uint32_t*>(vp + E * (4 * g2 + v) + 4 * q);
              const f32x2 lo = Float8<F>::template to_f32<false>(x);
              const f32x2 hi = Float8<F>::template to_f32<true>(x);
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
          // (a quarter each: four finite sums add up to a finite one)
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
            pk[q] = pack2<T>(lo, hi);
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
          if ((t & 15) == 0) {
            a.ml[2 * part] = M;
            a.ml[2 * part + 1] = L;
          }
        }
      }
    }
    left -= take;
    if (left <= 0) return;
    u = 0;
    if (++seg == tiles * pa.groups) {  // the next sequence with rows (there are units left)
      seg = 0;
      do sq = uniform_seq(paged_seq(a, ++b));
      while (sq.nq == 0);
      tiles = seq_tiles(a, sq);
      units = seq_units(pa.unit, sq);
    }
    __syncthreads();  // (the merge buffer)
  }
}

// One head of a segment per workgroup of 16 waves: its rows' partials, weighted by
// exp2(m - max m) and divided by their l. They are the first of workgroups w0 + 1 .. w1
// and the first or last of w0. As many waves as there are share a row's partials.
template <typename T, int D, int HP>
__global__ __launch_bounds__(1024) void k_paged8_merge(Paged8Args pa) {
  constexpr int XD = D / 64;  // dims per lane
  typedef float vec __attribute__((ext_vector_type(XD)));
  __shared__ float so[16][D], sl[16];
  const PagedArgs& a = pa.a;
  const Work work = find_work(pa, 0, blockIdx.x / HP);
  if (work.b < 0) return;
  const int tiles = seq_tiles(a, work.s), units = seq_units(pa.unit, work.s);
  const int seg = static_cast<int>(blockIdx.x / HP) - work.segs, hh = blockIdx.x % HP;
  const int x0 = work.units + seg * units;
  const int w0 = __builtin_amdgcn_readfirstlane(x0 / work.share);
  const int n = __builtin_amdgcn_readfirstlane((x0 + units - 1) / work.share) - w0 + 1;
  if (n == 1) return;  // written by k_paged8
  const int h = seg / tiles * HP + hh, tl = seg % tiles;
  const int rows = min(work.s.nq * a.G - 16 * tl, 16);
  const int lgr = rows > 1 ? 32 - __clz(rows - 1) : 0;  // rows as a power of two
  const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int row = w & ((1 << lgr) - 1), share = 16 >> lgr;
  if (row < rows) {
    const int first = 2 * w0 + (x0 != w0 * work.share);
    const auto part = [&](int j) {
      return static_cast<int64_t>(((j == 0 ? first : 2 * (w0 + j)) * HP + hh) * 16 + row);
    };
    float M = -INFINITY;
    for (int j = lane; j < n; j += 64) M = fmaxf(M, a.ml[2 * part(j)]);
    M = wave_max(M);
    vec acc{};
    float L = 0.0f;
#pragma unroll 4
    for (int j = w >> lgr; j < n; j += share) {
      const int64_t p = part(j);
      const vec x = *reinterpret_cast<const vec*>(a.part + p * D + XD * lane);
      const float m = a.ml[2 * p], l = a.ml[2 * p + 1];
      // (2^-10: the sum over the partials, at most 512, stays finite)
      static_assert(kPaged8Groups <= 1024, "weights");
      const float f = m == -INFINITY ? 0.0f : 0x1p-10f * __builtin_amdgcn_exp2f(m - M);
      L += m == -INFINITY ? l : f * l;
#pragma unroll
      for (int q = 0; q < XD; ++q) acc[q] = fmaf(f, x[q], acc[q]);
    }
#pragma unroll
    for (int q = 0; q < XD; ++q) so[w][XD * lane + q] = acc[q];
    if (lane == 0) sl[w] = L;
  }
  __syncthreads();
  const float vs = fixed_scale(pa.vs, h);
  for (int i = t; i < rows * D; i += 1024) {
    const int r = i / D, d = i % D;
    float o = 0.0f, L = 0.0f;
    for (int k = r; k < 16; k += 1 << lgr) {
      o += so[k][d];
      L += sl[k];
    }
    const int rr = 16 * tl + r;
    static_cast<uint16_t*>(a.o)[(work.s.q0 + rr / a.G) * a.ost +
                                static_cast<int64_t>(h * a.G + rr % a.G) * a.ohs + d] =
        T::from_f32(o / L * vs);
  }
}

// Many rows (prefill over a cached prefix): 128-row tiles as in k_paged_rows, over keys that are
// widened on their way into LDS. The 64 keys of a tile are loaded into registers
// (16 keys by each wave, a tile ahead), widened once per workgroup and written as
// 16-bit tiles, K in q's type and V in bf16; P s_v takes two bf16 parts, 2^-17 of
// each product: a 64th of what rounding the output to fp16 may lose of its value
// (2^-11; to bf16 2^-8) and an 8,192nd of what rounding to e4m3 may have lost of the
// cached one (2^-4; to e5m2 2^-3). A third part, as k_paged8 has it, would add half as
// many MFMAs to P.V again for errors below these; one part would save a fifth of the
// time and lose 2^-8 of each product, as much as a bf16 output's rounding.
//
// Chunks have the length of the call's longest sequence over its chunk slots. Chunks cut
// to each sequence, for an equal share of all keys per workgroup, balance the workgroups
// but split more rows: 118 -> 146 us (512 new of 8,192 tokens), 82 -> 102 (300 new of
// 5,500 and of 1,200), 157 -> 144 .. 159 (500 new of 6,144, 2,500 and 1,111).
//
// D = 256: one workgroup per CU (256 VGPRs and 240 AGPRs, 130 KB of LDS), one wave per
// SIMD: nothing runs beside its softmax. 3 sequences of 5,000 tokens with 600 new ones,
// 32 q / 4 kv heads: 570 us, 486 TFLOP/s (729 counting both parts of P).
template <typename T, int F, int D, bool P16, bool PS>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void k_paged8_rows(Paged8Args pa) {
  constexpr int KT = 64, TT = KT / 32;
  constexpr int KS = D / 16, DT = D / 32, CH = D / 8;
  constexpr int LPR = D / 16;        // lanes per key (16 bytes each)
  constexpr int NL = 16 * LPR / 64;  // load instructions per wave and tile
  constexpr int NP = 2;
  constexpr float kStep = 8.0f;
  constexpr bool kScaled = PS || !P16;
  __shared__ uint4 sk[2][KT * CH];
  __shared__ uint4 sv[2][KT * CH];
  __shared__ float ssk[kScaled ? 2 : 1][KT];  // scale * log2 e * s_k, and s_v
  __shared__ float ssv[kScaled ? 2 : 1][KT];
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
  // (a sequence's last rows see most keys and start first)
  const int tl = (rows + 127) / 128 - 1 - tile.tl;

  // this lane's query row and its last visible key
  const int rr = tl * 128 + 32 * w + l32;
  const bool rvalid = rr < rows;
  const int qi = (rvalid ? rr : rows - 1) / a.G;
  const int64_t tok = sq.q0 + qi;
  const int hq = h * a.G + (rvalid ? rr : rows - 1) % a.G;
  const int lim = nk - nq + qi;
  // the wave's first and last visible keys' bounds (wave-uniform)
  const int r0 = min(tl * 128 + 32 * w, rows - 1);
  const int r1 = min(tl * 128 + 32 * w + 31, rows - 1);
  const int lim_lo = __builtin_amdgcn_readfirstlane(nk - nq + r0 / a.G);
  const int lim_hi = __builtin_amdgcn_readfirstlane(nk - nq + r1 / a.G);
  // keys past the last row of the tile are visible to none of its rows
  const int last_row = min(tl * 128 + 127, rows - 1);
  const int k1 = __builtin_amdgcn_readfirstlane(
      min(min(k0 + tile.chunk, nk), max(nk - nq + last_row / a.G + 1, 0)));

  // (fixed scales: one factor, its sign in q, so that the largest score is that of the
  // largest product)
  const float signed_scale = a.scale_log2 * fixed_scale(pa.ks, h);
  // (not 0, by which a masked score would be NaN: by 2^-149 no score reaches 2^-21)
  const float scale = kScaled ? signed_scale
                              : signed_scale == 0.0f ? 0x1p-149f : fabsf(signed_scale);
  const uint32_t flip = !kScaled && signed_scale < 0.0f ? 0x80008000u : 0u;
  typename T::vec8 qb[KS];
  {
    const uint16_t* qp = static_cast<const uint16_t*>(a.q) + tok * a.qst +
                         static_cast<int64_t>(hq) * a.qhs + 8 * half;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const uint4 x = ld16(qp + 16 * s);
      qb[s] = as_vec8<T>(rvalid ? make_uint4(x.x ^ flip, x.y ^ flip, x.z ^ flip, x.w ^ flip)
                                : zero4());
    }
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

  // the lane's row of a load (d = 128: in an order in which the eight lanes of a row and
  // the next eight write to banks of their own, rows 0 4 1 5 2 6 3 7)
  const int lrow = D == 128 ? 4 * ((lane >> 3) & 1) + (lane >> 4) : lane / LPR;
  // 16 bytes per lane of the wave's 16 keys, and lane i's scales (every 16 lanes)
  uint4 kr[NL], vr[NL];
  float kscr = 1.0f, vscr = 1.0f;
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
        const int r = q * (64 / LPR) + lrow;
        kr[q] = ld16(kp + static_cast<uint32_t>(r * static_cast<int>(a.kcs) + 16 * (lane % LPR)));
        vr[q] = ld16(vp + static_cast<uint32_t>(r * static_cast<int>(a.vcs) + 16 * (lane % LPR)));
      }
      if constexpr (PS) {
        kscr = kss[pg * pa.ks.sb + in + (lane & 15)];
        vscr = vss[pg * pa.vs.sb + in + (lane & 15)];
      }
    } else {
#pragma unroll
      for (int q = 0; q < NL; ++q) {
        const int key = min(base + 16 * w + q * (64 / LPR) + lrow, nk - 1);
        const int64_t pg = paged_page<false>(a, row, key, bad);
        const int64_t in = key % a.bs;
        kr[q] = ld16(kc + pg * a.kcb + in * a.kcs + 16 * (lane % LPR));
        vr[q] = ld16(vc + pg * a.vcb + in * a.vcs + 16 * (lane % LPR));
      }
      if (pa.ks.slot || pa.vs.slot) {
        const int key = min(base + 16 * w + (lane & 15), nk - 1);
        const int64_t pg = paged_page<false>(a, row, key, bad);
        if (pa.ks.slot) kscr = kss[pg * pa.ks.sb + key % a.bs];
        if (pa.vs.slot) vscr = vss[pg * pa.vs.sb + key % a.bs];
      }
    }
  };
  // widened into buffer `buf`; V and its scales of slots past the sequence are 0
  // (they may hold anything)
  auto store = [&](int base, int buf) {
#pragma unroll
    for (int q = 0; q < NL; ++q) {
      const int r = 16 * w + q * (64 / LPR) + lrow;
      const int c0 = r * CH + ((2 * (lane % LPR)) ^ swz<D>(r));
      const uint4 u = kr[q], v = base + r < nk ? vr[q] : zero4();
      sk[buf][c0] = widen8<T, F>(u.x, u.y);
      sk[buf][c0 ^ 1] = widen8<T, F>(u.z, u.w);
      sv[buf][c0] = widen8<BF16, F>(v.x, v.y);
      sv[buf][c0 ^ 1] = widen8<BF16, F>(v.z, v.w);
    }
    if (kScaled && lane < 16) {
      ssk[buf][16 * w + lane] = scale * kscr;
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
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int t4 = 0; t4 < TT; ++t4) {
          const int r = 32 * t4 + l32;
          const uint4 kop = sk[buf][r * CH + ((2 * ks + half) ^ swz<D>(r))];
          s[t4] = T::mfma32(as_vec8<T>(kop), qb[ks], ks == 0 ? f32x16{} : s[t4]);
        }
      if constexpr (kScaled) {
#pragma unroll
        for (int t4 = 0; t4 < TT; ++t4)
#pragma unroll
          for (int g4 = 0; g4 < 4; ++g4) {
            const float4 f =
                *reinterpret_cast<const float4*>(&ssk[buf][32 * t4 + 8 * g4 + 4 * half]);
            s[t4][4 * g4] *= f.x;
            s[t4][4 * g4 + 1] *= f.y;
            s[t4][4 * g4 + 2] *= f.z;
            s[t4][4 * g4 + 3] *= f.w;
          }
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
      mx = pair32_max(mx);
      if constexpr (!kScaled) mx *= scale;
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
      const float ms = m_run == -INFINITY ? 0.0f : m_run;
#pragma unroll
      for (int t4 = 0; t4 < TT; ++t4) {
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const float x = kScaled ? s[t4][v] - ms : fmaf(s[t4][v], scale, -ms);
          s[t4][v] = __builtin_amdgcn_exp2f(x);
          l_part += s[t4][v];
        }
        if constexpr (kScaled) {
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
          __builtin_amdgcn_sched_barrier(0);
          typename BF16::vec8 va[DT];
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) va[dt] = read_vt<BF16, D>(sv16, r, 32 * dt + tr_col);
          // (a dim tile's two products apart: the second would wait for the first)
#pragma unroll
          for (int p = NP - 1; p >= 0; --p)
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) o[dt] = BF16::mfma32(va[dt], pb[p], o[dt]);
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
    // P (at most 2^kStep) and l 2^off times smaller (m larger): the sum of P V then stays
    // below the largest value, as that of normalised weights does
    const float off = static_cast<float>(32 - __clz(k1 - k0)) + kStep;
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
      d = pair32_sum(d) * (kScaled && pa.ks.slot ? scale * kss[pg * pa.ks.sb + in] : scale);
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
hipError_t launch_rows_t(const Paged8Args& p, int64_t tiles, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(tiles * p.a.Hkv), static_cast<unsigned>(p.a.nc)), b(256);
  if (p.a.bs % 16 != 0 || p.ks.slot != p.vs.slot)
    hipLaunchKernelGGL((k_paged8_rows<T, F, D, false, false>), grid, b, 0, s, p);
  else if (p.ks.slot)
    hipLaunchKernelGGL((k_paged8_rows<T, F, D, true, true>), grid, b, 0, s, p);
  else
    hipLaunchKernelGGL((k_paged8_rows<T, F, D, true, false>), grid, b, 0, s, p);
  return hipGetLastError();
}

template <typename T, int F, int D, int HP>
hipError_t launch_few_t(const Paged8Args& p, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(p.a.nc)), b(256);
  if (p.a.bs % 16 != 0 || p.ks.slot != p.vs.slot)
    hipLaunchKernelGGL((k_paged8<T, F, D, false, false, HP>), grid, b, 0, s, p);
  else if (p.ks.slot)
    hipLaunchKernelGGL((k_paged8<T, F, D, true, true, HP>), grid, b, 0, s, p);
  else
    hipLaunchKernelGGL((k_paged8<T, F, D, true, false, HP>), grid, b, 0, s, p);
  if (p.a.part != nullptr)
    hipLaunchKernelGGL((k_paged8_merge<T, D, HP>), dim3(static_cast<unsigned>(p.segs * HP)),
                       dim3(1024), 0, s, p);
  return hipGetLastError();
}

hipError_t launch_paged8(const Paged8Args& p, int dtype, int format, int head_dim, bool rows,
                         int64_t tiles, hipStream_t s) {
  const auto run = [&](auto t, auto f) -> hipError_t {
    using T = decltype(t);
    constexpr int F = decltype(f)::value;
    if (!rows)
      return with_head_dim(head_dim, [&](auto d) {
        constexpr int D = decltype(d)::value;
        if constexpr (D == 64) {
          if (p.groups < p.a.Hkv) return launch_few_t<T, F, D, 2>(p, s);
        }
        return launch_few_t<T, F, D, 1>(p, s);
      });
    const hipError_t e = with_head_dim(
        head_dim, [&](auto d) { return launch_rows_t<T, F, decltype(d)::value>(p, tiles, s); });
    if (e != hipSuccess || p.a.nc <= 1) return e;
    return launch_paged_merge8(p.a, dtype, head_dim, s);
  };
  if (dtype == FP_DTYPE_BF16)
    return format == FP_CACHE_E4M3 ? run(BF16{}, IntC<FP_CACHE_E4M3>{})
                                   : run(BF16{}, IntC<FP_CACHE_E5M2>{});
  return format == FP_CACHE_E4M3 ? run(F16{}, IntC<FP_CACHE_E4M3>{})
                                 : run(F16{}, IntC<FP_CACHE_E5M2>{});
}

}  // namespace fp

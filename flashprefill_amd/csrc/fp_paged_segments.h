// How few query rows over a paged cache of 8- or 4-bit values are shared out
// (fp_paged8.hip, fp_paged4.hip): the segments of a call, the workgroups' shares of their
// keys, and the merge of the segments that several workgroups served (k_paged8_merge,
// k_paged4_merge).
#pragma once

#include "fp_float8.h"
#include "fp_paged_common.h"

namespace fp {

// A segment is 16 rows of the queries of one (sequence, KV head or pair of them) with all
// its keys, in units of `unit` keys; the segments of a call lie behind each other
// (sequence, heads, row tile) and every workgroup takes an equal share of the units, whatever segments
// they belong to: a decode step reads each cached byte once, so equal bytes take equal
// times, and no workgroup starts for keys that are not there (the host cannot see the
// lengths without a synchronisation). A share is a whole number of units, so that a call of
// few leaves workgroups without any: 1,620 units are four for each of 405 workgroups of 512,
// 2,152 five for each of 431, 13,728 twenty-seven for each of 509. A segment that is one workgroup's is written out,
// the others as partials (O, m, l), the first and the last of a workgroup at most, which
// merge_segments combines. Where the table has room for few keys, a unit is a whole
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

// One head of a segment per workgroup of 16 waves: its rows' partials, weighted by
// exp2(m - max m) and divided by their l. They are the first of workgroups w0 + 1 .. w1
// and the first or last of w0. As many waves as there are share a row's partials.
// SPLIT (the 4-bit form): a segment's rows are shared by the gridDim.y workgroups (a power of
// two) of its head, each of which takes every gridDim.y-th.
template <typename T, int D, int HP, bool SPLIT = false>
__device__ __forceinline__ void merge_segments(const Paged8Args& pa) {
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
  if (n == 1) return;  // written already
  const int h = seg / tiles * HP + hh, tl = seg % tiles;
  const int first_row = SPLIT ? static_cast<int>(blockIdx.y) : 0;
  const int row_step = SPLIT ? static_cast<int>(gridDim.y) : 1;
  int rows = min(work.s.nq * a.G - 16 * tl, 16);
  if constexpr (SPLIT) rows = (rows - first_row + row_step - 1) / row_step;
  if (SPLIT && rows <= 0) return;
  const int lgr = rows > 1 ? 32 - __clz(rows - 1) : 0;  // rows as a power of two
  const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int row = w & ((1 << lgr) - 1), share = 16 >> lgr;
  const float vs = fixed_scale(pa.vs, h);
  if (row < rows) {
    const int first = 2 * w0 + (x0 != w0 * work.share);
    const auto part = [&](int j) {
      return static_cast<int64_t>(((j == 0 ? first : 2 * (w0 + j)) * HP + hh) * 16 +
                                  first_row + row * row_step);
    };
    float M = -INFINITY, L = 0.0f;
    vec acc{};
    if constexpr (SPLIT) {
      // What a row needs is on its way at once, since each trip is 1 to 2 us (other XCDs have
      // just written it): a wave's lanes hold the weights of up to 64 of its partials, U
      // of which are loaded at a time (past the last one, that again: its weight is 0 there).
      // 256 rows of up to 14 partials: 6.0 us, loaded in three trips 7.0; 32 rows of 512
      // partials 11.2 and 11.6 (one CU's loads of each, 128 KB).
      constexpr int MM = (kPaged4Groups + 63) / 64;
      const int j0 = w >> lgr, mine = j0 < n ? (n - 1 - j0) / share + 1 : 0;
      // a row's partials lie `step` rows apart, but for the first, a workgroup's last, `odd`
      // behind its place (fewer than 2 kPaged4Groups x 4 x 16 rows in all)
      constexpr uint32_t step = 2 * HP * 16;
      const uint32_t row0 = (2 * w0 * HP + hh) * 16 + first_row + row * row_step;
      const uint32_t odd = (first & 1) * HP * 16;
      const auto at = [&](int j) {
        return row0 + static_cast<uint32_t>(j) * step + (j == 0 ? odd : 0u);
      };
      const auto run = [&](auto uc) {
        constexpr int U = decltype(uc)::value, MU = U <= 4 ? 1 : MM;
        vec x[U];
        float m[MU], ml, l, f;
        const uint32_t gap = share * step, last = at(j0 + share * (mine - 1));
        const auto weights = [&](int k0) {
          const uint32_t p = at(j0 + share * min(k0 + lane, mine - 1));
          ml = a.ml[2 * p];
          l = a.ml[2 * p + 1];
        };
        const auto load = [&](int k) {
          uint32_t p = row0 + (j0 + share * k) * step;
#pragma unroll
          for (int i = 0; i < U; ++i) {
            const uint32_t r = i == 0 && k == 0 ? at(j0) : min(p, last);
            x[i] = *reinterpret_cast<const vec*>(a.part + (r * D + XD * lane));
            p += gap;
          }
        };
        const auto weigh = [&](int k0) {
          const bool in = k0 + lane < mine;
          // (2^-10: the sum over the partials, at most 768, stays finite)
          static_assert(kPaged4Groups <= 1024, "weights");
          f = ml == -INFINITY || !in ? 0.0f : 0x1p-10f * __builtin_amdgcn_exp2f(ml - M);
          L += !in ? 0.0f : ml == -INFINITY ? l : f * l;
        };
        const auto add = [&](int k) {
#pragma unroll
          for (int i = 0; i < U; ++i) {
            const float fi =
                __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f), (k + i) & 63));
            // (partials are finite, or the row is NaN)
#pragma unroll
            for (int q = 0; q < XD; ++q) acc[q] = fmaf(fi, x[i][q], acc[q]);
          }
        };
#pragma unroll
        for (int i = 0; i < MU; ++i) m[i] = a.ml[2 * at(min(lane + 64 * i, n - 1))];
        weights(0);
        load(0);
        asm volatile("" ::: "memory");
#pragma unroll
        for (int i = 0; i < MU; ++i) M = fmaxf(M, m[i]);
        M = wave_max(M);
        weigh(0);
        add(0);
        for (int k = U; k < mine; k += U) {
          if (k % 64 == 0) weights(k);
          load(k);
          if (k % 64 == 0) weigh(k);
          add(k);
        }
      };
      if (mine > 0) {
        if (n <= 64 && mine <= 4) run(IntC<4>{});
        else run(IntC<XD == 1 ? 16 : 8>{});
      }
      L = static_cast<float>(wave_sum_d(L));
    } else {
      for (int j = lane; j < n; j += 64) M = fmaxf(M, a.ml[2 * part(j)]);
      M = wave_max(M);
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
    }
#pragma unroll
    for (int q = 0; q < XD; ++q) so[w][XD * lane + q] = acc[q];
    if (lane == 0) sl[w] = L;
  }
  __syncthreads();
  for (int i = t; i < rows * D; i += 1024) {
    const int r = i / D, d = i % D;
    float o = 0.0f, L = 0.0f;
    for (int k = r; k < 16; k += 1 << lgr) {
      o += so[k][d];
      L += sl[k];
    }
    const int rr = 16 * tl + first_row + r * row_step;
    static_cast<uint16_t*>(a.o)[(work.s.q0 + rr / a.G) * a.ost +
                                static_cast<int64_t>(h * a.G + rr % a.G) * a.ohs + d] =
        T::from_f32(o / L * vs);
  }
}

}  // namespace fp

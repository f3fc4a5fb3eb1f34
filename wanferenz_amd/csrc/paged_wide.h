// paged_attn for trees with more than 64 rows of queries a KV head (heads of 64 and 128), where the products count as
// much as the cache: a worker is 4 or 8 waves of 32 rows each, which share tiles of 64 tokens.
//
// A wave's row tile is that of V_MFMA_F32_32X32X16: lane (row n, half h) of S^T = K Q^T holds tokens 8 j + 4 h + i, which
// are the k slots of its P operand in O^T += V^T P^T, so P stays in the lane, and a row's statistics are met by one swap
// of the wave's halves.  Two waves a SIMD: one's matrix instructions run beside the other's exponentials, whose
// time is about the same.  Every wave reads all of a tile from LDS (K and V once for its 32 rows), which takes as long as the
// products of bf16 rows; 64 rows a wave would halve that, and leave one wave a SIMD with nothing beside it.
//   * the loads fill a ring of NS tiles in LDS directly; a wave has T / NW rows of a tile, which lie in one page;
//   * one barrier a tile: a tile that a wave's loads have brought is there for all behind it, and the tile before it is free;
//   * p = 2^(y - m) as in paged_attn_kernel, m moved only when a tile's maximum exceeds it by more than 8.
// Units, shares, partials and the join are paged_attn_kernel's, but that units without a row of a sequence's own nodes are none.
// 8 trees of 64 nodes over 8191 tokens, 64 heads on 8 of 128 (268 MB, 137 GF) 157 to 195 us by card, mostly 161: 850 TFLOP/s,
// the matrix units busy two fifths of it, the vector units as long; a product of 8192^3 by the library does 1218.
#pragma once

#include <cfloat>

#include "paged_attn.h"

namespace wz {

typedef float pv16f __attribute__((ext_vector_type(16)));

constexpr int kWideTile = 64;

template <int D, bool FP8, bool SHARED, int NW>
struct WideCfg {
  static constexpr int RB = D * (FP8 ? 1 : 2);
  static constexpr int SIDE = kWideTile * RB;
  static constexpr int STAGE = SIDE * (SHARED ? 1 : 2);
  static constexpr int SCALES = FP8 ? 8 * kWideTile : 0;  // a tile's K and V scales
  static constexpr int RPW = kWideTile / NW;      // rows that a wave loads of each side
  static constexpr int LPS = RPW * RB / 1024;     // loads of them
  static constexpr int LOADS = LPS * (SHARED ? 1 : 2) + (FP8 ? 1 : 0);
  static constexpr int ROWS = 32 * NW;
  static constexpr int PER_CU = 8 / NW;                   // two waves a SIMD
  static constexpr int FIT = 150 * 1024 / PER_CU / (STAGE + SCALES);
  static constexpr int NS = FIT < 6 ? FIT : 6;
  static constexpr int RING = NS * (STAGE + SCALES);
  static constexpr int LDS = RING + NS * 8;  // valid masks
  static_assert(LPS * 1024 == RPW * RB && LPS >= 1 && NS >= 2 && NS * LOADS < 64, "whole loads, counted by the waits");
  static_assert(RPW <= 16 && RPW >= 8, "a wave's rows lie in one page, and fill bytes of the mask");
};

// 16-byte chunk c of row r at slot c ^ swz(r).  The fragments' 16-byte reads take one chunk of 32 rows, the transposing ones four
// neighbouring chunks (two of e4m3) of eight rows; both meet every bank equally often.
template <int RB>
__device__ __forceinline__ int wide_swz(int row) {
  if constexpr (RB == 256) return (row & 3) << 2 | ((row >> 2) & 3);
  if constexpr (RB == 128) return ((row >> 1) & 1) << 2 | ((row >> 2) & 3);
  return (row >> 2) & 3;
}

__device__ __forceinline__ pv16f wide_mfma(pv8s a, pv8s b, pv16f c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(pv8bf, a), __builtin_bit_cast(pv8bf, b), c, 0, 0, 0);
}

// The larger and the sum of a lane's value and that of the lane 32 apart.
__device__ __forceinline__ float wide_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float wide_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Units of a sequence that hold rows of its nodes, and all of their cost; paged_total and paged_find over them.
template <int ROWS>
__device__ __forceinline__ int wide_live(const PagedAttnArgs& a, int b) {
  return a.c.heads * ((paged_nodes(a, b) * (a.H / a.c.heads) + ROWS - 1) / ROWS);
}
template <int ROWS>
__device__ __forceinline__ int wide_cost(const PagedAttnArgs& a, int b) {
  return b < a.B ? paged_cost<kWideTile, kPagedStart>(paged_len(a, b)) * wide_live<ROWS>(a, b) : 0;
}
template <int ROWS>
__device__ __forceinline__ int wide_total(const PagedAttnArgs& a) {
  const int lane = threadIdx.x & 63;
  int sum = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) sum += wide_cost<ROWS>(a, b0 + lane);
  for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o, 64);
  return __builtin_amdgcn_readfirstlane(sum);
}
template <int ROWS>
__device__ __forceinline__ void wide_find(const PagedAttnArgs& a, int x, int* seq, int* before) {
  const int lane = threadIdx.x & 63;
  int sum = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const int g = wide_cost<ROWS>(a, b0 + lane);
    int inc = g;
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(inc, o, 64);
      if (lane >= o) inc += y;
    }
    const uint64_t past = __ballot(sum + inc > x);
    if (past) {
      const int l = __builtin_ctzll(past);
      *seq = b0 + l;
      *before = __builtin_amdgcn_readlane(sum + inc - g, l);
      return;
    }
    sum += __builtin_amdgcn_readlane(inc, 63);
  }
  *seq = a.B - 1;  // not reached: x is below the total
  *before = sum;
}

// The rows that are no node's, of the sequences w, w + a.W, ...: zeros, and no parts of the units that hold nothing else.
template <int ROWS>
__device__ __forceinline__ void wide_empty(const PagedAttnArgs& a, int w, int RG, int D) {
  const int grp = a.H / a.c.heads, upb = a.c.heads * RG;
  for (int b = w; b < a.B; b += a.W) {
    const int nodes = paged_len(a, b) > 0 ? paged_nodes(a, b) : 0, live = (nodes * grp + ROWS - 1) / ROWS;
    const int64_t node = int64_t(a.H) * (D / 8), end = (int64_t(b) + 1) * a.S * node;
    for (int64_t i = (int64_t(b) * a.S + nodes) * node + threadIdx.x; i < end; i += blockDim.x)
      *reinterpret_cast<v4i*>(a.o + i * 8) = v4i{0, 0, 0, 0};
    if (a.by_unit)
      for (int u = threadIdx.x; u < upb; u += blockDim.x)
        if (u % RG >= live) a.cut[int64_t(b) * upb + u] = PagedCut{b, u, 0, 0};
  }
}

template <int D, bool FP8, bool SHARED, int NW>
__global__ __launch_bounds__(64 * NW, 2) void paged_wide_kernel(PagedAttnArgs a) {
  using C = WideCfg<D, FP8, SHARED, NW>;
  constexpr int NS = C::NS, RB = C::RB, ROWS = C::ROWS, T = kWideTile;
  constexpr int KC = D / 16, NT = D / 32, CH = RB / 16;
  extern __shared__ __align__(1024) uint8_t lds[];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  uint8_t* const scales = lds + NS * C::STAGE;
  uint8_t* const s_valid = lds + C::RING;  // a bit a token, RPW bits a wave
  const uint32_t ring_lds = lds_addr(lds), scales_lds = lds_addr(scales);
  auto meet = [] { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };  // loads stay in flight

  const int grp = a.H / a.c.heads, R = a.S * grp, RG = (R + ROWS - 1) / ROWS, upb = a.c.heads * RG;
  const int w = blockIdx.x;
  wide_empty<ROWS>(a, w, RG, D);
  const PagedShares shares(wide_total<ROWS>(a), a.W);
  if (!a.by_unit && tid == 0) a.cut[w] = PagedCut{0, 0, 0, 0};
  if (w >= shares.workers) return;
  int x = shares.begin(w);
  const int x_end = shares.begin(w + 1);
  int b, before;  // sequence, and the granules before it
  wide_find<ROWS>(a, x, &b, &before);
  int n = __builtin_amdgcn_readfirstlane(paged_len(a, b)), cost = paged_cost<T, kPagedStart>(n);
  int live = __builtin_amdgcn_readfirstlane(wide_live<ROWS>(a, b));
  int u = (x - before) / cost, ubeg = before + u * cost;  // of the sequence's live units, and where it begins
  const int ps = a.c.shift, page = a.c.page;
  // the largest of the raw products is the largest of the scaled ones too: a negative scale turns Q's signs
  const float scale2 = a.scale2 == 0.0f ? FLT_MIN : fabsf(a.scale2);  // (masked products are -inf times it)
  const int flip = a.scale2 < 0.0f ? int(0x80008000u) : 0;

  auto next = [&] {  // the next unit that holds anything
    ubeg += cost;
    if (ubeg >= x_end) return false;
    x = ubeg;
    if (++u == live) {
      do {
        ++b;
        n = __builtin_amdgcn_readfirstlane(paged_len(a, b));
        live = __builtin_amdgcn_readfirstlane(wide_live<ROWS>(a, b));
      } while (n == 0 || live == 0);
      cost = paged_cost<T, kPagedStart>(n);
      u = 0;
    }
    return true;
  };
  // Of the two waves of a SIMD one goes first: its exponentials then run beside the other's products.  Taking turns they would do
  // the same at the same time.
  if (wave >= 4) __builtin_amdgcn_s_setprio(1);
  for (bool more = true; more; more = next()) {
    int lane = tid & 63;
    asm volatile("" : "+v"(lane));  // the lane's coordinates, made anew for each part
    const int nl = lane & 31, h = lane >> 5;
    // this worker's granules of the unit
    const int g0 = max(x - ubeg - kPagedStart, 0), g1 = min(x_end - ubeg, cost) - kPagedStart;
    if (g1 <= 0) continue;
    const bool whole = g0 == 0 && g1 == cost - kPagedStart;
    const int lrg = live / a.c.heads, hk = u / lrg, rg = u - hk * lrg;
    const int row0 = rg * ROWS + 32 * wave;  // this wave's first row
    const int t0 = g0 * T, tm = min(g1 * T, n);
    // the tree's tokens, from n0 on, are seen by some rows only (as in paged_attn_kernel)
    const int nodes = __builtin_amdgcn_readfirstlane(paged_nodes(a, b)), n0 = n - nodes;
    const bool busy = row0 < nodes * grp;  // or the wave has no row of the sequence's nodes
    const uint64_t masks = tm > n0 ? paged_tree_masks(a, b, nodes, lane) : 0ull;
    const int rq = min(row0 + nl, R - 1);  // this lane's row
    int odd0 = 0, odd1 = 0;
    if (g0 == 0 && tid == 0 && (a.by_unit || !whole))
      a.cut[a.by_unit ? int64_t(b) * upb + hk * RG + rg : w] =
          PagedCut{b, hk * RG + rg, whole ? 1 : shares.owner(ubeg + cost - 1) - w + 1, w};
    const int32_t* const trow = a.table + int64_t(b) * a.width;

    // ---- loads ----
    const int nk = (tm - t0 + T - 1) / T;
    const int wrow = C::RPW * wave;  // this wave's first row of a tile's loads
    int ids = -1, ids_base = 0;  // lane e: the page of this wave's rows of tile base + e
    auto fetch_ids = [&](int k0) {
      ids_base = k0;
      const int t = t0 + T * (k0 + lane) + wrow;
      int id = -1;
      if (k0 + lane < nk && t < tm) id = trow[t >> ps];
      ids = uint32_t(id) < uint32_t(a.c.pages) ? id : -1;
    };
    auto issue = [&](int k, int stage) {
      if (k - ids_base >= 64) fetch_ids(k);
      const int id = __builtin_amdgcn_readlane(ids, k - ids_base);
      const int t = t0 + T * k + wrow;
      const uint32_t valid = id < 0 ? 0u : tm - t >= C::RPW ? (1u << C::RPW) - 1u : (1u << max(tm - t, 0)) - 1u;
      if (lane == 0) {
        if constexpr (C::RPW == 8) s_valid[8 * stage + wave] = uint8_t(valid);
        else *reinterpret_cast<uint16_t*>(s_valid + 8 * stage + wrow / 8) = uint16_t(valid);
      }
      const int64_t row = (int64_t(max(id, 0)) * a.c.heads + hk) * page + (t & (page - 1));
      const int rin = lane / CH, slot = lane % CH;
      auto load = [&](const uint8_t* pool, int side) {
        const uint32_t dst = __builtin_amdgcn_readfirstlane(ring_lds + stage * C::STAGE + side * C::SIDE + wrow * RB);
#pragma unroll
        for (int j = 0; j < C::LPS; ++j) {
          const int r = j * (1024 / RB);  // of the wave's rows; the swizzle goes by the tile's
          const uint32_t voff = uint32_t(rin * RB + ((slot ^ wide_swz<RB>(wrow + r + rin)) << 4));
          paged_load16(pool + (row + r) * RB, voff, dst + j * 1024);
        }
      };
      load(a.c.k, 0);
      if constexpr (!SHARED) load(a.c.v, 1);
      if constexpr (FP8) {  // K's with the first RPW lanes, V's with the next
        const uint32_t sdst = __builtin_amdgcn_readfirstlane(scales_lds + stage * C::SCALES + 8 * wrow);
        if (lane < 2 * C::RPW) paged_load4((lane >= C::RPW ? a.c.vs : a.c.ks) + row + lane % C::RPW, sdst);
      }
    };
    if (nk > 0) fetch_ids(0);

    // ---- Q: lane (row n, half h) of step cc: d 16 cc + 8 h + e; e4m3 rows are read 16 codes at a time, so there steps 2 p and
    // 2 p + 1 have d 32 p + 16 h + e and + 8 ----
    pv8s qf[KC];
    {
      const uint16_t* const qrow = a.q + b * a.qb + (rq / grp) * a.qs + (hk * grp + rq % grp) * a.qh;
#pragma unroll
      for (int cc = 0; cc < KC; ++cc) {
        v4i q = load16(qrow + (FP8 ? 32 * (cc >> 1) + 16 * h + 8 * (cc & 1) : 16 * cc + 8 * h));
#pragma unroll
        for (int i = 0; i < 4; ++i) q[i] ^= flip;
        qf[cc] = __builtin_bit_cast(pv8s, q);
      }
    }
    pv16f acc[NT];  // acc[nt][i] = O[row n][32 nt + 8 (i >> 2) + 4 h + (i & 3)]
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) acc[nt] = pv16f(0.0f);
    float m_run = -INFINITY, l_run = 0.0f;

    __builtin_amdgcn_s_waitcnt(vmcnt_only(0));  // Q and the ids too: no wait for them is left inside the loop
#pragma unroll
    for (int k = 0; k < NS - 1; ++k)
      if (k < nk) issue(k, k);

    int stage = 0;
#pragma unroll 1
    for (int k = 0; k < nk; ++k) {
      if (k + NS - 2 < nk) __builtin_amdgcn_s_waitcnt(vmcnt_only((NS - 2) * C::LOADS));
      else __builtin_amdgcn_s_waitcnt(vmcnt_only(0));
      meet();  // every wave's part of tile k has landed, and tile k - 1 has been read out of its stage
      if (k + NS - 1 < nk) issue(k + NS - 1, stage == 0 ? NS - 1 : stage - 1);
      uint8_t* const kt = lds + stage * C::STAGE;
      uint8_t* const vt = SHARED ? kt : kt + C::SIDE;
      const float* const sc = reinterpret_cast<const float*>(scales + stage * C::SCALES);
      uint64_t valid = uint64_t(paged_uniform(*reinterpret_cast<const int64_t*>(s_valid + 8 * stage)));
      const int tk = t0 + T * k;
      // where token t's scale stands
      auto scale_at = [](int t, int side) { return t / C::RPW * 2 * C::RPW + side * C::RPW + t % C::RPW; };
      const bool last = tk + T > n0;
      if (last) {
        const uint64_t some = valid & ~((1ull << max(n0 - tk, 0)) - 1ull);  // tokens that some rows see
        bool odd = false;  // every wave looks at all of them, and comes to the same
        for (int i = lane; i < T * CH; i += 64)
          if ((some >> (i / CH)) & 1) odd |= paged_odd<FP8>(*reinterpret_cast<const v4i*>(vt + i * 16));
        if constexpr (FP8) odd |= ((some >> lane) & 1) && !is_finite_f32(sc[scale_at(lane, 1)]);
        if (__ballot(odd)) {
          odd0 = odd1 > 0 ? odd0 : max(n0, tk);
          odd1 = min(tk + T, tm);
          valid &= ~some;
        }
        meet();  // every wave has looked before the rows are cleared
      }
      if (~valid) {
        // rows that hold nothing become zeros, whatever bits their memory has
        for (int i = tid; i < T * CH; i += 64 * NW)
          if (!((valid >> (i / CH)) & 1)) {
            *reinterpret_cast<v4i*>(kt + i * 16) = v4i{0, 0, 0, 0};
            if (!SHARED) *reinterpret_cast<v4i*>(vt + i * 16) = v4i{0, 0, 0, 0};
          }
        meet();
      }
      stage = stage + 1 == NS ? 0 : stage + 1;
      if (!busy) continue;

      // ---- S^T: s[tt][i] = q . k of row n, token 32 tt + 8 (i >> 2) + 4 h + (i & 3) ----
      // Fragments are read kAhead steps ahead of their products: left to the compiler each read stood right before its product.
      constexpr int kAhead = 3;
      pv16f s[2] = {pv16f(0.0f), pv16f(0.0f)};
      {
        constexpr int STEPS = FP8 ? KC / 2 : KC;  // reads of a row
        const uint8_t* const krow = kt + nl * RB;
        const int sw = wide_swz<RB>(nl);
        v4i kf[kAhead + 1];
        auto kload = [&](int j) {  // j = 2 step + tt
          kf[j % (kAhead + 1)] = *reinterpret_cast<const v4i*>(krow + 32 * (j & 1) * RB + (((2 * (j >> 1) + h) ^ sw) << 4));
        };
#pragma unroll
        for (int j = 0; j < kAhead; ++j) kload(j);
#pragma unroll
        for (int j = 0; j < 2 * STEPS; ++j) {
          if (j + kAhead < 2 * STEPS) kload(j + kAhead);
          __builtin_amdgcn_sched_barrier(0);
          const v4i kc = kf[j % (kAhead + 1)];
          if constexpr (!FP8) {
            s[j & 1] = wide_mfma(__builtin_bit_cast(pv8s, kc), qf[j >> 1], s[j & 1]);
          } else {
            s[j & 1] = wide_mfma(paged_widen(kc[0], kc[1]), qf[2 * (j >> 1)], s[j & 1]);
            s[j & 1] = wide_mfma(paged_widen(kc[2], kc[3]), qf[2 * (j >> 1) + 1], s[j & 1]);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      if constexpr (FP8) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const v4f ks = *reinterpret_cast<const v4f*>(sc + scale_at(8 * j + 4 * h, 0));
#pragma unroll
          for (int i = 0; i < 4; ++i) s[j >> 2][4 * (j & 3) + i] *= ks[i];
        }
      }
      // ---- softmax ----
      if (~valid || last) {
        // bit t: this lane's row sees token t of the tile; the nodes' bits begin at n0
        const uint64_t mask = paged_tree_mask(masks, rq / grp);
        const int off = n0 - tk;
        const uint64_t prefix = off >= 64 ? ~0ull : off > 0 ? (1ull << off) - 1ull : 0ull;
        const uint64_t tree = off >= 64 || off <= -64 ? 0ull : off >= 0 ? mask << off : mask >> -off;
        const uint64_t seen = (valid & (prefix | tree)) >> (4 * h);
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) {
          const uint32_t word = uint32_t(seen >> (32 * tt));
#pragma unroll
          for (int i = 0; i < 16; ++i) s[tt][i] = word & (1u << (8 * (i >> 2) + (i & 3))) ? s[tt][i] : -INFINITY;
        }
      }
      float top = s[0][0];
#pragma unroll
      for (int i = 1; i < 32; ++i) top = fmaxf(top, s[i >> 4][i & 15]);
      top = wide_max(top) * scale2;
      const bool bump = top > m_run + kPagedLazy;
      if (__ballot(bump)) {
        const float resc = !bump ? 1.0f : (m_run == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_run - top));
        m_run = bump ? top : m_run;
        l_run *= resc;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) acc[nt] = acc[nt] * resc;
      }
      const float m = m_run == -INFINITY ? 0.0f : m_run;
      pv8s pf[4];  // of 16 tokens: 16 q + 4 h + i, then 16 q + 8 + 4 h + i
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float p[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = __builtin_amdgcn_exp2f(fmaf(s[q >> 1][8 * (q & 1) + i], scale2, -m));
        l_run += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
        if constexpr (FP8) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int t = 16 * q + 8 * j + 4 * h;
            const v4f vs = *reinterpret_cast<const v4f*>(sc + scale_at(t, 1));
#pragma unroll
            for (int i = 0; i < 4; ++i) p[4 * j + i] *= vs[i];
            if (~valid) {  // a row that holds nothing has any scale
              const uint32_t held = uint32_t(valid >> t);
#pragma unroll
              for (int i = 0; i < 4; ++i) p[4 * j + i] = held & (1u << i) ? p[4 * j + i] : 0.0f;
            }
          }
        }
        v4i d;
#pragma unroll
        for (int i = 0; i < 4; ++i) d[i] = int(f32x2_to_bf16x2(p[2 * i], p[2 * i + 1]));
        pf[q] = __builtin_bit_cast(pv8s, d);
      }
      // ---- O^T += V^T P^T, 16 tokens at a time ----
      const int l16 = lane & 15, side = (lane >> 4) & 1;  // column 16 side + l16 of 32
      v4i vf[kAhead + 1];
      auto vload = [&](int j) {  // j = NT q + nt
        const int q = j / NT, nt = j % NT;
        v4i& f = vf[j % (kAhead + 1)];
        if constexpr (!FP8) {
          const int row = 4 * h + (l16 >> 2), c = 4 * nt + 2 * side + ((l16 >> 1) & 1);  // 16 rows on the swizzle is the same
          const pv4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (lds_pv4s*)(vt + (16 * q + row) * RB + ((c ^ wide_swz<RB>(row)) << 4) + (l16 & 1) * 8));
          const pv4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (lds_pv4s*)(vt + (16 * q + row + 8) * RB + ((c ^ wide_swz<RB>(row + 8)) << 4) + (l16 & 1) * 8));
          f = __builtin_bit_cast(v4i, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
          const int row = 4 * h + ((l16 >> 1) & 3) + 8 * (l16 >> 3), c = 2 * nt + side;
          const pv2i c8 = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
              (lds_pv2i*)(vt + (16 * q + row) * RB + ((c ^ wide_swz<RB>(row)) << 4) + (l16 & 1) * 8));
          f[0] = c8[0];
          f[1] = c8[1];
        }
      };
#pragma unroll
      for (int j = 0; j < kAhead; ++j) vload(j);
#pragma unroll
      for (int j = 0; j < 4 * NT; ++j) {
        if (j + kAhead < 4 * NT) vload(j + kAhead);
        __builtin_amdgcn_sched_barrier(0);
        const v4i f = vf[j % (kAhead + 1)];
        acc[j % NT] = wide_mfma(FP8 ? paged_widen(f[0], f[1]) : __builtin_bit_cast(pv8s, f), pf[j / NT], acc[j % NT]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }

    // ---- tokens that only some rows see and whose V is not finite: a row takes nothing from one that it does not see ----
    for (int t = odd0; t < odd1; ++t) {
      const int64_t at = paged_row(a.c, trow, a.width, hk, t);
      if (at < 0) continue;
      const uint8_t* const kr = a.c.k + at * RB;
      const uint8_t* const vr = (SHARED ? a.c.k : a.c.v) + at * RB;
      const float ksc = FP8 ? a.c.ks[at] : 1.0f, vsc = FP8 ? a.c.vs[at] : 1.0f;
      const uint16_t* const qrow = a.q + b * a.qb + (rq / grp) * a.qs + (hk * grp + rq % grp) * a.qh;
      float dot = 0.0f;  // this half's share of the products
      for (int d = 4 * h; d < D; d += 8) {
        const v4f kv = paged_four<FP8>(kr, d);
        const uint2 q = *reinterpret_cast<const uint2*>(qrow + d);
        dot = fmaf(kv[0], bf16lo(q.x), fmaf(kv[1], bf16hi(q.x), fmaf(kv[2], bf16lo(q.y), fmaf(kv[3], bf16hi(q.y), dot))));
      }
      const float y = wide_sum(dot) * ksc * a.scale2;
      const uint64_t mask = paged_tree_mask(masks, rq / grp) >> ((t - n0) & 63);
      if (busy && (mask & 1)) {
        const float m_new = fmaxf(m_run, y);
        const float m = m_new == -INFINITY ? 0.0f : m_new;
        const float resc = m_run == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_run - m);
        const float p = __builtin_amdgcn_exp2f(y - m);
        m_run = m_new;
        l_run = l_run * resc + (h == 0 ? p : 0.0f);
        const float pv = p * vsc;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const v4f v = paged_four<FP8>(vr, 32 * nt + 8 * j + 4 * h);
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[nt][4 * j + i] = fmaf(pv, v[i], acc[nt][4 * j + i] * resc);
          }
      }
    }

    // ---- the part's end ----
    l_run = wide_sum(l_run);
    const int r = row0 + nl;
    if (r < nodes * grp) {  // the rest is zeros already (the join writes them again)
      if (whole) {
        const int head = hk * grp + r % grp, node = r / grp;
        float den = l_run, f = 1.0f;
        if (a.sink) {
          const float sk = a.sink[head] * kLog2e, M = fmaxf(m_run, sk), Me = M == -INFINITY ? 0.0f : M;
          f = m_run == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_run - Me);
          den = den * f + __builtin_amdgcn_exp2f(sk - Me);
        }
        const float inv = den == 0.0f ? 0.0f : f / den;
        uint16_t* const orow = a.o + ((int64_t(b) * a.S + node) * a.H + head) * D + 4 * h;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            *reinterpret_cast<uint2*>(orow + 32 * nt + 8 * j) =
                make_uint2(f32x2_to_bf16x2(acc[nt][4 * j] * inv, acc[nt][4 * j + 1] * inv),
                           f32x2_to_bf16x2(acc[nt][4 * j + 2] * inv, acc[nt][4 * j + 3] * inv));
          }
      } else {
        float* const part = a.part + (2 * int64_t(w) + (g0 == 0 ? 1 : 0)) * paged_slot(a.rows, D);
        const int rl = 32 * wave + nl;
        if (h == 0) {
          part[rl] = m_run;
          part[a.rows + rl] = l_run;
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            *reinterpret_cast<v4f*>(part + paged_head(a.rows) + rl * D + 32 * nt + 8 * j + 4 * h) =
                v4f{acc[nt][4 * j], acc[nt][4 * j + 1], acc[nt][4 * j + 2], acc[nt][4 * j + 3]};
      }
    }
    meet();  // the ring is free for the next part's tiles
  }
}

template <int D, bool FP8, bool SHARED, int NW>
int paged_wide_launch(PagedAttnArgs a, bool ask, int* workers, hipStream_t stream) {
  using C = WideCfg<D, FP8, SHARED, NW>;
  static_assert(C::LDS * C::PER_CU <= 160 * 1024, "a compute unit's LDS");
  const int R = a.S * (a.H / a.c.heads);
  a.W = std::min(cu_count() * C::PER_CU, kPagedMaxWorkers);
  a.unit_rows = C::ROWS;
  a.rows = std::min(R, C::ROWS);
  if (ask) {
    *workers = a.W;
    return a.rows;
  }
  a.by_unit = paged_units(a) <= a.W;
  static LdsGrant grant;
  auto* const kernel = paged_wide_kernel<D, FP8, SHARED, NW>;
  if (int rc = allow_lds("paged_attn", kernel, C::LDS, grant)) return rc;
  WZ_LAUNCH("paged_attn", stream, kernel, dim3{unsigned(a.W)}, dim3(64 * NW), C::LDS, a);
  if (int rc = check_launch("paged_attn")) return rc;
  return paged_attn_join<D>(a, stream);
}

// Rows beyond 64: workers of 4 waves, beyond 128 rows of 128 of 8, which read the cache half as often (8 x 8191 tokens, 512 rows:
// 164 us against 188).  Heads of 64 stay with 4: a tile's time there is one wave's way through it, and two workers a compute unit
// go theirs side by side (24 x 1125 .. 9001 e4m3 tokens, 8 to 192 rows: 65 us against 99).
template <int D, bool FP8, bool SHARED>
int paged_wide(const PagedAttnArgs& a, bool ask, int* workers, hipStream_t stream) {
  if constexpr (D == 128)
    if (a.S * (a.H / a.c.heads) > 128) return paged_wide_launch<D, FP8, SHARED, 8>(a, ask, workers, stream);
  return paged_wide_launch<D, FP8, SHARED, 4>(a, ask, workers, stream);
}

template <bool FP8>
int paged_tree_launch(int D, const PagedAttnArgs& a, bool ask, int* workers, hipStream_t stream) {
  if (a.S * (a.H / a.c.heads) > 64 && !paged_few(a)) {
    if (D == 64 && !a.c.shared) return paged_wide<64, FP8, false>(a, ask, workers, stream);
    if (D == 128 && a.c.shared) return paged_wide<128, FP8, true>(a, ask, workers, stream);
    if (D == 128) return paged_wide<128, FP8, false>(a, ask, workers, stream);
  }
  return paged_attn_launch<FP8, true>(D, a, ask, workers, stream);
}

}  // namespace wz

// Attention of a few new tokens over a paged cache: the kernel, compiled for bf16 and e4m3
// rows by the two sources that include it.
//
// One KV head's rows of queries (the S tokens' heads that share it, R = S H / kv_heads of them) are
// taken in groups of up to 64; a group of a sequence is a unit, and its n cached tokens are granules
// of 32.  All units' granules in a row are cut into one equal share per worker, so the chip is filled
// whatever the lengths: a unit inside one share is finished there, a cut one leaves (m, l, O) partials
// that paged_attn_join_kernel merges.  A worker's share holds at most two cut units, one
// that began before it and one that goes on after it, which own its partial slots 2w and 2w + 1; the
// worker that a cut unit begins in says so.
//
// A worker is one wave, or two that split 64 rows (RH = 2) and the loads.  One wave waits for nobody:
// while it begins a unit or ends one, the compute unit's other workers keep loading.  Tiles of 32 tokens
// go through a ring of NS in LDS that the loads fill directly, without registers:
//   * S^T = K Q^T and O^T += V^T P^T with V_MFMA_F32_16X16X32; lane (row n, group g) of S^T
//     holds tokens 4g + i and 16 + 4g + i, which are the k slots of its P operand, so P never
//     leaves the lane and the softmax statistics are one register a row tile;
//   * y = q . k scale log2(e), p = 2^(y - m), m moved only when a tile's maximum exceeds it by more
//     than 8 (the final quotient does not depend on m); p is rounded to bf16 for the product with V
//     (the sums keep it in 32 bits), which adds as much error as the output's own rounding.
// Reading the cache bounds it: 2 R / element-size flops a byte is far below the matrix units' rate
// for the usual group sizes.  At 5.5 to 5.8 TB/s: 131071 tokens of 8 heads of 128, 32 query heads (537 MB) 93 us, 64
// sequences of 16 to 16384 (647 MB) 118, four new tokens on 16 x 8191 (538 MB) 99 to 102; 48 of 1125 to 9001 e4m3 rows of 64 (207 MB) 44,
// 4.7 TB/s.  What is left is a worker's first tile and its last: 10 us whatever the length.  Latents of 512 have
// a kernel of their own (paged_latent.hip).
#pragma once

#include <algorithm>

#include "paged.h"

namespace wz {

typedef short pv4s __attribute__((ext_vector_type(4)));
typedef short pv8s __attribute__((ext_vector_type(8)));
typedef __bf16 pv8bf __attribute__((ext_vector_type(8)));
typedef __bf16 pv2bf __attribute__((ext_vector_type(2)));
typedef int pv2i __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) pv4s lds_pv4s;
typedef __attribute__((address_space(3))) pv2i lds_pv2i;

constexpr int kPagedTile = 32;           // tokens of a wave's tile
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kPagedLazy = 8.0f;       // the running maximum moves when a tile exceeds it by more
constexpr int kPagedMaxS = 16;
constexpr int kPagedMaxNodes = 64;       // of a tree: a lane each, a bit each
constexpr int kPagedStart = 3;           // a worker's start of a unit, in tiles (paged_cost)

// A unit's parts: np of them (1: nothing to join, 0: no unit), of worker w and those after it.
struct PagedCut {
  int32_t b, u, np, w;
};

struct PagedAttnArgs {
  PagedView c;
  const uint16_t* q;
  int64_t qb, qs, qh;  // elements between sequences, tokens, heads
  const float* sink;
  const int32_t* table;
  const int32_t* lens;
  uint16_t* o;
  float* part;    // 2 W slots of m[rows], l[rows] and O[rows][D] (paged_head, paged_slot)
  PagedCut* cut;  // a unit where by_unit, else the cut unit that begins in a worker's share
  float* ml;      // accumulate: per unit and row the final maximum and 1 / sum
  float* scores;  // accumulate: y [B, heads, R, capacity]
  const int32_t* parent;  // trees: [B, S]
  const int32_t* count;   // trees: nodes of each sequence, or null: S
  int width, B, S, H, W, rows, unit_rows, by_unit;  // rows: of a partial, min(R, unit_rows)
  int64_t capacity;  // slots of the table, width * page
  float scale2;      // softmax scale * log2(e)
};

// Floats of a partial before its O, and in all.  O is stored and read 16 bytes at a time, so with odd rows
// two floats are left out before it.
__host__ __device__ __forceinline__ int paged_head(int rows) { return (2 * rows + 3) & ~3; }
__host__ __device__ __forceinline__ int64_t paged_slot(int rows, int D) { return paged_head(rows) + int64_t(rows) * D; }

static inline int64_t paged_units(const PagedAttnArgs& a) {
  const int R = a.S * (a.H / a.c.heads);
  return int64_t(a.B) * a.c.heads * ((R + a.unit_rows - 1) / a.unit_rows);
}

// Tokens of a sequence, and its granules.
__device__ __forceinline__ int paged_len(const PagedAttnArgs& a, int b) {
  return int(min(int64_t(max(a.lens[b], 0)), a.capacity));
}

// Nodes of a sequence's tree.
__device__ __forceinline__ int paged_nodes(const PagedAttnArgs& a, int b) {
  return a.count ? min(max(a.count[b], 0), a.S) : a.S;
}

// A tree's visibility: bit j of lane i's mask says that node i sees node j, itself or one above it.  Each of six rounds
// doubles the steps up that a mask covers, so the order of the nodes does not matter, and a parent that is no node of the
// tree ends the way up.
__device__ __forceinline__ uint64_t paged_tree_masks(const PagedAttnArgs& a, int b, int nodes, int lane) {
  uint64_t seen = lane < nodes ? 1ull << lane : 0ull;
  int up = lane < nodes ? a.parent[int64_t(b) * a.S + lane] : -1;
  up = uint32_t(up) < uint32_t(nodes) ? up : -1;
  for (int i = 0; i < 6; ++i) {
    const uint32_t lo = __shfl(uint32_t(seen), up & 63, 64), hi = __shfl(uint32_t(seen >> 32), up & 63, 64);
    const int next = __shfl(up, up & 63, 64);
    if (up >= 0) {
      seen |= uint64_t(hi) << 32 | lo;
      up = next;
    }
  }
  return seen;
}
__device__ __forceinline__ uint64_t paged_tree_mask(uint64_t masks, int node) {
  return uint64_t(uint32_t(__shfl(uint32_t(masks >> 32), node, 64))) << 32 | uint32_t(__shfl(uint32_t(masks), node, 64));
}

// What a unit of n tokens counts for: its granules of G, and START more for the time in which a worker
// loads nothing (the query, the pages' ids, the first tile's way).  64 sequences of 16 to 16384 tokens took
// 133 us with START = 0, since some worker had to begin a dozen short ones, and 118 with 3 (128, 119, 118
// with 1, 2, 4).
template <int G, int START>
__device__ __forceinline__ int paged_cost(int n) {
  return n > 0 ? (n + G - 1) / G + START : 0;
}

// All of that: upb units a sequence (the host has checked that it fits 31 bits).  Every lane of a wave
// gets the result; B sequences are summed 64 at a time.
template <int G, int START>
__device__ __forceinline__ int paged_total(const PagedAttnArgs& a, int upb) {
  const int lane = threadIdx.x & 63;
  int sum = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    int g = b0 + lane < a.B ? paged_cost<G, START>(paged_len(a, b0 + lane)) : 0;
    for (int o = 1; o < 64; o <<= 1) g += __shfl_xor(g, o, 64);
    sum += g;
  }
  return __builtin_amdgcn_readfirstlane(sum * upb);
}

// The sequence that holds granule x (0 <= x < total) and the granules before it.
template <int G, int START>
__device__ __forceinline__ void paged_find(const PagedAttnArgs& a, int upb, int x, int* seq, int* before) {
  const int lane = threadIdx.x & 63;
  int sum = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const int g = b0 + lane < a.B ? paged_cost<G, START>(paged_len(a, b0 + lane)) : 0;
    int inc = g;
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(inc, o, 64);
      if (lane >= o) inc += y;
    }
    const uint64_t past = __ballot((sum + inc) * upb > x);  // granules up to and with this lane's sequence
    if (past) {
      const int l = __builtin_ctzll(past);
      *seq = b0 + l;
      *before = __builtin_amdgcn_readlane((sum + inc - g) * upb, l);
      return;
    }
    sum += __builtin_amdgcn_readlane(inc, 63);
  }
  *seq = a.B - 1;  // not reached: x < total
  *before = sum * upb;
}

// The workers' shares: `workers` of them (one granule at least each), the first `rest` one granule longer
// than `each`; where worker w's begins, and who holds granule x.  A total between W and 2 W has shares of two
// anyway, so all get two, and from W / 2 on half the partials to write and join outweigh a granule's time: the
// kernel and the join of 17000 latents of 32 heads 28.3 us with one each, 21.9 with two, 2 x 19247 tokens of one head
// 15.9 and 13.5, 4000 of 8 heads 15.4 and 14.1.  Below that a granule each: 999 tokens of 8 heads 11.2 against
// 11.7, 2 x 200 latents 17.4 against 20.
struct PagedShares {
  int workers, each, rest;
  __device__ __forceinline__ PagedShares(int total, int W)
      : workers(total <= W / 2 ? total : min((total + 1) / 2, W)), each(total / max(workers, 1)), rest(total - each * workers) {}
  __device__ __forceinline__ int begin(int w) const { return w * each + min(w, rest); }
  __device__ __forceinline__ int owner(int x) const {
    const int longer = rest * (each + 1);
    return x < longer ? x / (each + 1) : rest + (x - longer) / each;
  }
};

// LDS image of a tile: rows of RB bytes, 16-byte chunk c of row r at slot c ^ swz(r).  The
// fragments' 16-byte reads of one chunk of 16 rows are served in passes that mix rows 0-3 and 12-15
// with rows 4-11 of the neighbouring chunk; the transpose reads take two adjacent chunks of 8 rows.
template <int RB>
struct PagedRow {
  static constexpr int CH = RB / 16;     // chunks a row
  static constexpr int RPI = 1024 / RB;  // rows a load
  static __device__ __forceinline__ int swz(int row) {
    const int hi = (row >> 3) & 1;
    if constexpr (RB >= 256) return ((row ^ (hi << 2)) & 7) << 1 | hi;
    if constexpr (RB == 128) return ((((row >> 1) & 3) ^ (hi << 1)) << 1) | hi;
    const int q = (row >> 2) & 3;
    return (q << 1 ^ 3 * (q >> 1)) & 3;  // 0, 2, 3, 1
  }
};

// 1 KB straight into LDS, 16 bytes a lane, from a wave-uniform base and a lane's offset.  The
// compiler does not look into the block for hazards, so it waits itself for what the hardware does
// not check: an SGPR that a vector instruction wrote (a readlane) is readable by a load after five
// states, m0 after one.
__device__ __forceinline__ int64_t paged_uniform(int64_t x) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane(uint32_t(x)), hi = __builtin_amdgcn_readfirstlane(uint32_t(x >> 32));
  return int64_t(uint64_t(hi) << 32 | lo);
}
__device__ __forceinline__ void paged_load16(const uint8_t* base, uint32_t voff, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(lds), "v"(voff), "s"(base) : "memory", "m0");
}
// 4 bytes a lane.
__device__ __forceinline__ void paged_load4(const float* p, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" : : "s"(lds), "v"(p) : "memory", "m0");
}

__device__ __forceinline__ v4f paged_mfma(pv8s a, pv8s b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(pv8bf, a), __builtin_bit_cast(pv8bf, b), c, 0, 0, 0);
}

// 8 e4m3 codes as bf16 (exact).
__device__ __forceinline__ pv8s paged_widen(int lo, int hi) {
  union {
    pv2bf p[4];
    pv8s v;
  } u;
  u.p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false);
  u.p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
  u.p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false);
  u.p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
  return u.v;
}

// The sequences without tokens among w, w + a.W, ...: zeros, and nothing to join.
__device__ __forceinline__ void paged_empty(const PagedAttnArgs& a, int w, int upb, int D, int threads) {
  for (int b = w; b < a.B; b += a.W) {
    if (paged_len(a, b) > 0) continue;
    const int64_t chunks = int64_t(a.S) * a.H * (D / 8);
    for (int64_t i = threadIdx.x; i < chunks; i += threads)
      *reinterpret_cast<v4i*>(a.o + (b * chunks + i) * 8) = v4i{0, 0, 0, 0};
    if (a.by_unit)
      for (int u = threadIdx.x; u < upb; u += threads) a.cut[int64_t(b) * upb + u] = PagedCut{b, u, 0, 0};
  }
}

// Whether 16 bytes of V hold an infinity or a NaN.
template <bool FP8>
__device__ __forceinline__ bool paged_odd(v4i v) {
  bool odd = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = uint32_t(v[i]);
    if constexpr (FP8)  // e4m3's NaN: all ones but the sign
      odd |= (w & 0x7Fu) == 0x7Fu || (w & 0x7F00u) == 0x7F00u || (w & 0x7F0000u) == 0x7F0000u || (w & 0x7F000000u) == 0x7F000000u;
    else
      odd |= (w & 0x7F80u) == 0x7F80u || (w & 0x7F800000u) == 0x7F800000u;
  }
  return odd;
}

// One row of Q (bf16) against one row of the cache, this lane group's share g of the products; the rest of
// the row is with the lanes 16 apart.  For the few tokens that not every row sees: Q is read again.
template <int D, bool FP8>
__device__ __forceinline__ float paged_dot(const uint16_t* qrow, const uint8_t* krow, int g) {
  float dot = 0.0f;
#pragma unroll 2
  for (int cc = 0; cc < D / 32; ++cc) {
    const int d = 32 * cc + 8 * g;
    const pv8s q = *reinterpret_cast<const pv8s*>(qrow + d);
    pv8s k;
    if constexpr (FP8) {
      const pv2i c8 = *reinterpret_cast<const pv2i*>(krow + d);
      k = paged_widen(c8[0], c8[1]);
    } else {
      k = *reinterpret_cast<const pv8s*>(krow + 2 * d);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) dot = fmaf(bf16_to_f32(uint16_t(k[i])), bf16_to_f32(uint16_t(q[i])), dot);
  }
  dot += __shfl_xor(dot, 16, 64);
  dot += __shfl_xor(dot, 32, 64);
  return dot;
}

// Four neighbouring values of a row, from column d on.
template <bool FP8>
__device__ __forceinline__ v4f paged_four(const uint8_t* row, int d) {
  if constexpr (FP8) {
    const int c = *reinterpret_cast<const int*>(row + d);
    return v4f{__builtin_amdgcn_cvt_f32_fp8(c, 0), __builtin_amdgcn_cvt_f32_fp8(c, 1), __builtin_amdgcn_cvt_f32_fp8(c, 2),
               __builtin_amdgcn_cvt_f32_fp8(c, 3)};
  } else {
    const uint2 c = *reinterpret_cast<const uint2*>(row + 2 * d);
    return v4f{bf16lo(c.x), bf16hi(c.x), bf16lo(c.y), bf16hi(c.y)};
  }
}

// Sizes of one compiled kernel.
template <int D, bool FP8, bool SHARED, int RT, int RH>
struct PagedCfg {
  static constexpr int RB = D * (FP8 ? 1 : 2);
  static constexpr int SIDE = kPagedTile * RB;                 // one side of a tile
  static constexpr int STAGE = SIDE * (SHARED ? 1 : 2);
  static constexpr int SCALES = FP8 ? 256 : 0;                 // a tile's K and V scales
  static constexpr int NS = 2;                                 // one being read, one on its way
  static constexpr int LOADS = STAGE / 1024 / RH + (FP8 ? 1 : 0);  // a wave's loads of a tile
  static constexpr int WROWS = 16 * RT;                        // rows of a wave
  static constexpr int ROWS = WROWS * RH;                      // rows of a unit
  static constexpr int RING = NS * (STAGE + SCALES);
  static constexpr int LDS = RING + RH * NS * 4;               // valid masks
  // Waves a SIMD.  One of tiles of 8 KB and more keeps the memory busy, and a second adds partial results:
  // 48 sequences of 9001 tokens, 64 heads on 8, us with one / two: bf16 of 64 157 / 160, e4m3 of 128
  // 164 / 172; tiles of 4 KB need two: e4m3 of 64 111 / 91, with three
  // and four 100 / 96 (rings of four tiles 109 / 95).
  static constexpr int EU = STAGE <= 4096 ? 2 : 1;
  static constexpr int PER_CU = 160 * 1024 / LDS < 4 * EU / RH ? 160 * 1024 / LDS : 4 * EU / RH;
  static_assert(NS >= 2 && (NS - 1) * LOADS < 64, "the waits count the loads in flight");
  static_assert(PER_CU >= 1 && SIDE / 1024 % RH == 0, "a worker fits, and its waves share a tile's loads evenly");
};

// TREE: the new tokens are the nodes of a tree, which see the prefix, themselves and the nodes above them.
template <int D, bool FP8, bool SHARED, int RT, int RH, bool TREE>
__global__ __launch_bounds__(64 * RH, (PagedCfg<D, FP8, SHARED, RT, RH>::EU))
void paged_attn_kernel(PagedAttnArgs a) {
  using C = PagedCfg<D, FP8, SHARED, RT, RH>;
  using L = PagedRow<C::RB>;
  constexpr int NS = C::NS, RB = C::RB, ROWS = C::ROWS;
  constexpr int KC = D / 32, NT = D / 16;
  extern __shared__ __align__(1024) uint8_t lds[];
  const int tid = threadIdx.x, rh = RH == 1 ? 0 : __builtin_amdgcn_readfirstlane(tid >> 6);
  uint8_t* const ring = lds;
  uint8_t* const scales = ring + NS * C::STAGE;  // e4m3: 256 bytes a tile
  uint32_t* const s_valid = reinterpret_cast<uint32_t*>(lds + C::RING) + rh * NS;
  const uint32_t ring_lds = lds_addr(ring), scales_lds = lds_addr(scales);
  auto meet = [&]() {  // the worker's waves; loads stay in flight
    if constexpr (RH > 1) asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  };

  const int grp = a.H / a.c.heads, R = a.S * grp, RG = (R + ROWS - 1) / ROWS, upb = a.c.heads * RG;
  const int w = blockIdx.x;
  const PagedShares shares(paged_total<kPagedTile, kPagedStart>(a, upb), a.W);
  if (!a.by_unit && tid == 0) a.cut[w] = PagedCut{0, 0, 0, 0};
  if (w >= shares.workers) {
    paged_empty(a, w, upb, D, 64 * RH);
    return;
  }
  int x = shares.begin(w);
  const int x_end = shares.begin(w + 1);
  int b, before;  // sequence, and the granules before it
  paged_find<kPagedTile, kPagedStart>(a, upb, x, &b, &before);
  int n = __builtin_amdgcn_readfirstlane(paged_len(a, b)), cost = paged_cost<kPagedTile, kPagedStart>(n);
  int u = (x - before) / cost, ubeg = before + u * cost;  // unit of the sequence, and where it begins
  const int ps = a.c.shift, page = a.c.page;
  const int ish = page >= kPagedTile ? 0 : 1;  // page ids a tile: 1 or 2

  auto next = [&] {  // the next unit that holds anything
    ubeg += cost;
    if (ubeg >= x_end) return false;
    x = ubeg;
    if (++u == upb) {
      do {
        ++b;
        n = __builtin_amdgcn_readfirstlane(paged_len(a, b));
      } while (n == 0);
      cost = paged_cost<kPagedTile, kPagedStart>(n);
      u = 0;
    }
    return true;
  };
  for (bool more = true; more; more = next()) {
    // the lane's coordinates, made anew for each part: addresses computed from them stay inside it
    int lane = tid & 63;
    asm volatile("" : "+v"(lane));
    const int nl = lane & 15, g = lane >> 4;
    // this worker's granules of the unit
    const int g0 = max(x - ubeg - kPagedStart, 0), g1 = min(x_end - ubeg, cost) - kPagedStart;
    if (g1 <= 0) continue;
    const bool whole = g0 == 0 && g1 == cost - kPagedStart;
    const int hk = u / RG, rg = u - hk * RG;
    const int row0 = rg * ROWS + rh * C::WROWS;  // this wave's first row
    const int t0 = g0 * kPagedTile, tm = min(g1 * kPagedTile, n);
    // The last S - 1 tokens, from n0 on, are seen by some rows only.  The others' p is 0 there, which keeps
    // a finite value out of them; a token whose V is not finite is added by itself after the tiles.
    const int nodes = TREE ? __builtin_amdgcn_readfirstlane(paged_nodes(a, b)) : 0;
    const int n0 = TREE ? n - nodes : n - a.S + 1;  // a tree's first token need not be above the others
    const uint64_t masks = TREE && tm > n0 ? paged_tree_masks(a, b, nodes, lane) : 0ull;
    int odd0 = 0, odd1 = 0;  // those tokens
    if (g0 == 0 && tid == 0 && (a.by_unit || !whole))
      a.cut[a.by_unit ? int64_t(b) * upb + u : w] =
          PagedCut{b, u, whole ? 1 : shares.owner(ubeg + cost - 1) - w + 1, w};
    const int32_t* const trow = a.table + int64_t(b) * a.width;

    // Q fragments: lane (row nl, group g); e4m3 rows are read 16 codes at a time, so there the
    // chunks 2p and 2p + 1 hold d 64p + 16g .. +8 and +8 .. +16
    pv8s qf[RT][KC];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int r = min(row0 + 16 * rt + nl, R - 1);
      const uint16_t* const qrow = a.q + b * a.qb + (r / grp) * a.qs + (hk * grp + r % grp) * a.qh;
#pragma unroll
      for (int cc = 0; cc < KC; ++cc) {
        const int d = FP8 ? 64 * (cc >> 1) + 16 * g + 8 * (cc & 1) : 32 * cc + 8 * g;
        qf[rt][cc] = *reinterpret_cast<const pv8s*>(qrow + d);
      }
    }
    v4f acc[RT][NT];  // acc[rt][nt][i] = O[row 16rt + nl][16nt + 4g + i]
    float m_run[RT], l_run[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      m_run[rt] = -INFINITY;
      l_run[rt] = 0.0f;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) acc[rt][nt] = v4f{0.f, 0.f, 0.f, 0.f};
    }

    // ---- the tiles t0 + 32 k, k < nk ----
    const int nk = (tm - t0 + kPagedTile - 1) / kPagedTile;
    // page ids of the next 64 >> ish tiles, lane e: tile base + (e >> ish), part e & ish
    int ids = -1, ids_base = 0;
    auto fetch_ids = [&](int k0) {
      ids_base = k0;
      const int k = k0 + (lane >> ish);
      const int t = t0 + kPagedTile * k + ((lane & ish) << 4);
      int id = -1;
      if (k < nk && t < tm) id = trow[t >> ps];
      ids = uint32_t(id) < uint32_t(a.c.pages) ? id : -1;
    };
    auto issue = [&](int k, int stage) {
      if (((k - ids_base) << ish) >= 64) fetch_ids(k);
      const int t = t0 + kPagedTile * k;
      const int e = (k - ids_base) << ish;
      int id[2];
      id[0] = __builtin_amdgcn_readlane(ids, e);
      id[1] = ish ? __builtin_amdgcn_readlane(ids, e + 1) : id[0];
      uint32_t valid = tm - t >= 32 ? 0xFFFFFFFFu : (1u << (tm - t)) - 1u;
      if (id[0] < 0) valid &= ish ? 0xFFFF0000u : 0u;
      if (id[1] < 0) valid &= ish ? 0x0000FFFFu : 0u;
      if (lane == 0) s_valid[stage] = valid;
      const int off = ish ? 0 : t & (page - 1);
      int64_t row[2];  // of the tile's halves
#pragma unroll
      for (int i = 0; i < 2; ++i)
        row[i] = (int64_t(max(id[i], 0)) * a.c.heads + hk) * page + off + (ish ? 0 : 16 * i);
      const uint32_t dst = __builtin_amdgcn_readfirstlane(ring_lds + stage * C::STAGE);
      const int rin = lane / L::CH, slot = lane % L::CH;
#pragma unroll
      for (int side = 0; side < (SHARED ? 1 : 2); ++side) {
        const uint8_t* const pool = side ? a.c.v : a.c.k;
        constexpr int N = C::SIDE / 1024 / RH;  // consecutive loads of each of the waves that share the tile
#pragma unroll
        for (int jj = 0; jj < N; ++jj) {
          const int j = rh * N + jj;
          constexpr int HALF = 16 / L::RPI > 0 ? 16 / L::RPI : 1;  // loads of half a tile
          const int half = j / HALF, r = (j % HALF) * L::RPI;
          const uint32_t voff = uint32_t(rin * RB + ((slot ^ L::swz(r + rin)) << 4));
          paged_load16(pool + ((half ? row[1] : row[0]) + r) * RB, voff, dst + side * C::SIDE + j * 1024);
        }
      }
      if constexpr (FP8) {  // (each wave of the worker loads them: the same bytes)
        const int tok = lane & 31;
        const int64_t at = tok < 16 ? row[0] + tok : row[1] + tok - 16;
        paged_load4((lane < 32 ? a.c.ks : a.c.vs) + at,
                    __builtin_amdgcn_readfirstlane(scales_lds + stage * C::SCALES));
      }
    };
    if (nk > 0) fetch_ids(0);
    __builtin_amdgcn_s_waitcnt(vmcnt_only(0));  // Q too: no wait for it is left inside the loop
#pragma unroll
    for (int k = 0; k < NS - 1; ++k)
      if (k < nk) issue(k, k);

    int stage = 0;
#pragma unroll 1
    for (int k = 0; k < nk; ++k) {
      // the tile before has been read out of its stage, by every wave of the worker
      if constexpr (RH > 1) meet();
      else __builtin_amdgcn_s_waitcnt(lgkmcnt_only(0));
      if (k + NS - 1 < nk) {
        issue(k + NS - 1, stage == 0 ? NS - 1 : stage - 1);
        __builtin_amdgcn_s_waitcnt(vmcnt_only((NS - 1) * C::LOADS));
      } else {
        __builtin_amdgcn_s_waitcnt(vmcnt_only(0));
      }
      if constexpr (RH > 1) {
        meet();  // and every wave's part of this one has landed
      } else {
        asm volatile("" ::: "memory");
      }
      uint8_t* const kt = ring + stage * C::STAGE;
      uint8_t* const vt = SHARED ? kt : kt + C::SIDE;
      uint32_t valid = __builtin_amdgcn_readfirstlane(s_valid[stage]);
      const int t = t0 + kPagedTile * k;
      const bool last = (TREE || a.S > 1) && t + kPagedTile > n0;
      if (last) {
        const uint32_t some = valid & ~((1u << max(n0 - t, 0)) - 1u);  // tokens that some rows see
        bool odd = false;
        for (int i = lane; i < kPagedTile * L::CH; i += 64)
          if ((some >> (i / L::CH)) & 1) odd |= paged_odd<FP8>(*reinterpret_cast<const v4i*>(vt + i * 16));
        if constexpr (FP8) {
          const float sc = reinterpret_cast<const float*>(scales + stage * C::SCALES)[32 + (lane & 31)];
          odd |= ((some >> (lane & 31)) & 1) && !is_finite_f32(sc);
        }
        if (__ballot(odd)) {
          odd0 = odd1 > 0 ? odd0 : max(n0, t);
          odd1 = min(t + kPagedTile, tm);
          valid &= ~some;
        }
        meet();  // both waves have looked at V before its rows are cleared
      }
      if (valid != 0xFFFFFFFFu) {
        // rows that hold nothing become zeros, whatever bits their memory has
        for (int i = lane; i < kPagedTile * L::CH; i += 64)
          if (!((valid >> (i / L::CH)) & 1)) {
            *reinterpret_cast<v4i*>(kt + i * 16) = v4i{0, 0, 0, 0};
            if (!SHARED) *reinterpret_cast<v4i*>(vt + i * 16) = v4i{0, 0, 0, 0};
          }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      }
      // ---- S^T: sacc[rt][tt][i] = q . k of row nl, token 16tt + 4g + i ----
      v4f sacc[RT][2];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) sacc[rt][0] = sacc[rt][1] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int tt = 0; tt < 2; ++tt) {
        const uint8_t* const krow = kt + (16 * tt + nl) * RB;
        const int sw = L::swz(nl);
        if constexpr (!FP8) {
#pragma unroll
          for (int cc = 0; cc < KC; ++cc) {
            const pv8s kf = *reinterpret_cast<const pv8s*>(krow + (((4 * cc + g) ^ sw) << 4));
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) sacc[rt][tt] = paged_mfma(kf, qf[rt][cc], sacc[rt][tt]);
          }
        } else {
#pragma unroll
          for (int cp = 0; cp < KC / 2; ++cp) {
            const v4i kc = *reinterpret_cast<const v4i*>(krow + (((4 * cp + g) ^ sw) << 4));
            const pv8s k0 = paged_widen(kc[0], kc[1]), k1 = paged_widen(kc[2], kc[3]);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
              sacc[rt][tt] = paged_mfma(k0, qf[rt][2 * cp], sacc[rt][tt]);
              sacc[rt][tt] = paged_mfma(k1, qf[rt][2 * cp + 1], sacc[rt][tt]);
            }
          }
        }
      }
      v4f ksc[2], vsc[2];
      if constexpr (FP8) {
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) {
          ksc[tt] = *reinterpret_cast<const v4f*>(scales + stage * C::SCALES + 4 * (16 * tt + 4 * g));
          vsc[tt] = *reinterpret_cast<const v4f*>(scales + stage * C::SCALES + 128 + 4 * (16 * tt + 4 * g));
        }
      }
      // ---- softmax ----
      pv8s pf[RT];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        float y[8], top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          y[i] = sacc[rt][i >> 2][i & 3] * a.scale2;
          if constexpr (FP8) y[i] = sacc[rt][i >> 2][i & 3] * ksc[i >> 2][i & 3] * a.scale2;
        }
        if (valid != 0xFFFFFFFFu) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (!((valid >> (16 * (i >> 2) + 4 * g + (i & 3))) & 1)) y[i] = -INFINITY;
        }
        if (last) {
          if constexpr (TREE) {
            const uint64_t mask = paged_tree_mask(masks, min(row0 + 16 * rt + nl, R - 1) / grp);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int node = t + 16 * (i >> 2) + 4 * g + (i & 3) - n0;
              if (node >= 0 && !((mask >> (node & 63)) & 1)) y[i] = -INFINITY;
            }
          } else {
            const int sees = n0 + min(row0 + 16 * rt + nl, R - 1) / grp - t;  // tokens of the tile that the row sees
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (16 * (i >> 2) + 4 * g + (i & 3) >= sees) y[i] = -INFINITY;
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, y[i]);
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        if (a.scores) {
          const int r = row0 + 16 * rt + nl;
          if (r < R) {
            float* const row = a.scores + ((int64_t(b) * a.c.heads + hk) * R + r) * a.capacity + t + 4 * g;
            const int left = tm - t - 4 * g;
#pragma unroll
            for (int tt = 0; tt < 2; ++tt) {
              if (16 * tt + 3 < left) {
                *reinterpret_cast<v4f*>(row + 16 * tt) = v4f{y[4 * tt], y[4 * tt + 1], y[4 * tt + 2], y[4 * tt + 3]};
              } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  if (16 * tt + i < left) row[16 * tt + i] = y[4 * tt + i];
              }
            }
          }
        }
        const bool bump = top > m_run[rt] + kPagedLazy;
        if (__ballot(bump)) {
          const float resc = !bump ? 1.0f : (m_run[rt] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_run[rt] - top));
          m_run[rt] = bump ? top : m_run[rt];
          l_run[rt] *= resc;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) acc[rt][nt] = acc[rt][nt] * resc;
        }
        const float m = m_run[rt] == -INFINITY ? 0.0f : m_run[rt];
        float p[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = __builtin_amdgcn_exp2f(y[i] - m);
        l_run[rt] += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
        if constexpr (FP8) {
#pragma unroll
          for (int i = 0; i < 8; ++i) p[i] *= vsc[i >> 2][i & 3];
          if (valid != 0xFFFFFFFFu) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (!((valid >> (16 * (i >> 2) + 4 * g + (i & 3))) & 1)) p[i] = 0.0f;
          }
        }
        union {
          uint32_t d[4];
          pv8s v;
        } pk;
#pragma unroll
        for (int i = 0; i < 4; ++i) pk.d[i] = f32x2_to_bf16x2(p[2 * i], p[2 * i + 1]);
        pf[rt] = pk.v;
      }
      // ---- O^T += V^T P^T: k slots 0-3 tokens 4g + i, 4-7 tokens 16 + 4g + i ----
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        pv8s vf;
        if constexpr (!FP8) {
          const int row = 4 * g + (nl >> 2);
          const uint8_t* const p = vt + row * RB + (((2 * nt + ((nl >> 1) & 1)) ^ L::swz(row)) << 4) + (nl & 1) * 8;
          const pv4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_pv4s*)p);
          const pv4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_pv4s*)(p + 16 * RB));
          vf = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        } else {
          const int row = 4 * g + ((nl >> 1) & 3) + 16 * (nl >> 3);
          const uint8_t* const p = vt + row * RB + ((nt ^ L::swz(row)) << 4) + (nl & 1) * 8;
          const pv2i c8 = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_pv2i*)p);
          vf = paged_widen(c8[0], c8[1]);
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) acc[rt][nt] = paged_mfma(vf, pf[rt], acc[rt][nt]);
      }
      stage = stage + 1 == NS ? 0 : stage + 1;
    }

    // ---- tokens that only some rows see and whose V is not finite: a row takes nothing from one that
    // it does not see ----
    if (odd0 < odd1) {
      __builtin_amdgcn_s_waitcnt(vmcnt_only(0));  // scores that the tiles stored for these tokens
      for (int t = odd0; t < odd1; ++t) {
        const int64_t at = paged_row(a.c, trow, a.width, hk, t);
        if (at < 0) continue;
        const uint8_t* const kr = a.c.k + at * RB;
        const uint8_t* const vr = (SHARED ? a.c.k : a.c.v) + at * RB;
        const float ksc = FP8 ? a.c.ks[at] : 1.0f, vsc = FP8 ? a.c.vs[at] : 1.0f;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          const int rq = min(row0 + 16 * rt + nl, R - 1);
          const float dot =
              paged_dot<D, FP8>(a.q + b * a.qb + (rq / grp) * a.qs + (hk * grp + rq % grp) * a.qh, kr, g);
          const int r = row0 + 16 * rt + nl;
          const uint64_t mask = TREE ? paged_tree_mask(masks, rq / grp) >> ((t - n0) & 63) : 0ull;
          const bool sees = r < R && (TREE ? mask & 1 : t < n - (a.S - 1 - r / grp));
          const float y = FP8 ? dot * ksc * a.scale2 : dot * a.scale2;
          if (a.scores && r < R && g == 0)
            a.scores[((int64_t(b) * a.c.heads + hk) * R + r) * a.capacity + t] = y;
          if (sees) {
            const float m_new = fmaxf(m_run[rt], y);
            const float m = m_new == -INFINITY ? 0.0f : m_new;
            const float resc = m_run[rt] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_run[rt] - m);
            const float p = __builtin_amdgcn_exp2f(y - m);
            m_run[rt] = m_new;
            l_run[rt] = l_run[rt] * resc + (g == 0 ? p : 0.0f);
            const float pv = p * vsc;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              const v4f v = paged_four<FP8>(vr, 16 * nt + 4 * g);
#pragma unroll
              for (int i = 0; i < 4; ++i) acc[rt][nt][i] = fmaf(pv, v[i], acc[rt][nt][i] * resc);
            }
          }
        }
      }
    }

    // ---- the part's end ----
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      l_run[rt] += __shfl_xor(l_run[rt], 16, 64);
      l_run[rt] += __shfl_xor(l_run[rt], 32, 64);
    }
    {
      float* const part = a.part + (2 * int64_t(w) + (g0 == 0 ? 1 : 0)) * paged_slot(a.rows, D);
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const int rl = rh * C::WROWS + 16 * rt + nl, r = rg * ROWS + rl;
        if (r >= R) continue;
        if (whole) {
          const int head = hk * grp + r % grp, s = r / grp;
          float den = l_run[rt], f = 1.0f, M = m_run[rt];
          if (a.sink) {
            const float sk = a.sink[head] * kLog2e;
            M = fmaxf(M, sk);
            const float Me = M == -INFINITY ? 0.0f : M;
            f = m_run[rt] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_run[rt] - Me);
            den = den * f + __builtin_amdgcn_exp2f(sk - Me);
          }
          if (TREE && s >= nodes) {  // no node's row
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) acc[rt][nt] = v4f{0.f, 0.f, 0.f, 0.f};
            den = 0.0f;
          }
          const float inv = den == 0.0f ? 0.0f : f / den;
          uint16_t* const orow = a.o + ((int64_t(b) * a.S + s) * a.H + head) * D + 4 * g;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            *reinterpret_cast<uint2*>(orow + 16 * nt) =
                make_uint2(f32x2_to_bf16x2(acc[rt][nt][0] * inv, acc[rt][nt][1] * inv),
                           f32x2_to_bf16x2(acc[rt][nt][2] * inv, acc[rt][nt][3] * inv));
          if (a.ml && g == 0) {
            float* const e = a.ml + 2 * ((int64_t(b) * a.c.heads + hk) * R + r);
            e[0] = M == -INFINITY ? 0.0f : M;
            e[1] = den == 0.0f ? 0.0f : 1.0f / den;
          }
        } else {
          if (g == 0) {
            part[rl] = m_run[rt];
            part[a.rows + rl] = l_run[rt];
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            *reinterpret_cast<v4f*>(part + paged_head(a.rows) + rl * D + 16 * nt + 4 * g) = acc[rt][nt];
        }
      }
    }
    meet();  // the ring is free for the next part's tiles
  }
  paged_empty(a, w, upb, D, 64 * RH);
}

// Merges the cut units' partials.  WIDE: a workgroup a row of a unit, every partial's (m, l) at once,
// then O with GR partials in flight at a time, for units of eight parts and more (128 parts of 8 units 5.4 us against
// 35.7, 16 of 64 5.0 against 7.8, 8 of 128 4.6 against 5.8).  Else GR rows a workgroup, each by the CH threads that hold
// its columns, without a barrier (4 parts of 256 units 4.0 us against 4.3).
constexpr int kPagedMaxWorkers = 4096;

template <int D, bool WIDE>
__device__ __forceinline__ void paged_join(const PagedAttnArgs& a, int unit, int rows) {
  constexpr int CH = D / 4, GR = 256 / CH;
  const PagedCut cut = a.cut[unit];
  const int np = cut.np;
  if (np < 2) return;
  const int grp = a.H / a.c.heads, R = a.S * grp, RG = (R + a.unit_rows - 1) / a.unit_rows;
  const int hk = cut.u / RG, rg = cut.u - hk * RG, b = cut.b;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int ch = tid % CH, gr = tid / CH;
  const int rl = WIDE ? rows : rows * GR + gr, r = rg * a.unit_rows + rl;
  if (rl >= a.rows || r >= R) return;  // WIDE: the whole workgroup
  const int64_t slot = paged_slot(a.rows, D);
  const float* const part = a.part + rl;
  auto at = [&](int j) { return part + (2 * (int64_t(cut.w) + j) + (j == 0 ? 1 : 0)) * slot; };
  const int head = hk * grp + r % grp;
  const float sk = a.sink ? a.sink[head] * kLog2e : -INFINITY;
  const int off = paged_head(a.rows) + rl * (D - 1) + 4 * ch;
  float M = sk, den = 0.0f;
  v4f o = v4f{0.f, 0.f, 0.f, 0.f};
  float Me;
  if constexpr (WIDE) {
    __shared__ float s_f[kPagedMaxWorkers];
    __shared__ float s_red[2][4];
    __shared__ v4f s_o[256];
    float l0 = 0.0f;  // of this thread's first partial; there are seldom more
    for (int j = tid; j < np; j += 256) {
      const float m = at(j)[0];
      if (j == tid) l0 = at(j)[a.rows];
      s_f[j] = m;
      M = fmaxf(M, m);
    }
    for (int i = 1; i < 64; i <<= 1) M = fmaxf(M, __shfl_xor(M, i, 64));
    if (lane == 0) s_red[0][wave] = M;
    __syncthreads();
    M = fmaxf(fmaxf(s_red[0][0], s_red[0][1]), fmaxf(s_red[0][2], s_red[0][3]));
    Me = M == -INFINITY ? 0.0f : M;
    for (int j = tid; j < np; j += 256) {
      const float f = __builtin_amdgcn_exp2f(s_f[j] - Me);
      s_f[j] = f;
      den += f * (j == tid ? l0 : at(j)[a.rows]);
    }
    for (int i = 1; i < 64; i <<= 1) den += __shfl_xor(den, i, 64);
    if (lane == 0) s_red[1][wave] = den;
    __syncthreads();
    den = (s_red[1][0] + s_red[1][1]) + (s_red[1][2] + s_red[1][3]);
#pragma unroll 8
    for (int j = gr; j < np; j += GR) o += *reinterpret_cast<const v4f*>(at(j) + off) * s_f[j];
    s_o[tid] = o;
    __syncthreads();
    if (tid >= CH) return;
#pragma unroll
    for (int i = 1; i < GR; ++i) o += s_o[i * CH + tid];
  } else {
#pragma unroll 4
    for (int j = 0; j < np; ++j) M = fmaxf(M, at(j)[0]);
    Me = M == -INFINITY ? 0.0f : M;
#pragma unroll 4
    for (int j = 0; j < np; ++j) {
      const float f = __builtin_amdgcn_exp2f(at(j)[0] - Me);
      den += f * at(j)[a.rows];
      o += *reinterpret_cast<const v4f*>(at(j) + off) * f;
    }
  }
  if (a.sink) den += __builtin_amdgcn_exp2f(sk - Me);
  if (a.parent && r / grp >= paged_nodes(a, b)) {  // no node's row
    o = v4f{0.f, 0.f, 0.f, 0.f};
    den = 0.0f;
  }
  const float inv = den == 0.0f ? 0.0f : 1.0f / den;
  uint16_t* const orow = a.o + ((int64_t(b) * a.S + r / grp) * a.H + head) * D;
  *reinterpret_cast<uint2*>(orow + 4 * ch) =
      make_uint2(f32x2_to_bf16x2(o[0] * inv, o[1] * inv), f32x2_to_bf16x2(o[2] * inv, o[3] * inv));
  if (a.ml && ch == 0) {
    float* const e = a.ml + 2 * ((int64_t(b) * a.c.heads + hk) * R + r);
    e[0] = Me;
    e[1] = inv;
  }
}

template <int D, bool WIDE>
__global__ __launch_bounds__(256) void paged_attn_join_kernel(PagedAttnArgs a) {
  paged_join<D, WIDE>(a, blockIdx.x, blockIdx.y);
}

// weights[slot] += sum over the KV head's rows that see the slot of 2^(y - m) / sum, rows in ascending
// order.  A workgroup takes kWeighSlots slots of a head, four a thread.  Its bound is the launch: 4.3 us at 16 x
// 3000 tokens of 8 heads, one slot a thread 7.7.  JOIN: the rows' m and sum come from the cut units'
// partials, 16 threads a row, so that one launch does the join as well; that is for up to kWeighRows rows a KV
// head, which the workgroup takes at once (4 rows: 5.6 us against 8.5 in two launches, 131071 tokens 9.4 against 11.8;
// 64 rows 22.9 against 20.2).
constexpr int kWeighSlots = 1024;
constexpr int kWeighRows = 16;  // and no more than a unit's

template <int D, bool JOIN>
__device__ __forceinline__ void paged_weigh(const PagedAttnArgs& a, int bh, int block, float* s_ml) {
  const int b = bh / a.c.heads, hk = bh - b * a.c.heads;
  const int grp = a.H / a.c.heads, R = a.S * grp;
  const int n = paged_len(a, b);
  const int t = block * kWeighSlots + 4 * threadIdx.x;
  if (block * kWeighSlots >= n) return;
  const float* const ml = a.ml + 2 * int64_t(bh) * R;
  if constexpr (JOIN) {
    const int r = threadIdx.x >> 4, li = threadIdx.x & 15;  // one unit holds the rows
    if (r < R) {
      const PagedCut cut = a.cut[bh];
      float m, inv;
      if (cut.np < 2) {
        m = ml[2 * r];
        inv = ml[2 * r + 1];
      } else {
        const int64_t slot = paged_slot(a.rows, D);
        const float* const part = a.part + r;
        auto at = [&](int j) { return part + (2 * (int64_t(cut.w) + j) + (j == 0 ? 1 : 0)) * slot; };
        const float sk = a.sink ? a.sink[hk * grp + r % grp] * kLog2e : -INFINITY;
        float M = -INFINITY, l = 0.0f;  // of this thread's partials
        for (int j = li; j < cut.np; j += 16) {
          const float mj = at(j)[0], lj = at(j)[a.rows], Mn = fmaxf(M, mj), e = Mn == -INFINITY ? 0.0f : Mn;
          l = l * __builtin_amdgcn_exp2f(M - e) + lj * __builtin_amdgcn_exp2f(mj - e);
          M = Mn;
        }
        m = fmaxf(M, sk);
        for (int i = 1; i < 16; i <<= 1) m = fmaxf(m, __shfl_xor(m, i, 64));
        m = m == -INFINITY ? 0.0f : m;
        l *= __builtin_amdgcn_exp2f(M - m);
        for (int i = 1; i < 16; i <<= 1) l += __shfl_xor(l, i, 64);
        if (a.sink) l += __builtin_amdgcn_exp2f(sk - m);
        inv = l == 0.0f ? 0.0f : 1.0f / l;
      }
      if (li == 0) {
        s_ml[2 * r] = m;
        s_ml[2 * r + 1] = inv;
      }
    }
  } else {
    for (int i = threadIdx.x; i < 2 * R; i += 256) s_ml[i] = ml[i];
  }
  __syncthreads();
  if (t >= n) return;
  const int64_t at = paged_row(a.c, a.table + int64_t(b) * a.width, a.width, hk, t);  // of four slots of one page
  if (at < 0) return;
  const float* const y = a.scores + int64_t(bh) * R * a.capacity + t;
  v4f sum = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int r = 0; r < R; ++r) {
    const v4f v = *reinterpret_cast<const v4f*>(y + r * a.capacity);
    const int seen = n - (a.S - 1 - r / grp) - t;  // of the four
    const float m = s_ml[2 * r], inv = s_ml[2 * r + 1];
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[i] += i < seen ? __builtin_amdgcn_exp2f(v[i] - m) * inv : 0.0f;
  }
  float* const w = a.c.weights + at;
  if (t + 4 <= n) {
    *reinterpret_cast<v4f*>(w) += sum;
  } else {
    for (int i = 0; t + i < n; ++i) w[i] += sum[i];
  }
}

// The join and the weights in one launch.
template <int D, bool WIDE>
__global__ __launch_bounds__(256) void paged_attn_end_kernel(PagedAttnArgs a, int units, int row_blocks, int slot_blocks) {
  extern __shared__ float s_ml[];
  const int joins = units * row_blocks, block = blockIdx.x;
  if (block < joins) {
    paged_join<D, WIDE>(a, block / row_blocks, block % row_blocks);
  } else {
    const int i = block - joins;
    paged_weigh<D, true>(a, i / slot_blocks, i % slot_blocks, s_ml);
  }
}

template <int D>
__global__ __launch_bounds__(256) void paged_attn_weigh_kernel(PagedAttnArgs a) {
  extern __shared__ float s_ml[];
  paged_weigh<D, false>(a, blockIdx.y, blockIdx.x, s_ml);
}

// What follows the main kernel: the join, and the weights.
template <int D>
int paged_attn_join(const PagedAttnArgs& a, hipStream_t stream) {
  constexpr int GR = 256 / (D / 4);
  const int64_t units = paged_units(a);
  const bool wide = 8 * units <= a.W;
  const unsigned n = unsigned(std::min<int64_t>(units, a.W)), row_blocks = unsigned(wide ? a.rows : (a.rows + GR - 1) / GR);
  const int64_t heads = int64_t(a.B) * a.c.heads, slot_blocks = (a.capacity + kWeighSlots - 1) / kWeighSlots;
  const int64_t blocks = n * row_blocks + heads * slot_blocks;
  const int R = a.S * (a.H / a.c.heads);
  const size_t ml_bytes = 2 * sizeof(float) * R;
  if (a.scores && a.by_unit && R <= kWeighRows && blocks <= 0xFFFFFF) {
    if (wide)
      WZ_LAUNCH("paged_attn_end", stream, (paged_attn_end_kernel<D, true>), dim3{unsigned(blocks)}, dim3(256), ml_bytes, a,
                int(n), int(row_blocks), int(slot_blocks));
    else
      WZ_LAUNCH("paged_attn_end", stream, (paged_attn_end_kernel<D, false>), dim3{unsigned(blocks)}, dim3(256), ml_bytes, a,
                int(n), int(row_blocks), int(slot_blocks));
    return check_launch("paged_attn_end");
  }
  const dim3 grid(n, row_blocks);
  if (wide)
    WZ_LAUNCH("paged_attn_join", stream, (paged_attn_join_kernel<D, true>), grid, dim3(256), 0, a);
  else
    WZ_LAUNCH("paged_attn_join", stream, (paged_attn_join_kernel<D, false>), grid, dim3(256), 0, a);
  if (int rc = check_launch("paged_attn_join")) return rc;
  if (!a.scores || a.capacity == 0) return WZ_OK;
  WZ_LAUNCH("paged_attn_weigh", stream, paged_attn_weigh_kernel<D>, dim3(unsigned(slot_blocks), unsigned(heads)), dim3(256),
            ml_bytes, a);
  return check_launch("paged_attn_weigh");
}

// Whether a tree's units of 16 rows are so few, whatever the lengths that its table can hold, that there are six tiles a worker at
// most.  The time is a worker's way through its tiles then, and shorter with fewer rows: us with the kernel of the rows / with 16
// rows a unit (join in both), heads of 128: 1 x 1015 tokens, 64 rows on 8 KV heads 17.4 / 15.9, 1 x 4000 22.9 / 18.9, 8 x 300 26.1 /
// 19.2, 1 x 1000 with 256 rows 27.1 / 25.4, with 512 rows on 300 24.8 / 22.2; heads of 64: 1 x 3000, 192 rows on 8 20.9 / 20.2, 1 x
// 6000, 512 rows on one 16.3 / 18.5.
static inline bool paged_few(const PagedAttnArgs& a) {
  const int64_t R = a.S * (a.H / a.c.heads);
  return a.B * int64_t(a.c.heads) * ((R + 15) / 16) * (a.capacity / kPagedTile + kPagedStart) <= 24 * int64_t(cu_count());
}

// The kernel of R rows a KV head: 16, 32 or 64 rows a unit.  With 4 rows 16 x 8000 tokens take 94.5 / 97.6 / 121.7 us with
// each, 48 x 9001 e4m3 tokens of 128 with 8 rows 167 / 214 / 400.
template <int D, bool FP8, bool SHARED, int RT, int RH, bool TREE>
int paged_attn_launch_rt(PagedAttnArgs a, bool ask, int* workers, hipStream_t stream) {
  using C = PagedCfg<D, FP8, SHARED, RT, RH>;
  static_assert(C::LDS <= 160 * 1024, "a workgroup's LDS");
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
  auto* const kernel = paged_attn_kernel<D, FP8, SHARED, RT, RH, TREE>;
  if (int rc = allow_lds("paged_attn", kernel, C::LDS, grant)) return rc;
  WZ_LAUNCH("paged_attn", stream, kernel, dim3{unsigned(a.W)}, dim3(64 * RH), C::LDS, a);
  if (int rc = check_launch("paged_attn")) return rc;
  return paged_attn_join<D>(a, stream);
}

template <int D, bool FP8, bool SHARED, bool TREE>
int paged_attn_launch_d(const PagedAttnArgs& a, bool ask, int* workers, hipStream_t stream) {
  const int R = a.S * (a.H / a.c.heads);
  if constexpr (TREE)
    if (paged_few(a)) return paged_attn_launch_rt<D, FP8, SHARED, 1, 1, TREE>(a, ask, workers, stream);
  if (R <= 16) return paged_attn_launch_rt<D, FP8, SHARED, 1, 1, TREE>(a, ask, workers, stream);
  if (R <= 32) return paged_attn_launch_rt<D, FP8, SHARED, 2, 1, TREE>(a, ask, workers, stream);
  return paged_attn_launch_rt<D, FP8, SHARED, 2, 2, TREE>(a, ask, workers, stream);
}

int paged_latent(bool fp8, const PagedAttnArgs& a, bool ask, int* workers, hipStream_t stream);

// Launches, or with `ask` -> the rows of a partial, and *workers.
template <bool FP8, bool TREE>
int paged_attn_launch(int D, const PagedAttnArgs& a, bool ask, int* workers, hipStream_t stream) {
  if (a.c.shared) {
    if (D == 128) return paged_attn_launch_d<128, FP8, true, TREE>(a, ask, workers, stream);
    if (D == 256) return paged_attn_launch_d<256, FP8, true, TREE>(a, ask, workers, stream);
    return paged_latent(FP8, a, ask, workers, stream);
  }
  if (D == 64) return paged_attn_launch_d<64, FP8, false, TREE>(a, ask, workers, stream);
  if (D == 128) return paged_attn_launch_d<128, FP8, false, TREE>(a, ask, workers, stream);
  return paged_attn_launch_d<256, FP8, false, TREE>(a, ask, workers, stream);
}

// The kernels are compiled by four sources: for one to 16 new tokens in a row and for trees, of bf16 and of e4m3 rows.
int paged_attn_bf16(int D, const PagedAttnArgs& a, bool ask, int* workers, hipStream_t stream);
int paged_attn_e4m3(int D, const PagedAttnArgs& a, bool ask, int* workers, hipStream_t stream);
int paged_tree_bf16(int D, const PagedAttnArgs& a, bool ask, int* workers, hipStream_t stream);
int paged_tree_e4m3(int D, const PagedAttnArgs& a, bool ask, int* workers, hipStream_t stream);

}  // namespace wz

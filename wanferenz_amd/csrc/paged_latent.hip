// paged_attn on latents of 512 (K = V): a worker is a whole compute unit.
//
// 64 rows of queries on one latent (64 heads, or fewer heads of several tokens) make 128 flops a byte
// and 131 KB of partial O a cut unit, so the work is cut into as few parts as fill the chip, one a
// compute unit, of 8 waves that share a tile of 64 tokens.  What bounds a tile then is how often its rows
// are read from LDS; the waves split both products such that K is read twice, V once and P once:
//   * the tile sits in LDS row-major, loaded while the one before was computed (two buffers, the loads
//     fill them directly); wave w has the rows 8w .. +8 of the load, which lie in one page;
//   * S^T = K Q^T: wave w has tokens 16 (w & 3) .. +16 and SHT row tiles; lane (row n, group g) holds tokens
//     4g + i, and P goes to LDS in the order of the next product's k slots, 8 bytes a lane;
//   * P = 2^(y - m), m moved only when a tile's maximum exceeds it by more than 8.  Every wave writes its P
//     with the m of the tiles before and flags a row that needs a new one; only then a second barrier
//     follows, after the maxima have met, O is rescaled and P written again;
//   * O^T[512, rows] += V^T P^T: wave w has columns 64 w .. +64 of every row.
// 4 x 65536 latents (269 MB, 34 GF) take 68 to 81 us by card, 3.3 to 4 TB/s, and the join of the 131 KB partials 8.  A
// copy without the products takes 56 and one without the loads 58: a tile's chain from K to O is 3.6 us long, of which
// the matrix instructions are a fifth and LDS reads (K twice, V, Q's last chunks and P, 260 KB) a quarter, and one
// tile is in flight behind it.  With 16 heads 16 x 16000 latents (262 MB) take 52, 5.1 TB/s.
#include "paged_attn.h"

namespace wz {

constexpr int kLatentD = 512, kLatentTile = 64, kLatentWaves = 8;
// A unit's start in tiles (paged_cost): 64 sequences of 60 to 4000 latents, 64 heads, 40.1 / 31.1 / 29.3 / 31.6 us with 0 /
// 2 / 4 / 8, four of 65536 75.9 / 79.9 / 73.4 / 76.4.
constexpr int kLatentStart = 4;

template <bool FP8>
struct LatentCfg {
  static constexpr int RB = kLatentD * (FP8 ? 1 : 2);
  static constexpr int TILE = kLatentTile * RB;
  static constexpr int RPW = kLatentTile / kLatentWaves;      // rows that a wave loads
  static constexpr int LOADS = RPW * RB / 1024 + (FP8 ? 1 : 0);
};

// EXTRA: several new tokens, or weights to accumulate; without their code 64 rows just fit the registers (4 x 65536
// latents 73.4 us, with it 76.9).
template <bool FP8, int HT, bool EXTRA, bool TREE>
__global__ __launch_bounds__(64 * kLatentWaves, 2) void paged_latent_kernel(PagedAttnArgs a) {
  using C = LatentCfg<FP8>;
  using L = PagedRow<C::RB>;
  constexpr int D = kLatentD, RB = C::RB, ROWS = 16 * HT, T = kLatentTile;
  constexpr int KC = D / 32, NT = D / 16 / kLatentWaves;
  constexpr int SHT = HT == 4 ? 2 : 1;  // row tiles of S a wave
  // the last KQ chunks of Q are read from LDS for each tile: with all of 64 rows in registers some were
  // spilled, and a reload waits for the loads of the next tile (4 x 65536 latents 87.7 us; so 73.4)
  constexpr int KQ = HT == 4 ? 2 : 0;
  constexpr int QB = 2 * D;  // bytes of a row of Q
  __shared__ __align__(1024) uint8_t kb[2][C::TILE];
  __shared__ __align__(1024) uint8_t s_qf[FP8 ? ROWS * QB : 16];  // e4m3: 64 rows of Q are two tiles
  __shared__ __align__(16) uint8_t s_p[2][ROWS][64];  // [tokens / 32][row]: group g's 8 k slots at 16 g
  __shared__ float s_max[4][ROWS], s_l[4][ROWS];      // [token tile][row]
  __shared__ float s_scale[2][T], s_y[ROWS];
  __shared__ __align__(8) uint8_t s_valid[2][8];      // a bit a token
  __shared__ int s_bump[2];
  __shared__ __align__(16) uint8_t s_q[KQ ? ROWS : 1][128];  // [row]: chunk KC - 2 + c, group g at (4 c + g) ^ swz(row)

  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rt = wave & 3, ht0 = (wave >> 2) * SHT;  // this wave's token tile and first row tile of S
  const bool has_s = ht0 < HT;
  const uint32_t kb_lds = lds_addr(&kb[0][0]), sc_lds = lds_addr(&s_scale[0][0]);
  auto meet = [] { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };  // loads stay in flight

  const int grp = a.H / a.c.heads, R = a.S * grp, RG = (R + ROWS - 1) / ROWS, upb = a.c.heads * RG;
  const int w = blockIdx.x;
  const PagedShares shares(paged_total<T, kLatentStart>(a, upb), a.W);
  if (!a.by_unit && tid == 0) a.cut[w] = PagedCut{0, 0, 0, 0};
  if (w >= shares.workers) {
    paged_empty(a, w, upb, D, 64 * kLatentWaves);
    return;
  }
  int x = shares.begin(w);
  const int x_end = shares.begin(w + 1);
  int b, before;  // sequence, and the granules before it
  paged_find<T, kLatentStart>(a, upb, x, &b, &before);
  int n = __builtin_amdgcn_readfirstlane(paged_len(a, b)), cost = paged_cost<T, kLatentStart>(n);
  int u = (x - before) / cost, ubeg = before + u * cost;  // unit of the sequence, and where it begins
  const int ps = a.c.shift, page = a.c.page;

  auto next = [&] {  // the next unit that holds anything
    ubeg += cost;
    if (ubeg >= x_end) return false;
    x = ubeg;
    if (++u == upb) {
      do {
        ++b;
        n = __builtin_amdgcn_readfirstlane(paged_len(a, b));
      } while (n == 0);
      cost = paged_cost<T, kLatentStart>(n);
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
    const int g0 = max(x - ubeg - kLatentStart, 0), g1 = min(x_end - ubeg, cost) - kLatentStart;
    if (g1 <= 0) continue;
    const bool whole = g0 == 0 && g1 == cost - kLatentStart;
    const int hk = u / RG, rg = u - hk * RG, row0 = rg * ROWS;
    const int t0 = g0 * T, tm = min(g1 * T, n);
    // from n0 on a token is seen by some rows only, as in paged_attn_kernel
    const int nodes = TREE ? __builtin_amdgcn_readfirstlane(paged_nodes(a, b)) : 0;
    const int n0 = TREE ? n - nodes : n - a.S + 1;
    int odd0 = 0, odd1 = 0;
    if (g0 == 0 && tid == 0 && (a.by_unit || !whole))
      a.cut[a.by_unit ? int64_t(b) * upb + u : w] =
          PagedCut{b, u, whole ? 1 : shares.owner(ubeg + cost - 1) - w + 1, w};
    const int32_t* const trow = a.table + int64_t(b) * a.width;

    v4f acc[HT][NT];  // acc[ht][nt][i] = O[row 16ht + nl][64 wave + 16nt + 4g + i]
#pragma unroll
    for (int ht = 0; ht < HT; ++ht)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) acc[ht][nt] = v4f{0.f, 0.f, 0.f, 0.f};
    float m_run = -INFINITY, l_one = 0.0f;  // of row `lane`, the same in every wave: max, sum of the last tokens
    float m_s[SHT], l_s[SHT];               // of this lane's rows of S: the max, its tokens' share of the sum
#pragma unroll
    for (int h = 0; h < SHT; ++h) {
      m_s[h] = -INFINITY;
      l_s[h] = 0.0f;
    }

    const int nk = (tm - t0 + T - 1) / T;
    int ids = -1, ids_base = 0;  // lane e: the page of this wave's rows of tile base + e
    auto fetch_ids = [&](int k0) {
      ids_base = k0;
      const int t = t0 + T * (k0 + lane) + C::RPW * wave;
      int id = -1;
      if (k0 + lane < nk && t < tm) id = trow[t >> ps];
      ids = uint32_t(id) < uint32_t(a.c.pages) ? id : -1;
    };
    auto issue = [&](int k, int buf) {
      if (k - ids_base >= 64) fetch_ids(k);
      const int id = __builtin_amdgcn_readlane(ids, k - ids_base);
      const int t = t0 + T * k + C::RPW * wave;
      const uint32_t valid = id < 0 ? 0u : tm - t >= 8 ? 0xFFu : (1u << max(tm - t, 0)) - 1u;
      if (lane == 0) s_valid[buf][wave] = uint8_t(valid);
      const int64_t row = (int64_t(max(id, 0)) * a.c.heads + hk) * page + (t & (page - 1));
      const uint32_t dst = __builtin_amdgcn_readfirstlane(kb_lds + buf * C::TILE + C::RPW * wave * RB);
      int ln = lane;
      asm volatile("" : "+v"(ln));  // recomputed for each tile: the registers go to Q and O
      const int rin = ln / L::CH, slot = ln % L::CH;
#pragma unroll
      for (int j = 0; j < C::RPW / L::RPI; ++j) {
        const int r = j * L::RPI;  // of the wave's rows; the swizzle goes by the tile's
        const uint32_t voff = uint32_t(rin * RB + ((slot ^ L::swz(C::RPW * wave + r + rin)) << 4));
        paged_load16(a.c.k + (row + r) * RB, voff, dst + j * 1024);
      }
      if constexpr (FP8) {
        if (lane < C::RPW)
          paged_load4(a.c.ks + row + lane,
                      __builtin_amdgcn_readfirstlane(sc_lds + (buf * T + C::RPW * wave) * 4));
      }
    };
    // Q's rows in whole lines through the second buffer (fragments loaded by the four waves that share them
    // took 4 us more), while the first tile is on its way
    if (nk > 0) fetch_ids(0);
    __builtin_amdgcn_s_waitcnt(vmcnt_only(0));
    uint8_t* const qbuf = FP8 ? s_qf : kb[1];
    const uint32_t q_lds = lds_addr(qbuf);
    using QL = PagedRow<QB>;
#pragma unroll
    for (int j = 0; j < ROWS / kLatentWaves; ++j) {
      const int rl = j * kLatentWaves + wave, r = min(row0 + rl, R - 1);
      paged_load16(reinterpret_cast<const uint8_t*>(a.q + b * a.qb + (r / grp) * a.qs + (hk * grp + r % grp) * a.qh),
                   uint32_t((lane ^ QL::swz(rl)) << 4), __builtin_amdgcn_readfirstlane(q_lds + rl * QB));
    }
    if (tid < 2) s_bump[tid] = 0;
    if (nk > 0) {
      issue(0, 0);
      __builtin_amdgcn_s_waitcnt(vmcnt_only(C::LOADS));
    } else {
      __builtin_amdgcn_s_waitcnt(vmcnt_only(0));
    }
    meet();
    // fragments (B operand of S^T): lane (row nl, group g); the order of d as in paged_attn_kernel
    pv8s qb[SHT][KC - KQ];
#pragma unroll
    for (int h = 0; h < SHT; ++h) {
      const int rl = 16 * (has_s ? ht0 + h : 0) + nl;
#pragma unroll
      for (int cc = 0; cc < KC; ++cc) {
        const int ch = FP8 ? 8 * (cc >> 1) + 2 * g + (cc & 1) : 4 * cc + g;
        const pv8s q = *reinterpret_cast<const pv8s*>(qbuf + rl * QB + ((ch ^ QL::swz(rl)) << 4));
        if (cc < KC - KQ)
          qb[h][cc] = q;
        else if (rt == 0)
          *reinterpret_cast<pv8s*>(&s_q[rl][(((cc - (KC - KQ)) * 4 + g) ^ PagedRow<128>::swz(rl)) << 4]) = q;
      }
    }

#pragma unroll 1
    for (int k = 0; k < nk; ++k) {
      const int buf = k & 1;
      __builtin_amdgcn_s_waitcnt(vmcnt_only(0));  // this wave's loads of tile k have landed
      meet();                                     // ... and every wave's; the other buffer and s_p are free
      if (k + 1 < nk) issue(k + 1, buf ^ 1);
      uint8_t* const ks = kb[buf];
      uint64_t valid = uint64_t(paged_uniform(*reinterpret_cast<const int64_t*>(s_valid[buf])));
      const int tk = t0 + T * k;
      const bool last = EXTRA && (TREE || a.S > 1) && tk + T > n0;
      if (last) {
        const uint64_t some = valid & ~((1ull << max(n0 - tk, 0)) - 1ull);  // tokens that some rows see
        bool odd = false;  // every wave looks at all of them, and comes to the same
        for (int i = lane; i < T * L::CH; i += 64)
          if ((some >> (i / L::CH)) & 1) odd |= paged_odd<FP8>(*reinterpret_cast<const v4i*>(ks + i * 16));
        if constexpr (FP8) odd |= ((some >> lane) & 1) && !is_finite_f32(s_scale[buf][lane]);
        if (__ballot(odd)) {
          odd0 = odd1 > 0 ? odd0 : max(n0, tk);
          odd1 = min(tk + T, tm);
          valid &= ~some;
        }
        meet();  // every wave has looked before the rows are cleared
      }
      if (~valid) {
        // rows that hold nothing become zeros, whatever bits their memory has
        for (int i = tid; i < T * L::CH; i += 64 * kLatentWaves)
          if (!((valid >> (i / L::CH)) & 1)) *reinterpret_cast<v4i*>(ks + i * 16) = v4i{0, 0, 0, 0};
        meet();
      }
      int ln = lane;
      asm volatile("" : "+v"(ln));
      const int nl = ln & 15, g = ln >> 4;

      // ---- S^T[16 tokens, rows]: y[h][i] of token 16rt + 4g + i, row nl of tile h ----
      v4f y[SHT];
      float p_sum[SHT];
      v4f ksc = v4f{1.f, 1.f, 1.f, 1.f};
      if constexpr (FP8) ksc = *reinterpret_cast<const v4f*>(&s_scale[buf][16 * rt + 4 * g]);
      auto put_p = [&]() {  // P in bf16 to LDS, this lane's part of the row sum to p_sum
#pragma unroll
        for (int h = 0; h < SHT; ++h) {
          float pv[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) pv[i] = y[h][i] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(y[h][i] - m_s[h]);
          p_sum[h] = (pv[0] + pv[1]) + (pv[2] + pv[3]);
          if constexpr (FP8) {
#pragma unroll
            for (int i = 0; i < 4; ++i) pv[i] = y[h][i] == -INFINITY ? 0.0f : pv[i] * ksc[i];
          }
          *reinterpret_cast<uint2*>(&s_p[rt >> 1][16 * (ht0 + h) + nl][16 * g + 8 * (rt & 1)]) =
              make_uint2(f32x2_to_bf16x2(pv[0], pv[1]), f32x2_to_bf16x2(pv[2], pv[3]));
        }
      };
      if (has_s) {
#pragma unroll
        for (int h = 0; h < SHT; ++h) y[h] = v4f{0.f, 0.f, 0.f, 0.f};
        const uint8_t* const krow = ks + (16 * rt + nl) * RB;
        const int sw = L::swz(nl);
        // K fragments are read kAhead chunks ahead of their MFMAs
        constexpr int kAhead = 3, NC = FP8 ? KC / 2 : KC;
        v4i kf[kAhead + 1];
        auto kload = [&](int c) { kf[c % (kAhead + 1)] = *reinterpret_cast<const v4i*>(krow + (((4 * c + g) ^ sw) << 4)); };
#pragma unroll
        for (int c = 0; c < kAhead; ++c) kload(c);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          if (c + kAhead < NC) kload(c + kAhead);
          __builtin_amdgcn_sched_barrier(0);  // keep the reads ahead of their use
          const v4i kc = kf[c % (kAhead + 1)];
          auto q_of = [&](int h, int cc) -> pv8s {
            if (cc < KC - KQ) return qb[h][cc < KC - KQ ? cc : 0];
            const int rl = 16 * (ht0 + h) + nl;
            return *reinterpret_cast<const pv8s*>(&s_q[KQ ? rl : 0][(((cc - (KC - KQ)) * 4 + g) ^ PagedRow<128>::swz(rl)) << 4]);
          };
          if constexpr (FP8) {
            const pv8s k0 = paged_widen(kc[0], kc[1]), k1 = paged_widen(kc[2], kc[3]);
#pragma unroll
            for (int h = 0; h < SHT; ++h) {
              y[h] = paged_mfma(k0, q_of(h, 2 * c), y[h]);
              y[h] = paged_mfma(k1, q_of(h, 2 * c + 1), y[h]);
            }
          } else {
#pragma unroll
            for (int h = 0; h < SHT; ++h) y[h] = paged_mfma(__builtin_bit_cast(pv8s, kc), q_of(h, c), y[h]);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        bool bump = false;
#pragma unroll
        for (int h = 0; h < SHT; ++h) {
          float top = -INFINITY;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float s = FP8 ? y[h][i] * ksc[i] * a.scale2 : y[h][i] * a.scale2;
            y[h][i] = (valid >> (16 * rt + 4 * g + i)) & 1 ? s : -INFINITY;
          }
          if (last) {
            const int s = min(row0 + 16 * (ht0 + h) + nl, R - 1) / grp;
            if constexpr (TREE) {  // (the masks are made where they are used: held all along they cost a register too many)
              const uint64_t mask = paged_tree_mask(paged_tree_masks(a, b, nodes, ln), s);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int node = tk + 16 * rt + 4 * g + i - n0;
                if (node >= 0 && !((mask >> (node & 63)) & 1)) y[h][i] = -INFINITY;
              }
            } else {
              const int sees = n0 + s - tk;  // tokens that the row sees
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (16 * rt + 4 * g + i >= sees) y[h][i] = -INFINITY;
            }
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) top = fmaxf(top, y[h][i]);
          top = fmaxf(top, __shfl_xor(top, 16, 64));
          top = fmaxf(top, __shfl_xor(top, 32, 64));
          bump |= top > m_s[h] + kPagedLazy;
          if (g == 0) s_max[rt][16 * (ht0 + h) + nl] = top;
          if (EXTRA && a.scores) {
            const int r = row0 + 16 * (ht0 + h) + nl, t = t0 + T * k + 16 * rt + 4 * g;
            if (r < R) {
              float* const out = a.scores + ((int64_t(b) * a.c.heads + hk) * R + r) * a.capacity + t;
              if (t + 3 < tm) {
                *reinterpret_cast<v4f*>(out) = y[h];
              } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  if (t + i < tm) out[i] = y[h][i];
              }
            }
          }
        }
        if (__ballot(bump)) {
          if (lane == 0) s_bump[buf] = 1;
        }
        if (k > 0) put_p();
      }
      meet();
      const bool moved = k == 0 || s_bump[buf];
      if (tid == 0) s_bump[buf ^ 1] = 0;  // read by everyone before this barrier, written after the next
      if (moved) {
        // the tile's maxima have met: row `lane`
        const int hl = lane < ROWS ? lane : 0;
        const float bm = fmaxf(fmaxf(s_max[0][hl], s_max[1][hl]), fmaxf(s_max[2][hl], s_max[3][hl]));
        const bool bump = bm > m_run + kPagedLazy;
        const float resc = !bump ? 1.0f : (m_run == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_run - bm));
        m_run = bump ? bm : m_run;
#pragma unroll
        for (int h = 0; h < SHT; ++h) {
          m_s[h] = __shfl(m_run, (16 * (ht0 + h) + nl) & 63, 64);
          l_s[h] *= __shfl(resc, (16 * (ht0 + h) + nl) & 63, 64);
        }
        if (k > 0) {
#pragma unroll
          for (int ht = 0; ht < HT; ++ht) {
            const float r = __shfl(resc, 16 * ht + nl, 64);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) acc[ht][nt] = acc[ht][nt] * r;
          }
        }
        if (has_s) put_p();
        meet();
      }
      if (has_s) {
#pragma unroll
        for (int h = 0; h < SHT; ++h) l_s[h] += p_sum[h];
      }

      // ---- O^T[wave's columns, rows] += V^T[columns, 64 tokens] P^T[64 tokens, rows] ----
      pv8s vf[3];
      auto vload = [&](int j) {  // j = kc NT + nt, two column tiles ahead of their MFMAs
        const int row = 4 * g + (nl >> 2);  // rows 16 apart share their swizzle
        const uint8_t* const p = ks + ((j / NT) * 32 + row) * RB +
                                 (((wave * 2 * NT + 2 * (j % NT) + ((nl >> 1) & 1)) ^ L::swz(row)) << 4) + (nl & 1) * 8;
        const pv4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_pv4s*)p);
        const pv4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_pv4s*)(p + 16 * RB));
        vf[j % 3] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      };
      pv8s pb[HT];  // of 32 tokens kc; the second half's are read as the first half's are used up
      auto pload = [&](int kc, int ht) { pb[ht] = *reinterpret_cast<const pv8s*>(&s_p[kc][16 * ht + nl][16 * g]); };
#pragma unroll
      for (int ht = 0; ht < HT; ++ht) pload(0, ht);
      if constexpr (!FP8) {
        vload(0);
        vload(1);
#pragma unroll
        for (int j = 0; j < 2 * NT; ++j) {
          if (j + 2 < 2 * NT) vload(j + 2);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int ht = 0; ht < HT; ++ht) {
            acc[ht][j % NT] = paged_mfma(vf[j % 3], pb[ht], acc[ht][j % NT]);
            if (j == NT - 1) {
              __builtin_amdgcn_sched_barrier(0);
              pload(1, ht);
            }
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      } else {
        pv2i vc[2 * NT];
        const int row = 4 * g + ((nl >> 1) & 3) + 16 * (nl >> 3);
#pragma unroll
        for (int j = 0; j < 2 * NT; ++j)
          vc[j] = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
              (lds_pv2i*)(ks + ((j / NT) * 32 + row) * RB + (((wave * NT + j % NT) ^ L::swz(row)) << 4) + (nl & 1) * 8));
#pragma unroll
        for (int j = 0; j < 2 * NT; ++j) {
          const pv8s v = paged_widen(vc[j][0], vc[j][1]);
#pragma unroll
          for (int ht = 0; ht < HT; ++ht) {
            acc[ht][j % NT] = paged_mfma(v, pb[ht], acc[ht][j % NT]);
            if (j == NT - 1) pload(1, ht);
          }
        }
      }
    }

    // ---- tokens that only some rows see and that are not finite: a row takes nothing from one that it
    // does not see ----
    if (EXTRA && odd0 < odd1) __builtin_amdgcn_s_waitcnt(vmcnt_only(0));  // scores that the tiles stored for them
    for (int t = odd0; EXTRA && t < odd1; ++t) {
      const int64_t at = paged_row(a.c, trow, a.width, hk, t);
      if (at < 0) continue;  // the same in every wave
      const uint8_t* const kr = a.c.k + at * RB;
      const float sc = FP8 ? a.c.ks[at] : 1.0f;
      meet();  // s_y is free
      if (has_s && rt == 0) {
#pragma unroll
        for (int h = 0; h < SHT; ++h) {
          const int rq = min(row0 + 16 * (ht0 + h) + nl, R - 1);
          const float dot =
              paged_dot<D, FP8>(a.q + b * a.qb + (rq / grp) * a.qs + (hk * grp + rq % grp) * a.qh, kr, g);
          const int rl = 16 * (ht0 + h) + nl;
          const float yy = FP8 ? dot * sc * a.scale2 : dot * a.scale2;
          if (g == 0) {
            s_y[rl] = yy;
            if (a.scores && row0 + rl < R)
              a.scores[((int64_t(b) * a.c.heads + hk) * R + row0 + rl) * a.capacity + t] = yy;
          }
        }
      }
      meet();
      const int r = row0 + lane;
      const uint64_t mask =
          TREE ? paged_tree_mask(paged_tree_masks(a, b, nodes, lane), min(r, R - 1) / grp) >> ((t - n0) & 63) : 0ull;
      const bool sees = lane < ROWS && r < R && (TREE ? mask & 1 : t < n - (a.S - 1 - r / grp));
      const float yy = s_y[lane < ROWS ? lane : 0];
      const float m_new = sees ? fmaxf(m_run, yy) : m_run, m = m_new == -INFINITY ? 0.0f : m_new;
      const float resc = !sees ? 1.0f : m_run == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_run - m);
      const float p = sees ? __builtin_amdgcn_exp2f(yy - m) : 0.0f;
      m_run = m_new;
      l_one = l_one * resc + p;
#pragma unroll
      for (int h = 0; h < SHT; ++h) l_s[h] *= __shfl(resc, (16 * (ht0 + h) + nl) & 63, 64);
#pragma unroll
      for (int ht = 0; ht < HT; ++ht) {
        const float rr = __shfl(resc, 16 * ht + nl, 64), pv = __shfl(p, 16 * ht + nl, 64) * sc;
        const bool ok = __shfl(int(sees), 16 * ht + nl, 64);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const v4f v = paged_four<FP8>(kr, 16 * NT * wave + 16 * nt + 4 * g);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (ok) acc[ht][nt][i] = fmaf(pv, v[i], acc[ht][nt][i] * rr);
        }
      }
    }

    // ---- the part's end ----
    if (has_s) {
#pragma unroll
      for (int h = 0; h < SHT; ++h) {
        l_s[h] += __shfl_xor(l_s[h], 16, 64);
        l_s[h] += __shfl_xor(l_s[h], 32, 64);
        if (g == 0) s_l[rt][16 * (ht0 + h) + nl] = l_s[h];
      }
    }
    meet();
    const int hl = lane < ROWS ? lane : 0;
    const float l = ((s_l[0][hl] + s_l[1][hl]) + (s_l[2][hl] + s_l[3][hl])) + l_one;  // of row `lane`
    if (whole) {
      const int rr = min(row0 + hl, R - 1);
      float den = l, f = 1.0f, M = m_run;
      if (a.sink) {
        const float sk = a.sink[hk * grp + rr % grp] * kLog2e;
        M = fmaxf(M, sk);
        const float Me = M == -INFINITY ? 0.0f : M;
        f = m_run == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_run - Me);
        den = den * f + __builtin_amdgcn_exp2f(sk - Me);
      }
      const bool dead = TREE && rr / grp >= nodes;  // no node's row
      const float inv = den == 0.0f || dead ? 0.0f : f / den;
      if (a.ml && wave == 0 && lane < ROWS && row0 + lane < R) {
        float* const e = a.ml + 2 * ((int64_t(b) * a.c.heads + hk) * R + row0 + lane);
        e[0] = M == -INFINITY ? 0.0f : M;
        e[1] = den == 0.0f ? 0.0f : 1.0f / den;
      }
#pragma unroll
      for (int ht = 0; ht < HT; ++ht) {
        const float iv = __shfl(inv, 16 * ht + nl, 64);
        const int r = row0 + 16 * ht + nl;
        if (r >= R) continue;
        if (TREE && r / grp >= nodes) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) acc[ht][nt] = v4f{0.f, 0.f, 0.f, 0.f};
        }
        uint16_t* const orow =
            a.o + ((int64_t(b) * a.S + r / grp) * a.H + hk * grp + r % grp) * D + 16 * NT * wave + 4 * g;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          *reinterpret_cast<uint2*>(orow + 16 * nt) = make_uint2(f32x2_to_bf16x2(acc[ht][nt][0] * iv, acc[ht][nt][1] * iv),
                                                                 f32x2_to_bf16x2(acc[ht][nt][2] * iv, acc[ht][nt][3] * iv));
      }
    } else {
      float* const part = a.part + (2 * int64_t(w) + (g0 == 0 ? 1 : 0)) * paged_slot(a.rows, D);
      if (wave == 0 && lane < ROWS && row0 + lane < R) {
        part[lane] = m_run;
        part[a.rows + lane] = l;
      }
#pragma unroll
      for (int ht = 0; ht < HT; ++ht) {
        const int rl = 16 * ht + nl;
        if (row0 + rl >= R) continue;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          *reinterpret_cast<v4f*>(part + paged_head(a.rows) + rl * D + 16 * NT * wave + 16 * nt + 4 * g) = acc[ht][nt];
      }
    }
    meet();  // the buffers are free for the next part's tiles
  }
  paged_empty(a, w, upb, D, 64 * kLatentWaves);
}

template <bool FP8, int HT>
static int latent_launch(PagedAttnArgs a, bool ask, int* workers, hipStream_t stream) {
  const int R = a.S * (a.H / a.c.heads);
  a.W = std::min(cu_count(), kPagedMaxWorkers);
  a.unit_rows = 16 * HT;
  a.rows = std::min(R, a.unit_rows);
  if (ask) {
    *workers = a.W;
    return a.rows;
  }
  a.by_unit = paged_units(a) <= a.W;
  if (a.parent)
    WZ_LAUNCH("paged_attn", stream, (paged_latent_kernel<FP8, HT, true, true>), dim3{unsigned(a.W)}, dim3(64 * kLatentWaves), 0, a);
  else if (a.S > 1 || a.scores)
    WZ_LAUNCH("paged_attn", stream, (paged_latent_kernel<FP8, HT, true, false>), dim3{unsigned(a.W)}, dim3(64 * kLatentWaves), 0, a);
  else
    WZ_LAUNCH("paged_attn", stream, (paged_latent_kernel<FP8, HT, false, false>), dim3{unsigned(a.W)}, dim3(64 * kLatentWaves), 0, a);
  if (int rc = check_launch("paged_attn")) return rc;
  return paged_attn_join<kLatentD>(a, stream);
}

// The kernel of R rows: 16, 32 or 64 a unit.  16 x 16000 latents with 16 / 32 heads 51.6 / 54.2 us, in units of 64 rows 66.3 /
// 65.2.
int paged_latent(bool fp8, const PagedAttnArgs& a, bool ask, int* workers, hipStream_t stream) {
  const int R = a.S * (a.H / a.c.heads);
  if (R <= 16)
    return fp8 ? latent_launch<true, 1>(a, ask, workers, stream) : latent_launch<false, 1>(a, ask, workers, stream);
  if (R <= 32)
    return fp8 ? latent_launch<true, 2>(a, ask, workers, stream) : latent_launch<false, 2>(a, ask, workers, stream);
  return fp8 ? latent_launch<true, 4>(a, ask, workers, stream) : latent_launch<false, 4>(a, ask, workers, stream);
}

}  // namespace wz

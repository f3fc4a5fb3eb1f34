// New tokens of a projection into a paged cache: the norms of the queries' and keys' heads, the rotation by position and
// the write, in one pass over the rows; and the accepted path of a drafted tree, moved to the prefix's end.
#include <algorithm>

#include "paged.h"

namespace wz {

// Row x of a head: x' = x / sqrt(mean(x^2) + eps) w, then (a, b) -> (a c - b s, a s + b c) for the rotary dims' pairs, in
// 32 bits and rounded once.  A row has D / 16 threads; the two pieces of 8 that a thread loads are chosen such that it holds
// both halves of its pairs, so nothing but the sum of squares (and an e4m3 row's maximum) crosses lanes.  Rows are read and
// written once: 8191 tokens of 64 heads and a latent of 512 (1.09 GB) 237 us, 4.6 TB/s, where a copy runs at 5.0; loads that
// pass the caches by take 8 % more, such stores 1 %.  A step of 64 tokens (1.6 MB) takes 4 us, a launch and two ways to memory.
struct AppendArgs {
  const uint16_t* src[3];  // q, k, v
  int64_t sb[3], ss[3], sh[3];
  uint16_t* q_out;
  const float* norm[2];  // of q and k, or null
  const float2* freqs;   // [turns, R / 2] cos, sin
  const int32_t *table, *start, *count, *position;
  float eps;
  int turns, R, lo;  // the rotary dims [lo, lo + R)
  int each;          // whether position is [B, S] rather than [B]
  int width, S, H, rows;  // rows of a token: H, and the KV heads once or twice
  uint32_t total;         // rows in all
};

template <int D, bool FP8, bool HALVES>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedView c, AppendArgs a) {
  constexpr int LPR = D / 16, RPW = 256 / LPR;
  const uint32_t row = blockIdx.x * RPW + threadIdx.x / LPR;
  const int t = threadIdx.x % LPR;
  if (row >= a.total) return;  // a row's threads together
  const uint32_t token = row / uint32_t(a.rows), b = token / uint32_t(a.S);
  const int i = int(token - b * uint32_t(a.S)), r = int(row - token * uint32_t(a.rows));
  const int kind = r < a.H ? 0 : r < a.H + c.heads ? 1 : 2;
  const int h = kind == 0 ? r : kind == 1 ? r - a.H : r - a.H - c.heads;
  // this thread's pieces: rotary ones R / 16 apart, then the rest in order
  const int turned = a.R / 16, first = a.lo / 8;
  const bool turns = kind < 2 && t < turned;
  int p0, p1;
  if (t < turned) {
    p0 = first + t;
    p1 = p0 + turned;
  } else {
    p0 = 2 * (t - turned);
    if (p0 >= first) p0 += 2 * turned;
    p1 = p0 + 1;
  }
  const int n = a.count ? min(max(a.count[b], 0), a.S) : a.S;
  uint16_t* const qo = a.q_out + (int64_t(token) * a.H + h) * D;
  if (i >= n) {
    if (kind == 0) {
      *reinterpret_cast<v4i*>(qo + p0 * 8) = v4i{0, 0, 0, 0};
      *reinterpret_cast<v4i*>(qo + p1 * 8) = v4i{0, 0, 0, 0};
    }
    return;
  }
  const int start = a.start[b];
  int64_t at = 0;
  if (kind > 0) {
    const int64_t slot = int64_t(start) + i;
    at = slot > 0x7FFFFFFFLL ? -1 : paged_row(c, a.table + int64_t(b) * a.width, a.width, h, int(slot));
    if (at < 0) return;
  }
  const uint16_t* const src = a.src[kind] + b * a.sb[kind] + i * a.ss[kind] + h * a.sh[kind];
  const v4i x0 = load16(src + p0 * 8), x1 = load16(src + p1 * 8);
  const int pos = a.position ? (a.each ? a.position[int64_t(b) * a.S + i] : a.position[b] + i) : start + i;
  float f[2][8];
  bf16x8_unpack(x0, f[0]);
  bf16x8_unpack(x1, f[1]);
  const float* const w = kind == 0 ? a.norm[0] : kind == 1 ? a.norm[1] : nullptr;
  if (w) {
    float ss = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss += f[0][e] * f[0][e] + f[1][e] * f[1][e];
#pragma unroll
    for (int o = 1; o < LPR; o <<= 1) ss += __shfl_xor(ss, o, kWave);
    const float rs = 1.0f / sqrtf(ss / float(D) + a.eps);
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 8; e += 4) {
        const v4f ww = *reinterpret_cast<const v4f*>(w + (j ? p1 : p0) * 8 + e);
#pragma unroll
        for (int d = 0; d < 4; ++d) f[j][e + d] = f[j][e + d] * rs * ww[d];
      }
  }
  if (turns) {
    const bool known = uint32_t(pos) < uint32_t(a.turns);
    const float2* const z = a.freqs + int64_t(known ? pos : 0) * (a.R / 2);
    float cs[8], sn[8];
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      // halves: angle 8 t + e of both pieces; pairs: angles 4 t.. of the first piece, 4 (t + turned).. of the second
      const int ang = HALVES ? 8 * t + e : e < 4 ? 4 * t + e : 4 * (t + turned) + e - 4;
      const v4f v = *reinterpret_cast<const v4f*>(z + ang);
      cs[e] = known ? v[0] : NAN;
      sn[e] = known ? v[1] : NAN;
      cs[e + 1] = known ? v[2] : NAN;
      sn[e + 1] = known ? v[3] : NAN;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float& u = HALVES ? f[0][e] : f[e >> 2][2 * (e & 3)];
      float& v = HALVES ? f[1][e] : f[e >> 2][2 * (e & 3) + 1];
      const float x = u, y = v;
      u = x * cs[e] - y * sn[e];
      v = x * sn[e] + y * cs[e];
    }
  }
  auto pack = [](const float (&v)[8]) {
    return v4i{int(f32x2_to_bf16x2(v[0], v[1])), int(f32x2_to_bf16x2(v[2], v[3])), int(f32x2_to_bf16x2(v[4], v[5])),
               int(f32x2_to_bf16x2(v[6], v[7]))};
  };
  if (kind == 0) {
    *reinterpret_cast<v4i*>(qo + p0 * 8) = pack(f[0]);
    *reinterpret_cast<v4i*>(qo + p1 * 8) = pack(f[1]);
    return;
  }
  uint8_t* const dst = kind == 1 ? c.k : c.v;
  if constexpr (!FP8) {
    *reinterpret_cast<v4i*>(dst + (at * D + p0 * 8) * 2) = pack(f[0]);
    *reinterpret_cast<v4i*>(dst + (at * D + p1 * 8) * 2) = pack(f[1]);
  } else {
    float m = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = absmax(absmax(m, f[0][e]), f[1][e]);
#pragma unroll
    for (int o = 1; o < LPR; o <<= 1) m = wave_absmax_xor(m, o);
    const ActScale sc = act_scale(m, false);
    *reinterpret_cast<uint2*>(dst + at * D + p0 * 8) = quant8(f[0], sc, false, false);
    *reinterpret_cast<uint2*>(dst + at * D + p1 * 8) = quant8(f[1], sc, false, false);
    if (t == 0) (kind == 1 ? c.ks : c.vs)[at] = sc.s;
  }
  if (kind == 1 && t == 0 && c.weights) {
    c.weights[at] = 0.0f;
    c.positions[at] = pos;
  }
}

// ---- accept ----

struct AcceptArgs {
  const int32_t *drafted, *parent, *sampled, *table, *start, *count;
  int32_t *lens, *tokens, *path;
  int width, S, B;
  int row_bytes;
};

// The walk: node 0 is taken; from a taken node on to its first child, behind it in order, whose drafted token is the one
// sampled there.  Every wave walks for itself, a lane a node: a ballot a step.  Then the path's rows move down, node p_i to
// place i.  A node stands behind its parent, so p_i >= i, and place j is p_i's own only for a j > i: a thread that
// has its piece of all rows from the first to the last in that order, or loads before it stores, overwrites nothing it needs.
// kAcceptAhead rows are on their way together; 64 trees of 64 nodes (2.3 MB moved) take 6 us, one of 16 takes 4, a launch and
// the way to the table, to the rows and back.
constexpr int kAcceptAhead = 8;

__global__ __launch_bounds__(256) void paged_accept_kernel(PagedView c, AcceptArgs a) {
  const int b = blockIdx.x, lane = threadIdx.x & 63;
  const int S = a.S, nodes = a.count ? min(max(a.count[b], 0), S) : S;
  const int64_t base = int64_t(b) * S;
  const bool is = lane < nodes;
  const int drafted = is ? a.drafted[base + lane] : 0, sampled = is ? a.sampled[base + lane] : 0;
  const int parent = is ? a.parent[base + lane] : -1;
  const int start = a.start[b];
  int m = 0, mine = -1;  // nodes taken; lane i's: the i-th
  int cur = nodes > 0 ? 0 : -1;
  while (cur >= 0) {  // cur grows: S steps at most
    if (lane == m) mine = cur;
    ++m;
    const int token = __builtin_amdgcn_readlane(sampled, cur);
    const uint64_t next = __ballot(is && lane > cur && parent == cur && drafted == token);
    cur = next ? __builtin_ctzll(next) : -1;
  }
  if (blockIdx.y == 0 && threadIdx.x < 64) {
    const int token = __shfl(sampled, mine & 63, 64);
    if (lane < S) {
      a.tokens[base + lane] = lane < m ? token : -1;
      a.path[base + lane] = lane < m ? mine : -1;
    }
    if (lane == 0) a.lens[b] = start + m;
  }
  const uint64_t moved = __ballot(lane < m && mine != lane);
  if (!moved) return;
  // rows of head 0, or -1; a move needs both
  const int32_t* const trow = a.table + int64_t(b) * a.width;
  const int64_t f = int64_t(start) + mine, t = int64_t(start) + lane;
  int64_t from = -1, to = -1;
  if ((moved >> lane) & 1 && f <= 0x7FFFFFFFLL) {
    from = paged_row(c, trow, a.width, 0, int(f));
    to = paged_row(c, trow, a.width, 0, int(t));
    if (from < 0) to = -1;
  }
  const int chunks = a.row_bytes / 16, sides = c.shared ? 1 : 2, per = c.heads * chunks;  // 16-byte pieces
  const int first = __builtin_ctzll(moved);
  // whole waves go through the loop together: the rows come from other lanes
  const int pieces = sides * per;
  for (int x0 = blockIdx.y * 256 + (threadIdx.x & ~63); x0 < pieces; x0 += gridDim.y * 256) {
    const int x = x0 + lane;
    const bool on = x < pieces;
    const int side = on ? x / per : 0, y = on ? x - side * per : 0, h = y / chunks, ch = y - h * chunks;
    uint8_t* const pool = side ? c.v : c.k;
    float* const sc = side ? c.vs : c.ks;
    const bool extra = on && ch == 0 && (c.ks || (c.weights && side == 0));
    for (int i0 = first; i0 < m; i0 += kAcceptAhead) {
      v4i data[kAcceptAhead];
      float scale[kAcceptAhead], weight[kAcceptAhead];
      int pos[kAcceptAhead];
      int64_t dst[kAcceptAhead];
#pragma unroll
      for (int j = 0; j < kAcceptAhead; ++j) {
        const int i = i0 + j;
        const int64_t s = __shfl(from, i & 63, 64) + int64_t(h) * c.page;
        const int64_t d = __shfl(to, i & 63, 64);
        dst[j] = !on || i >= m || d < 0 ? -1 : d + int64_t(h) * c.page;
        if (dst[j] < 0) continue;
        data[j] = load16(pool + s * a.row_bytes + ch * 16);
        if (!extra) continue;
        if (c.ks) scale[j] = sc[s];
        if (c.weights && side == 0) {
          weight[j] = c.weights[s];
          pos[j] = c.positions[s];
        }
      }
#pragma unroll
      for (int j = 0; j < kAcceptAhead; ++j) {
        if (dst[j] < 0) continue;
        *reinterpret_cast<v4i*>(pool + dst[j] * a.row_bytes + ch * 16) = data[j];
        if (!extra) continue;
        if (c.ks) sc[dst[j]] = scale[j];
        if (c.weights && side == 0) {
          c.weights[dst[j]] = weight[j];
          c.positions[dst[j]] = pos[j];
        }
      }
    }
  }
}

}  // namespace wz

extern "C" int wz_paged_append(const wz_paged_kv* cache, const void* q_bf16, const int64_t* q_strides, const void* k_bf16,
                               const int64_t* k_strides, const void* v_bf16, const int64_t* v_strides, void* q_out_bf16,
                               int64_t H, const float* q_norm, const float* k_norm, float eps, const float* freqs,
                               int64_t turns, int64_t rotary, int halves, int64_t offset, const int32_t* table,
                               int64_t table_width, const int32_t* start, const int32_t* count, const int32_t* position,
                               int position_each, int64_t B, int64_t S, hipStream_t stream) {
  using namespace wz;
  PagedView c;
  if (int rc = paged_view("paged_append", cache, table_width, &c)) return rc;
  if (B < 0 || S < 0 || H <= 0 || H > 65536 || B > 0x7FFFFFFFLL || S > 0x7FFFFFFFLL)
    return set_error(WZ_EINVAL, "paged_append: bad shape B=%lld S=%lld H=%lld", (long long)B, (long long)S, (long long)H);
  const int D = cache->head_dim;
  if (rotary < 0 || rotary > D || offset < 0 || offset > D - rotary || (rotary | offset) % 16)
    return set_error(WZ_EINVAL, "paged_append: %lld rotary dims from %lld on (multiples of 16, up to %d)",
                     (long long)rotary, (long long)offset, D);
  if (turns < (rotary > 0 ? 1 : 0) || turns > 0x7FFFFFFFLL)  // a position outside the table reads its first row
    return set_error(WZ_EINVAL, "paged_append: %lld turns", (long long)turns);
  if (B == 0 || S == 0) return WZ_OK;
  const int sides = c.shared ? 1 : 2;
  const int64_t rows = H + sides * int64_t(c.heads);
  if (B > 0x7FFFFFFFLL / S || B * S > 0xFFFFFFFFLL / (rows * (D / 16)))  // a grid has 2^32 threads at most
    return set_error(WZ_EINVAL, "paged_append: %lld sequences of %lld tokens of %lld heads of %d", (long long)B, (long long)S,
                     (long long)rows, D);
  if (!q_bf16 || !k_bf16 || (!c.shared && !v_bf16) || !q_out_bf16 || !q_strides || !k_strides || (!c.shared && !v_strides) ||
      !start || (table_width > 0 && !table) || (rotary > 0 && !freqs))
    return set_error(WZ_EINVAL, "paged_append: null pointer");
  AppendArgs a{};
  const void* const src[3] = {q_bf16, k_bf16, c.shared ? nullptr : v_bf16};
  const int64_t* const strides[3] = {q_strides, k_strides, c.shared ? nullptr : v_strides};
  const int64_t heads[3] = {H, c.heads, c.heads};
  const int64_t out_bytes = B * S * H * D * 2;
  for (int i = 0; i < 1 + sides; ++i) {
    a.src[i] = static_cast<const uint16_t*>(src[i]);
    a.sb[i] = strides[i][0];
    a.ss[i] = strides[i][1];
    a.sh[i] = strides[i][2];
    if (reinterpret_cast<uintptr_t>(src[i]) & 15 || ((a.sb[i] | a.ss[i] | a.sh[i]) & 7) || a.sb[i] < 0 || a.ss[i] < 0 || a.sh[i] < 0)
      return set_error(WZ_EINVAL, "paged_append: rows must be 16-byte aligned (strides multiples of 8, not negative)");
    // q may be turned in its own place: a row's threads have read it before they write it
    const bool itself = i == 0 && src[i] == q_out_bf16 && a.sh[i] == D && a.ss[i] == H * D && (B == 1 || a.sb[i] == S * H * D);
    const int64_t span = 2 * ((B - 1) * a.sb[i] + (S - 1) * a.ss[i] + (heads[i] - 1) * a.sh[i] + D);
    if (!itself && overlap(q_out_bf16, out_bytes, src[i], span))
      return set_error(WZ_EINVAL, "paged_append: the rotated q overlaps an input (it may be q itself)");
  }
  if ((reinterpret_cast<uintptr_t>(q_out_bf16) | reinterpret_cast<uintptr_t>(q_norm) | reinterpret_cast<uintptr_t>(k_norm) |
       reinterpret_cast<uintptr_t>(freqs)) & 15)
    return set_error(WZ_EINVAL, "paged_append: the rotated q, the norms and the turns must be 16-byte aligned");
  a.q_out = static_cast<uint16_t*>(q_out_bf16);
  a.norm[0] = q_norm;
  a.norm[1] = k_norm;
  a.freqs = reinterpret_cast<const float2*>(freqs);
  a.table = table;
  a.start = start;
  a.count = count;
  a.position = position;
  a.each = position_each;
  a.eps = eps;
  a.turns = int(turns);
  a.R = int(rotary);
  a.lo = int(offset);
  a.width = int(table_width);
  a.S = int(S);
  a.H = int(H);
  a.rows = int(rows);
  a.total = uint32_t(B * S * rows);
  const int per = 256 / (D / 16);
  const dim3 grid(unsigned((B * S * rows + per - 1) / per));
#define WZ_APPEND(DD)                                                                                                  \
  do {                                                                                                                 \
    if (c.ks && halves)                                                                                                \
      WZ_LAUNCH("paged_append", stream, (paged_append_kernel<DD, true, true>), grid, dim3(256), 0, c, a);              \
    else if (c.ks)                                                                                                     \
      WZ_LAUNCH("paged_append", stream, (paged_append_kernel<DD, true, false>), grid, dim3(256), 0, c, a);             \
    else if (halves)                                                                                                   \
      WZ_LAUNCH("paged_append", stream, (paged_append_kernel<DD, false, true>), grid, dim3(256), 0, c, a);             \
    else                                                                                                               \
      WZ_LAUNCH("paged_append", stream, (paged_append_kernel<DD, false, false>), grid, dim3(256), 0, c, a);            \
  } while (0)
  if (D == 64) WZ_APPEND(64);
  else if (D == 128) WZ_APPEND(128);
  else if (D == 256) WZ_APPEND(256);
  else WZ_APPEND(512);
#undef WZ_APPEND
  return check_launch("paged_append");
}

extern "C" int wz_paged_accept(const wz_paged_kv* cache, const int32_t* drafted, const int32_t* parent,
                               const int32_t* sampled, const int32_t* table, int64_t table_width, const int32_t* start,
                               const int32_t* count, int32_t* lens, int32_t* tokens, int32_t* path, int64_t B, int64_t S,
                               hipStream_t stream) {
  using namespace wz;
  AcceptArgs a{};
  PagedView c;
  if (int rc = paged_view("paged_accept", cache, table_width, &c)) return rc;
  if (B < 0 || B > 0x7FFFFF || S < 0 || S > 64)
    return set_error(WZ_EINVAL, "paged_accept: bad shape B=%lld S=%lld (up to 64)", (long long)B, (long long)S);
  if (B == 0) return WZ_OK;
  if (!start || !lens || (S > 0 && (!drafted || !parent || !sampled || !tokens || !path)) || (table_width > 0 && !table))
    return set_error(WZ_EINVAL, "paged_accept: null pointer");
  // other workgroups read the inputs while the outputs are written
  const int64_t nodes = 4 * B * S, seqs = 4 * B;
  const struct { const void* p; int64_t n; } in[6] = {{drafted, nodes}, {parent, nodes}, {sampled, nodes}, {start, seqs},
                                                      {count, count ? seqs : 0}, {table, 4 * B * table_width}},
      out[3] = {{lens, seqs}, {tokens, nodes}, {path, nodes}};
  for (int i = 0; i < 3; ++i) {
    for (const auto& x : in)
      if (overlap(out[i].p, out[i].n, x.p, x.n)) return set_error(WZ_EINVAL, "paged_accept: an output overlaps an input");
    for (int j = 0; j < i; ++j)
      if (overlap(out[i].p, out[i].n, out[j].p, out[j].n)) return set_error(WZ_EINVAL, "paged_accept: outputs overlap");
  }
  a.drafted = drafted;
  a.parent = parent;
  a.sampled = sampled;
  a.table = table;
  a.start = start;
  a.count = count;
  a.lens = lens;
  a.tokens = tokens;
  a.path = path;
  a.width = int(table_width);
  a.S = int(S);
  a.B = int(B);
  a.row_bytes = cache->head_dim * (c.ks ? 1 : 2);
  const int64_t pieces = int64_t(c.shared ? 1 : 2) * c.heads * (a.row_bytes / 16);
  const unsigned splits = unsigned(std::min<int64_t>((pieces + 255) / 256, 1024));
  WZ_LAUNCH("paged_accept", stream, paged_accept_kernel, dim3(unsigned(B), splits), dim3(256), 0, c, a);
  return check_launch("paged_accept");
}

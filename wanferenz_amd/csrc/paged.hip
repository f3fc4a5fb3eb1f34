// The paged key-value cache: new tokens into their pages, and eviction by attention weight.
#include <algorithm>

#include "paged.h"

namespace wz {

int paged_view(const char* what, const wz_paged_kv* c, int64_t width, PagedView* v) {
  if (!c) return set_error(WZ_EINVAL, "%s: no cache", what);
  const int d = c->head_dim;
  const bool shared = c->v == nullptr;
  if (c->dtype != WZ_KV_BF16 && c->dtype != WZ_KV_E4M3) return set_error(WZ_EINVAL, "%s: cache type %d", what, c->dtype);
  if (shared ? (d != 128 && d != 256 && d != 512) : (d != 64 && d != 128 && d != 256))
    return set_error(WZ_EINVAL, "%s: head dim %d (64, 128, 256, or 128, 256, 512 where K = V)", what, d);
  if (c->page_size < 16 || c->page_size > 1024 || (c->page_size & (c->page_size - 1)))
    return set_error(WZ_EINVAL, "%s: page size %d (a power of two, 16 to 1024)", what, c->page_size);
  if (c->pages <= 0 || c->kv_heads <= 0 || c->kv_heads > 1024 || c->pages > 0x7FFFFFFFLL)
    return set_error(WZ_EINVAL, "%s: %lld pages of %d heads", what, (long long)c->pages, c->kv_heads);
  if (width < 0 || width > (int64_t(1) << 30) / c->page_size)
    return set_error(WZ_EINVAL, "%s: table width %lld (2^30 slots a sequence)", what, (long long)width);
  if (!c->k) return set_error(WZ_EINVAL, "%s: null pointer", what);
  if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15)
    return set_error(WZ_EINVAL, "%s: k and v must be 16-byte aligned", what);
  if (c->dtype == WZ_KV_E4M3 && (!c->k_scale || (!shared && !c->v_scale)))
    return set_error(WZ_EINVAL, "%s: an e4m3 cache needs its scales", what);
  if (!c->weights != !c->positions)
    return set_error(WZ_EINVAL, "%s: a tracked cache has weights and positions", what);
  v->k = static_cast<uint8_t*>(c->k);
  v->v = shared ? v->k : static_cast<uint8_t*>(c->v);
  v->ks = c->dtype == WZ_KV_E4M3 ? c->k_scale : nullptr;
  v->vs = c->dtype == WZ_KV_E4M3 ? (shared ? c->k_scale : c->v_scale) : nullptr;
  v->weights = c->weights;
  v->positions = c->positions;
  v->pages = int(c->pages);
  v->heads = c->kv_heads;
  v->page = c->page_size;
  v->shift = __builtin_ctz(unsigned(c->page_size));
  v->dtype = c->dtype;
  v->shared = shared;
  return WZ_OK;
}

// ---- write ----

struct WriteArgs {
  const uint16_t* src[2];
  int64_t sb[2], ss[2], sh[2];
  const int32_t *table, *start, *count, *position;
  int width, S;
  int64_t rows;  // B * S * heads
};

// A thread per 16 bytes of a new row, D / 8 threads a row; heads of one token are neighbours, as
// they are in the projection's output.  An e4m3 row's amax is the maximum over its threads, its
// scale and codes act_quant's (act_scale, quant_div) over the whole row.  blockIdx.y: K, V.
template <int D, bool FP8>
__global__ __launch_bounds__(256) void paged_write_kernel(PagedView c, WriteArgs a) {
  constexpr int LPR = D / 8;
  const int64_t t = int64_t(blockIdx.x) * 256 + threadIdx.x;
  const int64_t row = t / LPR;
  const int ch = int(t % LPR), side = blockIdx.y;
  if (row >= a.rows) return;
  const int h = int(row % c.heads), i = int(row / c.heads % a.S), b = int(row / c.heads / a.S);
  if (a.count && i >= a.count[b]) return;
  const int64_t slot64 = int64_t(a.start[b]) + i;
  if (slot64 < 0 || slot64 > 0x7FFFFFFFLL) return;
  const int slot = int(slot64);
  const int64_t at = paged_row(c, a.table + int64_t(b) * a.width, a.width, h, slot);
  if (at < 0) return;
  const v4i x = load16(a.src[side] + b * a.sb[side] + i * a.ss[side] + h * a.sh[side] + ch * 8);
  uint8_t* const dst = side ? c.v : c.k;
  if constexpr (!FP8) {
    *reinterpret_cast<v4i*>(dst + (at * D + ch * 8) * 2) = x;
  } else {
    float m = bf16x8_absmax(x);
#pragma unroll
    for (int o = 1; o < LPR; o <<= 1) m = wave_absmax_xor(m, o);
    const ActScale sc = act_scale(m, false);
    float f[8];
    bf16x8_unpack(x, f);
    *reinterpret_cast<uint2*>(dst + at * D + ch * 8) = quant8(f, sc, false, false);
    if (ch == 0) (side ? c.vs : c.ks)[at] = sc.s;
  }
  if (side == 0 && ch == 0 && c.weights) {
    c.weights[at] = 0.0f;
    c.positions[at] = (a.position ? a.position[b] : a.start[b]) + i;
  }
}

// ---- evict ----

constexpr int kEvictThreads = 1024;

// A slot's place in the order of what stays, as an unsigned number: the float's bits, ordered
// like the values (NaN lowest), a protected slot above them all.
__device__ __forceinline__ uint32_t evict_key(float w, bool safe) {
  if (safe) return 0xFFFFFFFFu;
  const uint32_t u = __float_as_uint(w);
  if ((u & 0x7FFFFFFFu) > 0x7F800000u) return 0u;
  const uint32_t k = u == 0x80000000u ? 0u : u;  // -0 and 0 weigh the same
  return (k & 0x80000000u) ? ~k : k | 0x80000000u;
}

// One workgroup per (sequence, head): the keep-th largest key by four rounds of 8 bits, then one
// pass in slot order that lists the holes below keep and the kept slots from keep on.
__global__ __launch_bounds__(kEvictThreads) void paged_evict_select_kernel(
    PagedView c, const int32_t* __restrict__ table, int width, const int32_t* __restrict__ lens,
    int32_t* __restrict__ counts, int32_t* __restrict__ holes, int32_t* __restrict__ movers, int64_t moves_max,
    int keep, int first, int recent) {
  __shared__ int s_hist[256];
  __shared__ int s_red[kEvictThreads / 64];
  __shared__ int s_pick[2];
  __shared__ int s_scan[3][kEvictThreads / 64];
  const int u = blockIdx.x, b = u / c.heads, h = u % c.heads;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int32_t* const trow = table + int64_t(b) * width;
  const int n = int(min(int64_t(max(lens[b], 0)), int64_t(width) << c.shift));
  if (n <= keep) {
    if (tid == 0) counts[u] = 0;
    return;
  }
  int last = -0x7FFFFFFF - 1;
  for (int t = tid; t < n; t += kEvictThreads) {
    const int64_t at = paged_row(c, trow, width, h, t);
    if (at >= 0) last = max(last, c.positions[at]);
  }
  for (int o = 1; o < 64; o <<= 1) last = max(last, __shfl_xor(last, o, 64));
  if (lane == 0) s_red[wave] = last;
  __syncthreads();
  for (int i = 0; i < kEvictThreads / 64; ++i) last = max(last, s_red[i]);
  auto key_of = [&](int t) -> uint32_t {
    const int64_t at = paged_row(c, trow, width, h, t);
    if (at < 0) return 0u;
    const int p = c.positions[at];
    return evict_key(c.weights[at], p < first || int64_t(p) > int64_t(last) - recent);
  };
  uint32_t prefix = 0, mask = 0;
  int need = keep;  // of the keys that match the prefix
  for (int sh = 24; sh >= 0; sh -= 8) {
    for (int i = tid; i < 256; i += kEvictThreads) s_hist[i] = 0;
    __syncthreads();
    for (int t = tid; t < n; t += kEvictThreads) {
      const uint32_t k = key_of(t);
      if ((k & mask) == prefix) atomicAdd(&s_hist[(k >> sh) & 255], 1);
    }
    __syncthreads();
    if (tid == 0) {
      int left = need, d = 255;
      while (d > 0 && s_hist[d] < left) left -= s_hist[d--];
      s_pick[0] = d;
      s_pick[1] = left;
    }
    __syncthreads();
    prefix |= uint32_t(s_pick[0]) << sh;
    mask |= 255u << sh;
    need = s_pick[1];
    __syncthreads();
  }
  // prefix: the keep-th largest key; `need` slots that have it stay, the lowest first
  int ties = 0, nh = 0, nm = 0;
  for (int t0 = 0; t0 < n; t0 += kEvictThreads) {
    const int t = t0 + tid;
    const uint32_t k = t < n ? key_of(t) : 0u;
    const bool tie = t < n && k == prefix;
    const uint64_t bt = __ballot(tie);
    const uint64_t below = (1ull << lane) - 1;
    if (lane == 0) s_scan[0][wave] = __popcll(bt);
    __syncthreads();
    int tb = ties + __popcll(bt & below);
    for (int i = 0; i < kEvictThreads / 64; ++i) {
      if (i < wave) tb += s_scan[0][i];
      ties += s_scan[0][i];
    }
    const bool kept = t < n && (k > prefix || (tie && tb < need));
    const bool hole = t < n && !kept && t < keep, mover = kept && t >= keep;
    const uint64_t bh = __ballot(hole), bm = __ballot(mover);
    if (lane == 0) {
      s_scan[1][wave] = __popcll(bh);
      s_scan[2][wave] = __popcll(bm);
    }
    __syncthreads();
    int ih = nh + __popcll(bh & below), im = nm + __popcll(bm & below);
    for (int i = 0; i < kEvictThreads / 64; ++i) {
      if (i < wave) {
        ih += s_scan[1][i];
        im += s_scan[2][i];
      }
      nh += s_scan[1][i];
      nm += s_scan[2][i];
    }
    if (hole && ih < moves_max) holes[u * moves_max + ih] = t;
    if (mover && im < moves_max) movers[u * moves_max + im] = t;
    __syncthreads();
  }
  if (tid == 0) counts[u] = min(nh, nm);
}

// The pairs' rows: D * element / 16 threads a row, K and V and what belongs to the slot.
__global__ __launch_bounds__(256) void paged_evict_move_kernel(
    PagedView c, const int32_t* __restrict__ table, int width, const int32_t* __restrict__ lens,
    int32_t* __restrict__ new_lens, const int32_t* __restrict__ counts, const int32_t* __restrict__ holes,
    const int32_t* __restrict__ movers, int64_t moves_max, int keep, int row_bytes) {
  const int u = blockIdx.y, b = u / c.heads, h = u % c.heads;
  if (blockIdx.x == 0 && h == 0 && threadIdx.x == 0)
    new_lens[b] = min(lens[b], keep);
  const int lpr = row_bytes / 16;
  const int count = counts[u];
  const int32_t* const trow = table + int64_t(b) * width;
  for (int64_t t = int64_t(blockIdx.x) * 256 + threadIdx.x; t < int64_t(count) * lpr; t += int64_t(gridDim.x) * 256) {
    const int i = int(t / lpr), ch = int(t % lpr);
    const int64_t to = paged_row(c, trow, width, h, holes[u * moves_max + i]);
    const int64_t fro = paged_row(c, trow, width, h, movers[u * moves_max + i]);
    if (to < 0 || fro < 0) continue;
    *reinterpret_cast<v4i*>(c.k + to * row_bytes + ch * 16) = load16(c.k + fro * row_bytes + ch * 16);
    if (!c.shared) *reinterpret_cast<v4i*>(c.v + to * row_bytes + ch * 16) = load16(c.v + fro * row_bytes + ch * 16);
    if (ch == 0) {
      c.weights[to] = c.weights[fro];
      c.positions[to] = c.positions[fro];
      if (c.ks) c.ks[to] = c.ks[fro];
      if (c.vs && !c.shared) c.vs[to] = c.vs[fro];
    }
  }
}

static int64_t evict_moves_max(const wz_paged_kv* c, int64_t width, int64_t keep) {
  return std::max<int64_t>(0, std::min(keep, width * c->page_size - keep));
}

}  // namespace wz

extern "C" int wz_paged_kv_write(const wz_paged_kv* cache, const void* k_bf16, const int64_t* k_strides,
                                 const void* v_bf16, const int64_t* v_strides, const int32_t* table,
                                 int64_t table_width, const int32_t* start, const int32_t* count,
                                 const int32_t* position, int64_t B, int64_t S, hipStream_t stream) {
  using namespace wz;
  PagedView c;
  if (int rc = paged_view("paged_kv_write", cache, table_width, &c)) return rc;
  if (B < 0 || S < 0 || B > 0x7FFFFFFFLL || S > 0x7FFFFFFFLL)
    return set_error(WZ_EINVAL, "paged_kv_write: bad shape B=%lld S=%lld", (long long)B, (long long)S);
  if (B == 0 || S == 0 || table_width == 0) return WZ_OK;
  if (!k_bf16 || !k_strides || !table || !start || (!c.shared && (!v_bf16 || !v_strides)))
    return set_error(WZ_EINVAL, "paged_kv_write: null pointer");
  WriteArgs a{};
  const void* src[2] = {k_bf16, c.shared ? k_bf16 : v_bf16};
  const int64_t* str[2] = {k_strides, c.shared ? k_strides : v_strides};
  for (int i = 0; i < 2; ++i) {
    if ((reinterpret_cast<uintptr_t>(src[i]) & 15) || ((str[i][0] | str[i][1] | str[i][2]) & 7))
      return set_error(WZ_EINVAL, "paged_kv_write: rows must be 16-byte aligned (strides multiples of 8)");
    a.src[i] = static_cast<const uint16_t*>(src[i]);
    a.sb[i] = str[i][0];
    a.ss[i] = str[i][1];
    a.sh[i] = str[i][2];
  }
  a.table = table;
  a.start = start;
  a.count = count;
  a.position = position;
  a.width = int(table_width);
  a.S = int(S);
  if (B > (int64_t(1) << 40) / (S * c.heads))
    return set_error(WZ_EINVAL, "paged_kv_write: %lld x %lld tokens", (long long)B, (long long)S);
  a.rows = B * S * c.heads;
  const int D = cache->head_dim;
  const int64_t blocks = (a.rows * (D / 8) + 255) / 256;
  if (blocks > 0x7FFFFFFFLL) return set_error(WZ_EINVAL, "paged_kv_write: %lld x %lld tokens", (long long)B, (long long)S);
  const dim3 grid{unsigned(blocks), c.shared ? 1u : 2u};
#define WZ_PAGED_WRITE(DD)                                                                                    \
  do {                                                                                                        \
    if (c.ks)                                                                                                 \
      WZ_LAUNCH("paged_write", stream, (paged_write_kernel<DD, true>), grid, dim3(256), 0, c, a);             \
    else                                                                                                      \
      WZ_LAUNCH("paged_write", stream, (paged_write_kernel<DD, false>), grid, dim3(256), 0, c, a);            \
  } while (0)
  if (D == 64) WZ_PAGED_WRITE(64);
  else if (D == 128) WZ_PAGED_WRITE(128);
  else if (D == 256) WZ_PAGED_WRITE(256);
  else WZ_PAGED_WRITE(512);
#undef WZ_PAGED_WRITE
  return check_launch("paged_kv_write");
}

extern "C" int64_t wz_paged_evict_workspace_bytes(const wz_paged_kv* cache, int64_t B, int64_t table_width,
                                                  int64_t keep) {
  using namespace wz;
  if (!cache || B <= 0 || table_width < 0 || keep < 0 || cache->page_size <= 0 || cache->kv_heads <= 0) return 0;
  const int64_t units = B * cache->kv_heads;
  return (units + 2 * units * evict_moves_max(cache, table_width, keep)) * int64_t(sizeof(int32_t));
}

extern "C" int wz_paged_evict(const wz_paged_kv* cache, const int32_t* table, int64_t table_width, const int32_t* lens,
                              int32_t* new_lens, int64_t B, int64_t keep, int64_t first, int64_t recent,
                              void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  using namespace wz;
  PagedView c;
  if (int rc = paged_view("paged_evict", cache, table_width, &c)) return rc;
  if (!c.weights) return set_error(WZ_EINVAL, "paged_evict: the cache is not tracked (weights and positions)");
  if (B < 0 || B * c.heads > 65535)
    return set_error(WZ_EINVAL, "paged_evict: %lld sequences of %d heads (65535 in all)", (long long)B, c.heads);
  if (keep < 0 || first < 0 || recent < 0 || keep > 0x7FFFFFFFLL || first > keep || recent > keep - first)
    return set_error(WZ_EINVAL, "paged_evict: keep %lld, first %lld, recent %lld (first + recent <= keep)",
                     (long long)keep, (long long)first, (long long)recent);
  if (B == 0) return WZ_OK;
  if (!lens || !new_lens || (table_width > 0 && !table)) return set_error(WZ_EINVAL, "paged_evict: null pointer");
  const int64_t need = wz_paged_evict_workspace_bytes(cache, B, table_width, keep);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return set_error(WZ_ESPACE, "paged_evict: workspace of %lld bytes, %lld needed",
                     (long long)(workspace ? workspace_bytes : 0), (long long)need);
  const int64_t units = B * c.heads, moves = evict_moves_max(cache, table_width, keep);
  int32_t* const counts = static_cast<int32_t*>(workspace);
  int32_t* const holes = counts + units;
  int32_t* const movers = holes + units * moves;
  const int width = int(table_width);
  if (reinterpret_cast<uintptr_t>(workspace) & 3) return set_error(WZ_EINVAL, "paged_evict: workspace alignment");
  WZ_LAUNCH("paged_evict_select", stream, paged_evict_select_kernel, dim3{unsigned(units)}, dim3(kEvictThreads), 0, c,
            table, width, lens, counts, holes, movers, moves, int(keep), int(first), int(recent));
  if (int rc = check_launch("paged_evict")) return rc;
  const int row_bytes = cache->head_dim * (c.ks ? 1 : 2);
  const int64_t blocks = std::min<int64_t>(std::max<int64_t>(1, (moves * (row_bytes / 16) + 255) / 256),
                                           std::max<int64_t>(1, 4096 / units));
  WZ_LAUNCH("paged_evict_move", stream, paged_evict_move_kernel, dim3(unsigned(blocks), unsigned(units)), dim3(256), 0,
            c, table, width, lens, new_lens, counts, holes, movers, moves, int(keep), row_bytes);
  return check_launch("paged_evict");
}

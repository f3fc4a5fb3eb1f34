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
  int width, B, S, block;  // block: tokens of a workgroup
};

// A workgroup takes a few new tokens of a sequence (`block`: 512 pieces of 16 bytes, if the batch has as
// many), D / 8 threads a row and a token's heads next to each other, so whole lines of the projection's
// rows are read.  An e4m3 row's amax is the maximum over its threads, its scale and codes act_quant's
// (act_scale, quant_div) over the whole row.  blockIdx.z: K, V.  Two loads of a thread are in flight
// together: 2 x 32767 tokens of 8 heads of 128 (537 MB) 116 us, with one 123, with four 164, since fewer
// workgroups are left to hide a load's way.  Nothing is read twice here, so loads and stores pass the
// caches by: 109 us, 4.9 TB/s, as a large copy.
constexpr int kWriteLoads = 2;

template <int D, bool FP8>
__global__ __launch_bounds__(256) void paged_write_kernel(PagedView c, WriteArgs a) {
  constexpr int LPR = D / 8, N = kWriteLoads;
  const int side = blockIdx.z, i0 = blockIdx.x * a.block;
  uint8_t* const dst = side ? c.v : c.k;
  const uint32_t per = uint32_t(c.heads) * LPR;  // 16-byte pieces of a token
  for (int b = blockIdx.y; b < a.B; b += gridDim.y) {
    const int count = a.count ? min(max(a.count[b], 0), a.S) : a.S;  // not negative: i0 is taken off it
    const int tokens = min(count - i0, a.block);
    if (tokens <= 0) continue;
    const int start = a.start[b];
    const int32_t* const trow = a.table + int64_t(b) * a.width;
    const uint16_t* const src = a.src[side] + b * a.sb[side] + i0 * a.ss[side];
    const uint32_t pieces = uint32_t(tokens) * per;  // 512 at most, or one token's 1024 x 64
    for (uint32_t p0 = 0; p0 < pieces; p0 += 256 * N) {
      v4i x[N];
      int64_t at[N];
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const uint32_t p = p0 + 256 * j + threadIdx.x;
        at[j] = -1;
        if (p >= pieces) continue;
        const uint32_t i = p / per, hc = p - i * per, h = hc / LPR, ch = hc % LPR;
        const int64_t slot = int64_t(start) + i0 + int(i);
        if (slot > 0x7FFFFFFFLL) continue;
        at[j] = paged_row(c, trow, a.width, int(h), int(slot));
        if (at[j] >= 0) x[j] = load16_nt(src + i * a.ss[side] + h * a.sh[side] + ch * 8);
      }
#pragma unroll
      for (int j = 0; j < N; ++j) {
        if (at[j] < 0) continue;  // the same in a row's threads
        const uint32_t p = p0 + 256 * j + threadIdx.x, ch = p % LPR;
        if constexpr (!FP8) {
          __builtin_nontemporal_store(x[j], reinterpret_cast<v4i*>(dst + (at[j] * D + ch * 8) * 2));
        } else {
          float m = bf16x8_absmax(x[j]);
#pragma unroll
          for (int o = 1; o < LPR; o <<= 1) m = wave_absmax_xor(m, o);
          const ActScale sc = act_scale(m, false);
          float f[8];
          bf16x8_unpack(x[j], f);
          *reinterpret_cast<uint2*>(dst + at[j] * D + ch * 8) = quant8(f, sc, false, false);
          if (ch == 0) (side ? c.vs : c.ks)[at[j]] = sc.s;
        }
        if (side == 0 && ch == 0 && c.weights) {
          c.weights[at[j]] = 0.0f;
          c.positions[at[j]] = (a.position ? a.position[b] : start) + i0 + int(p / per);
        }
      }
    }
  }
}

// ---- evict ----

constexpr int kEvictBins = 2048;         // keys are taken 11, 11 and 10 bits at a time
constexpr int kEvictSmall = 8192;        // slots of a table that one workgroup a unit goes through
constexpr int kEvictThreads = 1024;
constexpr int kEvictChunk = 1024;        // slots of a workgroup where several share a unit
constexpr int kEvictChunkThreads = 256;
constexpr int64_t kEvictUnits = 65535;   // of a call: the grid's second dimension
constexpr int64_t kEvictFused = 65536;   // bytes of K a unit's one workgroup moves itself,
constexpr int kEvictPairs = 1024;        // in up to as many rows
constexpr int kEvictTally = 1028;        // words of a chunk's sums over the last digit
constexpr int kNoPosition = -0x7FFFFFFF - 1;

// A slot's place in the order of what stays, as an unsigned number: the float's bits, ordered
// like the values (NaN lowest, 1), a protected slot above them all.  Slots without a page have 0: they are
// neither kept nor filled, so as many slots stay as have a page below keep.
__device__ __forceinline__ uint32_t evict_key(float w, bool safe) {
  if (safe) return 0xFFFFFFFFu;
  const uint32_t u = __float_as_uint(w);
  if ((u & 0x7FFFFFFFu) > 0x7F800000u) return 1u;
  const uint32_t k = u == 0x80000000u ? 0u : u;  // -0 and 0 weigh the same
  return (k & 0x80000000u) ? ~k : k | 0x80000000u;
}

// What the workgroups that share a unit tell each other.
struct alignas(16) EvictUnit {
  uint32_t hist[3][kEvictBins];  // of the keys' three digits, each under the digits before
  int32_t known[3][2];          // after each digit: the threshold's bits so far, and the keys still needed
};

struct EvictArgs {
  PagedView c;
  const int32_t* table;
  const int32_t* lens;
  int32_t* new_lens;
  int32_t* counts;  // pairs of a unit (sequence, head)
  int32_t* holes;   // [unit][moves]
  int32_t* movers;
  EvictUnit* unit;  // shared units only, as the rest
  int2* newest;     // [unit][chunk]: its newest position, its slots below keep that have a page
  uint32_t* tally;  // [unit][chunk][kEvictTally]
  uint32_t* keys;   // [unit][capacity]
  int64_t moves, capacity;
  int width, keep, first, recent;
};

__device__ __forceinline__ int evict_len(const EvictArgs& a, int b) {
  return int(min(int64_t(max(a.lens[b], 0)), a.capacity));
}

// A pair of rows (of [pages, heads, page]): `fro` over `to`, 16 bytes a thread.
__device__ __forceinline__ void evict_move(const EvictArgs& a, int64_t to, int64_t fro, int ch, int row_bytes) {
  const PagedView& c = a.c;
  if (to < 0 || fro < 0) return;
  const v4i k = load16(c.k + fro * row_bytes + ch * 16);
  v4i v = v4i{0, 0, 0, 0};
  if (!c.shared) v = load16(c.v + fro * row_bytes + ch * 16);
  if (ch == 0) {
    c.weights[to] = c.weights[fro];
    c.positions[to] = c.positions[fro];
    if (c.ks) c.ks[to] = c.ks[fro];
    if (c.vs && !c.shared) c.vs[to] = c.vs[fro];
  }
  *reinterpret_cast<v4i*>(c.k + to * row_bytes + ch * 16) = k;
  if (!c.shared) *reinterpret_cast<v4i*>(c.v + to * row_bytes + ch * 16) = v;
}

// A thread's keys, of the slots t0 + 64 i for i < per <= R (the same for the wave): their positions and
// weights, all loads in flight together.
template <int R>
__device__ __forceinline__ void evict_load(const EvictArgs& a, const int32_t* trow, int h, int n, int t0, int per,
                                           int64_t (&at)[R], int (&p)[R], float (&w)[R]) {
#pragma unroll
  for (int i = 0; i < R; ++i) {
    at[i] = -1;
    if (i < per && t0 + 64 * i < n) at[i] = paged_row(a.c, trow, a.width, h, t0 + 64 * i);
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    p[i] = at[i] >= 0 ? a.c.positions[at[i]] : kNoPosition;
    w[i] = at[i] >= 0 ? a.c.weights[at[i]] : 0.0f;
  }
}

__device__ __forceinline__ int wave_max(int x) {
  for (int o = 1; o < 64; o <<= 1) x = max(x, __shfl_xor(x, o, 64));
  return x;
}
__device__ __forceinline__ int wave_sum(int x) {
  for (int o = 1; o < 64; o <<= 1) x += __shfl_xor(x, o, 64);
  return x;
}

// Counts a wave's keys (the lanes with `in`) in their bins, in a word's upper half where `high`.  The lanes
// that share the first one's bin add up first: equal weights, as a prompt's zeros are, would meet in one
// word of LDS, an addition after the other (32 units of 8000 zeros 33.6 us, so 18.9, 128 of 4160 23.6 and 16.3;
// of random weights 16.2 to 17.2 and 18.2, 13.8 and 14.3).
__device__ __forceinline__ void evict_add(uint32_t* hist, int bin, bool in, bool high) {
  const uint64_t some = __ballot(in);
  if (!some) return;
  const int lead = __builtin_ctzll(some), first = __builtin_amdgcn_readlane(bin, lead);
  const bool same = in && bin == first;
  const uint32_t low = uint32_t(__popcll(__ballot(same && !high))), up = uint32_t(__popcll(__ballot(same && high)));
  if (int(threadIdx.x & 63) == lead) atomicAdd(&hist[first], low + (up << 16));
  if (in && !same) atomicAdd(&hist[bin], high ? 1u << 16 : 1u);
}

// A wave's slots below keep that have a page.
template <int R>
__device__ __forceinline__ int evict_places(const int64_t (&at)[R], int t0, int keep) {
  int have = 0;
#pragma unroll
  for (int i = 0; i < R; ++i) have += __popcll(__ballot(at[i] >= 0 && t0 + 64 * i < keep));
  return have;
}

// The bin, from the top, in which the need-th key lies, and how many of its keys are needed.  Called
// by a whole workgroup; the bins are not changed until everyone has read them.  -> whether all are needed
template <int THREADS>
__device__ __forceinline__ bool evict_pick(const uint32_t* hist, int* bin, int* need) {
  __shared__ int s_sum[THREADS / 64];
  __shared__ int s_out[3];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, want = *need;
  constexpr int P = kEvictBins / THREADS;
  int c[P], sum = 0;
#pragma unroll
  for (int j = 0; j < P; ++j) {
    c[j] = int(hist[kEvictBins - 1 - (tid * P + j)]);
    sum += c[j];
  }
  int up = sum;  // inclusive over the workgroup
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(up, o, 64);
    if (lane >= o) up += y;
  }
  if (lane == 63) s_sum[wave] = up;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < THREADS / 64; ++i) up += i < wave ? s_sum[i] : 0;
  int before = up - sum;
  // the keys are at least `want` in all, so one thread has the crossing (none wanted: the topmost bin)
  if ((up >= want && before < want) || (want == 0 && tid == 0)) {
    int j = 0;
    while (j < P - 1 && before + c[j] < want) before += c[j++];
    s_out[0] = kEvictBins - 1 - (tid * P + j);
    s_out[1] = want - before;
    s_out[2] = want - before == c[j];
  }
  __syncthreads();
  *bin = s_out[0];
  *need = s_out[1];
  return s_out[2] != 0;
}

// Digit d (0, 1, 2) of a key, its place, and whether a key has the threshold's digits before it.
__device__ __forceinline__ constexpr int evict_shift(int d) { return d == 0 ? 21 : d == 1 ? 10 : 0; }
__device__ __forceinline__ int evict_digit(uint32_t k, int d) {
  return int((k >> evict_shift(d)) & (d == 2 ? 1023u : 2047u));
}
__device__ __forceinline__ bool evict_under(uint32_t k, uint32_t prefix, int d) {
  return d == 0 || (d == 1 ? (k ^ prefix) >> 21 == 0 : (k ^ prefix) >> 10 == 0);
}

// A wave's counts of its R rounds: kept slots above the threshold and ties, below keep and past it.
template <int R>
__device__ __forceinline__ void evict_count(const uint32_t (&key)[R], int t0, int per, int keep, uint32_t top,
                                            int (&sum)[4]) {
#pragma unroll
  for (int i = 0; i < R; ++i) {
    if (i >= per) break;
    const int t = t0 + 64 * i;
    const bool low = t < keep, gt = key[i] > top, tie = key[i] != 0 && key[i] == top;
    sum[0] += __popcll(__ballot(gt && low));
    sum[1] += __popcll(__ballot(tie && low));
    sum[2] += __popcll(__ballot(gt && !low));
    sum[3] += __popcll(__ballot(tie && !low));
  }
}

// A wave's part of the lists: hole(i, r) and mover(i, r) take the i-th of the unit, which is in round r of
// this lane.  `before`: evict_count's sums of the slots before the wave's, `all`: of the unit, `have`:
// evict_places of the slots before the wave's.  Of the ties the lowest `need` stay, so those below keep go
// first.  -> the unit's pairs
template <int R, typename Hole, typename Mover>
__device__ __forceinline__ int evict_list(const EvictArgs& a, const uint32_t (&key)[R], int t0, int per, uint32_t top,
                                          int need, const int (&before)[4], const int (&all)[4], int have,
                                          Hole&& put_hole, Mover&& put_mover) {
  const int lane = threadIdx.x & 63;
  const uint64_t below = (1ull << lane) - 1;
  const int high = max(0, need - all[1]);  // ties past keep that stay
  const int pairs = int(min(int64_t(all[2] + min(all[3], high)), a.moves));
  int ties = before[1] + before[3];
  int ih = have - before[0] - min(before[1], need);  // dropped slots below keep
  int im = before[2] + min(before[3], high);                          // kept slots past it
#pragma unroll
  for (int i = 0; i < R; ++i) {
    if (i >= per) break;
    const int t = t0 + 64 * i;
    const bool in = key[i] != 0;
    const uint64_t tie = __ballot(in && key[i] == top);
    const bool kept = key[i] > top || (in && key[i] == top && ties + __popcll(tie & below) < need);
    ties += __popcll(tie);
    const bool hole = in && !kept && t < a.keep, mover = kept && t >= a.keep;
    const uint64_t bh = __ballot(hole), bm = __ballot(mover);
    const int x = ih + __popcll(bh & below), y = im + __popcll(bm & below);
    if (hole && x < pairs) put_hole(x, i);
    if (mover && y < pairs) put_mover(y, i);
    ih += __popcll(bh);
    im += __popcll(bm);
  }
  return pairs;
}

// A unit (sequence, head) of a table of up to kEvictSmall slots (the lengths are on the device, so the table's
// width decides, whatever a sequence holds): the keep-th largest key by three digits, then the
// holes below keep and the kept slots from keep on, in slot order.  Every wave has a range of
// consecutive slots, 64 a round with the keys in registers, so the ranks need one exchange between the
// waves.  MOVE: few pairs are moved here, which saves the second launch.  Its chain of dependent steps
// bounds it: 128 units of 4160 slots cut to 4096 take 14.2 to 14.9 us, 12.9 and a move of 5.2 without MOVE, and 32 to 36
// and a move of 6 as chunks.  16 rounds a thread, for 16384 slots, cost the short ones more than the long ones gain: 4160
// slots 19.3 to 20.4 us, 12000 slots of 32 units 25.8 against 28 to 31 as chunks.
template <bool MOVE>
__global__ __launch_bounds__(kEvictThreads) void paged_evict_small_kernel(EvictArgs a, int row_bytes) {
  constexpr int R = kEvictSmall / kEvictThreads, NW = kEvictThreads / 64;
  __shared__ uint32_t s_hist[3][kEvictBins];
  __shared__ int s_last[NW], s_have[NW];
  __shared__ __align__(16) uint2 s_count[NW];
  const int u = blockIdx.x, b = u / a.c.heads, h = u - b * a.c.heads;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int32_t* const trow = a.table + int64_t(b) * a.width;
  const int n = evict_len(a, b);
  if (MOVE && h == 0 && tid == 0) a.new_lens[b] = min(a.lens[b], a.keep);
  if (n <= a.keep) {
    if (!MOVE && tid == 0) a.counts[u] = 0;
    return;
  }
  const int per = ((n + 63) / 64 + NW - 1) / NW;  // rounds of a wave, up to R
  const int t0 = wave * per * 64 + lane;
  const int end = min(n, (wave + 1) * per * 64);
  int64_t at[R];
  int p[R];
  float w[R];
  evict_load<R>(a, trow, h, end, t0, per, at, p, w);
  for (int i = tid; i < 3 * kEvictBins; i += kEvictThreads) (&s_hist[0][0])[i] = 0;
  int last = kNoPosition;
#pragma unroll
  for (int i = 0; i < R; ++i) last = max(last, p[i]);
  last = wave_max(last);
  const int places = evict_places<R>(at, t0, a.keep);
  if (lane == 0) {
    s_last[wave] = last;
    s_have[wave] = places;
  }
  __syncthreads();
  int need = 0, have = 0;  // the unit's places, and those before the wave's slots
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    last = max(last, s_last[i]);
    have = i == wave ? need : have;
    need += s_have[i];
  }
  const int64_t old = int64_t(last) - a.recent;  // positions above it are protected
  uint32_t key[R];
#pragma unroll
  for (int i = 0; i < R; ++i) key[i] = at[i] < 0 ? 0u : evict_key(w[i], p[i] < a.first || int64_t(p[i]) > old);
  uint32_t top = 0;
#pragma unroll
  for (int d = 0; d < 3; ++d) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      if (i >= per) break;
      evict_add(s_hist[d], evict_digit(key[i], d), key[i] != 0 && evict_under(key[i], top, d), false);
    }
    __syncthreads();
    int bin;
    const bool whole = evict_pick<kEvictThreads>(s_hist[d], &bin, &need);
    top |= uint32_t(bin) << evict_shift(d);
    if (whole) break;  // the bin's keys all stay: the threshold is its lowest, the digits below 0
  }
  int sum[4] = {0, 0, 0, 0};
  evict_count<R>(key, t0, per, a.keep, top, sum);
  // two counts a word: they add up to kEvictSmall at most
  if (lane == 0) s_count[wave] = make_uint2(uint32_t(sum[0]) << 16 | uint32_t(sum[1]), uint32_t(sum[2]) << 16 | uint32_t(sum[3]));
  __syncthreads();
  uint2 total = make_uint2(0, 0), mine = total;
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    const uint2 x = s_count[i];
    mine = i == wave ? total : mine;
    total = make_uint2(total.x + x.x, total.y + x.y);
  }
  const int before[4] = {int(mine.x >> 16), int(mine.x & 0xFFFF), int(mine.y >> 16), int(mine.y & 0xFFFF)};
  const int all[4] = {int(total.x >> 16), int(total.x & 0xFFFF), int(total.y >> 16), int(total.y & 0xFFFF)};
  if constexpr (MOVE) {
    // the pairs' rows stay in LDS, in the histograms' place
    int64_t* const holes = reinterpret_cast<int64_t*>(&s_hist[0][0]);
    int64_t* const movers = holes + kEvictPairs;
    const int pairs = evict_list<R>(a, key, t0, per, top, need, before, all, have, [&](int i, int r) { holes[i] = at[r]; },
                                    [&](int i, int r) { movers[i] = at[r]; });
    __syncthreads();
    const int lpr = row_bytes / 16;
    for (int i = tid; i < pairs * lpr; i += kEvictThreads) evict_move(a, holes[i / lpr], movers[i / lpr], i % lpr, row_bytes);
  } else {
    int32_t* const holes = a.holes + u * a.moves;
    int32_t* const movers = a.movers + u * a.moves;
    const int pairs = evict_list<R>(a, key, t0, per, top, need, before, all, have,
                                    [&](int i, int r) { holes[i] = t0 + 64 * r; },
                                    [&](int i, int r) { movers[i] = t0 + 64 * r; });
    if (tid == 0) a.counts[u] = pairs;
  }
}

// The same for units of wider tables, which one compute unit's instruction rate would bound (32767 slots of 16
// units took it 87 us, 65535 of one 160): a workgroup per chunk of kEvictChunk slots of the table, a launch for
// each time that the workgroups have to meet.  Chunks past a sequence's length end at once, but they are launched
// five times: the 128 units of 4160 slots take 76 us and a move of 9.6 in a table of 131072 slots.  Every launch costs its 4 us whatever it does, so a chunk
// is what one workgroup of four waves does in that time: 26 us in all for both sizes with 1024 slots,
// 48 with 4096.  STEP 0: the chunk's newest position and places, and the unit's
// histograms cleared.  1: keys and the first digit's histogram.  2, 3: the second's and third's, the
// third with the chunk's own: tally[j] = its keys of at least the first two digits' threshold followed
// by j, those below keep in the low 16 bits and those past it in the high.  4: the threshold, what the other chunks
// have above it and at it from their tallies, and the chunk's part of the lists.
template <int STEP>
__global__ __launch_bounds__(kEvictChunkThreads) void paged_evict_chunk_kernel(EvictArgs a) {
  constexpr int R = kEvictChunk / kEvictChunkThreads, NW = kEvictChunkThreads / 64;
  const int u = blockIdx.y, chunk = blockIdx.x, nb = gridDim.x, b = u / a.c.heads, h = u - b * a.c.heads;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int32_t* const trow = a.table + int64_t(b) * a.width;
  const int n = evict_len(a, b);
  EvictUnit& st = a.unit[u];
  int2* const newest = a.newest + int64_t(u) * nb;
  uint32_t* const tally = a.tally + int64_t(u) * nb * kEvictTally;
  uint32_t* const keys = a.keys + u * a.capacity;
  if constexpr (STEP == 0)
    for (int i = chunk * kEvictChunkThreads + tid; i < 3 * kEvictBins; i += nb * kEvictChunkThreads)
      (&st.hist[0][0])[i] = 0;
  if (n <= a.keep) {
    if (STEP == 4 && chunk == 0 && tid == 0) a.counts[u] = 0;
    return;
  }
  const int chunks = (n + kEvictChunk - 1) / kEvictChunk;
  if (chunk >= chunks) return;
  const int t0 = chunk * kEvictChunk + wave * (64 * R) + lane;
  const int end = min(n, t0 - lane + 64 * R);
  __shared__ int s_wave[5][NW];
  uint32_t key[R];
  if constexpr (STEP <= 1) {
    int64_t at[R];
    int p[R];
    float w[R];
    evict_load<R>(a, trow, h, end, t0, R, at, p, w);
    if constexpr (STEP == 0) {
      int last = kNoPosition;
#pragma unroll
      for (int i = 0; i < R; ++i) last = max(last, p[i]);
      last = wave_max(last);
      const int places = evict_places<R>(at, t0, a.keep);
      if (lane == 0) {
        s_wave[0][wave] = last;
        s_wave[1][wave] = places;
      }
      __syncthreads();
      last = wave_max(s_wave[0][lane & (NW - 1)]);
      if (tid == 0) {
        int have = 0;
        for (int i = 0; i < NW; ++i) have += s_wave[1][i];
        newest[chunk] = make_int2(last, have);
      }
      return;
    }
    int last = kNoPosition;
    for (int i = lane; i < chunks; i += 64) last = max(last, newest[i].x);
    const int64_t old = int64_t(wave_max(last)) - a.recent;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      key[i] = at[i] < 0 ? 0u : evict_key(w[i], p[i] < a.first || int64_t(p[i]) > old);
      if (t0 + 64 * i < end) keys[t0 + 64 * i] = key[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < R; ++i) key[i] = t0 + 64 * i < end ? keys[t0 + 64 * i] : 0u;
  }
  // the threshold's digits so far; the launch before wrote what is read here
  uint32_t top = 0;
  int need = 0;
  if constexpr (STEP == 2) {
    for (int i = lane; i < chunks; i += 64) need += newest[i].y;
    need = wave_sum(need);
  }
  if constexpr (STEP > 2) {
    top = uint32_t(st.known[STEP - 3][0]);
    need = st.known[STEP - 3][1];
  }
  if constexpr (STEP >= 2 && STEP <= 4) {
    int bin;
    evict_pick<kEvictChunkThreads>(st.hist[STEP - 2], &bin, &need);
    top |= uint32_t(bin) << evict_shift(STEP - 2);
    if (chunk == 0 && tid == 0) {
      st.known[STEP - 2][0] = int32_t(top);
      st.known[STEP - 2][1] = need;
    }
  }
  if constexpr (STEP == 1 || STEP == 2) {
    constexpr int d = STEP - 1;
    __shared__ uint32_t s_hist[kEvictBins];
    for (int i = tid; i < kEvictBins; i += kEvictChunkThreads) s_hist[i] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < R; ++i)
      evict_add(s_hist, evict_digit(key[i], d), key[i] != 0 && evict_under(key[i], top, d), false);
    __syncthreads();
    for (int i = tid; i < kEvictBins; i += kEvictChunkThreads)
      if (s_hist[i]) atomicAdd(&st.hist[d][i], s_hist[i]);  // integers: the order does not matter
  }
  if constexpr (STEP == 3) {
    __shared__ uint32_t s_hist[1024];
    __shared__ uint32_t s_up[NW];
    static_assert(kEvictChunkThreads * 4 == 1024);
    for (int i = tid; i < 1024; i += kEvictChunkThreads) s_hist[i] = 0;
    __syncthreads();
    uint32_t more = 0;  // the wave's keys above the two digits
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int t = t0 + 64 * i;
      const bool gt = key[i] >> 10 > top >> 10;
      evict_add(s_hist, evict_digit(key[i], 2), key[i] != 0 && evict_under(key[i], top, 2), t >= a.keep);
      more += uint32_t(__popcll(__ballot(gt && t < a.keep))) + (uint32_t(__popcll(__ballot(gt && t >= a.keep))) << 16);
    }
    if (lane == 0) s_wave[0][wave] = int(more);
    __syncthreads();
    more = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) more += uint32_t(s_wave[0][i]);
    uint32_t c[4], sum = 0;  // of the bins from 1023 - 4 tid down
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      c[j] = s_hist[1023 - (4 * tid + j)];
      sum += c[j];
      if (c[j]) atomicAdd(&st.hist[2][1023 - (4 * tid + j)], (c[j] & 0xFFFF) + (c[j] >> 16));
    }
    uint32_t up = sum;  // inclusive over the workgroup
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t y = __shfl_up(up, o, 64);
      if (lane >= o) up += y;
    }
    if (lane == 63) s_up[wave] = up;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NW; ++i) up += i < wave ? s_up[i] : 0;
    uint32_t run = more + up - sum;
    v4i g;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      run += c[j];
      g[3 - j] = int(run);
    }
    *reinterpret_cast<v4i*>(tally + chunk * int64_t(kEvictTally) + 1020 - 4 * tid) = g;
    if (tid == 0) tally[chunk * int64_t(kEvictTally) + 1024] = more;
  }
  if constexpr (STEP == 4) {
    int sum[4] = {0, 0, 0, 0};
    evict_count<R>(key, t0, R, a.keep, top, sum);
    int have = 0;  // the places of the wave, then of those before it
#pragma unroll
    for (int i = 0; i < R; ++i) have += __popcll(__ballot(key[i] != 0 && t0 + 64 * i < a.keep));
    if (lane == 0) {
#pragma unroll
      for (int j = 0; j < 4; ++j) s_wave[j][wave] = sum[j];
      s_wave[4][wave] = have;
    }
    __syncthreads();
    have = 0;
    int before[4] = {0, 0, 0, 0}, all[4] = {0, 0, 0, 0};
    const int bin = evict_digit(top, 2);
    for (int i = lane; i < chunks; i += 64) {
      const uint32_t ge = tally[i * int64_t(kEvictTally) + bin], gt = tally[i * int64_t(kEvictTally) + bin + 1];
      const uint32_t tie = ge - gt;
      const int x[4] = {int(gt & 0xFFFF), int(tie & 0xFFFF), int(gt >> 16), int(tie >> 16)};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        all[j] += x[j];
        before[j] += i < chunk ? x[j] : 0;
      }
      have += i < chunk ? newest[i].y : 0;
    }
    have = wave_sum(have);
    for (int i = 0; i < wave; ++i) have += s_wave[4][i];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      all[j] = wave_sum(all[j]);
      before[j] = wave_sum(before[j]);
      for (int i = 0; i < wave; ++i) before[j] += s_wave[j][i];
    }
    int32_t* const holes = a.holes + u * a.moves;
    int32_t* const movers = a.movers + u * a.moves;
    const int pairs = evict_list<R>(a, key, t0, R, top, need, before, all, have,
                                    [&](int i, int r) { holes[i] = t0 + 64 * r; },
                                    [&](int i, int r) { movers[i] = t0 + 64 * r; });
    if (chunk == 0 && tid == 0) a.counts[u] = pairs;
  }
}

// The pairs' rows: D * element / 16 threads a row, K and V and what belongs to the slot.
__global__ __launch_bounds__(256) void paged_evict_move_kernel(EvictArgs a, int row_bytes) {
  const int u = blockIdx.y, b = u / a.c.heads, h = u - b * a.c.heads;
  if (blockIdx.x == 0 && h == 0 && threadIdx.x == 0) a.new_lens[b] = min(a.lens[b], a.keep);
  const int lpr = row_bytes / 16;
  const int count = a.counts[u];
  const int32_t* const trow = a.table + int64_t(b) * a.width;
  for (int64_t t = int64_t(blockIdx.x) * 256 + threadIdx.x; t < int64_t(count) * lpr; t += int64_t(gridDim.x) * 256) {
    const int64_t i = u * a.moves + t / lpr;
    evict_move(a, paged_row(a.c, trow, a.width, h, a.holes[i]), paged_row(a.c, trow, a.width, h, a.movers[i]), int(t % lpr),
               row_bytes);
  }
}

static int64_t evict_moves_max(const wz_paged_kv* c, int64_t width, int64_t keep) {
  return std::max<int64_t>(0, std::min(keep, width * c->page_size - keep));
}

// Bytes of the workspace's parts, in order: EvictUnit, newest, tally, keys (shared units only), counts,
// holes, movers.
struct EvictSizes {
  int64_t units, chunks, unit, newest, tally, keys, counts, moves, total;
};

static EvictSizes evict_sizes(const wz_paged_kv* c, int64_t B, int64_t width, int64_t keep) {
  EvictSizes z{};
  const int64_t capacity = width * c->page_size;
  z.units = B * c->kv_heads;
  z.moves = evict_moves_max(c, width, keep);
  if (capacity > kEvictSmall) {
    z.chunks = (capacity + kEvictChunk - 1) / kEvictChunk;
    z.unit = z.units * int64_t(sizeof(EvictUnit));
    z.newest = (8 * z.units * z.chunks + 15) / 16 * 16;
    z.tally = 4 * kEvictTally * z.units * z.chunks;
    z.keys = 4 * z.units * capacity;
  }
  z.counts = 4 * z.units;
  z.total = z.unit + z.newest + z.tally + z.keys + z.counts + 8 * z.units * z.moves;
  return z;
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
  a.B = int(B);
  const int D = cache->head_dim;
  a.block = std::max(1, 256 * kWriteLoads / (c.heads * (D / 8)));
  const int64_t blocks = (S + a.block - 1) / a.block;  // of 256 threads: a grid's side stays below 2^32
  if (B > (int64_t(1) << 40) / (S * c.heads) || blocks > 0xFFFFFF)
    return set_error(WZ_EINVAL, "paged_kv_write: %lld x %lld tokens", (long long)B, (long long)S);
  const dim3 grid(unsigned(blocks), unsigned(std::min<int64_t>(B, 65535)),
                  c.shared ? 1u : 2u);
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
  // the shape alone: a caller may ask before its pools exist
  if (!cache || cache->page_size <= 0 || cache->kv_heads <= 0 || cache->kv_heads > 1024) return 0;
  if (table_width < 0 || table_width > (int64_t(1) << 30) / cache->page_size) return 0;
  if (B <= 0 || B > kEvictUnits / cache->kv_heads || keep < 0 || keep > 0x7FFFFFFFLL) return 0;
  return evict_sizes(cache, B, table_width, keep).total;
}

extern "C" int wz_paged_evict(const wz_paged_kv* cache, const int32_t* table, int64_t table_width, const int32_t* lens,
                              int32_t* new_lens, int64_t B, int64_t keep, int64_t first, int64_t recent,
                              void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  using namespace wz;
  PagedView c;
  if (int rc = paged_view("paged_evict", cache, table_width, &c)) return rc;
  if (!c.weights) return set_error(WZ_EINVAL, "paged_evict: the cache is not tracked (weights and positions)");
  if (B < 0 || B > kEvictUnits / c.heads)
    return set_error(WZ_EINVAL, "paged_evict: %lld sequences of %d heads (%lld in all)", (long long)B, c.heads,
                     (long long)kEvictUnits);
  if (keep < 0 || first < 0 || recent < 0 || keep > 0x7FFFFFFFLL || first > keep || recent > keep - first)
    return set_error(WZ_EINVAL, "paged_evict: keep %lld, first %lld, recent %lld (first + recent <= keep)",
                     (long long)keep, (long long)first, (long long)recent);
  if (B == 0) return WZ_OK;
  if (!lens || !new_lens || (table_width > 0 && !table)) return set_error(WZ_EINVAL, "paged_evict: null pointer");
  // other workgroups read lens while new_lens is written: the same array is looked after, a shifted one is not
  if (const uintptr_t l = reinterpret_cast<uintptr_t>(lens), o = reinterpret_cast<uintptr_t>(new_lens);
      l != o && (l < o ? o - l : l - o) < 4 * uintptr_t(B))
    return set_error(WZ_EINVAL, "paged_evict: new_lens overlaps lens (it may be lens itself)");
  const int64_t need = wz_paged_evict_workspace_bytes(cache, B, table_width, keep);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return set_error(WZ_ESPACE, "paged_evict: workspace of %lld bytes, %lld needed",
                     (long long)(workspace ? workspace_bytes : 0), (long long)need);
  if (reinterpret_cast<uintptr_t>(workspace) & 15)
    return set_error(WZ_EINVAL, "paged_evict: the workspace must be 16-byte aligned");
  const EvictSizes z = evict_sizes(cache, B, table_width, keep);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  auto take = [&](int64_t bytes) {
    uint8_t* const p = ws;
    ws += bytes;
    return p;
  };
  EvictArgs a{};
  a.c = c;
  a.table = table;
  a.lens = lens;
  a.new_lens = new_lens;
  a.unit = reinterpret_cast<EvictUnit*>(take(z.unit));
  a.newest = reinterpret_cast<int2*>(take(z.newest));
  a.tally = reinterpret_cast<uint32_t*>(take(z.tally));
  a.keys = reinterpret_cast<uint32_t*>(take(z.keys));
  a.counts = reinterpret_cast<int32_t*>(take(z.counts));
  a.holes = reinterpret_cast<int32_t*>(take(4 * z.units * z.moves));
  a.movers = reinterpret_cast<int32_t*>(take(4 * z.units * z.moves));
  a.moves = z.moves;
  a.capacity = table_width * c.page;
  a.width = int(table_width);
  a.keep = int(keep);
  a.first = int(first);
  a.recent = int(recent);
  const int row_bytes = cache->head_dim * (c.ks ? 1 : 2);
  const unsigned units = unsigned(z.units);
  if (z.chunks == 0) {
    // Up to kEvictFused bytes of a unit are moved by the workgroup that chose them.  The lengths can
    // then be written there too, unless other heads' workgroups still read them.
    const bool move = z.moves * row_bytes <= kEvictFused && z.moves <= kEvictPairs && new_lens != lens;
    if (move)
      WZ_LAUNCH("paged_evict", stream, paged_evict_small_kernel<true>, dim3{units}, dim3(kEvictThreads), 0, a, row_bytes);
    else
      WZ_LAUNCH("paged_evict", stream, paged_evict_small_kernel<false>, dim3{units}, dim3(kEvictThreads), 0, a, row_bytes);
    if (int rc = check_launch("paged_evict")) return rc;
    if (move) return WZ_OK;
  } else {
#define WZ_EVICT(STEP)                                                                                               \
  do {                                                                                                               \
    WZ_LAUNCH("paged_evict", stream, paged_evict_chunk_kernel<STEP>, dim3(unsigned(z.chunks), units),                \
              dim3(kEvictChunkThreads), 0, a);                                                                       \
    if (int rc = check_launch("paged_evict")) return rc;                                                             \
  } while (0)
    WZ_EVICT(0);
    WZ_EVICT(1);
    WZ_EVICT(2);
    WZ_EVICT(3);
    WZ_EVICT(4);
#undef WZ_EVICT
  }
  const int64_t blocks = std::min<int64_t>(std::max<int64_t>(1, (z.moves * (row_bytes / 16) + 255) / 256),
                                           std::max<int64_t>(1, 4096 / z.units));
  WZ_LAUNCH("paged_evict_move", stream, paged_evict_move_kernel, dim3(unsigned(blocks), units), dim3(256), 0, a,
            row_bytes);
  return check_launch("paged_evict");
}

// One token a row of logits, from a given uniform number: temperature, min-p, top-k and top-p.
//
// The tokens of a row stand in one order, by logit and equal ones by index, and every filter keeps a first part of it, so a
// row is done with cumulated weights alone: with w_i = exp((l_i - max) / t) the first token whose cumulated weight exceeds
// u times the kept total.  Nothing is sorted as a whole.  The order's 2048 bins are even steps of log2(1 / w) down to 2^-42;
// a histogram of counts and weights over them says in which bins the cuts and the token lie, and only those bins' tokens are
// gathered and sorted, a few dozen as a rule.  Where they are too many (thousands of equal logits) the row's keys are
// counted digit by digit instead.
//
// Weights are whole multiples of 2^-42 of the largest, so sums have no order and the same call gives the same token: a
// cumulated weight is off by 2^-43 a token at most, and an exponential is within 1.5e-13 of its weight, which takes
// double precision.  32 bits would misplace the borders of 1e5 tokens so far that one row in a thousand got a neighbour.
//
// Its bound is the histogram: some 26 vector instructions and a 64-bit addition in LDS an element, on one of 2048 places
// that a wave's lanes often share.  512 rows of 100003 float32 by mass (205 MB, read three times, the second and third time
// mostly from beyond L2) take 104 to 107 us: 5.8 TB/s, the vector units three quarters busy.  One row is three launches' chains, 21 us.
#include <algorithm>

#include "common.h"

namespace wz {

constexpr int kSampleBins = 2048;
constexpr float kSampleRange = 42.0f;     // log2 of the smallest weight that counts
constexpr double kSampleOne = 4398046511104.0;  // 2^42
constexpr int kSampleList = 4096;         // tokens that are sorted
constexpr int kSampleThreads = 1024;
constexpr int64_t kSampleMaxV = 1 << 21;  // 2^21 weights of 2^42 fit 64 bits
constexpr int kSampleHead = 1024;         // top-k up to here: the first bins are gathered, and only their tokens get weights

constexpr int kSampleSteps = 256;         // of the table of 2^(42 - j / 256)
constexpr int kSampleChunk = 4096;        // logits that a workgroup takes at least where several share a row

constexpr int kSampleShare = 512;         // threads of a workgroup there

typedef unsigned long long u64;

// The bins to gather: the first ones to k's, or k's, p's and the token's own.
struct SampleBins {
  int from[3], to[3], last;
  int cut;  // by count
  u64 total;
  __device__ __forceinline__ bool wanted(int b) const {
    return (b >= from[0] && b <= to[0]) || (b >= from[1] && b <= to[1]) || (b >= from[2] && b <= to[2]);
  }
};

// What the workgroups that share a row tell each other.
struct alignas(16) SampleSpace {
  u64 mass[kSampleBins];  // of each bin, then of the bins before it
  u64 list[kSampleList];
  uint32_t count[kSampleBins];
  SampleBins bins;
  uint32_t listed, done;  // tokens in the list, workgroups that have put in what they have
  float top;              // the row's largest logit, and its first place
  int32_t first;
};

struct SampleArgs {
  const void* logits;
  int64_t stride;  // elements between rows
  const float* u;
  const float *t, *p, *m;  // of each row, or null: the values below
  const int32_t* k;
  float t1, p1, m1;
  int k1;
  int32_t* token;
  float* prob;
  int V;
  int chunks, chunk;   // workgroups a row, and the logits of each
  SampleSpace* space;  // [n], and of each row's chunks the largest logit and its first place:
  float* top;          // [n, chunks]
  int32_t* first;
};

// What a row asks for.
struct SampleRow {
  float t, p, m;
  int k;
  double u;
};

__device__ __forceinline__ SampleRow sample_row(const SampleArgs& a, int64_t row) {
  SampleRow r;
  r.t = a.t ? a.t[row] : a.t1;
  r.p = a.p ? a.p[row] : a.p1;
  r.m = a.m ? a.m[row] : a.m1;
  r.k = a.k ? a.k[row] : a.k1;
  const float u = a.u[row];
  r.u = u >= 0.0f ? double(fminf(u, 0x1.fffffep-1f)) : 0.0;  // a NaN is 0
  return r;
}

// 2^(42 - j / 256), by Taylor's polynomial of e^y.
struct SampleTable {
  double step[kSampleSteps];
  constexpr SampleTable() : step() {
    for (int j = 0; j < kSampleSteps; ++j) {
      const double y = -j * (0.69314718055994530942 / kSampleSteps);
      double e = 1.0;
      for (int i = 20; i > 0; --i) e = 1.0 + e * y / i;
      step[j] = e * kSampleOne;
    }
  }
};
__constant__ constexpr SampleTable kSampleTable;

// 2^-(x / 256) for 0 <= x < 256 * 44 in multiples of 2^-42: 2^-n from the exponent, 2^-(j / 256) from the table and e^(r c) for
// what is left, c = ln(2) / 256 and |r| <= 1 / 2, by Taylor's polynomial (the next term is 1.4e-13); then rounded by an
// addition that leaves no place for the fraction.
__device__ __forceinline__ uint64_t sample_weight(double x, const double* table) {
  constexpr double c = 0.69314718055994530942 / kSampleSteps;
  const double t = x + 0x1.8p52;  // the nearest whole number stands in its low bits
  const int k = __double2loint(t);
  const double r = (t - 0x1.8p52) - x;
  const double step = table[k & (kSampleSteps - 1)];
  const double scaled = __hiloint2double(__double2hiint(step) - ((k >> 8) << 20), __double2loint(step));
  double e = fma(r, c * c * c / 6.0, c * c / 2.0);
  e = fma(e, r, c);
  e = fma(e, r, 1.0);
  return uint64_t(__double_as_longlong(fma(e, scaled, 0x1p52)) & ((1ll << 52) - 1));
}

// How a row's logits are weighed.
struct SampleScale {
  float top;     // the largest logit
  float step;    // bins a logit
  double steps;  // steps of 2^(-1 / 256) a logit
  uint64_t least;  // the smallest weight that min-p keeps
  const double* table;
  __device__ SampleScale(float top, const SampleRow& r, const double* table) : top(top), table(table) {
    const double log2t = 1.44269504088896340736 / double(r.t);
    steps = log2t * kSampleSteps;
    step = float(fmin(log2t * (double(kSampleBins) / double(kSampleRange)), 3e38));
    least = uint64_t(fmin(fmax(rint(double(r.m) * kSampleOne), 0.0), kSampleOne));
  }
  // A temperature below 2e-37 or so, of which a bin's width has no 32-bit inverse: such rows are counted by their keys.
  __device__ bool cold() const { return step >= 3e38f; }
  // Bin of a logit, kSampleBins for one whose weight is nothing (a NaN's among them); lower logits have higher bins.
  __device__ int bin(float l) const {
    const float x = l == top ? 0.0f : (top - l) * step;
    return x < float(kSampleBins) ? int(x) : kSampleBins;
  }
  // The same without the question whether a logit is the largest one, for rows whose largest logit is finite.
  __device__ int bin_finite(float l) const { return int(fminf((top - l) * step, float(kSampleBins))); }
  __device__ uint64_t weight_finite(float l) const { return sample_weight((double(top) - double(l)) * steps, table); }
  __device__ uint64_t weight(float l) const {  // of a logit with a bin
    return l == top ? uint64_t(kSampleOne)
                    : sample_weight(fmin((double(top) - double(l)) * steps, double(kSampleRange + 1) * kSampleSteps), table);
  }
};

// A float's bits, ordered like the floats; -0 is 0.
__device__ __forceinline__ uint32_t sample_key(float l) {
  uint32_t x = __float_as_uint(l);
  if (x == 0x80000000u) x = 0;
  return x & 0x80000000u ? ~x : x | 0x80000000u;
}
__device__ __forceinline__ float sample_unkey(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

// f(logits[N], index of the first) for the row's tokens [begin, end), N of them at a time, each by one of the workgroup's threads;
// what stands outside is -inf.
template <bool BF16, typename F>
__device__ __forceinline__ void sample_each(const SampleArgs& a, int64_t row, int begin, int end, F&& f) {
  constexpr int ESZ = BF16 ? 2 : 4, N = 16 / ESZ;
  const char* const base = static_cast<const char*>(a.logits) + row * a.stride * ESZ;
  const int skew = int((reinterpret_cast<uintptr_t>(base) + int64_t(begin) * ESZ) & 15) / ESZ;
  const int first = begin - skew;  // index of the first 16-byte piece's first element
  const int pieces = (end - first + N - 1) / N;
  // pieces [w0, w0 + whole) lie inside: the first and the last need not
  const int w0 = skew ? 1 : 0, whole = (end - first) / N - w0;
  auto load = [&](int c) { return load16(base + int64_t(begin) * ESZ + (uint32_t(c) * 16u - uint32_t(skew * ESZ))); };
  // the body stands here once: unrolled over the pieces it did not fit the instruction cache; the next piece is on its way
  int c = threadIdx.x;
  v4i next = v4i{0, 0, 0, 0};
  if (uint32_t(c - w0) < uint32_t(max(whole, 0))) next = load(c);
#pragma unroll 1
  for (; c < pieces; c += blockDim.x) {
    const v4i now = next;
    const int later = c + int(blockDim.x), i = first + c * N;
    const bool inside = uint32_t(c - w0) < uint32_t(max(whole, 0));
    if (uint32_t(later - w0) < uint32_t(max(whole, 0))) next = load(later);
    float l[N];
    if (inside) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (BF16) {
          l[2 * e] = bf16lo(uint32_t(now[e]));
          l[2 * e + 1] = bf16hi(uint32_t(now[e]));
        } else {
          l[e] = __int_as_float(now[e]);
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        l[e] = -INFINITY;
        if (i + e >= begin && i + e < end)
          l[e] = BF16 ? bf16_to_f32(*reinterpret_cast<const uint16_t*>(base + int64_t(i + e) * 2))
                      : *reinterpret_cast<const float*>(base + int64_t(i + e) * 4);
      }
    }
    f(l, i);
  }
}

// x of the lanes before, by one of the moves within a wave; nothing where there is none (ROWS: the rows of 16 lanes that get it).
template <int MOVE, int ROWS = 0xF, typename T>
__device__ __forceinline__ T sample_moved(T x) {
  if constexpr (sizeof(T) == 4) {
    return T(__builtin_amdgcn_update_dpp(0, int(x), MOVE, ROWS, 0xF, false));
  } else {
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, int(uint32_t(x)), MOVE, ROWS, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, int(uint32_t(x >> 32)), MOVE, ROWS, 0xF, false);
    return T(hi) << 32 | lo;
  }
}
// Inclusive sums over a row's 16 lanes, and over a wave.
template <typename T>
__device__ __forceinline__ T sample_row_scan(T x) {
  x += sample_moved<0x111>(x);  // row_shr 1, 2, 4, 8
  x += sample_moved<0x112>(x);
  x += sample_moved<0x114>(x);
  return x + sample_moved<0x118>(x);
}
template <typename T>
__device__ __forceinline__ T sample_wave_scan(T x) {
  x = sample_row_scan(x);
  x += sample_moved<0x142, 0xA>(x);  // row_bcast 15 into rows 1 and 3
  return x + sample_moved<0x143, 0xC>(x);  // row_bcast 31 into rows 2 and 3
}
template <typename T>
__device__ __forceinline__ T sample_lane(T x, int lane) {
  const uint32_t lo = __builtin_amdgcn_readlane(int(uint32_t(x)), lane);
  if constexpr (sizeof(T) == 4) return T(lo);
  else return T(uint32_t(__builtin_amdgcn_readlane(int(uint32_t(x >> 32)), lane))) << 32 | lo;
}

// Sums before this thread's x over the workgroup's threads (16 waves at most), in their order; *total: of all.
template <typename T>
__device__ __forceinline__ T sample_over_waves(T x, T in, const T* s_wave, T* total) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const T y = sample_row_scan(lane < waves ? s_wave[lane] : T(0));
  *total = sample_lane(y, waves - 1);
  return (wave ? sample_lane(y, wave - 1) : T(0)) + in - x;
}
template <typename T>
__device__ __forceinline__ T sample_scan(T x, T* s_wave, T* total) {
  const T in = sample_wave_scan(x);
  __syncthreads();  // s_wave is free
  if ((threadIdx.x & 63) == 63) s_wave[threadIdx.x >> 6] = in;
  __syncthreads();
  return sample_over_waves(x, in, s_wave, total);
}

constexpr int kSampleRanked = 512;  // tokens of a list that are sorted by counting
static_assert(kSampleRanked <= kSampleShare && kSampleSteps <= kSampleShare, "a thread each");

struct SampleShared {
  uint32_t count[kSampleBins];  // of each bin, then of the bins before it
  u64 mass[kSampleBins];
  u64 list[kSampleList];        // key << 32 | ~index: descending is the row's order
  int rank[kSampleRanked];
  u64 wave64[16];
  float wavef[16];
  uint32_t wave32[16];
  int at;
  double table[kSampleSteps];
  u64 value[2];  // the weight that the cut by count keeps, and the cut by weight
  int bin[4];
  uint32_t listed;
};

__device__ __forceinline__ float sample_block_max(float x, SampleShared& s) {
  for (int o = 1; o < 64; o <<= 1) x = fmaxf(x, __shfl_xor(x, o, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s.wavef[threadIdx.x >> 6] = x;
  __syncthreads();
  x = s.wavef[0];
  for (int w = 1; w < int(blockDim.x >> 6); ++w) x = fmaxf(x, s.wavef[w]);
  return x;
}

// s.count and s.mass become the sums before each bin; -> the totals.
__device__ __forceinline__ void sample_prefix(SampleShared& s, uint32_t* tokens, u64* total) {
  const int per = kSampleBins / blockDim.x, b0 = threadIdx.x * per;
  uint32_t c = 0;
  u64 w = 0;
#pragma unroll 2
  for (int i = 0; i < per; ++i) {
    c += s.count[b0 + i];
    w += s.mass[b0 + i];
  }
  const uint32_t cin = sample_wave_scan(c);
  const u64 win = sample_wave_scan(w);
  if ((threadIdx.x & 63) == 63) {
    s.wave32[threadIdx.x >> 6] = cin;
    s.wave64[threadIdx.x >> 6] = win;
  }
  __syncthreads();
  uint32_t cs = sample_over_waves(c, cin, s.wave32, tokens);
  u64 ws = sample_over_waves(w, win, s.wave64, total);
#pragma unroll 2
  for (int i = 0; i < per; ++i) {
    const uint32_t x = s.count[b0 + i];
    const u64 y = s.mass[b0 + i];
    s.count[b0 + i] = cs;
    s.mass[b0 + i] = ws;
    cs += x;
    ws += y;
  }
  __syncthreads();
}

// Sorts the list, descending.  A short one by each token's rank: the threads that have the same token count in a part of the list
// each (200 tokens 2 us; sorted 9).  Else to a power of two of places (zeros behind), a pair of places a thread: pairs up to
// 64 apart stay with one wave, which waits for nobody.
__device__ __forceinline__ void sample_sort(SampleShared& s, int n) {
  if (n <= kSampleRanked) {
    int places = 64;
    while (places < n) places <<= 1;
    const int parts = blockDim.x / places, i = threadIdx.x & (places - 1), part = threadIdx.x / places;
    const int share = (n + parts - 1) / parts, j1 = min((part + 1) * share, n);
    const u64 x = s.list[max(min(i, n - 1), 0)];
    int rank = 0;
#pragma unroll 8
    for (int j = part * share; j < j1; ++j) rank += s.list[j] > x;
    if (part == 0) s.rank[i] = 0;
    __syncthreads();
    if (i < n && rank) atomicAdd(&s.rank[i], rank);
    __syncthreads();
    if (int(threadIdx.x) < n) s.list[s.rank[i]] = x;
    __syncthreads();
    return;
  }
  int size = 2 * kSampleRanked;
  while (size < n) size <<= 1;
  for (int i = n + threadIdx.x; i < size; i += blockDim.x) s.list[i] = 0;
  __syncthreads();
#pragma unroll 1
  for (int k = 2; k <= size; k <<= 1)
#pragma unroll 1
    for (int j = k >> 1; j > 0; j >>= 1) {
#pragma unroll 1
      for (int i = threadIdx.x; i < size / 2; i += blockDim.x) {
        const int x = 2 * i - (i & (j - 1)), y = x + j;  // pairs j apart
        const u64 p = s.list[x], q = s.list[y];
        if ((p < q) == !(x & k)) {
          s.list[x] = q;
          s.list[y] = p;
        }
      }
      if (j > 64 || (j == 1 && k >= 128)) __syncthreads();
      else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}

// Digit by digit over the keys of all tokens that have a bin and a weight that min-p keeps: the key at which the count (by
// weight: the weight) cumulated in the order reaches `target`.  -> the key, the count and the weight before it.
template <bool BF16>
__device__ void sample_locate(const SampleArgs& a, int64_t row, const SampleScale& sc, SampleShared& s, bool by_weight,
                              double target, uint32_t* key, uint32_t* count, u64* mass) {
  uint32_t prefix = 0, mask = 0, before = 0;
  u64 lighter = 0;
  for (int d = 0; d < 3; ++d) {
    const int shift = d == 0 ? 21 : d == 1 ? 10 : 0;
    const uint32_t digit = d == 2 ? 1023u : 2047u;
    __syncthreads();
    for (int i = threadIdx.x; i < kSampleBins; i += blockDim.x) {
      s.count[i] = 0;
      s.mass[i] = 0;
    }
    __syncthreads();
    sample_each<BF16>(a, row, 0, a.V, [&](auto& l, int) {
#pragma unroll
      for (const float x : l) {
        if (sc.bin(x) == kSampleBins) continue;
        const uint32_t k = sample_key(x);
        if ((k & mask) != prefix) continue;
        const uint64_t w = sc.weight(x);
        if (w < sc.least) continue;
        const uint32_t at = digit - ((k >> shift) & digit);  // the highest first
        atomicAdd(&s.count[at], 1u);
        atomicAdd(&s.mass[at], u64(w));
      }
    });
    __syncthreads();
    uint32_t tokens;
    u64 total;
    sample_prefix(s, &tokens, &total);
    // the first digit whose sum reaches the target; the last one that holds anything where rounding keeps all below it
    if (threadIdx.x == 0) s.at = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < kSampleBins; i += blockDim.x) {
      const uint32_t c0 = s.count[i], c1 = i + 1 < kSampleBins ? s.count[i + 1] : tokens;
      const double x = by_weight ? double(lighter + s.mass[i]) : double(before + c0);
      if (c1 > c0 && (x < target || c0 == 0)) atomicMax(&s.at, i);
    }
    __syncthreads();
    const int at = s.at;
    before += s.count[at];
    lighter += s.mass[at];
    prefix |= (digit - uint32_t(at)) << shift;
    mask |= digit << shift;
  }
  __syncthreads();
  *key = prefix;
  *count = before;
  *mass = lighter;
}

// A row whose cuts lie among more tokens than are sorted.
template <bool BF16>
__device__ __forceinline__ void sample_dense(const SampleArgs& a, int64_t row, const SampleRow& r, const SampleScale& sc,
                                          SampleShared& s) {
  uint32_t key = 0, before = 0;
  u64 lighter = 0, w = 0;
  double total = 0.0, target = 0.0;
#pragma unroll 1
  for (int step = 0; step < 3; ++step) {  // the cut by count (or the last token), the cut by weight, the token
    if (step == 1 && r.p >= 1.0f) continue;
    target = step == 0 ? (r.k > 0 ? double(r.k) : 4e9) : step == 1 ? fmax(double(r.p) * total, 1.0) : floor(r.u * total) + 1.0;
    sample_locate<BF16>(a, row, sc, s, step > 0, target, &key, &before, &lighter);
    w = sc.weight(sample_unkey(key));
    if (step == 0) {  // tokens of this key: as many as the cut wants, or all
      uint32_t same = 0, all;
      sample_each<BF16>(a, row, 0, a.V, [&](auto& l, int) {
        for (const float x : l) same += sample_key(x) == key && x == x;
      });
      sample_scan(same, s.wave32, &all);
      const uint32_t want = r.k > 0 && uint32_t(r.k) - before < all ? uint32_t(r.k) - before : all;
      total = double(lighter + w * want);
    } else if (step == 1) {
      const double want = fmax(ceil((target - double(lighter)) / double(w)), 1.0);
      total = fmin(double(lighter) + want * double(w), total);
    }
  }
  const uint32_t nth = uint32_t(fmax(floor((r.u * total - double(lighter)) / double(w)), 0.0));
  // the nth token of this key, by index: each thread counts a run of them, then the run that holds it is walked
  const int per = (a.V + int(blockDim.x) - 1) / int(blockDim.x);
  const int i0 = min(int(threadIdx.x) * per, a.V), i1 = min(i0 + per, a.V);
  const char* const base = static_cast<const char*>(a.logits) + row * a.stride * (BF16 ? 2 : 4);
  auto is = [&](int i) {
    const float l = BF16 ? bf16_to_f32(*reinterpret_cast<const uint16_t*>(base + int64_t(i) * 2))
                         : *reinterpret_cast<const float*>(base + int64_t(i) * 4);
    return l == l && sample_key(l) == key;
  };
  uint32_t mine = 0, all;
  for (int i = i0; i < i1; ++i) mine += is(i);
  const uint32_t ahead = sample_scan(mine, s.wave32, &all);
  const uint32_t n = min(nth, all - 1);
  if (ahead <= n && n < ahead + mine) {
    uint32_t left = n - ahead;
    for (int i = i0; i < i1; ++i)
      if (is(i) && left-- == 0) {
        a.token[row] = i;
        a.prob[row] = float(double(w) / total);
        break;
      }
  }
}

// The largest logit of [begin, end) and its first place; every thread gets both.
template <bool BF16>
__device__ __forceinline__ float sample_top(const SampleArgs& a, int64_t row, int begin, int end, SampleShared& s, int* first) {
  float top = -INFINITY;
  int at = 0x7FFFFFFF;
  sample_each<BF16>(a, row, begin, end, [&](auto& l, int i) {  // a thread's indexes grow
    float m = l[0];
    for (const float x : l) m = fmaxf(m, x);
    if (m > top) {
      top = m;
      at = i;
      int e = 0;
      bool past = false;
      for (const float x : l) {
        past |= x == m;
        e += !past;
      }
      at += e;
    }
  });
  const float all = sample_block_max(top, s);
  if (threadIdx.x == 0) s.at = 0x7FFFFFFF;
  __syncthreads();
  if (top == all && at != 0x7FFFFFFF) atomicMin(&s.at, at);
  __syncthreads();
  *first = s.at;
  return all;
}

__device__ __forceinline__ void sample_clear(SampleShared& s) {
  for (int i = threadIdx.x; i < kSampleBins; i += blockDim.x) {
    s.count[i] = 0;
    s.mass[i] = 0;
  }
  if (int(threadIdx.x) < kSampleSteps) s.table[threadIdx.x] = kSampleTable.step[threadIdx.x];
  __syncthreads();
}

// Counts where a cut by count asks for them, weights where the cuts by weight or the token do before the list is there.
__device__ __forceinline__ bool sample_head(const SampleRow& r) { return r.k > 0 && r.k <= kSampleHead; }

template <bool BF16>
__device__ __forceinline__ void sample_histogram(const SampleArgs& a, int64_t row, int begin, int end, const SampleRow& r,
                                                 const SampleScale& sc, SampleShared& s) {
  constexpr int N = BF16 ? 8 : 4;  // a piece's tokens side by side, so that their steps overlap
  if (sample_head(r)) {
    sample_each<BF16>(a, row, begin, end, [&](auto& l, int) {
      int b[N];
#pragma unroll
      for (int e = 0; e < N; ++e) b[e] = sc.bin_finite(l[e]);
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (b[e] < kSampleBins) atomicAdd(&s.count[b[e]], 1u);
    });
  } else {
    const bool counted = r.k > 0;
    sample_each<BF16>(a, row, begin, end, [&](auto& l, int) {
#pragma unroll
      for (int h = 0; h < N; h += 4) {
        int b[4];
        uint64_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) b[e] = sc.bin_finite(l[h + e]);
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = sc.weight_finite(l[h + e]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (b[e] == kSampleBins || w[e] < sc.least) continue;
          if (counted) atomicAdd(&s.count[b[e]], 1u);
          atomicAdd(&s.mass[b[e]], u64(w[e]));
        }
      }
    });
  }
  __syncthreads();
}

// The bins in which the cumulated weight first reaches lo and hi, or with `past` exceeds them: each thread looks at its own.  The
// same comparison in doubles places the token itself, so that those bins hold it.
__device__ __forceinline__ void sample_cross(SampleShared& s, double lo, double hi, bool past, u64 total, int* from, int* to) {
  const int per = kSampleBins / blockDim.x, b0 = threadIdx.x * per;
  if (threadIdx.x == 0) s.bin[0] = s.bin[1] = kSampleBins - 1;
  __syncthreads();
  auto over = [&](u64 w, double target) { return past ? double(w) > target : double(w) >= target; };
  u64 w = s.mass[b0];
#pragma unroll 2
  for (int i = 0; i < per; ++i) {
    const int b = b0 + i;
    const u64 next = b + 1 < kSampleBins ? s.mass[b + 1] : total;
    if (next != w) {
      if (over(next, lo) && !over(w, lo)) s.bin[0] = b;
      if (over(next, hi) && !over(w, hi)) s.bin[1] = b;
    }
    w = next;
  }
  __syncthreads();
  *from = s.bin[0];
  *to = s.bin[1];
  __syncthreads();
}

// From the sums before each bin.
__device__ __forceinline__ SampleBins sample_bins(const SampleRow& r, SampleShared& s, uint32_t tokens, u64 total) {
  SampleBins g{{0, 0, 0}, {-1, -1, -1}, 0, r.k > 0 && uint32_t(r.k) < tokens, total};
  int kb = kSampleBins - 1;
  if (g.cut) {  // the bin of the k-th token
    const int per = kSampleBins / blockDim.x, b0 = threadIdx.x * per;
#pragma unroll 2
    for (int b = b0; b < b0 + per; ++b) {
      const uint32_t through = b + 1 < kSampleBins ? s.count[b + 1] : tokens;
      if (s.count[b] < uint32_t(r.k) && through >= uint32_t(r.k)) s.bin[2] = b;
    }
    __syncthreads();
    kb = s.bin[2];
  }
  if (sample_head(r)) {
    g.to[0] = kb;
  } else {
    auto through = [&](int b) { return double(b + 1 < kSampleBins ? s.mass[b + 1] : total); };
    double lo = double(total), hi = double(total);  // the kept weight is within
    if (g.cut) {
      g.from[0] = g.to[0] = kb;
      lo = double(s.mass[kb]);
      hi = through(kb);
    }
    if (r.p < 1.0f) {
      sample_cross(s, fmax(double(r.p) * lo, 1.0), fmax(double(r.p) * hi, 1.0), false, total, &g.from[1], &g.to[1]);
      lo = fmin(lo, double(s.mass[g.from[1]]));
      hi = fmin(hi, through(g.to[1]));
    }
    sample_cross(s, r.u * lo, r.u * hi, true, total, &g.from[2], &g.to[2]);
  }
  g.last = max(g.to[0], max(g.to[1], g.to[2]));
  return g;
}

// The tokens of the wanted bins, into s.list as far as it reaches; s.listed counts them all.
template <bool BF16>
__device__ __forceinline__ void sample_gather(const SampleArgs& a, int64_t row, int begin, int end, const SampleRow& r,
                                              const SampleScale& sc, const SampleBins& g, SampleShared& s) {
  const bool head = sample_head(r);
  if (threadIdx.x == 0) s.listed = 0;
  __syncthreads();
  sample_each<BF16>(a, row, begin, end, [&](auto& l, int i) {
    constexpr int N = BF16 ? 8 : 4;
    float top = l[0];
#pragma unroll
    for (int e = 1; e < N; ++e) top = fmaxf(top, l[e]);
    if (sc.bin_finite(top) > g.last) return;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const int b = sc.bin_finite(l[e]);
      if (b > g.last || !g.wanted(b)) continue;
      if (!head && sc.weight_finite(l[e]) < sc.least) continue;
      const uint32_t at = atomicAdd(&s.listed, 1u);
      if (at < uint32_t(kSampleList)) s.list[at] = u64(sample_key(l[e])) << 32 | uint32_t(~(i + e));
    }
  });
  __syncthreads();
}

// The cuts and the token from the n tokens in s.list and the sums before each bin.  A thread has a run of the sorted list.
__device__ __forceinline__ void sample_finish(const SampleArgs& a, int64_t row, const SampleRow& r, const SampleScale& sc,
                                              const SampleBins& g, SampleShared& s, int n) {
  const bool head = sample_head(r);
  sample_sort(s, n);
  const int per = (n + int(blockDim.x) - 1) / int(blockDim.x);
  const int i0 = min(int(threadIdx.x) * per, n), i1 = min(i0 + per, n);
  auto logit = [&](int i) { return sample_unkey(uint32_t(s.list[i] >> 32)); };
  auto weigh = [&](int i) -> u64 {
    const uint64_t w = sc.weight(logit(i));
    return w < sc.least ? 0 : w;  // head: min-p keeps another first part
  };
  u64 sum = 0, listed;
  for (int i = i0; i < i1; ++i) sum += weigh(i);
  const u64 before = sample_scan(sum, s.wave64, &listed);
  if (!head) {  // what the list has before a bin's first token, taken off the sums before the bin: an offset for all of its tokens
    u64 cum = before;
    for (int i = i0; i < i1; ++i) {
      const int b = sc.bin(logit(i));
      if (i == 0 || sc.bin(logit(i - 1)) != b) {
        s.mass[b] -= cum;
        s.count[b] -= uint32_t(i);
      }
      cum += weigh(i);
    }
  }
  if (threadIdx.x == 0) {
    s.value[0] = g.total;  // head: there is one token to be kept at least
    s.value[1] = ~0ull;
  }
  __syncthreads();
  // f(place, rank, weight, cumulated weight in the whole order)
  auto each = [&](auto&& f) {
    u64 cum = before;
    for (int i = i0; i < i1; ++i) {
      const u64 w = weigh(i);
      cum += w;
      const int b = head ? 0 : sc.bin(logit(i));
      f(i, uint32_t(i) + (head ? 0u : s.count[b]), w, cum + (head ? 0ull : s.mass[b]));
    }
  };
  if (head) {  // the last token that k and min-p keep
    const int keep = g.cut ? min(r.k, n) : n;
    each([&](int i, uint32_t, u64 w, u64 cum) {
      if (i < keep && w > 0 && (i + 1 == keep || weigh(i + 1) == 0)) s.value[0] = cum;
    });
  } else if (g.cut) {
    each([&](int, uint32_t rank, u64, u64 cum) {
      if (rank == uint32_t(r.k) - 1) s.value[0] = cum;
    });
  }
  __syncthreads();
  u64 kept = s.value[0];
  if (r.p < 1.0f) {
    const double target = fmax(double(r.p) * double(kept), 1.0);
    each([&](int, uint32_t, u64 w, u64 cum) {
      if (double(cum) >= target && double(cum - w) < target) s.value[1] = cum;  // one token of the order
    });
    __syncthreads();
    kept = min(kept, s.value[1]);
  }
  const double target = r.u * double(kept);
  each([&](int i, uint32_t, u64 w, u64 cum) {
    if (double(cum) > target && double(cum - w) <= target) {
      a.token[row] = int32_t(~uint32_t(s.list[i]));
      a.prob[row] = float(double(w) / double(kept));
    }
  });
}

// Rows that need no weights: nothing to choose from, or the first token.
__device__ __forceinline__ bool sample_plain(const SampleArgs& a, int64_t row, const SampleRow& r, float top, int first) {
  const bool none = top == -INFINITY;
  if (!none && r.t > 0.0f) return false;
  if (threadIdx.x == 0) {
    a.token[row] = none ? -1 : first;
    a.prob[row] = none ? 0.0f : 1.0f;
  }
  return true;
}

// A row by one workgroup.  A row whose cuts lie among too many tokens is left to the launch that follows: a kernel that holds the
// code for it too does not fit 64 registers, and one with scratch memory starts its workgroups 16 us apart.
constexpr int kSampleLeft = -2;  // in place of the token

template <bool BF16>
__global__ __launch_bounds__(kSampleThreads, 8) void sample_kernel(SampleArgs a) {
  __shared__ SampleShared s;
  const int64_t row = blockIdx.x;
  const SampleRow r = sample_row(a, row);
  int first;
  const float top = sample_top<BF16>(a, row, 0, a.V, s, &first);
  if (sample_plain(a, row, r, top, first)) return;
  const SampleScale sc(top, r, s.table);
  sample_clear(s);
  if (top != INFINITY && !sc.cold()) {
    sample_histogram<BF16>(a, row, 0, a.V, r, sc, s);
    uint32_t tokens;
    u64 total;
    sample_prefix(s, &tokens, &total);
    const SampleBins g = sample_bins(r, s, tokens, total);
    sample_gather<BF16>(a, row, 0, a.V, r, sc, g, s);
    if (s.listed <= uint32_t(kSampleList)) {
      sample_finish(a, row, r, sc, g, s, int(s.listed));
      return;
    }
  }
  if (threadIdx.x == 0) a.token[row] = kSampleLeft;
}

template <bool BF16>
__global__ __launch_bounds__(kSampleThreads, 4) void sample_dense_kernel(SampleArgs a) {
  __shared__ SampleShared s;
  const int64_t row = blockIdx.x;
  if (a.token[row] != kSampleLeft) return;
  const SampleRow r = sample_row(a, row);
  int first;
  const float top = sample_top<BF16>(a, row, 0, a.V, s, &first);
  const SampleScale sc(top, r, s.table);
  sample_clear(s);
  sample_dense<BF16>(a, row, r, sc, s);
}

// A row by several workgroups, in three launches: the largest logit; the histogram, from which the workgroup that comes last
// chooses the bins; their tokens, which again the last one sorts and finishes.  What a workgroup leaves for
// the last one is written and read with atomics of the device's scope, which pass by the L2 of its own die, and has
// arrived before the workgroup is counted.  (A fence would write all of the L2 back, one workgroup after another: the third launch of
// 64 rows of 131072 took 270 us.)
__device__ __forceinline__ bool sample_last(const SampleArgs& a, SampleSpace& z, SampleShared& s) {
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  if (threadIdx.x == 0)
    s.at = __hip_atomic_fetch_add(&z.done, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == uint32_t(a.chunks) - 1;
  __syncthreads();
  return s.at;
}

template <typename T>
__device__ __forceinline__ T sample_read(T* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

template <bool BF16>
__global__ __launch_bounds__(kSampleShare, 8) void sample_top_kernel(SampleArgs a) {
  __shared__ SampleShared s;
  const int64_t row = blockIdx.y;
  const int c = blockIdx.x, begin = c * a.chunk, end = min(begin + a.chunk, a.V);
  SampleSpace& z = a.space[row];
  const int per = (kSampleBins + a.chunks - 1) / a.chunks;
  for (int i = c * per + threadIdx.x; i < min((c + 1) * per, kSampleBins); i += blockDim.x) {
    z.mass[i] = 0;
    z.count[i] = 0;
  }
  if (c == 0 && threadIdx.x == 0) z.listed = z.done = 0;
  int first;
  const float top = sample_top<BF16>(a, row, begin, end, s, &first);
  if (threadIdx.x == 0) {
    a.top[row * a.chunks + c] = top;
    a.first[row * a.chunks + c] = first;
  }
}

// The row's largest logit and its first place, from its chunks'.
__device__ __forceinline__ float sample_row_top(const SampleArgs& a, int64_t row, int* first) {
  const int lane = threadIdx.x & 63;
  float top = -INFINITY;
  int at = 0x7FFFFFFF;
  for (int c = lane; c < a.chunks; c += 64) {
    const float x = a.top[row * a.chunks + c];
    const int i = a.first[row * a.chunks + c];
    at = x > top ? i : at;
    top = fmaxf(top, x);
  }
#pragma unroll 1
  for (int o = 1; o < 64; o <<= 1) {
    const float x = __shfl_xor(top, o, 64);
    const int y = __shfl_xor(at, o, 64);
    at = x > top ? y : x == top ? min(at, y) : at;
    top = fmaxf(top, x);
  }
  *first = at;
  return top;
}

template <bool BF16>
__global__ __launch_bounds__(kSampleShare, 8) void sample_histogram_kernel(SampleArgs a) {
  __shared__ SampleShared s;
  const int64_t row = blockIdx.y;
  const int begin = blockIdx.x * a.chunk, end = min(begin + a.chunk, a.V);
  const SampleRow r = sample_row(a, row);
  int first;
  const float top = sample_row_top(a, row, &first);
  SampleSpace& z = a.space[row];
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    z.top = top;
    z.first = first;
  }
  if (!is_finite_f32(top) || !(r.t > 0.0f)) return;
  const SampleScale sc(top, r, s.table);
  if (sc.cold()) return;
  sample_clear(s);
  sample_histogram<BF16>(a, row, begin, end, r, sc, s);
  for (int i = threadIdx.x; i < kSampleBins; i += blockDim.x) {
    if (s.count[i]) atomicAdd(&z.count[i], s.count[i]);
    if (s.mass[i]) atomicAdd(&z.mass[i], s.mass[i]);
  }
  if (!sample_last(a, z, s)) return;
#pragma unroll
  for (int j = 0; j < kSampleBins / kSampleShare; ++j) {
    const int i = j * kSampleShare + threadIdx.x;
    s.count[i] = sample_read(&z.count[i]);
    s.mass[i] = sample_read(&z.mass[i]);
  }
  __syncthreads();
  uint32_t tokens;
  u64 total;
  sample_prefix(s, &tokens, &total);
  const SampleBins g = sample_bins(r, s, tokens, total);
  if (threadIdx.x == 0) {
    z.bins = g;
    z.done = 0;
  }
  if (sample_head(r)) return;  // its tokens need no sums before them
  for (int i = threadIdx.x; i < kSampleBins; i += kSampleShare) {
    z.count[i] = s.count[i];
    z.mass[i] = s.mass[i];
  }
}

template <bool BF16>
__global__ __launch_bounds__(kSampleShare, 4) void sample_pick_kernel(SampleArgs a) {
  __shared__ SampleShared s;
  const int64_t row = blockIdx.y;
  const int begin = blockIdx.x * a.chunk, end = min(begin + a.chunk, a.V);
  SampleSpace& z = a.space[row];
  const SampleRow r = sample_row(a, row);
  const SampleBins g = z.bins;  // (of no meaning where the histogram's launch had nothing to do)
  float top = z.top;
  int first = z.first;
  if (!a.t && !(a.t1 > 0.0f)) top = sample_row_top(a, row, &first);  // there was none
  if (top == -INFINITY || !(r.t > 0.0f)) {
    if (blockIdx.x == 0) sample_plain(a, row, r, top, first);
    return;
  }
  const SampleScale sc(top, r, s.table);
  if (int(threadIdx.x) < kSampleSteps) s.table[threadIdx.x] = kSampleTable.step[threadIdx.x];
  if (top == INFINITY || sc.cold()) {
    __syncthreads();
    if (blockIdx.x == 0) sample_dense<BF16>(a, row, r, sc, s);
    return;
  }
  sample_gather<BF16>(a, row, begin, end, r, sc, g, s);
  const int mine = int(s.listed);
  if (threadIdx.x == 0 && mine > 0)
    s.at = int(min(__hip_atomic_fetch_add(&z.listed, uint32_t(mine), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT),
                   uint32_t(kSampleList)));
  __syncthreads();
  if (mine > 0)
    for (int i = threadIdx.x; i < min(mine, kSampleList - s.at); i += blockDim.x)
      __hip_atomic_store(&z.list[s.at + i], s.list[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  if (!sample_last(a, z, s)) return;
  const uint32_t listed = sample_read(&z.listed);
  if (listed > uint32_t(kSampleList)) {
    sample_dense<BF16>(a, row, r, sc, s);
    return;
  }
  for (int i = threadIdx.x; i < int(listed); i += blockDim.x) s.list[i] = sample_read(&z.list[i]);
  if (!sample_head(r))
    for (int i = threadIdx.x; i < kSampleBins; i += kSampleShare) {
      s.count[i] = z.count[i];
      s.mass[i] = z.mass[i];
    }
  __syncthreads();
  sample_finish(a, row, r, sc, g, s, int(listed));
}

// Workgroups a row, and the logits of each.  A row is shared where it is long and rows are few: as many workgroups as fill the chip
// twice, none below kSampleChunk logits.  us shared / by one workgroup each, top-p: 1, 64, 128, 192, 256 rows of 100003 float32
// 25 / 49, 42 / 68, 61 / 76, 89 / 78, 98 / 87; of 131072 bf16 24 / 52, 45 / 78, 66 / 86, 93 / 83, 97 / 85; 1, 64, 256 rows of 20000
// 24 / 19, 29 / 19, 37 / 21.
constexpr int64_t kSampleLong = 32768;

static int sample_chunks(int64_t n, int64_t V, int64_t* chunk) {
  *chunk = V;
  const int64_t want = 2 * cu_count() / std::max<int64_t>(n, 1), most = (V + kSampleChunk - 1) / kSampleChunk;
  if (want < 4 || V < kSampleLong) return 1;
  const int64_t c = std::min(want, most);
  *chunk = ((V + c - 1) / c + 7) / 8 * 8;  // whole 16-byte pieces
  return int((V + *chunk - 1) / *chunk);
}

static int64_t sample_space(int64_t n, int64_t V) {
  if (n <= 0 || n > 0x3FFFFF || V <= 0 || V > kSampleMaxV) return 0;
  int64_t chunk;
  const int64_t c = sample_chunks(n, V, &chunk);
  return c > 1 ? n * (int64_t(sizeof(SampleSpace)) + 8 * c) : 0;
}

}  // namespace wz

extern "C" int64_t wz_sample_workspace_bytes(int64_t n, int64_t V) { return wz::sample_space(n, V); }

extern "C" int wz_sample(const void* logits, int logits_bf16, int64_t row_stride, const float* uniform,
                         const float* temperature, float temperature_all, const int32_t* top_k, int32_t top_k_all,
                         const float* top_p, float top_p_all, const float* min_p, float min_p_all, int32_t* tokens,
                         float* probs, int64_t n, int64_t V, void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  using namespace wz;
  if (n < 0 || n > 0x3FFFFF || V <= 0 || V > kSampleMaxV)
    return set_error(WZ_EINVAL, "sample: %lld rows of %lld logits (up to 2^22 and 2^21)", (long long)n, (long long)V);
  if (row_stride < V) return set_error(WZ_EINVAL, "sample: rows of %lld logits %lld apart", (long long)V, (long long)row_stride);
  if (n == 0) return WZ_OK;
  if (!logits || !uniform || !tokens || !probs) return set_error(WZ_EINVAL, "sample: null pointer");
  if (reinterpret_cast<uintptr_t>(logits) & (logits_bf16 ? 1 : 3)) return set_error(WZ_EINVAL, "sample: logits are not aligned");
  SampleArgs a{};
  a.logits = logits;
  a.stride = row_stride;
  a.u = uniform;
  a.t = temperature;
  a.p = top_p;
  a.m = min_p;
  a.k = top_k;
  a.t1 = temperature_all;
  a.p1 = top_p_all;
  a.m1 = min_p_all;
  a.k1 = top_k_all;
  a.token = tokens;
  a.prob = probs;
  a.V = int(V);
  const int64_t need = sample_space(n, V);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return set_error(WZ_ESPACE, "sample: workspace of %lld bytes, %lld needed",
                     (long long)(workspace ? workspace_bytes : 0), (long long)need);
  if (reinterpret_cast<uintptr_t>(workspace) & 15)
    return set_error(WZ_EINVAL, "sample: the workspace must be 16-byte aligned");
  const int64_t bytes = n * 4;
  const struct { const void* p; int64_t n; } in[] = {{logits, ((n - 1) * row_stride + V) * (logits_bf16 ? 2 : 4)},
                                                     {uniform, bytes}, {temperature, bytes}, {top_k, bytes},
                                                     {top_p, bytes}, {min_p, bytes}};
  for (const auto& x : in)
    if (x.p && (overlap(tokens, bytes, x.p, x.n) || overlap(probs, bytes, x.p, x.n)))
      return set_error(WZ_EINVAL, "sample: an output overlaps an input");
  if (overlap(tokens, bytes, probs, bytes)) return set_error(WZ_EINVAL, "sample: the outputs overlap");
  int64_t chunk;
  a.chunks = sample_chunks(n, V, &chunk);
  a.chunk = int(chunk);
  if (a.chunks == 1) {
    const dim3 block(kSampleThreads);
    if (logits_bf16) WZ_LAUNCH("sample", stream, sample_kernel<true>, dim3(unsigned(n)), block, 0, a);
    else WZ_LAUNCH("sample", stream, sample_kernel<false>, dim3(unsigned(n)), block, 0, a);
    if (int rc = check_launch("sample")) return rc;
    if (!temperature && !(temperature_all > 0.0f)) return WZ_OK;  // no row is left
    if (logits_bf16) WZ_LAUNCH("sample_dense", stream, sample_dense_kernel<true>, dim3(unsigned(n)), block, 0, a);
    else WZ_LAUNCH("sample_dense", stream, sample_dense_kernel<false>, dim3(unsigned(n)), block, 0, a);
    return check_launch("sample");
  }
  a.space = static_cast<SampleSpace*>(workspace);
  a.top = reinterpret_cast<float*>(a.space + n);
  a.first = reinterpret_cast<int32_t*>(a.top + n * a.chunks);
  const dim3 grid(unsigned(a.chunks), unsigned(n)), block(kSampleShare);
  if (logits_bf16) WZ_LAUNCH("sample_top", stream, sample_top_kernel<true>, grid, block, 0, a);
  else WZ_LAUNCH("sample_top", stream, sample_top_kernel<false>, grid, block, 0, a);
  if (int rc = check_launch("sample")) return rc;
  if (temperature || temperature_all > 0.0f) {
    if (logits_bf16) WZ_LAUNCH("sample_histogram", stream, sample_histogram_kernel<true>, grid, block, 0, a);
    else WZ_LAUNCH("sample_histogram", stream, sample_histogram_kernel<false>, grid, block, 0, a);
    if (int rc = check_launch("sample")) return rc;
  }
  if (logits_bf16) WZ_LAUNCH("sample_pick", stream, sample_pick_kernel<true>, grid, block, 0, a);
  else WZ_LAUNCH("sample_pick", stream, sample_pick_kernel<false>, grid, block, 0, a);
  return check_launch("sample");
}

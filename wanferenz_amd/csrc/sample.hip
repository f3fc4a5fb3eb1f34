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
// cumulated weight is off by 2^-43 a token at most, and an exponential's own error, 2e-13 of the weight, comes from double
// precision.  32 bits would misplace the borders of 1e5 tokens so far that one row in a thousand got a neighbour.
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

// 2^-x for 0 <= x < 44 in multiples of 2^-42: Taylor's polynomial of e^y for |y| <= ln(2) / 2 (the next
// term is 2e-13), then rounded by an addition that leaves no place for the fraction.
__device__ __forceinline__ uint64_t sample_weight(double x) {
  const double n = rint(x), y = (n - x) * 0.69314718055994530942;
  double e = 1.0 / 3628800.0;
  e = fma(e, y, 1.0 / 362880.0);
  e = fma(e, y, 1.0 / 40320.0);
  e = fma(e, y, 1.0 / 5040.0);
  e = fma(e, y, 1.0 / 720.0);
  e = fma(e, y, 1.0 / 120.0);
  e = fma(e, y, 1.0 / 24.0);
  e = fma(e, y, 1.0 / 6.0);
  e = fma(e, y, 0.5);
  e = fma(e, y, 1.0);
  e = fma(e, y, 1.0);
  const double s = __hiloint2double((1023 + 42 - int(n)) << 20, 0);  // 2^(42 - n)
  return uint64_t(__double_as_longlong(fma(e, s, 0x1p52)) & ((1ll << 52) - 1));
}

// How a row's logits are weighed.
struct SampleScale {
  float top;     // the largest logit
  float step;    // bins a logit
  double log2t;  // log2(e) / t
  uint64_t least;  // the smallest weight that min-p keeps
  __device__ SampleScale(float top, const SampleRow& r) : top(top) {
    log2t = 1.44269504088896340736 / double(r.t);
    step = float(fmin(log2t * (double(kSampleBins) / double(kSampleRange)), 3e38));
    least = uint64_t(fmin(fmax(rint(double(r.m) * kSampleOne), 0.0), kSampleOne));
  }
  // Bin of a logit, kSampleBins for one whose weight is nothing (a NaN's among them); lower logits have higher bins.
  __device__ int bin(float l) const {
    const float x = l == top ? 0.0f : (top - l) * step;
    return x < float(kSampleBins) ? int(x) : kSampleBins;
  }
  __device__ uint64_t weight(float l) const {  // of a logit with a bin
    return l == top ? uint64_t(kSampleOne) : sample_weight((double(top) - double(l)) * log2t);
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

// f(logit, index) for the row's tokens [begin, end), each by one of the workgroup's threads.
template <bool BF16, typename F>
__device__ __forceinline__ void sample_each(const SampleArgs& a, int64_t row, int begin, int end, F&& f) {
  constexpr int ESZ = BF16 ? 2 : 4, VEC = 16 / ESZ, DEEP = 4;
  const char* const base = static_cast<const char*>(a.logits) + row * a.stride * ESZ;
  const int skew = int((reinterpret_cast<uintptr_t>(base) + int64_t(begin) * ESZ) & 15) / ESZ;
  const int first = begin - skew;  // index of the first 16-byte piece's first element
  const int pieces = (end - first + VEC - 1) / VEC;
  auto one = [&](int i) {
    return BF16 ? bf16_to_f32(*reinterpret_cast<const uint16_t*>(base + int64_t(i) * 2))
                : *reinterpret_cast<const float*>(base + int64_t(i) * 4);
  };
  auto use = [&](const v4i& x, int i) {
    if constexpr (BF16) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f(bf16lo(uint32_t(x[e])), i + 2 * e);
        f(bf16hi(uint32_t(x[e])), i + 2 * e + 1);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) f(__int_as_float(x[e]), i + e);
    }
  };
  for (int c0 = threadIdx.x; c0 < pieces; c0 += DEEP * blockDim.x) {
    v4i x[DEEP];
#pragma unroll
    for (int d = 0; d < DEEP; ++d) {
      const int c = c0 + d * int(blockDim.x), i = first + c * VEC;
      if (i >= begin && i + VEC <= end) x[d] = load16(base + int64_t(i) * ESZ);
    }
#pragma unroll
    for (int d = 0; d < DEEP; ++d) {
      const int c = c0 + d * int(blockDim.x), i = first + c * VEC;
      if (i >= begin && i + VEC <= end) {
        use(x[d], i);
      } else if (c < pieces) {
        for (int e = max(i, begin); e < min(i + VEC, end); ++e) f(one(e), e);
      }
    }
  }
}

// Inclusive sums over the workgroup's threads, in their order; every thread gets the total too.
template <typename T>
__device__ __forceinline__ T sample_scan(T x, T* s_wave, T* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  for (int o = 1; o < 64; o <<= 1) {
    const T y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  __syncthreads();  // s_wave is free
  if (lane == 63) s_wave[wave] = x;
  __syncthreads();
  T before = 0, all = 0;
  for (int w = 0; w < waves; ++w) {
    const T y = s_wave[w];
    if (w < wave) before += y;
    all += y;
  }
  *total = all;
  return before + x;
}

typedef unsigned long long u64;

struct SampleShared {
  uint32_t count[kSampleBins];  // of each bin, then of the bins before it
  u64 mass[kSampleBins];
  u64 list[kSampleList];        // key << 32 | ~index: descending is the row's order
  u64 wave64[16];
  float wavef[16];
  uint32_t wave32[16];
  int at;
  u64 value[2];  // the weight that the cut by count keeps, and the cut by weight
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
  for (int i = 0; i < per; ++i) {
    c += s.count[b0 + i];
    w += s.mass[b0 + i];
  }
  uint32_t cs = sample_scan(c, s.wave32, tokens) - c;
  u64 ws = sample_scan(w, s.wave64, total) - w;
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

// Sorts the list, descending, to a power of two of places (zeros behind).
__device__ __forceinline__ void sample_sort(SampleShared& s, int n) {
  int size = 64;
  while (size < n) size <<= 1;
  for (int i = n + threadIdx.x; i < size; i += blockDim.x) s.list[i] = 0;
  __syncthreads();
  for (int k = 2; k <= size; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      for (int i = threadIdx.x; i < size / 2; i += blockDim.x) {
        const int x = 2 * i - (i & (j - 1)), y = x + j;  // pairs j apart
        const u64 p = s.list[x], q = s.list[y];
        if ((p < q) == !(x & k)) {
          s.list[x] = q;
          s.list[y] = p;
        }
      }
      __syncthreads();
    }
}

// The first bin whose cumulated weight reaches `target`, or with `past` exceeds it, from the sums before each bin; the
// last bin where none does.  The same comparison in doubles places the token itself, so that bin holds it.
__device__ __forceinline__ int sample_bin_of(const SampleShared& s, double target, bool past, u64 total) {
  int lo = 0, hi = kSampleBins - 1;  // the sum through bin b is the sum before b + 1
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    const double through = double(mid + 1 < kSampleBins ? s.mass[mid + 1] : total);
    if (past ? through > target : through >= target) hi = mid;
    else lo = mid + 1;
  }
  return lo;
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
    sample_each<BF16>(a, row, 0, a.V, [&](float l, int) {
      if (sc.bin(l) == kSampleBins) return;
      const uint32_t k = sample_key(l);
      if ((k & mask) != prefix) return;
      const uint64_t w = sc.weight(l);
      if (w < sc.least) return;
      const uint32_t at = digit - ((k >> shift) & digit);  // the highest first
      atomicAdd(&s.count[at], 1u);
      atomicAdd(&s.mass[at], u64(w));
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

template <bool BF16>
__device__ void sample_dense(const SampleArgs& a, int64_t row, const SampleRow& r, const SampleScale& sc, SampleShared& s) {
  uint32_t key, before;
  u64 lighter;
  double total;
  u64 w;
  // all of them, then the cut by count
  sample_locate<BF16>(a, row, sc, s, false, r.k > 0 ? double(r.k) : 4e9, &key, &before, &lighter);
  {
    // tokens of this key: as many as the cut wants, or all
    w = sc.weight(sample_unkey(key));
    uint32_t same = 0, all;
    sample_each<BF16>(a, row, 0, a.V, [&](float l, int) { same += sample_key(l) == key && l == l; });
    sample_scan(same, s.wave32, &all);
    const uint32_t want = r.k > 0 && uint32_t(r.k) - before < all ? uint32_t(r.k) - before : all;
    total = double(lighter + w * want);
  }
  if (r.p < 1.0f) {
    const double target = fmax(double(r.p) * total, 1.0);
    sample_locate<BF16>(a, row, sc, s, true, target, &key, &before, &lighter);
    w = sc.weight(sample_unkey(key));
    const double want = fmax(ceil((target - double(lighter)) / double(w)), 1.0);
    total = fmin(double(lighter) + want * double(w), total);
  }
  const double target = r.u * total;
  sample_locate<BF16>(a, row, sc, s, true, floor(target) + 1.0, &key, &before, &lighter);
  w = sc.weight(sample_unkey(key));
  const uint32_t nth = uint32_t(fmax(floor((target - double(lighter)) / double(w)), 0.0));
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
  const uint32_t through = sample_scan(mine, s.wave32, &all);
  const uint32_t n = min(nth, all - 1);
  if (through > n && through - mine <= n) {
    uint32_t left = n - (through - mine);
    for (int i = i0; i < i1; ++i)
      if (is(i) && left-- == 0) {
        a.token[row] = i;
        a.prob[row] = float(double(w) / total);
        break;
      }
  }
}

// A row by one workgroup.
template <bool BF16>
__global__ __launch_bounds__(kSampleThreads) void sample_kernel(SampleArgs a) {
  __shared__ SampleShared s;
  const int64_t row = blockIdx.x;
  const SampleRow r = sample_row(a, row);
  const bool greedy = !(r.t > 0.0f);
  float top = -INFINITY;
  sample_each<BF16>(a, row, 0, a.V, [&](float l, int) { top = fmaxf(top, l); });
  top = sample_block_max(top, s);
  if (top == -INFINITY) {  // nothing to choose from
    if (threadIdx.x == 0) {
      a.token[row] = -1;
      a.prob[row] = 0.0f;
    }
    return;
  }
  if (greedy) {
    if (threadIdx.x == 0) s.at = 0x7FFFFFFF;
    __syncthreads();
    int at = 0x7FFFFFFF;
    sample_each<BF16>(a, row, 0, a.V, [&](float l, int i) { at = l == top ? min(at, i) : at; });
    if (at != 0x7FFFFFFF) atomicMin(&s.at, at);
    __syncthreads();
    if (threadIdx.x == 0) {
      a.token[row] = s.at;
      a.prob[row] = 1.0f;
    }
    return;
  }
  const SampleScale sc(top, r);
  const bool head = r.k > 0 && r.k <= kSampleHead;
  for (int i = threadIdx.x; i < kSampleBins; i += blockDim.x) {
    s.count[i] = 0;
    s.mass[i] = 0;
  }
  __syncthreads();
  if (head) {
    sample_each<BF16>(a, row, 0, a.V, [&](float l, int) {
      const int b = sc.bin(l);
      if (b < kSampleBins) atomicAdd(&s.count[b], 1u);
    });
  } else {
    sample_each<BF16>(a, row, 0, a.V, [&](float l, int) {
      const int b = sc.bin(l);
      if (b == kSampleBins) return;
      const uint64_t w = sc.weight(l);
      if (w < sc.least) return;
      atomicAdd(&s.count[b], 1u);
      atomicAdd(&s.mass[b], u64(w));
    });
  }
  __syncthreads();
  uint32_t tokens;
  u64 total;
  sample_prefix(s, &tokens, &total);
  // ---- the bins to gather: the first to k's, or k's, p's and u's own ----
  const bool cut = r.k > 0 && uint32_t(r.k) < tokens;
  int kb = -1;
  if (cut) {  // the last bin with fewer than k tokens before it
    int lo = 0, hi = kSampleBins - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (s.count[mid] < uint32_t(r.k)) lo = mid;
      else hi = mid - 1;
    }
    kb = lo;
  }
  int from[3] = {0, 0, 0}, to[3] = {-1, -1, -1};
  auto through = [&](int b) { return b + 1 < kSampleBins ? s.mass[b + 1] : total; };
  if (head) {
    to[0] = cut ? kb : kSampleBins - 1;
  } else {
    double lo = double(total), hi = double(total);  // the kept total is within
    if (cut) {
      from[0] = to[0] = kb;
      lo = double(s.mass[kb]);
      hi = double(through(kb));
    }
    if (r.p < 1.0f) {
      from[1] = sample_bin_of(s, fmax(double(r.p) * lo, 1.0), false, total);
      to[1] = sample_bin_of(s, fmax(double(r.p) * hi, 1.0), false, total);
      lo = fmin(lo, double(s.mass[from[1]]));
      hi = fmin(hi, double(through(to[1])));
    }
    from[2] = sample_bin_of(s, r.u * lo, true, total);
    to[2] = sample_bin_of(s, r.u * hi, true, total);
  }
  auto wanted = [&](int b) {
    return (b >= from[0] && b <= to[0]) || (b >= from[1] && b <= to[1]) || (b >= from[2] && b <= to[2]);
  };
  const int last = max(to[0], max(to[1], to[2]));
  uint32_t many = 0;
  for (int b = threadIdx.x; b < kSampleBins; b += blockDim.x)
    if (wanted(b)) many += (b + 1 < kSampleBins ? s.count[b + 1] : tokens) - s.count[b];
  uint32_t all;
  sample_scan(many, s.wave32, &all);
  if (all > uint32_t(kSampleList)) {
    sample_dense<BF16>(a, row, r, sc, s);
    return;
  }
  if (threadIdx.x == 0) s.listed = 0;
  __syncthreads();
  sample_each<BF16>(a, row, 0, a.V, [&](float l, int i) {
    const int b = sc.bin(l);
    if (b > last || !wanted(b)) return;
    if (!head && sc.weight(l) < sc.least) return;
    const uint32_t at = atomicAdd(&s.listed, 1u);
    if (at < uint32_t(kSampleList)) s.list[at] = u64(sample_key(l)) << 32 | uint32_t(~i);
  });
  __syncthreads();
  const int n = min(int(s.listed), kSampleList);
  sample_sort(s, n);
  // ---- places 4 threadIdx.x .. +4 of the list: each token's rank, and its weight cumulated in the whole order ----
  constexpr int PER = kSampleList / kSampleThreads;
  const int i0 = threadIdx.x * PER;
  uint64_t w[PER];
  u64 cum[PER], sum = 0;
  int bin[PER];
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    const float l = sample_unkey(uint32_t(s.list[max(min(i0 + e, n - 1), 0)] >> 32));
    bin[e] = sc.bin(l);
    w[e] = i0 + e < n ? sc.weight(l) : 0;
    if (w[e] < sc.least) w[e] = 0;  // head: min-p is another first part
    sum += w[e];
    cum[e] = sum;
  }
  u64 listed;
  const u64 before = sample_scan(sum, s.wave64, &listed) - sum;
#pragma unroll
  for (int e = 0; e < PER; ++e) cum[e] += before;
  // where a bin begins in the list its sums before are known: an offset for all of its tokens
  uint32_t rank[PER];
  if (head) {
#pragma unroll
    for (int e = 0; e < PER; ++e) rank[e] = uint32_t(i0 + e);
  } else {
    // (bins that the list holds have their list's sums turned into offsets, by the token that begins them)
    __syncthreads();
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const int i = i0 + e;
      if (i >= n) continue;
      const bool begins = i == 0 || sc.bin(sample_unkey(uint32_t(s.list[i - 1] >> 32))) != bin[e];
      if (begins) {
        s.mass[bin[e]] -= cum[e] - w[e];
        s.count[bin[e]] -= uint32_t(i);
      }
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const int i = i0 + e;
      rank[e] = i < n ? s.count[bin[e]] + uint32_t(i) : 0;
      if (i < n) cum[e] += s.mass[bin[e]];
    }
  }
  // ---- the cut by count, the cut by weight, the token ----
  if (threadIdx.x == 0) {
    s.value[0] = head ? 0 : total;
    s.value[1] = ~0ull;
  }
  __syncthreads();
  if (head) {  // the last token that k and min-p keep
    const uint32_t keep = cut ? uint32_t(r.k) : uint32_t(n);
#pragma unroll
    for (int e = 0; e < PER; ++e)
      if (i0 + e < n && rank[e] < keep && w[e] > 0) atomicMax(&s.value[0], cum[e]);
  } else if (cut) {
#pragma unroll
    for (int e = 0; e < PER; ++e)
      if (i0 + e < n && rank[e] == uint32_t(r.k) - 1) s.value[0] = cum[e];
  }
  __syncthreads();
  u64 kept = s.value[0];
  if (r.p < 1.0f) {
    const double target = fmax(double(r.p) * double(kept), 1.0);
#pragma unroll
    for (int e = 0; e < PER; ++e)
      if (i0 + e < n && double(cum[e]) >= target && double(cum[e] - w[e]) < target) {
        s.value[1] = cum[e];  // one token of the order
      }
    __syncthreads();
    kept = min(kept, s.value[1]);
  }
  const double target = r.u * double(kept);
#pragma unroll
  for (int e = 0; e < PER; ++e)
    if (i0 + e < n && double(cum[e]) > target && double(cum[e] - w[e]) <= target) {
      a.token[row] = int32_t(~uint32_t(s.list[i0 + e]));
      a.prob[row] = float(double(w[e]) / double(kept));
    }
}

}  // namespace wz

extern "C" int wz_sample(const void* logits, int logits_bf16, int64_t row_stride, const float* uniform,
                         const float* temperature, float temperature_all, const int32_t* top_k, int32_t top_k_all,
                         const float* top_p, float top_p_all, const float* min_p, float min_p_all, int32_t* tokens,
                         float* probs, int64_t n, int64_t V, hipStream_t stream) {
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
  if (logits_bf16)
    WZ_LAUNCH("sample", stream, sample_kernel<true>, dim3(unsigned(n)), dim3(kSampleThreads), 0, a);
  else
    WZ_LAUNCH("sample", stream, sample_kernel<false>, dim3(unsigned(n)), dim3(kSampleThreads), 0, a);
  return check_launch("sample");
}

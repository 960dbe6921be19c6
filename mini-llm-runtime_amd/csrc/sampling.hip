// Sampling from logits with temperature, top-k, top-p and min-p, one given
// random number a row, in one launch.
//
// Row of logits x_i, T > 0, in descending order with ties by index:
//   w_i = exp((x_i - max x) / T)
//   kept: the first k; of those the shortest head with weight >= p times
//   theirs; of those the ones with w_i >= min_p. All are heads of the order.
//   S = sum of the kept; token = the first whose running sum exceeds u S.
//
// No sort of the row: since every filter and the draw ask for "the element at
// which the running count or weight reaches a target", the row is cut into
// kBins bins of equal distance from the maximum (monotone in x, so bins are in
// order), counts and weights of the bins are summed in LDS, and only the bin
// that holds the target is collected and sorted. A bin with more than kList
// elements (equal logits, T large) is narrowed by the bits of the FP32 value,
// and equal values by index.
//
// Weights are integers: w_i = round(2^shift exp(...)), 44 bits below the
// largest (past 2^18 tokens 62 - log2 of their number), from 64-bit arithmetic (a
// table of 2^(-j/1024) and the first three terms of the series for the rest: within
// 7e-12 relative). A token of less than 2^-45 of the largest weighs 0 and is not
// drawn. So sums are exact, no matter in which order atomics and scans add, the same
// logits and random numbers give the same token always, and a token differs from the
// formula's in exact arithmetic only where u S is next to a border: within 7e-12 S
// and the roundings of the weights between, each at most 2^-45 of the largest.
//
// One workgroup of 1,024 threads per row, which reads it three times (maximum,
// bins, collecting), the later times from the caches. What bounds a large batch is
// the 64-bit arithmetic of the weights, once per element. With few rows one CU
// each would be the bound; then a row is cut over several workgroups and the
// steps are launches of their own, the bins summed by integer atomics. 256 bf16 rows
// of 151,936 logits (77.8 MB) with top-p: 111 us, 0.7 TB/s, of which the maximum 14,
// the bins 39, collecting 10 to 30 and sorting 11 to 19; 48 FP32 rows in four
// launches: 60 us, more than half of it the sort and the bins' scan of the last.
//
// What a list cannot hold is done by one workgroup a row, step by step: a top_k past
// 2,048, and rows whose borders' bins hold more elements (equal logits, temperatures
// that level the row). 1 and 256 bf16 rows of 151,936: top_k = 50 and top_p = 0.9 38
// and 69 us, top_k = 5,000 208 and 227 us, a temperature of 20 214 and 297 us, with
// top_p = 0.9 beside it 366 and 470 us.
#include "mlr_common.h"

#include <algorithm>

namespace mlr {
namespace {

constexpr int kThreads = 1024;
constexpr int kWavesWg = kThreads / 64;
constexpr int kBins = 4096;  // 4 per thread; the last holds what weighs nothing
constexpr int kList = 2048;  // 2 per thread
constexpr int kTable = 1024;
constexpr int kMaxParts = 64, kPartMin = 2048;
constexpr int64_t kMaxVocab = int64_t(1) << 23;  // a segment of 1 / kBins of it fits the list

struct RowSpace;

struct SampleParams {
  const void *logits;
  int64_t row_st, num_logit_rows;
  const int64_t *row_ids;
  const void *uniforms;
  const float *temperature, *top_p, *min_p;
  const void *top_k;
  double temperature_v, top_p_v, min_p_v;
  int64_t top_k_v;
  int64_t *tokens;
  float *logprobs;
  int vocab, shift;
  bool uniforms_f64, top_k_i64;
  int parts;        // workgroups a row is cut over
  RowSpace *space;  // [rows], if parts > 1
};

template <typename T>
struct alignas(16) Row16 {
  T v[16 / sizeof(T)];
};

struct Shared {
  double table[kTable];
  uint64_t wsum[kBins + 64];  // from kBins on: a slot per lane for what has no bin
  uint64_t list[kList];  // sorted: ~key in the upper half, index in the lower
  uint32_t cnt[kBins + 64];
  uint64_t scan_w[kWavesWg];
  uint32_t scan_c[kWavesWg];
  uint64_t found_w;
  uint32_t found_c, found_at, found_n;
  uint32_t fill;
  float red_x[kWavesWg];
};

// FP32 values in unsigned order; both zeros alike.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b ^ (b & 0x80000000u ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float of_key(uint32_t k) {
  return __uint_as_float(k ^ (k & 0x80000000u ? 0x80000000u : 0xffffffffu));
}

// f(x, first index, count) over a row in runs of count <= N neighbours: 16 bytes
// a load, four loads of a thread in flight. A thread's indices ascend.
template <typename T, typename F>
__device__ __forceinline__ void each_run(const T *row, int n, F f) {
  constexpr int kVec = 16 / sizeof(T), kDeep = 4;
  const int tid = threadIdx.x;
  const int head = min(n, static_cast<int>(((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) /
                                           sizeof(T)));
  float x[kVec] = {};
  if (tid < head) {
    x[0] = Elem<T>::to_f32(row[tid]);
    f(x, tid, std::integral_constant<int, 1>{});
  }
  const int nv = (n - head) / kVec;
  const Row16<T> *vec = reinterpret_cast<const Row16<T> *>(row + head);
  for (int v0 = tid; v0 < nv; v0 += kDeep * kThreads) {
    Row16<T> r[kDeep];
#pragma unroll
    for (int k = 0; k < kDeep; ++k) r[k] = vec[min(v0 + k * kThreads, nv - 1)];
#pragma unroll
    for (int k = 0; k < kDeep; ++k) {
      const int v = v0 + k * kThreads;
      if (v < nv) {
#pragma unroll
        for (int j = 0; j < kVec; ++j) x[j] = Elem<T>::to_f32(r[k].v[j]);
        f(x, head + v * kVec, std::integral_constant<int, kVec>{});
      }
    }
  }
  const int rest = head + nv * kVec + tid;
  if (rest < n) {
    x[0] = Elem<T>::to_f32(row[rest]);
    f(x, rest, std::integral_constant<int, 1>{});
  }
}
// f(x, index) over a row.
template <typename T, typename F>
__device__ __forceinline__ void each(const T *row, int n, F f) {
  each_run(row, n, [&](const float *x, int i, auto count) {
#pragma unroll
    for (int j = 0; j < decltype(count)::value; ++j) f(x[j], i + j);
  });
}

// What turns a logit into its weight and its bin.
struct Scale {
  float mx, bins;        // the row's maximum; bins per unit of distance
  double mxd, c, far;    // c: 1024ths of a halving per unit of distance; far: 60 halvings
  int shift;

  __device__ __forceinline__ int bin(float x) const {
    return static_cast<int>(fminf((mx - x) * bins, static_cast<float>(kBins - 1)));
  }
  __device__ __forceinline__ uint64_t weight(float x, const double *table) const {
    constexpr double kMagic = 6755399441055744.0;  // 1.5 * 2^52: rounds to integer
    constexpr double kStep = 0.69314718055994530942 / kTable;
    // Past 60 halvings every weight rounds to 0; fmin also takes a NaN there.
    const double d = fmin(mxd - static_cast<double>(x), far);
    const double whole = fma(d, c, kMagic);
    const int k = __double2loint(whole);
    const double r = fma(d, c, kMagic - whole);
    const double series = fma(r, fma(r, 0.5 * kStep * kStep, -kStep), 1.0);
    const double w = ldexp(series * table[k & (kTable - 1)], shift - (k >> 10));
    return __double_as_longlong(w + 4503599627370496.0) & 0xFFFFFFFFFFFFFull;
  }
};

// Per-thread neighbours of an array of counts and weights with what lies
// before them.
template <int N>
struct Scan {
  uint32_t c[N], before_c, total_c;
  uint64_t w[N], before_w, total_w;
};

template <int N>
__device__ void scan_block(Scan<N> &s, Shared &sh) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  uint32_t c = 0;
  uint64_t w = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    c += s.c[i];
    w += s.w[i];
  }
  const uint32_t own_c = c;
  const uint64_t own_w = w;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t pc = __shfl_up(c, o);
    const uint64_t pw = __shfl_up(static_cast<unsigned long long>(w), o);
    if (lane >= o) {
      c += pc;
      w += pw;
    }
  }
  __syncthreads();  // the last use of scan_c, scan_w
  if (lane == 63) {
    sh.scan_c[wv] = c;
    sh.scan_w[wv] = w;
  }
  __syncthreads();
  uint32_t bc = 0, tc = 0;
  uint64_t bw = 0, tw = 0;
  for (int i = 0; i < kWavesWg; ++i) {
    if (i == wv) {
      bc = tc;
      bw = tw;
    }
    tc += sh.scan_c[i];
    tw += sh.scan_w[i];
  }
  s.before_c = bc + c - own_c;
  s.before_w = bw + w - own_w;
  s.total_c = tc;
  s.total_w = tw;
}

// Sum and largest of the threads' values, the same in all of them.
__device__ uint64_t total_of(uint64_t w, Shared &sh) {
  Scan<1> s;
  s.c[0] = 0;
  s.w[0] = w;
  scan_block(s, sh);
  return s.total_w;
}
__device__ uint64_t max_of(uint64_t w, Shared &sh) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1)
    w = max(w, static_cast<uint64_t>(__shfl_xor(static_cast<unsigned long long>(w), o)));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh.scan_w[threadIdx.x >> 6] = w;
  __syncthreads();
  for (int i = 0; i < kWavesWg; ++i) w = max(w, sh.scan_w[i]);
  return w;
}

// A place in the order: the array's entry at which the running count (kCount)
// or weight reaches `target` (1 <= target <= total), what lies before it and
// the entry itself. The same in all threads.
struct Place {
  int at;
  uint32_t before_c, c;
  uint64_t before_w, w;
};

template <bool kCount, int N>
__device__ Place find(const Scan<N> &s, uint64_t target, Shared &sh) {
  __syncthreads();  // the last use of found_*
  uint32_t bc = s.before_c;
  uint64_t bw = s.before_w;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint64_t b = kCount ? bc : bw, own = kCount ? s.c[i] : s.w[i];
    if (b < target && target <= b + own) {
      sh.found_at = threadIdx.x * N + i;
      sh.found_c = bc;
      sh.found_w = bw;
      sh.found_n = s.c[i];
      sh.scan_w[0] = s.w[i];
    }
    bc += s.c[i];
    bw += s.w[i];
  }
  __syncthreads();
  Place r{static_cast<int>(sh.found_at), sh.found_c, sh.found_n, sh.found_w, sh.scan_w[0]};
  return r;
}

__device__ __forceinline__ Scan<4> scan_bins(Shared &sh, bool weights) {
  Scan<4> s;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    s.c[i] = sh.cnt[threadIdx.x * 4 + i];
    s.w[i] = weights ? sh.wsum[threadIdx.x * 4 + i] : 0;
  }
  scan_block(s, sh);
  return s;
}

__device__ __forceinline__ void clear_bins(Shared &sh) {
  __syncthreads();
  for (int i = threadIdx.x; i < kBins; i += kThreads) {
    sh.cnt[i] = 0;
    sh.wsum[i] = 0;
  }
  __syncthreads();
}

__device__ __forceinline__ uint64_t entry_of(float x, int i) {
  return (static_cast<uint64_t>(~key_of(x)) << 32) | static_cast<uint32_t>(i);
}
__device__ __forceinline__ float value_of(uint64_t entry) {
  return of_key(~static_cast<uint32_t>(entry >> 32));
}

// Sorts the first `count` entries of the list; the result holds them two to a
// thread, with `base` before them.
__device__ Scan<2> sort_list(const Scale &sc, Shared &sh, int count, uint32_t base_c,
                             uint64_t base_w) {
  int size = 128;
  while (size < count) size *= 2;
  // Bitonic sort, two neighbours a thread in registers: partners within 128
  // entries are lanes of one wave; further ones meet in LDS.
  const int at0 = threadIdx.x * 2;
  uint64_t e[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) e[i] = at0 + i < count ? sh.list[at0 + i] : ~uint64_t(0);
  for (int k = 2; k <= size; k *= 2) {
    const bool up = (at0 & k) == 0;
    for (int j = k / 2; j > 1; j /= 2) {
      uint64_t o[2];
      if (j < 128) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
          o[i] = __shfl_xor(static_cast<unsigned long long>(e[i]), j / 2);
      } else {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; ++i) sh.list[at0 + i] = e[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; ++i) o[i] = sh.list[(at0 + i) ^ j];
      }
      const bool least = ((at0 & j) == 0) == up;
#pragma unroll
      for (int i = 0; i < 2; ++i) e[i] = (o[i] < e[i]) == least ? o[i] : e[i];
    }
    if ((e[1] < e[0]) == up) {
      const uint64_t x = e[0];
      e[0] = e[1];
      e[1] = x;
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) sh.list[at0 + i] = e[i];
  __syncthreads();
  Scan<2> s;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int at = threadIdx.x * 2 + i;
    s.c[i] = at < count;
    s.w[i] = at < count ? sc.weight(value_of(sh.list[at]), sh.table) : 0;
  }
  scan_block(s, sh);
  s.before_c += base_c;
  s.before_w += base_w;
  s.total_c += base_c;
  s.total_w += base_w;
  return s;
}

// Collects the elements that `take` accepts, as many as the list holds; how many
// there were.
template <typename T, typename F>
__device__ int gather(const T *row, int n, Shared &sh, F take) {
  __syncthreads();
  if (threadIdx.x == 0) sh.fill = 0;
  __syncthreads();
  each_run(row, n, [&](const float *x, int i, auto count) {
    // One branch for a run of neighbours, most of which take no part.
    uint32_t taken = 0;
#pragma unroll
    for (int j = 0; j < decltype(count)::value; ++j) taken |= (take(x[j], i + j) ? 1u : 0u) << j;
    if (taken == 0) return;
#pragma unroll
    for (int j = 0; j < decltype(count)::value; ++j)
      if (taken >> j & 1) {
        const uint32_t at = atomicAdd(&sh.fill, 1u);
        if (at < kList) sh.list[at] = entry_of(x[j], i + j);
      }
  });
  __syncthreads();
  return static_cast<int>(sh.fill);
}

template <typename T, typename F>
__device__ Scan<2> collect(const T *row, int n, const Scale &sc, Shared &sh, uint32_t base_c,
                           uint64_t base_w, F take) {
  const int count = min(gather(row, n, sh, take), kList);
  return sort_list(sc, sh, count, base_c, base_w);
}

// The element of the row at which the running count or weight reaches target.
struct Element {
  float x;
  int index;
  uint64_t through_w;  // weight up to and with it
};

// An element among those of `bin`, which hold it; more than kList of them. Its
// index only if kIndex: a border needs the weight up to it alone.
template <bool kCount, bool kIndex, typename T>
__device__ Element find_crowded(const T *row, int n, const Scale &sc, Shared &sh, const Place &bin,
                                uint64_t target) {
  // 16-bit logits crowd a bin with one value alone: then there is nothing to
  // narrow down, and the same pass has counted the value by runs of 2^seg indices.
  int seg = 0;
  while ((n - 1) >> seg >= kBins) ++seg;
  uint64_t low = ~uint64_t(0), high = 0;
  if (kIndex) clear_bins(sh);
  each(row, n, [&](float x, int i) {
    if (sc.bin(x) == bin.at) {
      const uint64_t k = key_of(x);
      low = min(low, k);
      high = max(high, k);
      if (kIndex) atomicAdd(&sh.cnt[i >> seg], 1u);
    }
  });
  high = max_of(high, sh);
  low = ~max_of(~low, sh);
  const bool one = low == high;
  uint32_t key = 0, mask = 0;
  Place at = bin;
  if (one) key = static_cast<uint32_t>(low);
  for (int shift = one ? -1 : 20; shift >= 0; shift = shift > 8 ? shift - 12 : shift - 8) {
    // 12, 12 and 8 bits of the key, in descending order.
    const int bits = shift == 0 ? 8 : 12;
    clear_bins(sh);
    each(row, n, [&](float x, int) {
      const uint32_t k = key_of(x);
      if (sc.bin(x) == bin.at && (k & mask) == key) {
        const int digit = (1 << bits) - 1 - ((k >> shift) & ((1 << bits) - 1));
        atomicAdd(&sh.cnt[digit], 1u);
        atomicAdd(reinterpret_cast<unsigned long long *>(&sh.wsum[digit]),
                  static_cast<unsigned long long>(sc.weight(x, sh.table)));
      }
    });
    __syncthreads();
    Scan<4> s = scan_bins(sh, true);
    s.before_c += at.before_c;
    s.before_w += at.before_w;
    at = find<kCount>(s, target, sh);
    key |= static_cast<uint32_t>((1 << bits) - 1 - at.at) << shift;
    mask |= static_cast<uint32_t>((1 << bits) - 1) << shift;
  }
  // All c elements left are equal, of weight w / c each; by index.
  const float x = of_key(key);
  const uint64_t each_w = at.w / at.c;
  const uint64_t m = kCount ? target - at.before_c
                            : (target - at.before_w + each_w - 1) / each_w;
  Element e{x, -1, at.before_w + m * each_w};
  if (!kIndex) return e;
  if (!one) {
    clear_bins(sh);
    each(row, n, [&](float y, int i) {
      if (y == x) atomicAdd(&sh.cnt[i >> seg], 1u);
    });
    __syncthreads();
  }
  const Scan<4> s = scan_bins(sh, false);
  const Place part = find<true>(s, m, sh);
  const int from = part.at << seg;
  const Scan<2> l = collect(row + from, min(1 << seg, n - from), sc, sh, part.before_c, 0,
                            [&](float y, int) { return y == x; });
  const Place found = find<true>(l, m, sh);
  e.index = from + static_cast<int>(static_cast<uint32_t>(sh.list[found.at]));
  return e;
}

template <bool kCount>
__device__ Element find_listed(const Scan<2> &l, uint64_t target, Shared &sh) {
  const Place e = find<kCount>(l, target, sh);
  const uint64_t v = sh.list[e.at];
  return {value_of(v), static_cast<int>(static_cast<uint32_t>(v)), e.before_w + e.w};
}

// Temperatures are held between these: below the least, every FP32 logit but those
// equal to the largest weighs 0, and above the most all weigh the same, while the
// 64-bit arithmetic stays clear of infinities.
constexpr double kLeastTemp = 1e-290, kMostTemp = 1e290;

// A row's source and parameters.
template <typename T>
struct Row {
  const T *x;
  double temp, top_p, min_p, u;
  int64_t top_k;
};

template <typename T>
__device__ __forceinline__ bool row_of(const SampleParams &p, int64_t out, Row<T> &r) {
  const int64_t src = p.row_ids ? p.row_ids[out] : out;
  if (src < 0 || src >= p.num_logit_rows) return false;
  r.x = static_cast<const T *>(p.logits) + src * p.row_st;
  r.temp = p.temperature ? static_cast<double>(p.temperature[out]) : p.temperature_v;
  if (r.temp > 0) r.temp = fmin(fmax(r.temp, kLeastTemp), kMostTemp);
  r.top_p = p.top_p ? static_cast<double>(p.top_p[out]) : p.top_p_v;
  r.min_p = p.min_p ? static_cast<double>(p.min_p[out]) : p.min_p_v;
  r.top_k = !p.top_k       ? p.top_k_v
            : p.top_k_i64 ? static_cast<const int64_t *>(p.top_k)[out]
                          : static_cast<const int32_t *>(p.top_k)[out];
  r.u = p.uniforms_f64 ? static_cast<const double *>(p.uniforms)[out]
                       : static_cast<const float *>(p.uniforms)[out];
  return true;
}

__device__ __forceinline__ void put(const SampleParams &p, int64_t out, int token, float logprob) {
  if (threadIdx.x == 0) {
    p.tokens[out] = token;
    if (p.logprobs) p.logprobs[out] = logprob;
  }
}

__device__ __forceinline__ float wave_top(float x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor(x, o));
  return x;
}
// The largest value (NaNs aside; -inf where there is none) and the index of the
// first that equals it, which only some rows need.
template <typename T>
__device__ float top_of(const T *row, int n, Shared &sh) {
  float t = -INFINITY;
  each(row, n, [&](float x, int) { t = fmaxf(t, x); });
  t = wave_top(t);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh.red_x[threadIdx.x >> 6] = t;
  __syncthreads();
  for (int i = 0; i < kWavesWg; ++i) t = fmaxf(t, sh.red_x[i]);
  return t;
}
template <typename T>
__device__ int index_of(const T *row, int n, float top, Shared &sh) {
  uint64_t first = 0x7fffffff;
  each(row, n, [&](float x, int i) {
    if (x == top) first = min(first, static_cast<uint64_t>(i));
  });
  return static_cast<int>(~max_of(~first, sh));
}

// Rows whose token is the first of the order whatever the random number: no
// temperature, the first kept only, or an infinite logit.
template <typename T>
__device__ __forceinline__ bool only_first(const Row<T> &r, float top) {
  return top == -INFINITY || !(r.temp > 0) || r.top_k == 1 || r.top_p <= 0 || r.min_p > 1 ||
         top == INFINITY;
}
template <typename T>
__device__ __forceinline__ void put_first(const SampleParams &p, int64_t out, const Row<T> &r,
                                          float top, Shared &sh) {
  if (top == -INFINITY) put(p, out, -1, -INFINITY);
  else put(p, out, index_of(r.x, p.vocab, top, sh), 0.f);
}

__device__ __forceinline__ Scale scale_of(float top, double temp, int shift) {
  Scale sc;
  sc.mx = top;
  sc.mxd = top;
  sc.shift = shift;
  sc.c = kTable / (temp * 0.69314718055994530942);
  sc.far = 60.0 * kTable / sc.c;
  // The last bin starts past 46 halvings, where every weight rounds to 0.
  sc.bins = static_cast<float>(fmin((kBins - 1) / (46.0 * 0.69314718055994530942 * temp), 1e30));
  return sc;
}

__device__ __forceinline__ void make_table(Shared &sh) {
  for (int i = threadIdx.x; i < kTable; i += kThreads)
    sh.table[i] = exp2(-static_cast<double>(i) / kTable);
}

// Counts, and weights if asked for, of a row's (or a part's) bins into LDS.
template <typename T>
__device__ void fill_bins(const T *row, int n, const Scale &sc, Shared &sh, bool weights) {
  clear_bins(sh);
  const int spare = kBins + (threadIdx.x & 63);
  auto fill = [&](auto weigh) {
    each(row, n, [&](float x, int) {
      // Without branches: what lies in the last bin (a NaN too) goes to the
      // lane's spare slot.
      const int b = sc.bin(x), slot = b < kBins - 1 ? b : spare;
      atomicAdd(&sh.cnt[slot], 1u);
      if constexpr (decltype(weigh)::value)
        atomicAdd(reinterpret_cast<unsigned long long *>(&sh.wsum[slot]),
                  static_cast<unsigned long long>(sc.weight(x, sh.table)));
    });
  };
  if (weights) fill(std::true_type{});
  else fill(std::false_type{});
  __syncthreads();
}

__device__ __forceinline__ uint64_t whole(double x) {  // 0 for a NaN
  return x >= 1 ? (x < 9.0e18 ? static_cast<uint64_t>(x) : static_cast<uint64_t>(9.0e18)) : 0;
}
__device__ __forceinline__ uint64_t top_p_target(double top_p, uint64_t kept) {
  return min(max(whole(ceil(top_p * static_cast<double>(kept))), uint64_t(1)), kept);
}
// In integers "exceeds u S" is "reaches floor(u S) + 1" (not added in 64-bit
// floating point, which has no such neighbour past 2^53).
__device__ __forceinline__ uint64_t draw_target(double u, uint64_t kept) {
  return min(whole(u * static_cast<double>(kept)) + 1, kept);
}

// Up to which distance from the maximum min-p keeps, and the bin of that.
struct Far {
  double far;
  int bin;
};
__device__ __forceinline__ Far far_of(double min_p, double temp, const Scale &sc) {
  const double far = temp < kMostTemp ? -temp * log(min_p) : INFINITY;
  return {far, static_cast<int>(fmin(far * static_cast<double>(sc.bins), kBins - 1.0))};
}

// Elements of the row before bin b and their weight.
struct Before {
  uint32_t c;
  uint64_t w;
};
__device__ Before before_bin(const Scan<4> &h, int b, Shared &sh) {
  __syncthreads();
  if (b / 4 == static_cast<int>(threadIdx.x)) {
    Before x{h.before_c, h.before_w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < (b & 3)) {
        x.c += h.c[i];
        x.w += h.w[i];
      }
    sh.found_c = x.c;
    sh.found_w = x.w;
  }
  __syncthreads();
  return {sh.found_c, sh.found_w};
}

__device__ __forceinline__ void put_drawn(const SampleParams &p, int64_t out, double temp,
                                          const Scale &sc, const Element &e, uint64_t kept) {
  put(p, out, e.index,
      static_cast<float>(-(sc.mxd - e.x) / temp - log(ldexp(static_cast<double>(kept), -p.shift))));
}

// A row step by step, each border by a pass of its own: for top-k past the list
// and rows whose borders lie in crowded bins. h: the row's bins, if `weighed`.
template <typename T>
__device__ void sample_stepwise(const SampleParams &p, int64_t out, const Row<T> &r,
                                const Scale &sc, Shared &sh, Scan<4> h, bool weighed) {
  const int n = p.vocab;
  if (!weighed) {
    fill_bins(r.x, n, sc, sh, true);
    h = scan_bins(sh, true);
  }
  auto only = [&](const Place &b) {
    return collect(r.x, n, sc, sh, b.before_c, b.before_w,
                   [&](float x, int) { return sc.bin(x) == b.at; });
  };
  // A weight's place in the order; its index for the draw alone.
  auto reach = [&](uint64_t target, auto index) {
    const Place b = find<false>(h, target, sh);
    if (b.c > kList)
      return find_crowded<false, decltype(index)::value>(r.x, n, sc, sh, b, target);
    return find_listed<false>(only(b), target, sh);
  };
  uint64_t kept = h.total_w;
  if (r.top_k > 0 && r.top_k < h.total_c) {
    const Place b = find<true>(h, r.top_k, sh);
    kept = b.c > kList ? find_crowded<true, false>(r.x, n, sc, sh, b, r.top_k).through_w
                       : find_listed<true>(only(b), r.top_k, sh).through_w;
  }
  if (r.top_p < 1) kept = reach(top_p_target(r.top_p, kept), std::false_type{}).through_w;
  if (r.min_p > 0) {
    // What the bins next to the border hold of such elements is added one by one.
    const Far f = far_of(r.min_p, r.temp, sc);
    uint64_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (static_cast<int>(threadIdx.x) * 4 + i < f.bin - 1) w += h.w[i];
    each(r.x, n, [&](float x, int) {
      const int bx = sc.bin(x);
      if (bx >= f.bin - 1 && bx <= f.bin + 1 && bx < kBins - 1 && sc.mxd - x <= f.far)
        w += sc.weight(x, sh.table);
    });
    kept = min(kept, total_of(w, sh));
  }
  const Element e = reach(draw_target(r.u, kept), std::true_type{});
  put_drawn(p, out, r.temp, sc, e, kept);
}

// Which elements decide a row, from its bins alone: a head of the order (top-k),
// or up to three runs of bins: those of the borders of top-p and min-p, and those
// in which the draw can fall given what the borders' bins leave open.
struct Plan {
  bool listed;  // whether there is such a plan at all
  bool head;
  int lo[3], hi[3];       // ascending, apart from each other; kBins: none
  uint64_t before_w[3];   // weight of the row before each run

  __device__ __forceinline__ bool takes(int b) const {
    auto in = [&](int i) {
      return static_cast<uint32_t>(b - lo[i]) <= static_cast<uint32_t>(hi[i] - lo[i]);
    };
    return in(0) | in(1) | in(2);
  }
};

template <typename T>
__device__ Plan plan_of(const Row<T> &r, int n, const Scale &sc, const Scan<4> &h, Shared &sh) {
  Plan pl;
  pl.listed = true;
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    pl.lo[i] = pl.hi[i] = kBins;
    pl.before_w[i] = 0;
  }
  pl.head = r.top_k > 0 && r.top_k < n;
  if (pl.head) {
    pl.lo[0] = 0;
    pl.hi[0] = kBins - 2;
    uint32_t through = h.total_c;
    if (r.top_k < h.total_c) {
      const Place b = find<true>(h, r.top_k, sh);
      pl.hi[0] = b.at;
      through = b.before_c + b.c;
    }
    pl.listed = through <= kList;
    return pl;
  }
  uint64_t least = h.total_w, most = h.total_w;
  if (r.top_p < 1) {
    const uint64_t target = top_p_target(r.top_p, h.total_w);
    const Place b = find<false>(h, target, sh);
    least = target;
    most = b.before_w + b.w;
    pl.lo[0] = pl.hi[0] = b.at;
  }
  if (r.min_p > 0) {
    const int b = far_of(r.min_p, r.temp, sc).bin;
    const int lo = min(max(b - 1, 0), kBins - 2), hi = min(b + 1, kBins - 2);
    least = min(least, max(before_bin(h, lo, sh).w, uint64_t(1)));
    most = min(most, max(before_bin(h, hi + 1, sh).w, uint64_t(1)));
    pl.lo[1] = lo;
    pl.hi[1] = hi;
  }
  pl.lo[2] = find<false>(h, draw_target(r.u, least), sh).at;
  pl.hi[2] = find<false>(h, draw_target(r.u, most), sh).at;
  // Ascending, then joined where they meet.
  auto order = [&](int i, int j) {
    if (pl.lo[j] < pl.lo[i]) {
      const int lo = pl.lo[i], hi = pl.hi[i];
      pl.lo[i] = pl.lo[j];
      pl.hi[i] = pl.hi[j];
      pl.lo[j] = lo;
      pl.hi[j] = hi;
    }
  };
  auto join = [&](int i, int j) {
    if (pl.lo[j] < kBins && pl.lo[j] <= pl.hi[i] + 1) {
      pl.hi[i] = max(pl.hi[i], pl.hi[j]);
      pl.lo[j] = pl.hi[j] = kBins;
    }
  };
  order(0, 1);
  order(1, 2);
  order(0, 1);
  join(0, 1);
  join(pl.lo[1] < kBins ? 1 : 0, 2);
  uint32_t count = 0;
#pragma unroll
  for (int i = 0; i < 3; ++i)
    if (pl.lo[i] < kBins) {
      const Before x = before_bin(h, pl.lo[i], sh);
      pl.before_w[i] = x.w;
      count += before_bin(h, pl.hi[i] + 1, sh).c - x.c;
    }
  pl.listed = count <= kList;
  return pl;
}

// Ends a row whose plan's elements, `count` of them, are in the list.
template <typename T>
__device__ void sample_listed(const SampleParams &p, int64_t out, const Row<T> &r, const Scale &sc,
                              const Plan &pl, int count, uint64_t total_w, Shared &sh) {
  Scan<2> l = sort_list(sc, sh, count, 0, 0);
  uint64_t kept = total_w;
  uint64_t before[2] = {l.before_w, l.before_w + l.w[0]};
  if (pl.head) {
    kept = l.total_w;
    if (r.top_k > 0 && r.top_k < l.total_c) kept = find_listed<true>(l, r.top_k, sh).through_w;
  } else {
    // An entry's place in the row: its place in its run, after what precedes the
    // run. Runs are in the list whole.
    uint64_t in_list[3] = {0, 0, 0};  // weight of the list before each run
#pragma unroll
    for (int i = 1; i < 3; ++i) {
      if (pl.lo[i] >= kBins) continue;  // uniform
      uint64_t w = 0;
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (l.c[e] && sc.bin(value_of(sh.list[threadIdx.x * 2 + e])) < pl.lo[i]) w += l.w[e];
      in_list[i] = total_of(w, sh);
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      if (!l.c[e]) continue;
      const int b = sc.bin(value_of(sh.list[threadIdx.x * 2 + e]));
      const int i = b >= pl.lo[2] ? 2 : b >= pl.lo[1] ? 1 : 0;
      before[e] = before[e] - in_list[i] + pl.before_w[i];
    }
  }
  // The entry at which the running weight reaches target.
  auto reach = [&](uint64_t target) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (before[e] < target && target <= before[e] + l.w[e]) {
        sh.found_at = threadIdx.x * 2 + e;
        sh.found_w = before[e] + l.w[e];
      }
    __syncthreads();
    const uint64_t v = sh.list[sh.found_at];
    return Element{value_of(v), static_cast<int>(static_cast<uint32_t>(v)), sh.found_w};
  };
  if (r.top_p < 1) kept = reach(top_p_target(r.top_p, kept)).through_w;
  if (r.min_p > 0) {
    // Weight up to the last entry within the distance. Where the list is a head it
    // holds all that is kept; else the bins about the distance are a part of it.
    const Far f = far_of(r.min_p, r.temp, sc);
    uint64_t w = 0;
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (l.c[e] && sc.mxd - value_of(sh.list[threadIdx.x * 2 + e]) <= f.far)
        w = max(w, before[e] + l.w[e]);
    w = max_of(w, sh);
    // At least all that lies before the run of those bins.
    if (!pl.head) {
      const int lo = min(max(f.bin - 1, 0), kBins - 2);
      w = max(w, pl.before_w[lo >= pl.lo[2] ? 2 : lo >= pl.lo[1] ? 1 : 0]);
    }
    kept = min(kept, w);
  }
  put_drawn(p, out, r.temp, sc, reach(draw_target(r.u, kept)), kept);
}

// Whether a row is ended in steps by one workgroup from the start.
template <typename T>
__device__ __forceinline__ bool stepwise(const Row<T> &r, int n) {
  return r.top_k > kList && r.top_k < n;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_kernel(SampleParams p) {
  __shared__ Shared sh;
  const int64_t out = blockIdx.x;
  const int n = p.vocab;
  Row<T> r;
  if (!row_of(p, out, r)) {
    put(p, out, -1, -INFINITY);
    return;
  }
  make_table(sh);
  const float top = top_of(r.x, n, sh);
  if (only_first(r, top)) {
    put_first(p, out, r, top, sh);
    return;
  }
  const Scale sc = scale_of(top, r.temp, p.shift);
  if (n <= kList) {  // all of it
    Plan pl{};
    pl.head = true;
    const int count = gather(r.x, n, sh, [&](float x, int) { return sc.bin(x) < kBins - 1; });
    sample_listed(p, out, r, sc, pl, count, 0, sh);
    return;
  }
  const bool weights = !(r.top_k > 0 && r.top_k < n);
  Scan<4> h{};
  if (!stepwise(r, n)) {
    fill_bins(r.x, n, sc, sh, weights);
    h = scan_bins(sh, weights);
    const Plan pl = plan_of(r, n, sc, h, sh);
    if (pl.listed) {
      const int count = gather(r.x, n, sh, [&](float x, int) { return pl.takes(sc.bin(x)); });
      sample_listed(p, out, r, sc, pl, count, h.total_w, sh);
      return;
    }
  }
  sample_stepwise(p, out, r, sc, sh, h, weights);
}

// A row cut over workgroups. What they share of it; every entry is written before
// it is read, the bins and the counter by split_top.
struct RowSpace {
  uint64_t wsum[kBins];
  uint64_t list[kList];
  uint32_t cnt[kBins];
  float top[kMaxParts];
  uint32_t fill;
  uint32_t first;  // least index of the largest value, for rows that need it
};

// The part of a row that workgroup `part` reads: [from, from + count).
struct Part {
  int64_t out;
  int part, from, count;
};
__device__ __forceinline__ Part part_of(const SampleParams &p) {
  Part t;
  t.out = blockIdx.x / p.parts;
  t.part = static_cast<int>(blockIdx.x - t.out * p.parts);
  const int size = ((p.vocab + p.parts - 1) / p.parts + 7) & ~7;
  t.from = min(t.part * size, p.vocab);
  t.count = min(size, p.vocab - t.from);
  return t;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void split_top(SampleParams p) {
  __shared__ Shared sh;
  const Part t = part_of(p);
  RowSpace &sp = p.space[t.out];
  for (int i = t.part * kThreads + threadIdx.x; i < kBins; i += p.parts * kThreads) {
    sp.wsum[i] = 0;
    sp.cnt[i] = 0;
  }
  if (t.part == 0 && threadIdx.x == 0) {
    sp.fill = 0;
    sp.first = 0x7fffffff;
  }
  Row<T> r;
  if (!row_of(p, t.out, r)) return;
  const float top = top_of(r.x + t.from, t.count, sh);
  if (threadIdx.x == 0) sp.top[t.part] = top;
}

// A lane per part.
__device__ __forceinline__ float top_of_parts(const SampleParams &p, const RowSpace &sp) {
  static_assert(kMaxParts <= 64, "a lane per part");
  const int lane = threadIdx.x & 63;
  return wave_top(lane < p.parts ? sp.top[lane] : -INFINITY);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void split_bins(SampleParams p) {
  __shared__ Shared sh;
  const Part t = part_of(p);
  RowSpace &sp = p.space[t.out];
  Row<T> r;
  if (!row_of(p, t.out, r)) return;
  const float top = top_of_parts(p, sp);
  if (only_first(r, top)) {
    if (top == -INFINITY || sp.top[t.part] != top) return;  // uniform
    const int at = index_of(r.x + t.from, t.count, top, sh);
    if (threadIdx.x == 0) atomicMin(&sp.first, static_cast<uint32_t>(t.from + at));
    return;
  }
  if (stepwise(r, p.vocab)) return;
  make_table(sh);
  const Scale sc = scale_of(top, r.temp, p.shift);
  const bool weights = !(r.top_k > 0 && r.top_k < p.vocab);
  fill_bins(r.x + t.from, t.count, sc, sh, weights);
  for (int i = threadIdx.x; i < kBins; i += kThreads)
    if (sh.cnt[i] != 0) {
      atomicAdd(&sp.cnt[i], sh.cnt[i]);
      if (weights)
        atomicAdd(reinterpret_cast<unsigned long long *>(&sp.wsum[i]),
                  static_cast<unsigned long long>(sh.wsum[i]));
    }
}

__device__ __forceinline__ Scan<4> bins_of(const RowSpace &sp, Shared &sh) {
  Scan<4> s;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    s.c[i] = sp.cnt[threadIdx.x * 4 + i];
    s.w[i] = sp.wsum[threadIdx.x * 4 + i];
  }
  scan_block(s, sh);
  return s;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void split_gather(SampleParams p) {
  __shared__ Shared sh;
  const Part t = part_of(p);
  RowSpace &sp = p.space[t.out];
  Row<T> r;
  if (!row_of(p, t.out, r)) return;
  const float top = top_of_parts(p, sp);
  if (only_first(r, top) || stepwise(r, p.vocab)) return;
  const Scale sc = scale_of(top, r.temp, p.shift);
  const Scan<4> h = bins_of(sp, sh);
  const Plan pl = plan_of(r, p.vocab, sc, h, sh);
  if (!pl.listed) return;
  const int count = gather(r.x + t.from, t.count, sh,
                           [&](float x, int) { return pl.takes(sc.bin(x)); });
  if (threadIdx.x == 0) sh.found_n = atomicAdd(&sp.fill, static_cast<uint32_t>(count));
  __syncthreads();
  const int base = static_cast<int>(sh.found_n);
  for (int i = threadIdx.x; i < min(count, kList); i += kThreads)
    if (base + i < kList) sp.list[base + i] = sh.list[i] + static_cast<uint64_t>(t.from);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void split_end(SampleParams p) {
  __shared__ Shared sh;
  const int64_t out = blockIdx.x;
  const RowSpace &sp = p.space[out];
  Row<T> r;
  if (!row_of(p, out, r)) {
    put(p, out, -1, -INFINITY);
    return;
  }
  const float top = top_of_parts(p, sp);
  if (only_first(r, top)) {
    const bool none = top == -INFINITY;
    put(p, out, none ? -1 : static_cast<int>(sp.first), none ? -INFINITY : 0.f);
    return;
  }
  make_table(sh);
  const Scale sc = scale_of(top, r.temp, p.shift);
  Scan<4> h{};
  if (!stepwise(r, p.vocab)) {
    h = bins_of(sp, sh);
    const Plan pl = plan_of(r, p.vocab, sc, h, sh);
    if (pl.listed) {
      const int count = static_cast<int>(sp.fill);
      for (int i = threadIdx.x; i < count; i += kThreads) sh.list[i] = sp.list[i];
      __syncthreads();
      sample_listed(p, out, r, sc, pl, count, h.total_w, sh);
      return;
    }
  }
  __syncthreads();  // the table
  sample_stepwise(p, out, r, sc, sh, h, !(r.top_k > 0 && r.top_k < p.vocab));
}

template <typename T>
int launch_sample(const SampleParams &p, unsigned rows, hipStream_t stream) {
  if (p.parts == 1) {
    sample_kernel<T><<<rows, kThreads, 0, stream>>>(p);
    return check_launch("mlr_sample_tokens");
  }
  const unsigned grid = rows * p.parts;
  split_top<T><<<grid, kThreads, 0, stream>>>(p);
  split_bins<T><<<grid, kThreads, 0, stream>>>(p);
  split_gather<T><<<grid, kThreads, 0, stream>>>(p);
  split_end<T><<<rows, kThreads, 0, stream>>>(p);
  return check_launch("mlr_sample_tokens");
}

// Workgroups a row is cut over: so many that the batch has one for every CU, each
// with at least kPartMin elements. The further launches take longer than they save
// where the row is short or the batch leaves few parts; one workgroup against the
// cut, top_k = 50 and top_p = 0.9, FP32, us:
//              32,000 logits       151,936 logits
//    1 row     31.3 / 36.8         53.2 / 38.6
//   48 rows    33.3 / 45.7         59.5 / 52.1
//   64 rows    34.0 / 47.6         60.2 / 58.9
//   85 rows    34.8 / 48.2         61.2 / 65.2
int parts_of(int64_t rows, int64_t vocab) {
  const int cus = current_device_cus() > 0 ? current_device_cus() : 256;
  const int64_t n = std::min({cus / std::max<int64_t>(rows, 1), vocab / kPartMin,
                              static_cast<int64_t>(kMaxParts)});
  return n >= 3 && vocab >= 1300 * (32 + rows) ? static_cast<int>(n) : 1;
}

}  // namespace
}  // namespace mlr

extern "C" size_t mlr_sample_tokens_workspace_size(int64_t num_rows, int64_t vocab) {
  if (num_rows <= 0 || vocab <= 0 || mlr::parts_of(num_rows, vocab) == 1) return 0;
  return static_cast<size_t>(num_rows) * sizeof(mlr::RowSpace);
}

extern "C" int mlr_sample_tokens(const void *logits, int64_t row_stride, int64_t num_logit_rows,
                                 int dtype, const int64_t *row_ids, const void *uniforms,
                                 int uniforms_f64, const float *temperature,
                                 double temperature_value, const void *top_k, int top_k_dtype,
                                 int64_t top_k_value, const float *top_p, double top_p_value,
                                 const float *min_p, double min_p_value, int64_t *tokens,
                                 float *logprobs, int64_t num_rows, int64_t vocab,
                                 void *workspace, size_t workspace_bytes, void *stream) {
  using namespace mlr;
  clear_error();
  MLR_REQUIRE(num_rows >= 0 && num_rows < (int64_t(1) << 31),
              "mlr_sample_tokens: num_rows must be in [0, 2^31)");
  MLR_REQUIRE(vocab > 0 && vocab <= kMaxVocab, "mlr_sample_tokens: vocab must be in [1, 2^23]");
  MLR_REQUIRE(num_logit_rows >= 0, "mlr_sample_tokens: num_logit_rows must be >= 0");
  MLR_REQUIRE(row_ids || num_logit_rows >= num_rows,
              "mlr_sample_tokens: fewer logit rows than rows to sample");
  MLR_REQUIRE(num_logit_rows <= 1 || row_stride >= vocab,
              "mlr_sample_tokens: row stride smaller than a row");
  MLR_REQUIRE(!top_k || top_k_dtype == MLR_INDEX_I32 || top_k_dtype == MLR_INDEX_I64,
              "mlr_sample_tokens: unknown index dtype %d", top_k_dtype);
  MLR_REQUIRE(dtype == MLR_DTYPE_F32 || dtype == MLR_DTYPE_F16 || dtype == MLR_DTYPE_BF16,
              "mlr_sample_tokens: unsupported dtype %d", dtype);
  if (num_rows == 0) return MLR_OK;
  MLR_REQUIRE((logits || num_logit_rows == 0) && uniforms && tokens,
              "mlr_sample_tokens: null pointer");
  const size_t need = mlr_sample_tokens_workspace_size(num_rows, vocab);
  MLR_REQUIRE(need == 0 || (workspace && workspace_bytes >= need &&
                            reinterpret_cast<uintptr_t>(workspace) % 8 == 0),
              "mlr_sample_tokens: workspace of %zu bytes, %zu needed, 8-byte aligned",
              workspace_bytes, need);
  SampleParams p;
  p.parts = parts_of(num_rows, vocab);
  p.space = static_cast<RowSpace *>(workspace);
  p.logits = logits;
  p.row_st = row_stride;
  p.num_logit_rows = num_logit_rows;
  p.row_ids = row_ids;
  p.uniforms = uniforms;
  p.temperature = temperature;
  p.top_p = top_p;
  p.min_p = min_p;
  p.top_k = top_k;
  p.temperature_v = temperature_value;
  p.top_p_v = top_p_value;
  p.min_p_v = min_p_value;
  p.top_k_v = top_k_value;
  p.tokens = tokens;
  p.logprobs = logprobs;
  p.vocab = static_cast<int>(vocab);
  int bits = 0;
  while ((int64_t(1) << bits) < vocab) ++bits;
  p.shift = 62 - bits < 44 ? 62 - bits : 44;  // sums stay below 2^63
  p.uniforms_f64 = uniforms_f64 != 0;
  p.top_k_i64 = top_k_dtype == MLR_INDEX_I64;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const unsigned grid = static_cast<unsigned>(num_rows);
  switch (dtype) {
    case MLR_DTYPE_F32: return launch_sample<float>(p, grid, s);
    case MLR_DTYPE_F16: return launch_sample<f16_t>(p, grid, s);
    default: return launch_sample<bf16_t>(p, grid, s);
  }
}

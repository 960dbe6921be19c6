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
// largest, from 64-bit arithmetic (a table of 2^(-j/1024) and the first three
// terms of the series for the rest: within 7e-12 relative). So sums are exact, no matter in
// which order atomics and scans add, the same logits and random numbers give
// the same token always, and a token differs from the formula's in exact
// arithmetic only where u S is within about 1e-11 S of a border.
//
// One workgroup of 1,024 threads per row: a row is read three times (maximum,
// bins, collecting the bin), the later times from the caches.
#include "mlr_common.h"

#include <cfloat>

namespace mlr {
namespace {

constexpr int kThreads = 1024;
constexpr int kWavesWg = kThreads / 64;
constexpr int kBins = 4096;  // 4 per thread; the last holds what weighs nothing
constexpr int kList = 2048;  // 2 per thread
constexpr int kTable = 1024;
constexpr int64_t kMaxVocab = int64_t(1) << 23;  // a segment of 1 / kBins of it fits the list

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
};

template <typename T>
struct alignas(16) Row16 {
  T v[16 / sizeof(T)];
};

struct Shared {
  double table[kTable];
  uint64_t wsum[kBins];
  uint64_t list[kList];  // sorted: ~key in the upper half, index in the lower
  uint32_t cnt[kBins];
  uint64_t scan_w[kWavesWg];
  uint32_t scan_c[kWavesWg];
  uint64_t found_w;
  uint32_t found_c, found_at, found_n;
  uint32_t fill;
  float red_x[kWavesWg];
  int red_i[kWavesWg];
};

// FP32 values in unsigned order; both zeros alike.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b ^ (b & 0x80000000u ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float of_key(uint32_t k) {
  return __uint_as_float(k ^ (k & 0x80000000u ? 0x80000000u : 0xffffffffu));
}

// f(x, index) over a row, 16 bytes a load, four loads of a thread in flight.
template <typename T, typename F>
__device__ __forceinline__ void each(const T *row, int n, F f) {
  constexpr int kVec = 16 / sizeof(T), kDeep = 4;
  const int tid = threadIdx.x;
  const int head = min(n, static_cast<int>(((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) /
                                           sizeof(T)));
  if (tid < head) f(Elem<T>::to_f32(row[tid]), tid);
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
        for (int j = 0; j < kVec; ++j) f(Elem<T>::to_f32(r[k].v[j]), head + v * kVec + j);
      }
    }
  }
  const int rest = head + nv * kVec + tid;
  if (rest < n) f(Elem<T>::to_f32(row[rest]), rest);
}

// What turns a logit into its weight and its bin.
struct Scale {
  float mx, bins;  // the row's maximum; bins per unit of distance
  double mxd, c;   // c: 1024ths of a halving per unit of distance
  int shift;

  __device__ __forceinline__ int bin(float x) const {
    return static_cast<int>(fminf((mx - x) * bins, static_cast<float>(kBins - 1)));
  }
  __device__ __forceinline__ uint64_t weight(float x, const double *table) const {
    constexpr double kMagic = 6755399441055744.0;  // 1.5 * 2^52: rounds to integer
    constexpr double kStep = 0.69314718055994530942 / kTable;
    // Past 60 halvings every weight rounds to 0; fmin also takes a NaN there.
    const double t = fmin((mxd - static_cast<double>(x)) * c, 60.0 * kTable);
    const double whole = t + kMagic;
    const int k = __double2loint(whole);
    const double r = t - (whole - kMagic);
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

// Collects the elements that `take` accepts (at most kList) and sorts them;
// the result holds the list's entries two to a thread, with `base` before them.
template <typename T, typename F>
__device__ Scan<2> collect(const T *row, int n, const Scale &sc, Shared &sh, uint32_t base_c,
                           uint64_t base_w, F take) {
  __syncthreads();
  if (threadIdx.x == 0) sh.fill = 0;
  __syncthreads();
  each(row, n, [&](float x, int i) {
    if (take(x, i)) {
      const uint32_t at = atomicAdd(&sh.fill, 1u);
      if (at < kList) sh.list[at] = (static_cast<uint64_t>(~key_of(x)) << 32) | static_cast<uint32_t>(i);
    }
  });
  __syncthreads();
  const int count = min(static_cast<int>(sh.fill), kList);
  int size = 128;
  while (size < count) size *= 2;
  for (int i = threadIdx.x + count; i < size; i += kThreads) sh.list[i] = ~uint64_t(0);
  __syncthreads();
  // Bitonic sort: every thread compares one pair a step.
  for (int k = 2; k <= size; k *= 2)
    for (int j = k / 2; j > 0; j /= 2) {
      for (int t = threadIdx.x; t < size / 2; t += kThreads) {
        const int a = 2 * t - (t & (j - 1)), b = a + j;
        const uint64_t x = sh.list[a], y = sh.list[b];
        if ((x > y) == ((a & k) == 0)) {
          sh.list[a] = y;
          sh.list[b] = x;
        }
      }
      __syncthreads();
    }
  Scan<2> s;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int at = threadIdx.x * 2 + i;
    s.c[i] = at < count;
    s.w[i] = at < count ? sc.weight(of_key(~static_cast<uint32_t>(sh.list[at] >> 32)), sh.table) : 0;
  }
  scan_block(s, sh);
  s.before_c += base_c;
  s.before_w += base_w;
  s.total_c += base_c;
  s.total_w += base_w;
  return s;
}

// The element of the row at which the running count or weight reaches target.
struct Element {
  float x;
  int index;
  uint64_t through_w;  // weight up to and with it
};

// An element among those of `bin`, which hold it; more than kList of them.
template <bool kCount, typename T>
__device__ Element find_crowded(const T *row, int n, const Scale &sc, Shared &sh, const Place &bin,
                                uint64_t target) {
  uint32_t key = 0, mask = 0;
  Place at = bin;
  for (int shift = 20; shift >= 0; shift = shift > 8 ? shift - 12 : shift - 8) {
    // 12, 12 and 8 bits of the key, in descending order.
    const int bits = shift == 0 ? 8 : 12;
    clear_bins(sh);
    each(row, n, [&](float x, int) {
      const uint32_t k = key_of(x);
      if (x == x && sc.bin(x) == bin.at && (k & mask) == key) {
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
  int seg = 0;  // segments of 2^seg indices
  while ((n - 1) >> seg >= kBins) ++seg;
  clear_bins(sh);
  each(row, n, [&](float y, int i) {
    if (y == x) atomicAdd(&sh.cnt[i >> seg], 1u);
  });
  __syncthreads();
  const Scan<4> s = scan_bins(sh, false);
  const Place part = find<true>(s, m, sh);
  const Scan<2> l = collect(row, n, sc, sh, part.before_c, 0,
                            [&](float y, int i) { return y == x && i >> seg == part.at; });
  const Place e = find<true>(l, m, sh);
  return {x, static_cast<int>(static_cast<uint32_t>(sh.list[e.at])), at.before_w + m * each_w};
}

template <bool kCount>
__device__ Element find_listed(const Scan<2> &l, uint64_t target, Shared &sh) {
  const Place e = find<kCount>(l, target, sh);
  const uint64_t v = sh.list[e.at];
  return {of_key(~static_cast<uint32_t>(v >> 32)), static_cast<int>(static_cast<uint32_t>(v)),
          e.before_w + e.w};
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_kernel(SampleParams p) {
  __shared__ Shared sh;
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const int64_t out = blockIdx.x;
  const int n = p.vocab;
  const int64_t src = p.row_ids ? p.row_ids[out] : out;
  if (src < 0 || src >= p.num_logit_rows) {
    if (tid == 0) {
      p.tokens[out] = -1;
      if (p.logprobs) p.logprobs[out] = -INFINITY;
    }
    return;
  }
  const T *row = static_cast<const T *>(p.logits) + src * p.row_st;
  const double temp = p.temperature ? static_cast<double>(p.temperature[out]) : p.temperature_v;
  const double top_p = p.top_p ? static_cast<double>(p.top_p[out]) : p.top_p_v;
  const double min_p = p.min_p ? static_cast<double>(p.min_p[out]) : p.min_p_v;
  const int64_t top_k = !p.top_k       ? p.top_k_v
                        : p.top_k_i64 ? static_cast<const int64_t *>(p.top_k)[out]
                                      : static_cast<const int32_t *>(p.top_k)[out];
  const double u = p.uniforms_f64 ? static_cast<const double *>(p.uniforms)[out]
                                  : static_cast<const float *>(p.uniforms)[out];
  for (int i = tid; i < kTable; i += kThreads)
    sh.table[i] = exp2(-static_cast<double>(i) / kTable);

  // The maximum and its first index.
  float best = -INFINITY;
  int best_i = 0x7fffffff;
  each(row, n, [&](float x, int i) {
    if (x > best) {  // a thread's indices ascend
      best = x;
      best_i = i;
    }
  });
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float x = __shfl_xor(best, o);
    const int i = __shfl_xor(best_i, o);
    if (x > best || (x == best && i < best_i)) {
      best = x;
      best_i = i;
    }
  }
  if (lane == 0) {
    sh.red_x[wv] = best;
    sh.red_i[wv] = best_i;
  }
  __syncthreads();
  best = sh.red_x[0];
  best_i = sh.red_i[0];
  for (int i = 1; i < kWavesWg; ++i)
    if (sh.red_x[i] > best || (sh.red_x[i] == best && sh.red_i[i] < best_i)) {
      best = sh.red_x[i];
      best_i = sh.red_i[i];
    }
  // One token alone: no temperature, the first kept only, or an infinite logit.
  if (best_i == 0x7fffffff || !(temp > 0) || top_k == 1 || top_p <= 0 || min_p > 1 ||
      best == INFINITY) {
    if (tid == 0) {
      const bool none = best_i == 0x7fffffff;
      p.tokens[out] = none ? -1 : best_i;
      if (p.logprobs) p.logprobs[out] = none ? -INFINITY : 0.f;
    }
    return;
  }

  Scale sc;
  sc.mx = best;
  sc.mxd = best;
  sc.shift = p.shift;
  sc.c = kTable / (temp * 0.69314718055994530942);
  // The last bin starts past 46 halvings, where every weight rounds to 0.
  sc.bins = static_cast<float>(fmin((kBins - 1) / (46.0 * 0.69314718055994530942 * temp), 1e30));
  auto bins = [&](bool weights) {
    clear_bins(sh);
    each(row, n, [&](float x, int) {
      const int b = sc.bin(x);  // a NaN goes to the last bin
      if (b < kBins - 1) {
        atomicAdd(&sh.cnt[b], 1u);
        if (weights)
          atomicAdd(reinterpret_cast<unsigned long long *>(&sh.wsum[b]),
                    static_cast<unsigned long long>(sc.weight(x, sh.table)));
      }
    });
    __syncthreads();
    return scan_bins(sh, weights);
  };
  auto up_to = [&](int b) {
    return collect(row, n, sc, sh, 0, 0, [&](float x, int) { return sc.bin(x) <= b; });
  };
  auto only = [&](const Place &b) {
    return collect(row, n, sc, sh, b.before_c, b.before_w,
                   [&](float x, int) { return sc.bin(x) == b.at; });
  };

  Scan<4> h;        // the bins
  Scan<2> l;        // the list
  bool listed = false;  // whether the list holds all that can be kept
  uint64_t kept;    // weight of what is kept
  bool need_k = top_k > 0 && top_k < n;
  if (n <= kList) {
    l = up_to(kBins - 2);
    listed = true;
    kept = l.total_w;
    if (need_k && top_k < l.total_c) kept = find_listed<true>(l, top_k, sh).through_w;
  } else if (need_k && top_k <= kList) {
    h = bins(false);
    Place b{kBins - 2, 0, 0, 0, 0};
    uint32_t through = h.total_c;
    if (top_k < h.total_c) {
      b = find<true>(h, top_k, sh);
      through = b.before_c + b.c;
    }
    if (through <= kList) {
      l = up_to(b.at);
      listed = true;
      kept = top_k < l.total_c ? find_listed<true>(l, top_k, sh).through_w : l.total_w;
    }
  }
  auto reach = [&](uint64_t target) {  // a weight's place in the order
    if (listed) return find_listed<false>(l, target, sh);
    const Place b = find<false>(h, target, sh);
    if (b.c > kList) return find_crowded<false>(row, n, sc, sh, b, target);
    l = only(b);
    return find_listed<false>(l, target, sh);
  };
  if (!listed) {
    h = bins(true);
    kept = h.total_w;
    if (need_k && top_k < h.total_c) {
      const Place b = find<true>(h, top_k, sh);
      if (b.c > kList) {
        kept = find_crowded<true>(row, n, sc, sh, b, top_k).through_w;
      } else {
        l = only(b);
        kept = find_listed<true>(l, top_k, sh).through_w;
      }
    }
  }
  auto whole = [&](double x) {  // 0 for a NaN
    return x >= 1 ? (x < 9.0e18 ? static_cast<uint64_t>(x) : static_cast<uint64_t>(9.0e18)) : 0;
  };
  if (top_p < 1) {
    const uint64_t target =
        min(max(whole(ceil(top_p * static_cast<double>(kept))), uint64_t(1)), kept);
    if (!listed) {
      const Place b = find<false>(h, target, sh);
      if (b.before_c + b.c <= kList) {
        l = up_to(b.at);
        listed = true;
      }
    }
    kept = reach(target).through_w;
  }
  if (min_p > 0) {
    // Up to this distance from the maximum; what the bins next to it hold of
    // such elements is added one by one.
    const double far = -temp * log(min_p);
    const int b = static_cast<int>(fmin(far * static_cast<double>(sc.bins), kBins - 1.0));
    uint64_t w = 0;
    if (listed) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (l.c[i]) {
          const float x = of_key(~static_cast<uint32_t>(sh.list[tid * 2 + i] >> 32));
          if (sc.mxd - x <= far) w += l.w[i];
        }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (tid * 4 + i < b - 1) w += h.w[i];
      each(row, n, [&](float x, int) {
        const int bx = sc.bin(x);
        if (bx >= b - 1 && bx <= b + 1 && bx < kBins - 1 && sc.mxd - x <= far)
          w += sc.weight(x, sh.table);
      });
    }
    Scan<1> s;
    s.c[0] = 0;
    s.w[0] = w;
    scan_block(s, sh);
    if (s.total_w < kept) kept = s.total_w;
  }
  // In integers "exceeds u S" is "reaches floor(u S) + 1" (not added in 64-bit
  // floating point, which has no such neighbour past 2^53).
  const uint64_t target = min(whole(u * static_cast<double>(kept)) + 1, kept);
  const Element e = reach(target);
  if (tid == 0) {
    p.tokens[out] = e.index;
    if (p.logprobs)
      p.logprobs[out] = static_cast<float>(-(sc.mxd - e.x) / temp -
                                           log(ldexp(static_cast<double>(kept), -p.shift)));
  }
}

}  // namespace
}  // namespace mlr

extern "C" int mlr_sample_tokens(const void *logits, int64_t row_stride, int64_t num_logit_rows,
                                 int dtype, const int64_t *row_ids, const void *uniforms,
                                 int uniforms_f64, const float *temperature,
                                 double temperature_value, const void *top_k, int top_k_dtype,
                                 int64_t top_k_value, const float *top_p, double top_p_value,
                                 const float *min_p, double min_p_value, int64_t *tokens,
                                 float *logprobs, int64_t num_rows, int64_t vocab, void *stream) {
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
  MLR_REQUIRE(logits && uniforms && tokens, "mlr_sample_tokens: null pointer");
  SampleParams p;
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
    case MLR_DTYPE_F32: sample_kernel<float><<<grid, kThreads, 0, s>>>(p); break;
    case MLR_DTYPE_F16: sample_kernel<f16_t><<<grid, kThreads, 0, s>>>(p); break;
    default: sample_kernel<bf16_t><<<grid, kThreads, 0, s>>>(p); break;
  }
  return check_launch("mlr_sample_tokens");
}

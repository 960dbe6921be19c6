// The best places of a row of keys, in order: what key eviction and block selection
// share.
//
// Of n places the first `sinks` and the last `recent` are chosen, and of those between
// as many with the largest keys as make up `budget`, ties by the lower place. One
// workgroup looks for the smallest chosen one among the (key, place from the end)
// between: a histogram in LDS of the keys from the smallest to the largest gives the bin
// that holds it, one of that bin's keys the next, until the keys of a bin are all chosen,
// or so few that each is compared with all. 2,048 bins of equal width: mostly one
// histogram is enough for a few thousand keys, as scores and weights lie close together.
// Integers alone, so the order of the atomics does not matter. A wave holds a run of
// neighbouring places, so the chosen are counted wave by wave and written in order. (4,096 and
// 8,192 bins, which leave fewer keys in the last, took as long: 16,384 keys 20 us each.)
#pragma once

#include "mlr_common.h"

namespace mlr {

constexpr int kBinBits = 11;
constexpr int kBins = 1 << kBinBits;
constexpr int kFew = 64;  // places that are compared with each other

// Numbers as unsigned keys of the same order; NaN counts as -infinity, -0 as 0.
__device__ __forceinline__ uint32_t order_key(float x) {
  x = x != x ? -INFINITY : x + 0.f;
  const uint32_t b = __float_as_uint(x);
  return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t order_key(double x) {
  x = x != x ? -INFINITY : x + 0.;
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  return b >> 63 ? ~b : b | 0x8000000000000000u;
}

struct SelectShared {
  int hist[kBins];
  uint64_t few_key[kFew], low[16], high[16], last_key;
  int few_place[kFew], wave_sum[16];
  int bin, left, count, last_place;
};

// How many of the first `count` lanes' (key, place) come before this lane's.
__device__ __forceinline__ int rank_few(uint64_t key, int place, int count) {
  const uint32_t low = static_cast<uint32_t>(key), high = static_cast<uint32_t>(key >> 32);
  int better = 0;
  for (int o = 0; o < count; ++o) {
    const uint64_t x = static_cast<uint64_t>(__builtin_amdgcn_readlane(high, o)) << 32 |
                       static_cast<uint32_t>(__builtin_amdgcn_readlane(low, o));
    better += x > key || (x == key && __builtin_amdgcn_readlane(place, o) < place);
  }
  return better;
}

// How the places of a row are dealt to the threads of a workgroup: each wave has a run of
// neighbours, in steps of 256, four to a lane. load(keys, place) fills keys[j][e] with the
// key of place(j) + e, for places up to n - 1 (what it gives for others is not used).
// Keys of places outside [lo, hi) become 0, which order_key never gives. The first kHeld
// steps stay in registers; a wave with more reads them again each time.
template <typename Key, int kThreads, int kHeld, class Load>
struct Places {
  int n, lo, hi, first, steps;
  bool held, inner;  // inner: the wave's places all lie in [lo, hi)
  Key keys[kHeld][4];
  Load load;

  __device__ __forceinline__ Places(int n_, int lo_, int hi_, Load l)
      : n(n_), lo(lo_), hi(hi_), load(l) {
    constexpr int kWaves = kThreads / 64;
    steps = ((n + kWaves - 1) / kWaves + 255) / 256;
    const int start = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * steps * 256;
    first = start + 4 * (threadIdx.x & 63);
    held = steps <= kHeld;
    inner = start >= lo && start + 256 * steps <= hi;
    if (held) {
      const int at = first;
      load(keys, [at](int j) __attribute__((always_inline)) { return at + 256 * j; });
      if (!inner) {
#pragma unroll
        for (int j = 0; j < kHeld; ++j) clear(keys[j], first + 256 * j);
      }
    }
  }
  __device__ __forceinline__ void clear(Key (&k)[4], int i) const {
#pragma unroll
    for (int e = 0; e < 4; ++e) k[e] = i + e >= lo && i + e < hi ? k[e] : Key(0);
  }
  // f(place, the four keys from there on), for all steps in order.
  template <class F>
  __device__ __forceinline__ void each(F f) {
    if (held) {
#pragma unroll
      for (int j = 0; j < kHeld; ++j)
        if (j < steps) f(first + 256 * j, keys[j]);
    } else {
      for (int j = 0; j < steps; ++j) {
        Key one[1][4];
        const int at = first + 256 * j;
        load(one, [at](int) __attribute__((always_inline)) { return at; });
        clear(one[0], at);
        f(at, one[0]);
      }
    }
  }
  // Whether place i is chosen whatever its key: one before lo or from hi on.
  __device__ __forceinline__ bool forced(int i) const {
    return !inner && i < n && (i < lo || i >= hi);
  }
};

// A value that all lanes share, in scalar registers: what depends on it branches once a wave.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ uint32_t uniform(uint32_t x) {
  return __builtin_amdgcn_readfirstlane(x);
}
__device__ __forceinline__ uint64_t uniform(uint64_t x) {
  const uint32_t low = uniform(static_cast<uint32_t>(x));
  return static_cast<uint64_t>(uniform(static_cast<uint32_t>(x >> 32))) << 32 | low;
}

// The `left`-th best, left > 0, of the places in [lo, hi), which are at least so many: the
// largest key first, ties by the lower place. All threads of the workgroup call it.
template <typename Key, int kThreads, class P>
__device__ __forceinline__ void find_last(SelectShared &s, P &places, int left, Key &last_key,
                                          int &last_place) {
  constexpr int kWaves = kThreads / 64;
  const int tid = threadIdx.x, lane = tid & 63, n = places.n;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // In question: keys from base on, `span` of them further, and once that is one key, places
  // (counted from the end) from place_base on, below 2^place_bits of them.
  Key least = ~Key(0), most = 0;  // least: less 1, so that 0 is the largest
  places.each([&](int, const Key(&k)[4]) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      least = k[e] - 1 < least ? k[e] - 1 : least;
      most = k[e] > most ? k[e] : most;
    }
  });
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const Key a = __shfl_xor(least, o), b = __shfl_xor(most, o);
    least = a < least ? a : least;
    most = b > most ? b : most;
  }
  if (lane == 0) {
    s.low[wave] = least;
    s.high[wave] = most;
  }
  for (int i = tid; i < kBins; i += kThreads) s.hist[i] = 0;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    least = static_cast<Key>(s.low[w]) < least ? static_cast<Key>(s.low[w]) : least;
    most = static_cast<Key>(s.high[w]) > most ? static_cast<Key>(s.high[w]) : most;
  }
  most = uniform(most);
  Key base = uniform(static_cast<Key>(least + 1)), span = most - base;
  int bits = span > 0 ? 64 - __clzll(static_cast<uint64_t>(span)) : 0;
  uint32_t place_base = 0;
  int place_bits = 32 - __clz(n);
  auto from_end = [&](int i) __attribute__((always_inline)) {
    return static_cast<uint32_t>(n - 1 - i);
  };
  // A key of 0 is further from base than the largest.
  auto in_span = [&](Key k) __attribute__((always_inline)) { return k - base <= span; };
  auto in_places = [&](int i, Key k) __attribute__((always_inline)) {
    return k == base && from_end(i) >= place_base && (from_end(i) - place_base) >> place_bits == 0;
  };
  for (;;) {
    const bool by_key = bits > 0;
    const int shift = max((by_key ? bits : place_bits) - kBinBits, 0);
    if (by_key) {
      places.each([&](int, const Key(&k)[4]) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (in_span(k[e])) atomicAdd(&s.hist[static_cast<int>((k[e] - base) >> shift)], 1);
      });
    } else {
      places.each([&](int i, const Key(&k)[4]) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (in_places(i + e, k[e]))
            atomicAdd(&s.hist[static_cast<int>((from_end(i + e) - place_base) >> shift)], 1);
      });
    }
    __syncthreads();
    // Thread t has the bins kBins - 1 - kOwn t and those below.
    constexpr int kOwn = kBins / kThreads;
    int own[kOwn], sum = 0;
#pragma unroll
    for (int b = 0; b < kOwn; ++b) sum += own[b] = s.hist[kBins - 1 - kOwn * tid - b];
    int upto = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int x = __shfl_up(upto, o);
      if (lane >= o) upto += x;
    }
    if (lane == 63) s.wave_sum[wave] = upto;
    if (tid == 0) s.count = 0;
    __syncthreads();
    int over = upto - sum;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) over += w < wave ? s.wave_sum[w] : 0;
    if (over < left && over + sum >= left) {
#pragma unroll
      for (int b = 0; b < kOwn; ++b) {
        if (over < left && over + own[b] >= left) {
          s.bin = kBins - 1 - kOwn * tid - b;
          s.left = left - over;
        }
        over += own[b];
      }
    }
    __syncthreads();
    const int bin = uniform(s.bin), count = uniform(s.hist[bin]);
    left = uniform(s.left);
    if (by_key) {
      base += static_cast<Key>(bin) << shift;
      bits = shift;
      span = min(static_cast<Key>((Key(1) << shift) - 1), static_cast<Key>(most - base));
    } else {
      place_base += static_cast<uint32_t>(bin) << shift;
      place_bits = shift;
    }
    if (count == left) {  // all of them
      last_key = base;
      last_place = by_key ? 0x7fffffff : n - 1 - static_cast<int>(place_base);
      break;
    }
    if (count <= kFew) {
      const bool whole = bits > 0;  // places do not matter yet
      places.each([&](int i, const Key(&k)[4]) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (whole ? in_span(k[e]) : in_places(i + e, k[e])) {
            const int at = atomicAdd(&s.count, 1);
            s.few_key[at] = k[e];
            s.few_place[at] = i + e;
          }
      });
      __syncthreads();
      if (wave == 0) {
        const uint64_t k = s.few_key[min(lane, count - 1)];
        const int i = s.few_place[min(lane, count - 1)];
        const int better = rank_few(k, i, count);
        if (lane < count && better == left - 1) {
          s.last_key = k;
          s.last_place = i;
        }
      }
      __syncthreads();
      last_key = static_cast<Key>(s.last_key);
      last_place = s.last_place;
      break;
    }
    __syncthreads();
    for (int i = tid; i < kBins; i += kThreads) s.hist[i] = 0;
    __syncthreads();
  }
}

// emit(r, i, at) for each place i with chosen(i, its key), r counting them in order; `at` is
// where the thread holds the place's key, 4 j + e, or -1.
template <typename Key, int kThreads, int kHeld, class P, class Chosen, class Emit>
__device__ __forceinline__ void emit_places(SelectShared &s, P &places, Chosen chosen, Emit emit) {
  static_assert(kHeld <= 8, "a bit for each key that a thread holds");
  constexpr int kWaves = kThreads / 64;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int before = 0;
  uint32_t taken = 0;
  if (places.held) {
#pragma unroll
    for (int j = 0; j < kHeld; ++j)
      if (j < places.steps) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool yes = chosen(places.first + 256 * j + e, places.keys[j][e]);
          taken |= yes ? 1u << (4 * j + e) : 0u;
          before += __popcll(__ballot(yes));
        }
      }
  } else {
    places.each([&](int i, const Key(&k)[4]) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < 4; ++e) before += __popcll(__ballot(chosen(i + e, k[e])));
    });
  }
  __syncthreads();  // wave_sum has been read
  if (lane == 0) s.wave_sum[wave] = before;
  __syncthreads();
  before = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) before += w < wave ? s.wave_sum[w] : 0;
  const uint64_t below = (uint64_t(1) << lane) - 1;
  if (places.held) {
#pragma unroll
    for (int j = 0; j < kHeld; ++j)
      if (j < places.steps) {
        int r = before;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint64_t all = __ballot(taken >> (4 * j + e) & 1);
          r += __popcll(all & below);
          before += __popcll(all);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (taken >> (4 * j + e) & 1) emit(r++, places.first + 256 * j + e, 4 * j + e);
      }
  } else {
    places.each([&](int i, const Key(&k)[4]) __attribute__((always_inline)) {
      int r = before;
      bool yes[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        yes[e] = chosen(i + e, k[e]);
        const uint64_t all = __ballot(yes[e]);
        r += __popcll(all & below);
        before += __popcll(all);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (yes[e]) emit(r++, i + e, -1);
    });
  }
}

// The choice by keys alone; emit as in emit_places. Returns the number of the chosen. All
// threads of a workgroup of kThreads call it, with the same sizes: 0 <= n, sinks + recent
// <= budget.
template <typename Key, int kThreads, int kHeld, class Load, class Emit>
__device__ __forceinline__ int select_places(SelectShared &s, int n, int sinks, int recent,
                                             int budget, Load load, Emit emit) {
  if (n <= budget) {
    for (int i = threadIdx.x; i < n; i += kThreads) emit(i, i, -1);
    return n;
  }
  const int left = budget - sinks - recent;
  Places<Key, kThreads, kHeld, Load> places(n, sinks, n - recent, load);
  Key last_key = ~Key(0);  // with no place left no key is large enough
  int last_place = -1;
  if (left > 0) find_last<Key, kThreads>(s, places, left, last_key, last_place);
  emit_places<Key, kThreads, kHeld>(
      s, places,
      [&](int i, Key k) __attribute__((always_inline)) {
        return k > last_key || (k == last_key && i <= last_place) || places.forced(i);
      },
      emit);
  return budget;
}

}  // namespace mlr

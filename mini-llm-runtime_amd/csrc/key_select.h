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
// neighbouring places, so the chosen are counted wave by wave and written in order.
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

// load(keys, place) fills keys[j][e] with the key of place(j) + e, for places up to n - 1
// (what it gives for others is not used); emit(r, i) is called once for each chosen place
// i, r counting them in order. Returns their number. All threads of a workgroup of
// kThreads call it, with the same sizes: 0 <= n, sinks + recent <= budget. The keys of
// the first kHeld * 4 * kThreads places stay in registers, further ones are read again.
template <typename Key, int kThreads, int kHeld, class Load, class Emit>
__device__ __forceinline__ int select_places(SelectShared &s, int n, int sinks, int recent,
                                             int budget, Load load, Emit emit) {
  constexpr int kWaves = kThreads / 64;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  if (n <= budget) {
    for (int i = tid; i < n; i += kThreads) emit(i, i);
    return n;
  }
  const int lo = sinks, hi = n - recent;
  // Of each wave, in steps of 256 places, four to a lane, kHeld of them at a time.
  const int steps = ((n + kWaves - 1) / kWaves + 255) / 256;
  const int first = wave * steps * 256 + 4 * lane;
  const bool held = steps <= kHeld;
  Key keys[kHeld][4];
  if (held) load(keys, [&](int j) __attribute__((always_inline)) { return first + 256 * j; });
  // f(place, the four keys from there on), for all steps in order.
  auto each = [&](auto &&f) __attribute__((always_inline)) {
    if (held) {
#pragma unroll
      for (int j = 0; j < kHeld; ++j)
        if (j < steps) f(first + 256 * j, keys[j]);
    } else {
      for (int j = 0; j < steps; ++j) {
        Key one[1][4];
        load(one, [&](int) __attribute__((always_inline)) { return first + 256 * j; });
        f(first + 256 * j, one[0]);
      }
    }
  };
  auto between = [&](int i) __attribute__((always_inline)) { return i >= lo && i < hi; };
  int left = budget - sinks - recent;  // still to be chosen among those in question
  // The last chosen one between: key and place. Without one no key is large enough.
  Key last_key = ~Key(0);
  int last_place = -1;
  if (left > 0) {
    // In question: keys from base on, below 2^bits of them, and once that is one key,
    // places (counted from the end) from place_base on, below 2^place_bits of them.
    Key least = ~Key(0), most = 0;
    each([&](int i, const Key(&k)[4]) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        least = between(i + e) && k[e] < least ? k[e] : least;
        most = between(i + e) && k[e] > most ? k[e] : most;
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
    Key base = least;
    int bits = most > least ? 64 - __clzll(static_cast<uint64_t>(most - least)) : 0;
    uint32_t place_base = 0;
    int place_bits = 32 - __clz(n);
    auto from_end = [&](int i) __attribute__((always_inline)) {
      return static_cast<uint32_t>(n - 1 - i);
    };
    auto asked = [&](int i, Key k) __attribute__((always_inline)) {
      // Shifts in two steps, as `bits` may be that of the whole type.
      return between(i) && k >= base && (k - base) >> (bits / 2) >> (bits - bits / 2) == 0 &&
             from_end(i) >= place_base && (from_end(i) - place_base) >> place_bits == 0;
    };
    for (;;) {
      const bool by_key = bits > 0;
      const int shift = max((by_key ? bits : place_bits) - kBinBits, 0);
      auto bin_of = [&](int i, Key k) __attribute__((always_inline)) {
        return by_key ? static_cast<int>((k - base) >> shift)
                      : static_cast<int>((from_end(i) - place_base) >> shift);
      };
      each([&](int i, const Key(&k)[4]) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (asked(i + e, k[e])) atomicAdd(&s.hist[bin_of(i + e, k[e])], 1);
      });
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
      const int count = s.hist[s.bin];
      left = s.left;
      if (by_key) {
        base += static_cast<Key>(s.bin) << shift;
        bits = shift;
      } else {
        place_base += static_cast<uint32_t>(s.bin) << shift;
        place_bits = shift;
      }
      if (count == left) {  // all of them
        last_key = base;
        last_place = by_key ? 0x7fffffff : n - 1 - static_cast<int>(place_base);
        break;
      }
      if (count <= kFew) {
        each([&](int i, const Key(&k)[4]) __attribute__((always_inline)) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (asked(i + e, k[e])) {
              const int at = atomicAdd(&s.count, 1);
              s.few_key[at] = k[e];
              s.few_place[at] = i + e;
            }
        });
        __syncthreads();
        if (wave == 0) {
          const uint64_t k = s.few_key[min(lane, count - 1)];
          const int i = s.few_place[min(lane, count - 1)];
          int better = 0;
          for (int o = 0; o < count; ++o) {
            const uint64_t x = s.few_key[o];
            better += x > k || (x == k && s.few_place[o] < i);
          }
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
  auto chosen = [&](int i, Key k) __attribute__((always_inline)) {
    return i < n && (!between(i) || k > last_key || (k == last_key && i <= last_place));
  };
  int before = 0;
  each([&](int i, const Key(&k)[4]) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 4; ++e) before += __popcll(__ballot(chosen(i + e, k[e])));
  });
  __syncthreads();  // wave_sum has been read
  if (lane == 0) s.wave_sum[wave] = before;
  __syncthreads();
  before = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) before += w < wave ? s.wave_sum[w] : 0;
  const uint64_t below = (uint64_t(1) << lane) - 1;
  each([&](int i, const Key(&k)[4]) __attribute__((always_inline)) {
    int r = before;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint64_t all = __ballot(chosen(i + e, k[e]));
      r += __popcll(all & below);
      before += __popcll(all);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (chosen(i + e, k[e])) emit(r++, i + e);
  });
  return budget;
}

}  // namespace mlr

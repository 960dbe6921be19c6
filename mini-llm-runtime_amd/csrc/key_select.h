// The best places of a row of keys, in order: what key eviction and block selection
// share.
//
// Of n places the first `sinks` and the last `recent` are chosen, and of those between
// as many with the largest keys as make up `budget`, ties by the lower place. One
// workgroup finds the smallest chosen key digit by digit from the top: a histogram in
// LDS of the keys that share the digits found so far gives the next one, until the
// keys of a bin are all chosen. A wave holds a run of neighbouring places, so the
// chosen are counted wave by wave and then written in order.
#pragma once

#include "mlr_common.h"

namespace mlr {

constexpr int kSelectThreads = 1024;

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
  int hist[256];
  int above[kSelectThreads / 64], equal[kSelectThreads / 64];
  int bin, left, whole;
};

// load(i) is the key of place i; emit(r, i) is called once for each chosen place, r
// counting them in order. Returns their number. kHeld keys of a thread stay in
// registers; rows past that are read again for each digit. All threads of a workgroup of
// kSelectThreads call it, with the same sizes: 0 <= n, sinks + recent <= budget.
template <typename Key, int kHeld, class Load, class Emit>
__device__ __forceinline__ int select_places(SelectShared &s, int n, int sinks, int recent,
                                             int budget, Load load, Emit emit) {
  constexpr int kWaves = kSelectThreads / 64;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  if (n <= budget) {
    for (int i = tid; i < n; i += kSelectThreads) emit(i, i);
    return n;
  }
  const int lo = sinks, hi = n - recent;
  const int steps = ((n + kWaves - 1) / kWaves + 63) / 64;  // of 64 places, of each wave
  const int first = wave * steps * 64 + lane;
  const bool held = steps <= kHeld;
  Key keys[kHeld];
  if (held) {
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
      const int i = first + 64 * j;
      keys[j] = j < steps && i >= lo && i < hi ? load(i) : Key(0);
    }
  }
  auto each = [&](auto &&f) __attribute__((always_inline)) {
    if (held) {
#pragma unroll
      for (int j = 0; j < kHeld; ++j)
        if (j < steps) f(first + 64 * j, keys[j]);
    } else {
      for (int j = 0; j < steps; ++j) {
        const int i = first + 64 * j;
        f(i, i >= lo && i < hi ? load(i) : Key(0));
      }
    }
  };

  int left = budget - sinks - recent;  // still to be chosen among the keys of `top`
  Key top = 0, mask = 0;
  for (int shift = 8 * static_cast<int>(sizeof(Key)) - 8; shift >= 0 && left > 0; shift -= 8) {
    for (int i = tid; i < 256; i += kSelectThreads) s.hist[i] = 0;
    __syncthreads();
    each([&](int i, Key k) __attribute__((always_inline)) {
      if (i >= lo && i < hi && (k & mask) == top)
        atomicAdd(&s.hist[static_cast<int>(k >> shift) & 255], 1);
    });
    __syncthreads();
    if (wave == 0) {
      // Lane l has the bins 255 - 4 l and the three below; the keys above them.
      int h[4], sum = 0;
#pragma unroll
      for (int b = 0; b < 4; ++b) sum += h[b] = s.hist[255 - 4 * lane - b];
      int upto = sum;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int x = __shfl_up(upto, o);
        if (lane >= o) upto += x;
      }
      int over = upto - sum;
      if (over < left && upto >= left) {
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          if (over < left && over + h[b] >= left) {
            s.bin = 255 - 4 * lane - b;
            s.left = left - over;
            s.whole = over + h[b] == left;
          }
          over += h[b];
        }
      }
    }
    __syncthreads();
    top |= static_cast<Key>(s.bin) << shift;
    mask |= static_cast<Key>(255) << shift;
    left = s.left;
    const bool whole = s.whole;
    __syncthreads();
    if (whole) break;
  }
  // Chosen: keys above `top` in the digits found, and the first `left` equal to it.
  const bool none = left <= 0;  // the sinks and the recent places are all
  int above = 0, equal = 0;
  auto kind = [&](int i, Key k, bool &over, bool &same) __attribute__((always_inline)) {
    const bool mid = i >= lo && i < hi;
    over = i < n && (!mid || (!none && (k & mask) > top));
    same = mid && !none && (k & mask) == top;
  };
  each([&](int i, Key k) __attribute__((always_inline)) {
    bool over, same;
    kind(i, k, over, same);
    above += __popcll(__ballot(over));
    equal += __popcll(__ballot(same));
  });
  if (lane == 0) {
    s.above[wave] = above;
    s.equal[wave] = equal;
  }
  __syncthreads();
  above = equal = 0;
  for (int w = 0; w < wave; ++w) {
    above += s.above[w];
    equal += s.equal[w];
  }
  const uint64_t below = (uint64_t(1) << lane) - 1;
  each([&](int i, Key k) __attribute__((always_inline)) {
    bool over, same;
    kind(i, k, over, same);
    const uint64_t a = __ballot(over), e = __ballot(same);
    const int eq = equal + __popcll(e & below);
    if (over || (same && eq < left)) emit(above + __popcll(a & below) + min(eq, left), i);
    above += __popcll(a);
    equal += __popcll(e);
  });
  return budget;
}

}  // namespace mlr

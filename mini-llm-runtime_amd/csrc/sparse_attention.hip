// Decode over the blocks of a cache that a cheap score selects.
//
//   bounds: for each block and KV head the elementwise minimum and maximum of its keys.
//   score of block j for request and KV head: the largest, over the heads h of the
//     group, of sum_d max(q_hd min_jd, q_hd max_jd), which no q_h.k of its keys exceeds
//   chosen: the first `sinks` blocks, the last `recent`, and of the others the best, up to
//     `budget`; attention over the keys of the chosen blocks.
//
// Scores are 64-bit sums of exact products, so which blocks are read does not
// depend on the order of a sum in 32 bits. The chosen blocks of a request and KV head
// become a block table of their own, in order, with which the decode of
// scored_rows.hip runs as over any other.
#include "key_select.h"
#include "scored_attention.h"

#include <algorithm>

namespace mlr {
namespace {

struct BoundParams {
  const void *k;
  void *bounds;  // [num_blocks, 2, hkv, d]
  int64_t num_blocks, block_size, hkv, d;
  const int64_t *bt;
  int64_t bt_st, bt_width;
  const int64_t *ctx, *starts;
  int64_t seqs, most;  // most: changed blocks of a request at most
};

template <typename T>
__device__ __forceinline__ void unpack(uint4 w, float *x) {
  if constexpr (sizeof(T) == 4) {
    x[0] = __uint_as_float(w.x);
    x[1] = __uint_as_float(w.y);
    x[2] = __uint_as_float(w.z);
    x[3] = __uint_as_float(w.w);
  } else {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = Elem<T>::to_f32(T{static_cast<uint16_t>(u[i])});
      x[2 * i + 1] = Elem<T>::to_f32(T{static_cast<uint16_t>(u[i] >> 16)});
    }
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack(const float *x) {
  if constexpr (sizeof(T) == 4) {
    return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]),
                      __float_as_uint(x[3]));
  } else {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      u[i] = Elem<T>::from_f32(x[2 * i]).bits |
             static_cast<uint32_t>(Elem<T>::from_f32(x[2 * i + 1]).bits) << 16;
    return make_uint4(u[0], u[1], u[2], u[3]);
  }
}

// Thread: 16 bytes of a row of one changed block and KV head; a block's keys are read once.
// Bound by the read: 4 requests of 7,000 to 8,192 keys, 8 KV heads of 128: 71 MB in 12.7 us,
// some from the caches; one new key of 64 requests, 2 KV heads of 64, 4.3 us of latency (7.1 us
// the call).
template <typename T>
__global__ __launch_bounds__(256) void bound_keys(BoundParams p) {
  constexpr int kE = 16 / sizeof(T);
  const int64_t pieces = p.hkv * p.d / kE;
  const int64_t total = p.seqs * p.most * pieces;
  for (int64_t at = blockIdx.x * int64_t(256) + threadIdx.x; at < total;
       at += gridDim.x * int64_t(256)) {
    const int64_t piece = at % pieces, which = at / pieces;
    const int64_t seq = which / p.most;
    const int64_t ctx = clamp64(p.ctx[seq], 0, p.bt_width * p.block_size);
    const int64_t start = p.starts ? clamp64(p.starts[seq], 0, ctx) : 0;
    const int64_t block = start / p.block_size + which % p.most;
    const int64_t keys = min(ctx - block * p.block_size, p.block_size);
    if (keys <= 0 || (p.starts && start >= ctx)) continue;
    const int64_t id = p.bt[seq * p.bt_st + block];
    if (id < 0 || id >= p.num_blocks) continue;
    const int64_t row = p.hkv * p.d;
    const T *k = static_cast<const T *>(p.k) + id * p.block_size * row + piece * kE;
    float low[kE], high[kE];
#pragma unroll
    for (int e = 0; e < kE; ++e) {
      low[e] = INFINITY;
      high[e] = -INFINITY;
    }
#pragma unroll 8
    for (int64_t i = 0; i < keys; ++i) {
      float x[kE];
      unpack<T>(*reinterpret_cast<const uint4 *>(k + i * row), x);
#pragma unroll
      for (int e = 0; e < kE; ++e) {  // a NaN stays
        low[e] = __builtin_elementwise_minimum(low[e], x[e]);
        high[e] = __builtin_elementwise_maximum(high[e], x[e]);
      }
    }
    T *out = static_cast<T *>(p.bounds) + id * 2 * row + piece * kE;
    *reinterpret_cast<uint4 *>(out) = pack<T>(low);
    *reinterpret_cast<uint4 *>(out + row) = pack<T>(high);
  }
}

struct SparseParams {
  const void *q, *bounds;
  int64_t q_st, q_sh;
  int64_t num_blocks, block_size, hkv, group, d;
  const int64_t *bt;
  int64_t bt_st, bt_width;
  const int64_t *ctx;
  int64_t seqs;
  bool flip;  // a negative scale: the largest score is that of -q
  int sinks, recent, budget, list;  // list: columns of `table`, min(budget, bt_width)
  uint64_t *keys;                   // [seqs, hkv, keys_st] scores as ordered keys, or in
                                    // 32 bits with their errors
  uint64_t *exact;                  // as many, for choose_rough
  int64_t keys_st;                  // bt_width, in whole fours
  int64_t *table;                   // [seqs, hkv, list] physical blocks of the chosen
  int64_t *lens;                    // [seqs] keys of the chosen blocks
  int64_t *chosen;                  // [seqs, hkv, budget] their places, may be null
};

typedef double f64x4_t __attribute__((ext_vector_type(4)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

// Whether a 32-bit word of a row holds an infinity or NaN.
template <typename T>
__device__ __forceinline__ bool odd(uint32_t w) {
  if constexpr (sizeof(T) == 4) return (w & 0x7f800000u) == 0x7f800000u;
  else if constexpr (std::is_same_v<T, bf16_t>)
    return (((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u) != 0;
  else return (((w & 0x7c007c00u) + 0x04000400u) & 0x80008000u) != 0;
}
template <typename T>
__device__ __forceinline__ bool odd(uint4 w) {
  return odd<T>(w.x) || odd<T>(w.y) || odd<T>(w.z) || odd<T>(w.w);
}

// One request and KV head. Of a row, lane group l / 16 has every fourth piece of 16 bytes,
// so that its k-th elements are those of a head (lane l: head l % 16) and of a block
// (block l % 16) alike.
template <typename T, int kT>
struct Pair {
  static constexpr int kE = 16 / sizeof(T);
  int64_t seq, kvh, n;  // n: blocks of the request
  const int64_t *table;
  const T *q, *bounds;
  int64_t q_sh, row, d, num_blocks;
  int heads, col, g;
  bool flip;

  __device__ __forceinline__ Pair(const SparseParams &p, int64_t pair_seq, int64_t pair_kvh)
      : seq(pair_seq), kvh(pair_kvh), q_sh(p.q_sh), row(p.hkv * p.d), d(p.d),
        num_blocks(p.num_blocks), heads(static_cast<int>(p.group)), col(threadIdx.x & 15),
        g((threadIdx.x & 63) >> 4), flip(p.flip) {
    const int64_t ctx = clamp64(p.ctx[seq], 0, p.bt_width * p.block_size);
    n = (ctx + p.block_size - 1) / p.block_size;
    table = p.bt + seq * p.bt_st;
    q = static_cast<const T *>(p.q) + seq * p.q_st + kvh * p.group * p.q_sh;
    bounds = static_cast<const T *>(p.bounds) + kvh * d;
  }
  // The lane's pieces of a block's bounds, zeros where there is none.
  __device__ __forceinline__ bool read(uint4 (&low)[kT], uint4 (&high)[kT], int64_t id) const {
    const bool there = id >= 0 && id < num_blocks;
    const T *at = bounds + (there ? id : 0) * 2 * row;
#pragma unroll
    for (int t = 0; t < kT; ++t) {
      const int e = (g + 4 * t) * kE;
      low[t] = high[t] = make_uint4(0, 0, 0, 0);
      if (e < d && there) {
        low[t] = *reinterpret_cast<const uint4 *>(at + e);
        high[t] = *reinterpret_cast<const uint4 *>(at + row + e);
      }
    }
    return there;
  }
  // And of head h0 + l % 16; a group of fewer heads repeats its last one, so that a
  // maximum over heads needs no mask.
  __device__ __forceinline__ void read_q(uint4 (&x)[kT], int h0) const {
    const T *mine = q + min(h0 + col, heads - 1) * q_sh;
#pragma unroll
    for (int t = 0; t < kT; ++t) {
      const int e = (g + 4 * t) * kE;
      x[t] = make_uint4(0, 0, 0, 0);
      if (e < d) x[t] = *reinterpret_cast<const uint4 *>(mine + e);
    }
  }

  // The scores of a wave's 16 blocks, block l % 16's in lane l, in 64 bits on
  // v_mfma_f64_16x16x4: sum_d max(q low, q high) = [q-, q+].[low, high] with q- = min(q, 0)
  // and q+ = max(q, 0), heads as operand A, blocks as operand B. Where a bound or q is not
  // finite, 0 times it would be NaN where the larger of both products is not: such tiles
  // take a head at a time, in every row of A, and only the bound that it asks for; a sum
  // that is NaN does not count. Both add up the same products in the same order, so that
  // blocks of the same score have it to the last bit wherever they stand.
  __device__ __forceinline__ double score(int64_t id) const {
    uint4 low[kT], high[kT];
    const bool there = read(low, high, id);
    double best = -INFINITY;
    for (int h0 = 0; h0 < heads; h0 += 16) {
      uint4 x[kT];
      read_q(x, h0);
      bool strange = false;
#pragma unroll
      for (int t = 0; t < kT; ++t)
        strange = strange || odd<T>(x[t]) || odd<T>(low[t]) || odd<T>(high[t]);
      if (__builtin_expect(!__any(strange), 1)) {
        f64x4_t sum0 = {0., 0., 0., 0.}, sum1 = {0., 0., 0., 0.};
#pragma unroll
        for (int t = 0; t < kT; ++t) {
          float f[kE], l[kE], u[kE];
          unpack<T>(x[t], f);
          unpack<T>(low[t], l);
          unpack<T>(high[t], u);
#pragma unroll
          for (int e = 0; e < kE; ++e) {
            const float v = flip ? -f[e] : f[e];
            sum0 = __builtin_amdgcn_mfma_f64_16x16x4f64(fminf(v, 0.f), l[e], sum0, 0, 0, 0);
            sum1 = __builtin_amdgcn_mfma_f64_16x16x4f64(fmaxf(v, 0.f), u[e], sum1, 0, 0, 0);
          }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) best = fmax(best, sum0[r] + sum1[r]);
      } else {
        for (int h = h0; h < min(h0 + 16, heads); ++h) {
          f64x4_t sum0 = {0., 0., 0., 0.}, sum1 = {0., 0., 0., 0.};
#pragma unroll
          for (int t = 0; t < kT; ++t) {
            float l[kE], u[kE];
            unpack<T>(low[t], l);
            unpack<T>(high[t], u);
#pragma unroll
            for (int e = 0; e < kE; ++e) {
              const int at = (g + 4 * t) * kE + e;
              const float f = at < d ? Elem<T>::to_f32(q[h * q_sh + at]) : 0.f;
              const float v = flip ? -f : f;
              const bool below = v < 0.f;
              sum0 = __builtin_amdgcn_mfma_f64_16x16x4f64(below ? v : 0.f, below ? l[e] : 0.f, sum0,
                                                          0, 0, 0);
              sum1 = __builtin_amdgcn_mfma_f64_16x16x4f64(below ? 0.f : v, below ? 0.f : u[e], sum1,
                                                          0, 0, 0);
            }
          }
          const double sum = sum0[0] + sum1[0];
          best = sum > best ? sum : best;
        }
      }
    }
    best = fmax(best, __shfl_xor(best, 16));
    best = fmax(best, __shfl_xor(best, 32));
    return there ? best : -INFINITY;
  }
};

// Scores in 64 bits of all blocks (FP32, and where score_rough is not taken), a wave for 16.
// Bound by the 64-bit matrix instructions, half of whose work is with zeros: 8 requests of
// 2,048 blocks, 4 KV heads of 128: 8.6 GFLOP of 16 heads in 26 us.
template <typename T, int kT>
__global__ __launch_bounds__(256) void score_blocks(SparseParams p) {
  const int64_t b = blockIdx.x;
  const Pair<T, kT> x(p, b % p.seqs, b / p.seqs % p.hkv);
  const int64_t first = (b / p.seqs / p.hkv * 4 + (threadIdx.x >> 6)) * 16;
  if (first >= x.n || x.n <= p.budget) return;  // nothing there, or nothing to choose
  const int64_t j = first + x.col;
  const double best = x.score(j < x.n ? x.table[j] : -1);
  if (x.g == 0 && j < x.n)
    p.keys[(x.seq * p.hkv + x.kvh) * p.keys_st + j] = order_key(best);
}

// For the 16-bit types, scores in 32 bits on the matrix instructions of the type, with how
// far at most they are from those in 64: what that leaves undecided, a few blocks around the
// last chosen one, is scored in 64 bits by choose_rough.
//   |error| <= (2 d + 8) 2^-22 (sum_d |q_d|) (max_d |bound_d|)
// for 2 d products, exact in 32 bits, added in any order with a relative error of 2^-22 each
// (four times that of rounding to nearest), and 1e-30 of each factor for operands that
// the matrix unit may take for 0. Not finite, or (sum_d |q_d|) (max_d |bound_d|) so large that a
// sum may overflow on its way to a smaller one: no bound.
// Bound by reading the bounds: 8 requests of 2,048 blocks, 4 KV heads of 128: 33 MB in
// 13.6 us, where score_blocks takes 26 us.
template <typename T> struct Rough;
template <> struct Rough<bf16_t> {
  __device__ static f32x4_t mfma(uint4 a, uint4 b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                   __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  }
};
template <> struct Rough<f16_t> {
  __device__ static f32x4_t mfma(uint4 a, uint4 b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a),
                                                  __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  }
};

template <typename T, int kT>
__global__ __launch_bounds__(256) void score_rough(SparseParams p, int tiles) {
  constexpr int kE = 8;
  const int64_t b = blockIdx.x;
  const Pair<T, kT> x(p, b % p.seqs, b / p.seqs % p.hkv);
  // A wave's tiles of 16 blocks: the workgroup's in turn.
  const int64_t first = (b / p.seqs / p.hkv * 4 * tiles + (threadIdx.x >> 6)) * 16;
  if (first >= x.n || x.n <= p.budget) return;
  auto id_of = [&](int i) __attribute__((always_inline)) {
    const int64_t j = first + 64 * i + x.col;
    const int64_t id = x.table[min(j, x.n - 1)];
    return j < x.n ? id : int64_t(-1);
  };
  auto sizes = [&](const uint4 (&w)[kT], bool add, float &v) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < kT; ++t) {
      float f[kE];
      unpack<T>(w[t], f);
#pragma unroll
      for (int e = 0; e < kE; ++e) v = add ? v + fabsf(f[e]) : fmaxf(v, fabsf(f[e]));
    }
  };
  // Halves of w whose sign is set, or is not; -0 makes no difference.
  auto part = [&](uint4 w, bool negative) __attribute__((always_inline)) {
    auto one = [&](uint32_t v) __attribute__((always_inline)) {
      const uint32_t minus = (v >> 15 & 0x00010001u) * 0xffffu;
      return negative ? v & minus : v & ~minus;
    };
    return make_uint4(one(w.x), one(w.y), one(w.z), one(w.w));
  };
  uint4 qw[kT];
  float q_size = 0.f;  // the largest sum of |q| of a head
  bool q_odd = false;
  auto read_q = [&](int h0) __attribute__((always_inline)) {
    x.read_q(qw, h0);
    const uint32_t turn = x.flip ? 0x80008000u : 0u;
#pragma unroll
    for (int t = 0; t < kT; ++t) {
      q_odd = q_odd || odd<T>(qw[t]);
      qw[t] = make_uint4(qw[t].x ^ turn, qw[t].y ^ turn, qw[t].z ^ turn, qw[t].w ^ turn);
    }
    float sum = 0.f;
    sizes(qw, true, sum);
    sum += __shfl_xor(sum, 16);
    q_size = fmaxf(q_size, sum + __shfl_xor(sum, 32));
  };
  uint4 low[2][kT], high[2][kT];
  bool there[2];
  auto score = [&](const uint4 (&l)[kT], const uint4 (&u)[kT], bool exists, int i)
      __attribute__((always_inline)) {
    float best = -INFINITY;
    for (int h0 = 0; h0 < x.heads; h0 += 16) {
      if (x.heads > 16) read_q(h0);
      f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int t = 0; t < kT; ++t) {
        sum = Rough<T>::mfma(part(qw[t], true), l[t], sum);
        sum = Rough<T>::mfma(part(qw[t], false), u[t], sum);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) best = __builtin_elementwise_maximum(best, sum[r]);  // NaN stays
    }
    best = __builtin_elementwise_maximum(best, __shfl_xor(best, 16));
    best = __builtin_elementwise_maximum(best, __shfl_xor(best, 32));
    float size = 0.f, most = q_size;
    bool strange = q_odd;
    sizes(l, false, size);
    sizes(u, false, size);
#pragma unroll
    for (int t = 0; t < kT; ++t) strange = strange || odd<T>(l[t]) || odd<T>(u[t]);
    size = fmaxf(size, __shfl_xor(size, 16));
    size = fmaxf(size, __shfl_xor(size, 32));
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) most = fmaxf(most, __shfl_xor(most, o));
    strange = __any(strange);  // of the whole tile, for q is everyone's
    const float d = static_cast<float>(x.d);
    float off = (2.f * d + 8.f) * 0x1p-22f * most * size + 1e-30f * (most + d * size + d);
    if (strange || !(most * size < 1e37f) || !(off < 1e37f)) {
      best = 0.f;
      off = INFINITY;
    }
    const int64_t j = first + 64 * i + x.col;
    if (x.g == 0 && j < x.n)
      reinterpret_cast<float2 *>(p.keys)[(x.seq * p.hkv + x.kvh) * p.keys_st + j] =
          exists ? make_float2(best, off) : make_float2(-INFINITY, 0.f);
  };
  const int count = static_cast<int>(min(int64_t(tiles), (x.n - first + 63) / 64));
  there[0] = x.read(low[0], high[0], id_of(0));
  int64_t id = id_of(1);
  if (x.heads <= 16) read_q(0);
  for (int i = 0; i < count; i += 2) {
    if (i + 1 < count) there[1] = x.read(low[1], high[1], id);
    id = id_of(i + 2);
    score(low[0], high[0], there[0], i);
    if (i + 1 >= count) break;
    if (i + 2 < count) there[0] = x.read(low[0], high[0], id);
    id = id_of(i + 3);
    score(low[1], high[1], there[1], i + 1);
  }
}

// Where the chosen of a request and KV head go: a block table of their own, and their places.
struct Chosen {
  const int64_t *row;
  int64_t *table, *chosen;
  __device__ __forceinline__ Chosen(const SparseParams &p, int64_t seq, int64_t kvh)
      : row(p.bt + seq * p.bt_st), table(p.table + (seq * p.hkv + kvh) * p.list),
        chosen(p.chosen ? p.chosen + (seq * p.hkv + kvh) * p.budget : nullptr) {}
  __device__ __forceinline__ void put(int r, int i, int64_t id) const {
    table[r] = id;
    if (chosen) chosen[r] = i;
  }
  __device__ __forceinline__ void operator()(int r, int i, int) const { put(r, i, row[i]); }
  // The last block is always chosen, and the only one that may not be full.
  __device__ __forceinline__ void finish(const SparseParams &p, int64_t seq, int64_t kvh,
                                         int count, int threads) const {
    if (chosen)
      for (int i = count + threadIdx.x; i < p.budget; i += threads) chosen[i] = -1;
    if (p.lens && kvh == 0 && threadIdx.x == 0) {
      const int64_t ctx = clamp64(p.ctx[seq], 0, p.bt_width * p.block_size);
      const int64_t n = (ctx + p.block_size - 1) / p.block_size;
      p.lens[seq] = count > 0 ? ctx - (n - count) * p.block_size : 0;
    }
  }
};

__device__ __forceinline__ int blocks_of(const SparseParams &p, int64_t seq) {
  const int64_t ctx = clamp64(p.ctx[seq], 0, p.bt_width * p.block_size);
  return static_cast<int>((ctx + p.block_size - 1) / p.block_size);
}

// Loads four neighbouring keys of 64 bits at a time.
__device__ __forceinline__ auto keys_from(const uint64_t *keys, int n) {
  return [keys, n](auto &held, auto place) __attribute__((always_inline)) {
    constexpr int kMany = sizeof(held) / sizeof(held[0]);
#pragma unroll
    for (int j = 0; j < kMany; ++j) {
      const ulonglong2 *at = reinterpret_cast<const ulonglong2 *>(keys + (min(place(j), n - 1) & ~3));
      const ulonglong2 a = at[0], b = at[1];
      held[j][0] = a.x;
      held[j][1] = a.y;
      held[j][2] = b.x;
      held[j][3] = b.y;
    }
  };
}

// A workgroup chooses the blocks of one request and KV head, from keys in the workspace.
template <int kThreads, int kHeld>
__global__ __launch_bounds__(kThreads) void choose_blocks(SparseParams p) {
  __shared__ SelectShared s;
  const int64_t seq = blockIdx.x % p.seqs, kvh = blockIdx.x / p.seqs;
  const int n = blocks_of(p, seq);
  const Chosen out(p, seq, kvh);
  const int count = select_places<uint64_t, kThreads, kHeld>(
      s, n, p.sinks, p.recent, p.budget,
      keys_from(p.keys + (seq * p.hkv + kvh) * p.keys_st, n), out);
  out.finish(p, seq, kvh, count, kThreads);
}

// The same for tables of few blocks, with their scores: one launch. Eight waves with a tile
// each; past that the scores of one request keep one CU too long. So few blocks need no
// histogram: each is compared with all. us of one launch and of two, 16 requests, 4 KV heads
// of 128, by blocks: 64 10.4 and 15.8, 128 14.0 and 15.1, 256 (sixteen waves) 36.6 and 15.8.
constexpr int kSmall = 128, kSmallThreads = 512;
template <typename T, int kT>
__global__ __launch_bounds__(kSmallThreads) void choose_small(SparseParams p) {
  static_assert(kSmallThreads == 4 * kSmall, "a tile a wave, four threads a block");
  __shared__ uint64_t s_keys[kSmall];
  __shared__ int s_count[kSmallThreads / 64];
  const Pair<T, kT> x(p, blockIdx.x % p.seqs, blockIdx.x / p.seqs);
  const int n = static_cast<int>(x.n), lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Chosen out(p, x.seq, x.kvh);
  const int i = threadIdx.x / 4;
  bool chosen = i < n && threadIdx.x % 4 == 0;
  if (n > p.budget) {  // uniform
    const int j = 16 * wave + x.col;
    if (16 * wave < n) {
      const double best = x.score(j < n ? x.table[j] : -1);
      if (x.g == 0) s_keys[j] = order_key(best);
    }
    __syncthreads();
    // A block is compared with all that are asked, by four threads.
    const int lo = p.sinks, hi = n - p.recent;
    const uint64_t key = s_keys[min(i, n - 1)];
    int better = 0;
#pragma unroll 8
    for (int o = lo + threadIdx.x % 4; o < hi; o += 4) {
      const uint64_t other = s_keys[o];
      better += other > key || (other == key && o < i);
    }
    better += __shfl_xor(better, 1);
    better += __shfl_xor(better, 2);
    chosen = chosen && (i < lo || i >= hi || better < p.budget - p.sinks - p.recent);
  }
  const uint64_t all = __ballot(chosen);
  if (lane == 0) s_count[wave] = __popcll(all);
  __syncthreads();
  int r = __popcll(all & ((uint64_t(1) << lane) - 1));
#pragma unroll
  for (int w = 0; w < kSmallThreads / 64; ++w) r += w < wave ? s_count[w] : 0;
  if (chosen) out(r, i, -1);
  out.finish(p, x.seq, x.kvh, min(n, p.budget), kSmallThreads);
}

// The choice from scores in 32 bits and how far off they may be. With T the last chosen of
// them and R the largest error, a block below T - 2 R is worse than all down to T, and one
// above T + 2 R is better than all from T on; those in between are scored in 64 bits. Where
// they are more than kFew, all blocks are. Bound by latency, a dozen steps of 1 us, 16.5 us
// for 32 lists of 2,048 blocks: what a later step needs of memory (block ids, q) is read with the
// scores.
constexpr int kRoughThreads = 512, kRoughHeld = 2;
constexpr int kRoughBlocks = 4 * kRoughThreads * kRoughHeld;  // at most, as they stay in registers

// The second look costs some 6 us more than choose_blocks, so that 32 bits pay where the
// scores in 64 take longer than that. us of scores and choice in 64 bits and in 32, by
// lists x blocks x elements x tiles of 16 heads: 8 x 512 x 128 14 and 20, 4 x 4,096 x 128 20 and
// 27, 128 x 512 x 64 20 and 20, 32 x 2,048 x 128 38 and 31, 64 x 4,096 x 128 98 and 66.
bool takes_rough(int64_t pairs, int64_t group, int64_t d, int64_t width, int64_t budget,
                 int dtype) {
  return dtype != MLR_DTYPE_F32 && width > std::max<int64_t>(budget, kSmall) &&
         width <= kRoughBlocks && pairs * width * d * ceil_div(group, 16) >= int64_t(6) << 20;
}
template <typename T, int kT>
__global__ __launch_bounds__(kRoughThreads) void choose_rough(SparseParams p) {
  constexpr int kWaves = kRoughThreads / 64;
  __shared__ SelectShared s;
  __shared__ float s_off[kWaves];
  __shared__ int64_t s_id[kFew];
  __shared__ int s_sure[kWaves], s_open[kWaves], s_taken[kFew];
  const Pair<T, kT> x(p, blockIdx.x % p.seqs, blockIdx.x / p.seqs);
  const int n = static_cast<int>(x.n), lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Chosen out(p, x.seq, x.kvh);
  const int left = p.budget - p.sinks - p.recent;
  if (n <= p.budget || left == 0) {  // uniform
    const int count = min(n, p.budget);
    for (int i = threadIdx.x; i < count; i += kRoughThreads)
      out(i, n <= p.budget || i < p.sinks ? i : n - p.budget + i, -1);
    out.finish(p, x.seq, x.kvh, count, kRoughThreads);
    return;
  }
  const int lo = p.sinks, hi = n - p.recent;
  const int64_t pair = x.seq * p.hkv + x.kvh;
  const float2 *rough = reinterpret_cast<const float2 *>(p.keys) + pair * p.keys_st;
  float off = 0.f;
  int64_t ids[4 * kRoughHeld];
  auto load = [&](auto &held, auto place) __attribute__((always_inline)) {
    constexpr int kMany = sizeof(held) / sizeof(held[0]);
    float4 a[kMany], b[kMany];
#pragma unroll
    for (int j = 0; j < kMany; ++j) {
      const int at = min(place(j), n - 1) & ~3;
      a[j] = *reinterpret_cast<const float4 *>(rough + at);
      b[j] = *reinterpret_cast<const float4 *>(rough + at + 2);
#pragma unroll
      for (int e = 0; e < 4; ++e) ids[4 * j + e] = x.table[min(at + e, n - 1)];
    }
#pragma unroll
    for (int j = 0; j < kMany; ++j) {
      const int at = min(place(j), n - 1) & ~3;
      const float v[4] = {a[j].x, a[j].z, b[j].x, b[j].z};
      const float r[4] = {a[j].y, a[j].w, b[j].y, b[j].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        held[j][e] = order_key(v[e]);
        if (at + e >= lo && at + e < hi) off = fmaxf(off, r[e]);
      }
    }
  };
  Places<uint32_t, kRoughThreads, kRoughHeld, decltype(load)> places(n, lo, hi, load);
  off = wave_max(off);
  if (lane == 0) s_off[wave] = off;
  uint32_t last_key = 0;
  int last_place = 0;
  find_last<uint32_t, kRoughThreads>(s, places, left, last_key, last_place);
#pragma unroll
  for (int w = 0; w < kWaves; ++w) off = fmaxf(off, s_off[w]);
  // That key may be below the last chosen one's, with none between: the window is as well
  // around any score from there on.
  const float last = __uint_as_float(last_key >> 31 ? last_key & 0x7fffffffu : ~last_key);
  const float reach = 2.02f * off + 4e-7f * fabsf(last);
  const bool bound = off < INFINITY;
  const uint32_t from = bound ? order_key(last - reach) : 1u;
  // Room for kFew numbers in between.
  const uint32_t to = bound ? max(order_key(last + reach), from + kFew) : ~0u;
  int sure = 0, open = 0;
  places.each([&](int, const uint32_t(&k)[4]) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      sure += __popcll(__ballot(k[e] > to));
      open += __popcll(__ballot(k[e] >= from && k[e] <= to));
    }
  });
  if (lane == 0) {
    s_sure[wave] = sure;
    s_open[wave] = open;
  }
  if (threadIdx.x == 0) s.count = 0;
  __syncthreads();
  sure = open = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    sure += s_sure[w];
    open += s_open[w];
  }
  const int need = left - sure;
  if (open > kFew) {  // uniform
    uint64_t *keys = p.exact + pair * p.keys_st;
    for (int at = 16 * wave; at < n; at += 16 * kWaves) {
      const int j = at + x.col;
      const double best = x.score(j < n ? x.table[j] : -1);
      if (x.g == 0 && j < n) keys[j] = order_key(best);
    }
    __threadfence_block();
    __syncthreads();
    const int count = select_places<uint64_t, kRoughThreads, 1>(s, n, p.sinks, p.recent, p.budget,
                                                                keys_from(keys, n), out);
    out.finish(p, x.seq, x.kvh, count, kRoughThreads);
    return;
  }
  const bool few = open > need;
  if (few) {
    // The open ones in a list; a key of theirs becomes from + its place in it.
#pragma unroll
    for (int j = 0; j < kRoughHeld; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = places.first + 256 * j + e;
        uint32_t &k = places.keys[j][e];
        if (j < places.steps && k >= from && k <= to) {
          const int at = atomicAdd(&s.count, 1);
          s.few_place[at] = i;
          s_id[at] = ids[4 * j + e];
          k = from + at;
        }
      }
    __syncthreads();
    if (16 * wave < open) {
      const int at = 16 * wave + x.col;
      const double best = x.score(at < open ? s_id[min(at, open - 1)] : -1);
      if (x.g == 0 && at < open) s.few_key[at] = order_key(best);
    }
    __syncthreads();
    if (wave == 0) {
      const int at = min(lane, open - 1);
      const int better = rank_few(s.few_key[at], s.few_place[at], open);
      if (lane < open) s_taken[lane] = better < need;
    }
    __syncthreads();
  }
  emit_places<uint32_t, kRoughThreads, kRoughHeld>(
      s, places,
      [&](int i, uint32_t k) __attribute__((always_inline)) {
        if (k > to || places.forced(i)) return true;
        return k >= from && (!few || s_taken[k - from] != 0);
      },
      [&](int r, int i, int at) __attribute__((always_inline)) {
        out.put(r, i, at < 0 ? out.row[i] : ids[at]);
      });
  out.finish(p, x.seq, x.kvh, p.budget, kRoughThreads);
}

template <typename T>
int launch_choice(const SparseParams &p, bool rough, hipStream_t stream) {
  const int64_t pairs = p.hkv * p.seqs;
  const unsigned lists = static_cast<unsigned>(pairs);
  const int64_t pieces = ceil_div(p.d * static_cast<int64_t>(sizeof(T)), 16);
#define MLR_BY_PIECES(LAUNCH)                   \
  if (pieces <= 4) LAUNCH(1);                   \
  else if (pieces <= 8) LAUNCH(2);              \
  else if (sizeof(T) == 2 || pieces <= 16) LAUNCH(4); \
  else LAUNCH((sizeof(T) == 4 ? 8 : 4))
  if (p.bt_width <= kSmall) {
#define MLR_SMALL(N) choose_small<T, N><<<lists, kSmallThreads, 0, stream>>>(p)
    MLR_BY_PIECES(MLR_SMALL);
#undef MLR_SMALL
    return check_launch("choose_small");
  }
  if (rough) {
    if constexpr (sizeof(T) == 2) {
      // Tiles of a wave: q is read once for all of them, but two waves for every SIMD come
      // first (us by 1, 2, 4 and as many as that: 128 lists of 512 blocks of 64 elements 9.0,
      // -, 10.8 and 8.6; 64 of 4,096 of 128 58, -, 45 and 43).
      const int64_t cus = current_device_cus() > 0 ? current_device_cus() : 256;
      const int tiles = static_cast<int>(
          std::max<int64_t>(1, std::min<int64_t>(8, ceil_div(p.bt_width, 64) * pairs / (2 * cus))));
      const unsigned grid = static_cast<unsigned>(ceil_div(p.bt_width, 64 * tiles) * pairs);
#define MLR_ROUGH(N)                                             \
  {                                                              \
    score_rough<T, N><<<grid, 256, 0, stream>>>(p, tiles);       \
    choose_rough<T, N><<<lists, kRoughThreads, 0, stream>>>(p);  \
  }
      if (pieces <= 4) MLR_ROUGH(1) else if (pieces <= 8) MLR_ROUGH(2) else MLR_ROUGH(4)
#undef MLR_ROUGH
    }
    return check_launch("choose_rough");
  }
  if (p.bt_width > p.budget) {  // something to choose
    const unsigned grid = static_cast<unsigned>(ceil_div(p.bt_width, 64) * pairs);
#define MLR_SCORE(N) score_blocks<T, N><<<grid, 256, 0, stream>>>(p)
    MLR_BY_PIECES(MLR_SCORE);
#undef MLR_SCORE
  }
#undef MLR_BY_PIECES
  // As many waves as hold the keys in registers: fewer meet sooner (us of 256 and 1,024
  // threads: 16 lists of 512 blocks 6.6 and 11.3).
  if (p.bt_width <= 1024) choose_blocks<256, 1><<<lists, 256, 0, stream>>>(p);
  else choose_blocks<1024, 2><<<lists, 1024, 0, stream>>>(p);
  return check_launch("choose_blocks");
}

int64_t whole_fours(int64_t n) { return (n + 3) & ~int64_t(3); }

struct Layout {
  size_t keys, exact, table, lens, decode;
  size_t total() const { return keys + exact + table + lens + decode; }
};
Layout layout_of(int64_t batch, int64_t hq, int64_t hkv, int64_t d, int64_t width,
                 int64_t block_size, int64_t budget, int dtype) {
  const int64_t list = std::min(budget, width);
  const bool rough = takes_rough(batch * hkv, hq / hkv, d, width, budget, dtype);
  const size_t keys =
      width > kSmall ? align256(batch * hkv * whole_fours(width) * sizeof(uint64_t)) : 0;
  return Layout{keys, rough ? keys : 0,
                align256(batch * hkv * list * sizeof(int64_t)), align256(batch * sizeof(int64_t)),
                short_keys(list * block_size, d, dtype)
                    ? 0
                    : decode_workspace(batch, hq, hkv, d, list * block_size)};
}

}  // namespace
}  // namespace mlr

using namespace mlr;

extern "C" int mlr_update_key_bounds(const void *k_cache, void *key_bounds, int64_t num_blocks,
                                     int64_t block_size, int64_t num_kv_heads, int64_t head_dim,
                                     const int64_t *block_tables, int64_t bt_stride,
                                     int64_t max_blocks, const int64_t *seq_lens,
                                     const int64_t *starts, int64_t max_new, int64_t batch,
                                     int dtype, void *stream) {
  clear_error();
  const char *w = "mlr_update_key_bounds";
  MLR_REQUIRE(dtype == MLR_DTYPE_F32 || dtype == MLR_DTYPE_F16 || dtype == MLR_DTYPE_BF16,
              "%s: unsupported dtype %d", w, dtype);
  MLR_REQUIRE(batch >= 0 && batch < (1 << 24), "%s: number of sequences must be in [0, 2^24)", w);
  MLR_REQUIRE(num_kv_heads > 0 && num_kv_heads < (1 << 16) && head_dim > 0 && head_dim <= 1024 &&
                  head_dim * dtype_size(dtype) % 16 == 0,
              "%s: rows must be multiples of 16 bytes, of at most 1024 elements", w);
  MLR_REQUIRE(num_blocks > 0 && num_blocks < (int64_t(1) << 31) && block_size > 0 &&
                  max_blocks >= 0 && max_blocks < (int64_t(1) << 31) / block_size,
              "%s: a block table must cover fewer than 2^31 positions", w);
  MLR_REQUIRE(max_new >= 0, "%s: max_new must be >= 0", w);
  if (batch == 0 || max_blocks == 0 || (starts && max_new == 0)) return MLR_OK;
  MLR_REQUIRE(k_cache && key_bounds && block_tables && seq_lens, "%s: null pointer", w);
  MLR_REQUIRE((reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(key_bounds)) %
                      16 == 0, "%s: operands must be 16-byte aligned", w);
  // `max_new` positions touch one block more than they fill.
  const int64_t most =
      starts ? std::min(max_blocks, ceil_div(std::min(max_new, max_blocks * block_size) - 1,
                                             block_size) + 1)
             : max_blocks;
  const BoundParams p{k_cache, key_bounds, num_blocks, block_size, num_kv_heads, head_dim,
                      block_tables, bt_stride, max_blocks, seq_lens, starts, batch, most};
  const int64_t threads = batch * most * num_kv_heads * head_dim * dtype_size(dtype) / 16;
  const unsigned grid =
      static_cast<unsigned>(std::min<int64_t>(ceil_div(threads, 256), int64_t(1) << 20));
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == MLR_DTYPE_F32) bound_keys<float><<<grid, 256, 0, s>>>(p);
  else if (dtype == MLR_DTYPE_F16) bound_keys<f16_t><<<grid, 256, 0, s>>>(p);
  else bound_keys<bf16_t><<<grid, 256, 0, s>>>(p);
  return check_launch("bound_keys");
}

extern "C" size_t mlr_paged_decode_sparse_workspace_size(int64_t batch, int64_t num_q_heads,
                                                         int64_t num_kv_heads, int64_t head_dim,
                                                         int64_t max_blocks, int64_t block_size,
                                                         int64_t budget, int dtype) {
  if (batch <= 0 || num_kv_heads <= 0 || num_q_heads <= 0 || max_blocks <= 0 || block_size <= 0 ||
      budget <= 0)
    return 0;
  return layout_of(batch, num_q_heads, num_kv_heads, head_dim, max_blocks, block_size, budget, dtype)
      .total();
}

extern "C" int mlr_paged_decode_sparse(
    const void *q, int64_t q_stride_b, int64_t q_stride_h, const void *k_cache,
    const void *v_cache, const void *key_bounds, int64_t num_blocks, int64_t block_size,
    int64_t num_kv_heads, int64_t head_dim, const int64_t *block_tables, int64_t bt_stride,
    int64_t max_blocks, const int64_t *seq_lens, int64_t batch, int64_t num_q_heads,
    int64_t budget, int64_t sinks, int64_t recent, double scale, double softcap, int dtype,
    int64_t *chosen, void *workspace, size_t workspace_bytes, void *out, int64_t out_stride_b,
    int64_t out_stride_h, void *stream) {
  clear_error();
  Operands o{"mlr_paged_decode_sparse", q, q_stride_b, q_stride_h, k_cache, v_cache,
             num_blocks, block_size, num_kv_heads, head_dim, block_tables, bt_stride,
             max_blocks, seq_lens, batch, num_q_heads, scale, softcap, nullptr, dtype,
             out, out_stride_b, out_stride_h};
  if (const int rc = check_operands(o)) return rc;
  MLR_REQUIRE(sinks >= 0 && recent >= 1 && budget < (int64_t(1) << 31) && recent <= budget &&
                  sinks <= budget - recent,
              "%s: budget must cover sinks and recent, which is at least 1", o.what);
  if (batch == 0) return MLR_OK;
  const int64_t group = num_q_heads / num_kv_heads;
  MLR_REQUIRE(batch * num_q_heads < (int64_t(1) << 28), "%s: too many query rows", o.what);
  MLR_REQUIRE(q && k_cache && v_cache && key_bounds && (block_tables || max_blocks == 0) &&
                  seq_lens && out, "%s: null pointer", o.what);
  MLR_REQUIRE(reinterpret_cast<uintptr_t>(key_bounds) % 16 == 0,
              "%s: bounds must be 16-byte aligned", o.what);
  MLR_REQUIRE(ceil_div(max_blocks, 64) * num_kv_heads * batch < (int64_t(1) << 31),
              "%s: too many blocks", o.what);
  const size_t need = mlr_paged_decode_sparse_workspace_size(
      batch, num_q_heads, num_kv_heads, head_dim, max_blocks, block_size, budget, dtype);
  MLR_REQUIRE(need == 0 || (workspace && workspace_bytes >= need),
              "%s: workspace of %zu bytes, %zu needed", o.what, workspace_bytes, need);
  hipStream_t s = static_cast<hipStream_t>(stream);
  char *ws = static_cast<char *>(workspace);
  const int64_t list = std::min(budget, max_blocks);
  SparseParams x{q, key_bounds, q_stride_b, q_stride_h, num_blocks, block_size, num_kv_heads,
                 group, head_dim, block_tables, bt_stride, max_blocks, seq_lens, batch, scale < 0,
                 static_cast<int>(sinks), static_cast<int>(recent), static_cast<int>(budget),
                 static_cast<int>(list), nullptr, nullptr, whole_fours(max_blocks), nullptr, nullptr,
                 chosen};
  int64_t max_keys = 0;
  if (need) {
    const Layout l = layout_of(batch, num_q_heads, num_kv_heads, head_dim, max_blocks, block_size,
                               budget, dtype);
    x.keys = reinterpret_cast<uint64_t *>(ws);
    x.exact = reinterpret_cast<uint64_t *>(ws += l.keys);
    x.table = reinterpret_cast<int64_t *>(ws += l.exact);
    x.lens = reinterpret_cast<int64_t *>(ws += l.table);
    ws += l.lens;
    max_keys = list * block_size;
    o.bt = x.table;
    o.bt_st = num_kv_heads * list;
    o.bt_width = list;
    o.ctx = x.lens;
  }
  const bool rough = need && takes_rough(batch * num_kv_heads, group, head_dim, max_blocks, budget,
                                         dtype);
  int rc = MLR_OK;
  if (dtype == MLR_DTYPE_F32) rc = launch_choice<float>(x, rough, s);
  else if (dtype == MLR_DTYPE_F16) rc = launch_choice<f16_t>(x, rough, s);
  else rc = launch_choice<bf16_t>(x, rough, s);
  if (rc) return rc;
  ScoredParams p = params_of(o, kModeDecode);
  p.bt_sh = need ? list : 0;
  p.fine = true;
  p.whole = short_keys(max_keys, head_dim, dtype);
  const bool parts = !p.whole;
  const int64_t items = plan_decode(p, max_keys, parts ? ws : nullptr);
  rc = launch_scored_rows(p, dtype, grid_of(items), s);
  if (rc) return rc;
  return parts ? merge_decode(p, dtype, s) : MLR_OK;
}

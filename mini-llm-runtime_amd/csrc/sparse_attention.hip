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

// Thread: 16 bytes of a row of one changed block and KV head.
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
  uint64_t *keys;                   // [seqs, hkv, keys_st] scores as ordered keys
  int64_t keys_st;                  // bt_width, in whole fours
  int64_t *table;                   // [seqs, hkv, list] physical blocks of the chosen
  int64_t *lens;                    // [seqs] keys of the chosen blocks
  int64_t *chosen;                  // [seqs, hkv, budget] their places, may be null
};

typedef double f64x4_t __attribute__((ext_vector_type(4)));

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

// Scores on v_mfma_f64_16x16x4: sum_d max(q low, q high) = [q-, q+].[low, high] with q- =
// min(q, 0) and q+ = max(q, 0), 16 heads times 16 blocks. Operand A is q (lane l: head
// l % 16), B the bounds (lane l: block l % 16); of a row lane group l / 16 has every
// fourth piece of 16 bytes, so that its k-th elements are those of A and B alike. A
// group of fewer heads repeats its last one, and the maximum over heads needs no mask.
// Where a bound or q is not finite, 0 times it would be NaN where the larger of both
// products is not: such tiles are added up product by product.
//
// Bound by the matrix unit where the heads of a group are many, by the reads of the bounds
// where they are few: 8 requests of 2,048 blocks, 28/4 heads of 128, bf16, 33 MB in 26 us.
template <typename T, int kT>
__global__ __launch_bounds__(256) void score_blocks(SparseParams p, int tiles) {
  constexpr int kE = 16 / sizeof(T);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, g = lane >> 4;
  const int64_t b = blockIdx.x;
  const int64_t seq = b % p.seqs, kvh = b / p.seqs % p.hkv;
  // A wave's tiles of 16 blocks: the workgroup's in turn.
  const int64_t first = (b / p.seqs / p.hkv * 4 * tiles + wave) * 16;
  const int64_t ctx = clamp64(p.ctx[seq], 0, p.bt_width * p.block_size);
  const int64_t n = (ctx + p.block_size - 1) / p.block_size;
  if (first >= n || n <= p.budget) return;  // nothing there, or nothing to choose
  const int64_t *table = p.bt + seq * p.bt_st;
  const T *bounds = static_cast<const T *>(p.bounds) + kvh * p.d;
  const int64_t row = p.hkv * p.d;
  const T *q = static_cast<const T *>(p.q) + seq * p.q_st + kvh * p.group * p.q_sh;
  auto id_of = [&](int i) __attribute__((always_inline)) {
    return table[min(first + 64 * i + col, n - 1)];
  };
  struct Tile {
    uint4 low[kT], high[kT];
    bool there;
  };
  auto read = [&](Tile &x, int i, int64_t id) __attribute__((always_inline)) {
    x.there = first + 64 * i + col < n && id >= 0 && id < p.num_blocks;
    const T *at = bounds + (x.there ? id : 0) * 2 * row;
#pragma unroll
    for (int t = 0; t < kT; ++t) {
      const int e = (g + 4 * t) * kE;
      x.low[t] = x.high[t] = make_uint4(0, 0, 0, 0);
      if (e < p.d && x.there) {
        x.low[t] = *reinterpret_cast<const uint4 *>(at + e);
        x.high[t] = *reinterpret_cast<const uint4 *>(at + row + e);
      }
    }
  };
  const int heads = static_cast<int>(p.group);
  const bool many = heads > 16;
  // q of heads h0 ..: its negative and its positive part, in 64 bits.
  double below[kT][kE], above[kT][kE];
  bool q_odd = false;
  auto read_q = [&](int h0) __attribute__((always_inline)) {
    const T *mine = q + min(h0 + col, heads - 1) * p.q_sh;
    q_odd = false;
#pragma unroll
    for (int t = 0; t < kT; ++t) {
      const int e0 = (g + 4 * t) * kE;
      uint4 x = make_uint4(0, 0, 0, 0);
      if (e0 < p.d) x = *reinterpret_cast<const uint4 *>(mine + e0);
      q_odd = q_odd || odd<T>(x);
      float f[kE];
      unpack<T>(x, f);
#pragma unroll
      for (int e = 0; e < kE; ++e) {
        const float v = p.flip ? -f[e] : f[e];
        below[t][e] = fminf(v, 0.f);
        above[t][e] = fmaxf(v, 0.f);
      }
    }
  };
  auto score = [&](const Tile &x, int i) __attribute__((always_inline)) {
    bool bound_odd = false;
#pragma unroll
    for (int t = 0; t < kT; ++t)
      bound_odd = bound_odd || odd<T>(x.low[t]) || odd<T>(x.high[t]);
    double best = -INFINITY;
    for (int h0 = 0; h0 < heads; h0 += 16) {
      if (many) read_q(h0);
      if (__builtin_expect(!__any(bound_odd || q_odd), 1)) {
        f64x4_t sum0 = {0., 0., 0., 0.}, sum1 = {0., 0., 0., 0.};
#pragma unroll
        for (int t = 0; t < kT; ++t) {
          float l[kE], u[kE];
          unpack<T>(x.low[t], l);
          unpack<T>(x.high[t], u);
#pragma unroll
          for (int e = 0; e < kE; ++e) {
            sum0 = __builtin_amdgcn_mfma_f64_16x16x4f64(below[t][e], l[e], sum0, 0, 0, 0);
            sum1 = __builtin_amdgcn_mfma_f64_16x16x4f64(above[t][e], u[e], sum1, 0, 0, 0);
          }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) best = fmax(best, sum0[r] + sum1[r]);
      } else {
        for (int h = h0; h < min(h0 + 16, heads); ++h) {
          double sum = 0.;
#pragma unroll
          for (int t = 0; t < kT; ++t) {
            float l[kE], u[kE];
            unpack<T>(x.low[t], l);
            unpack<T>(x.high[t], u);
#pragma unroll
            for (int e = 0; e < kE; ++e) {
              const int at = (g + 4 * t) * kE + e;
              if (at >= p.d) continue;
              const float f = Elem<T>::to_f32(q[h * p.q_sh + at]);
              const double v = p.flip ? -f : f;
              sum = fma(v, v >= 0. ? u[e] : l[e], sum);
            }
          }
          sum += __shfl_xor(sum, 16);
          sum += __shfl_xor(sum, 32);
          best = sum > best ? sum : best;  // a sum that is NaN does not count
        }
      }
    }
    best = fmax(best, __shfl_xor(best, 16));
    best = fmax(best, __shfl_xor(best, 32));
    const int64_t j = first + 64 * i + col;
    if (g == 0 && j < n)
      p.keys[(seq * p.hkv + kvh) * p.keys_st + j] = order_key(x.there ? best : -INFINITY);
  };
  Tile even, other;
  const int count = static_cast<int>(min(int64_t(tiles), (n - first + 63) / 64));
  read(even, 0, id_of(0));
  int64_t id = id_of(1);
  if (!many) read_q(0);
  for (int i = 0; i < count; i += 2) {
    if (i + 1 < count) read(other, i + 1, id);
    id = id_of(i + 2);
    score(even, i);
    if (i + 1 >= count) break;
    if (i + 2 < count) read(even, i + 2, id);
    id = id_of(i + 3);
    score(other, i + 1);
  }
}

// A workgroup chooses the blocks of one request and KV head.
template <int kThreads, int kHeld>
__global__ __launch_bounds__(kThreads) void choose_blocks(SparseParams p) {
  __shared__ SelectShared s;
  const int64_t seq = blockIdx.x % p.seqs, kvh = blockIdx.x / p.seqs;
  const int64_t pair = seq * p.hkv + kvh;
  const int64_t ctx = clamp64(p.ctx[seq], 0, p.bt_width * p.block_size);
  const int n = static_cast<int>((ctx + p.block_size - 1) / p.block_size);
  const uint64_t *keys = p.keys + pair * p.keys_st;
  const int64_t *row = p.bt + seq * p.bt_st;
  int64_t *table = p.table + pair * p.list;
  int64_t *chosen = p.chosen ? p.chosen + pair * p.budget : nullptr;
  const int count = select_places<uint64_t, kThreads, kHeld>(
      s, n, p.sinks, p.recent, p.budget,
      [&](auto &held, auto place) __attribute__((always_inline)) {
        constexpr int kMany = sizeof(held) / sizeof(held[0]);
#pragma unroll
        for (int j = 0; j < kMany; ++j) {
          const ulonglong2 *at =
              reinterpret_cast<const ulonglong2 *>(keys + (min(place(j), n - 1) & ~3));
          const ulonglong2 a = at[0], b = at[1];
          held[j][0] = a.x;
          held[j][1] = a.y;
          held[j][2] = b.x;
          held[j][3] = b.y;
        }
      },
      [&](int r, int i) __attribute__((always_inline)) {
        table[r] = row[i];
        if (chosen) chosen[r] = i;
      });
  if (chosen)
    for (int i = count + threadIdx.x; i < p.budget; i += kThreads) chosen[i] = -1;
  // The last block is always chosen, and the only one that may not be full.
  if (p.lens && kvh == 0 && threadIdx.x == 0)
    p.lens[seq] = count > 0 ? ctx - static_cast<int64_t>(n - count) * p.block_size : 0;
}

template <typename T>
int launch_scores(const SparseParams &p, hipStream_t stream) {
  // Tiles of a wave: q is converted once for all of them, but a wave for every SIMD comes
  // first.
  const int64_t all = ceil_div(p.bt_width, 64) * p.hkv * p.seqs;  // of four waves
  const int64_t cus = current_device_cus() > 0 ? current_device_cus() : 256;
  const int tiles = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(8, all / cus)));
  const unsigned grid =
      static_cast<unsigned>(ceil_div(p.bt_width, 64 * tiles) * p.hkv * p.seqs);
  const int64_t pieces = ceil_div(p.d * static_cast<int64_t>(sizeof(T)), 16);
  if (pieces <= 4) score_blocks<T, 1><<<grid, 256, 0, stream>>>(p, tiles);
  else if (pieces <= 8) score_blocks<T, 2><<<grid, 256, 0, stream>>>(p, tiles);
  else if (pieces <= 16) score_blocks<T, 4><<<grid, 256, 0, stream>>>(p, tiles);
  else score_blocks<T, 8><<<grid, 256, 0, stream>>>(p, tiles);
  return check_launch("score_blocks");
}

int64_t whole_fours(int64_t n) { return (n + 3) & ~int64_t(3); }

struct Layout {
  size_t keys, table, lens, decode;
  size_t total() const { return keys + table + lens + decode; }
};
Layout layout_of(int64_t batch, int64_t hq, int64_t hkv, int64_t d, int64_t width,
                 int64_t block_size, int64_t budget, int dtype) {
  const int64_t list = std::min(budget, width);
  return Layout{align256(batch * hkv * whole_fours(width) * sizeof(uint64_t)),
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
  if (batch == 0 || max_blocks == 0 || max_new == 0) return MLR_OK;
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
                 static_cast<int>(list), nullptr, whole_fours(max_blocks), nullptr, nullptr, chosen};
  int64_t max_keys = 0;
  if (need) {
    const Layout l = layout_of(batch, num_q_heads, num_kv_heads, head_dim, max_blocks, block_size,
                               budget, dtype);
    x.keys = reinterpret_cast<uint64_t *>(ws);
    x.table = reinterpret_cast<int64_t *>(ws += l.keys);
    x.lens = reinterpret_cast<int64_t *>(ws += l.table);
    ws += l.lens;
    int rc = MLR_OK;
    if (max_blocks > budget) {
      if (dtype == MLR_DTYPE_F32) rc = launch_scores<float>(x, s);
      else if (dtype == MLR_DTYPE_F16) rc = launch_scores<f16_t>(x, s);
      else rc = launch_scores<bf16_t>(x, s);
      if (rc) return rc;
    }
    max_keys = list * block_size;
    o.bt = x.table;
    o.bt_st = num_kv_heads * list;
    o.bt_width = list;
    o.ctx = x.lens;
  }
  if (need || chosen) {
    const unsigned lists = static_cast<unsigned>(batch * num_kv_heads);
    if (max_blocks <= 1024) choose_blocks<256, 1><<<lists, 256, 0, s>>>(x);
    else choose_blocks<1024, 2><<<lists, 1024, 0, s>>>(x);
    if (const int rc = check_launch("choose_blocks")) return rc;
  }
  ScoredParams p = params_of(o, kModeDecode);
  p.bt_sh = need ? list : 0;
  p.whole = short_keys(max_keys, head_dim, dtype);
  const bool parts = !p.whole;
  const int64_t items = plan_decode(p, max_keys, parts ? ws : nullptr);
  if (const int rc = launch_scored_rows(p, dtype, grid_of(items), s)) return rc;
  return parts ? merge_decode(p, dtype, s) : MLR_OK;
}

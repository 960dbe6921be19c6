// Paged attention with capped or biased scores, for few query rows per key: single
// tokens, short chunks and small trees of drafted tokens, and everything in FP32 or with a
// block_size that is no power of two from 16 on.
//
//   x_ij = scale q_i.k_j;  cap: x = cap tanh(x / cap);  x -= slope_h |i - j|
//   j visible iff lo <= j < limit_i;  out_i = softmax_j(x_ij) v_j
//
// A unit is 16 query rows (all heads of a KV group of one token; in FP32 also
// rows of several tokens). Four waves share a split of its keys, 16-key tiles
// dealt in turn. Per tile and wave, on matrix cores:
//   S^T[16 keys x 16 rows] = K Q^T, K rows straight from memory as operand A
//     (lane l: key l % 16), Q^T in registers. Lane l then holds row l % 16 and
//     keys 4 (l / 16) + i, i < 4.
//   running maximum and sum of each row (FP32, one pass over the keys)
//   O^T[D x 16 rows] += V^T P^T with P^T straight from the S^T registers: the
//     k index of operand B is the key 4 (l / 16) + i. V as operand A: a lane
//     holds D / 16 neighbouring elements of rows 4 (l / 16) + i.
// In 16-bit types P is an operand of their type. Chunks, plain decodes and shared prefixes
// round it (by at most 2^-8 of it in bf16, 2^-11 in fp16), at every head size, which makes
// the error against 64 bits 1.4 times that of the one rounding of the result (bf16 0.0023
// and 0.0017 of the outputs' size). Drafted trees, weighing and sparse decodes hold it in
// two parts (two_parts below), to 2^-15 and 2^-21 of it: the instruction with twice as many
// keys takes both in the time of one. Scores, statistics and sums are FP32, and the result
// is rounded once.
// Drafted tokens see the keys before them and those that their bits name; a decode
// that weighs its keys leaves the scores in the workspace (64 requests as below: 22 us).
// The waves' results are joined through LDS. Splits of one unit leave (m, l, O)
// in the workspace, added up by scored_merge in the next launch.
//
// Bound by memory: a unit's K and V rows are read once for all of its rows (64
// requests of 128 to 4,096 keys, 14/2 heads of 64, bf16: 70.7 MB in 24.3 us with the
// merge's launch, 2.9 TB/s).
#include "scored_attention.h"

namespace mlr {
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4_t __attribute__((ext_vector_type(4)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

constexpr int kWavesWg = 4;
constexpr float kLog2e = 1.4426950408889634f;

template <typename T> struct Mma16;
template <> struct Mma16<bf16_t> {
  using v8 = bf16x8_t;
  __device__ static f32x4_t qk(uint4 k, uint4 q, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8, k),
                                                   __builtin_bit_cast(v8, q), c, 0, 0, 0);
  }
  __device__ static f32x4_t pv(uint2 v, uint2 p, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4_t, v),
                                                     __builtin_bit_cast(s16x4_t, p), c, 0, 0, 0);
  }
  __device__ static f32x4_t pv2(uint2 v, uint4 p, f32x4_t c) {
    return qk(make_uint4(v.x, v.y, v.x, v.y), p, c);
  }
};
template <> struct Mma16<f16_t> {
  using v8 = f16x8_t;
  __device__ static f32x4_t qk(uint4 k, uint4 q, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8, k),
                                                  __builtin_bit_cast(v8, q), c, 0, 0, 0);
  }
  __device__ static f32x4_t pv(uint2 v, uint2 p, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4_t, v),
                                                 __builtin_bit_cast(f16x4_t, p), c, 0, 0, 0);
  }
  __device__ static f32x4_t pv2(uint2 v, uint4 p, f32x4_t c) {
    return qk(make_uint4(v.x, v.y, v.x, v.y), p, c);
  }
};

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  typedef float f32x2_v __attribute__((ext_vector_type(2)));
  using H = std::conditional_t<std::is_same_v<T, bf16_t>, __bf16, _Float16>;
  typedef H h2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_v{a, b}, h2));
}

__device__ __forceinline__ float max_groups(float x) {  // over lanes l ^ 16, l ^ 32
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_groups(float x) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// One loaded tile: K as kK 16-byte chunks of key l % 16 (elements 64 / size *
// j + 16 / size * (l / 16)), V as D / 16 elements of keys 4 (l / 16) + i.
template <typename T, int D>
struct Tile {
  static constexpr int kK = D * sizeof(T) / 64;
  static constexpr int kV = D * sizeof(T) / 64;  // 32-bit words of a V row piece
  uint4 k[kK];
  uint32_t v[4][kV];
};

template <typename T, int D>
__device__ __forceinline__ void load_piece(uint32_t *dst, const T *src, int dim, int d) {
  constexpr int kV = Tile<T, D>::kV;
  if constexpr (kV == 2) {
    uint2 w = make_uint2(0, 0);
    if (dim < d) w = *reinterpret_cast<const uint2 *>(src);
    dst[0] = w.x;
    dst[1] = w.y;
  } else {
    constexpr int kPer = 16 / sizeof(T);
#pragma unroll
    for (int c = 0; c < kV / 4; ++c) {
      uint4 w = make_uint4(0, 0, 0, 0);
      if (dim + c * kPer < d) w = *reinterpret_cast<const uint4 *>(src + c * kPer);
      dst[4 * c] = w.x;
      dst[4 * c + 1] = w.y;
      dst[4 * c + 2] = w.z;
      dst[4 * c + 3] = w.w;
    }
  }
}

// The K and V rows of a tile. kPaged16: block_size is a multiple of 16, so a
// tile lies in one block.
template <typename T, int D, bool kPaged16>
struct Rows {
  const ScoredParams &p;
  const T *k, *v;
  const int64_t *table;
  int covered, bs;  // positions of the table, below 2^31; block_size, if it is less
  int m16, g, kvh;

  __device__ __forceinline__ int64_t slot_of(int key, bool &ok) const {
    ok = key < covered;
    const int at = !ok ? 0 : p.bs_log2 >= 0 ? key >> p.bs_log2 : key / bs;
    const int64_t blk = table[at];
    ok = ok && blk >= 0 && blk < p.num_blocks;
    return ok ? blk * p.block_size + (key - at * bs) : 0;
  }

  // The tile of keys [key0, key0 + 16), key0 a multiple of 16; only keys in
  // [lo, end) count. Absent K rows are read from slot 0 (their scores are
  // masked), absent V rows are zeros. Returns, as bit i, whether the lane's key
  // 4 g + i exists.
  __device__ __forceinline__ uint32_t load(Tile<T, D> &t, int key0, int lo, int end) const {
    int64_t ks, vs[4];
    bool kok, vok[4];
    if constexpr (kPaged16) {
      bool ok;
      const int64_t s = slot_of(key0, ok);
      kok = ok;
      ks = ok ? s + m16 : 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        vok[i] = ok && key0 + 4 * g + i >= lo && key0 + 4 * g + i < end;
        vs[i] = s + 4 * g + i;
      }
    } else {
      ks = slot_of(min(key0 + m16, end - 1), kok);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = key0 + 4 * g + i;
        vs[i] = slot_of(min(key, end - 1), vok[i]);
        vok[i] = vok[i] && key >= lo && key < end;
      }
    }
    constexpr int kE = 16 / sizeof(T);
    const T *kr = k + (ks * p.hkv + kvh) * p.d;
#pragma unroll
    for (int j = 0; j < Tile<T, D>::kK; ++j) {
      const int dim = 4 * kE * j + kE * g;
      t.k[j] = make_uint4(0, 0, 0, 0);
      if (D == p.d || dim < p.d) t.k[j] = *reinterpret_cast<const uint4 *>(kr + dim);
    }
    uint32_t bits = 0;
    constexpr int kVe = D / 16;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int dim = kVe * m16;
      load_piece<T, D>(t.v[i], v + ((vok[i] ? vs[i] : 0) * p.hkv + kvh) * p.d + dim, dim,
                       vok[i] ? p.d : 0);
      bits |= static_cast<uint32_t>(vok[i]) << i;
    }
    return bits;
  }
};

// Caps four scores of a lane, in units of the natural exponent. In 16-bit types y P(y^2)
// near 0, which keeps scores that lie far below the cap, and from 1/2 on 1 - 2 /
// (exp(2 y) + 1), an absolute error of 4e-7. Either is within 9e-7 of the score,
// whatever the cap. The wave leaves out the second where no score needs it.
template <typename T>
__device__ __forceinline__ void cap_scores(float (&x)[4], float cap, float inv_cap) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = cap * tanhf(x[i] * inv_cap);
  } else {
    float y[4], t[4];
    bool near = true;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      y[i] = x[i] * inv_cap;
      near = near && fabsf(y[i]) <= 0.5f;
      const float u = y[i] * y[i];
      t[i] = y[i] * fmaf(u, fmaf(u, fmaf(u, kTanh3, kTanh2), kTanh1), kTanh0);
    }
    if (__any(!near)) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float e = __builtin_amdgcn_exp2f(y[i] * (2.f * kLog2e));
        const float far = 1.f - 2.f * __builtin_amdgcn_rcpf(e + 1.f);
        t[i] = fabsf(y[i]) <= 0.5f ? t[i] : far;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = cap * t[i];
  }
}

// kPrefill: the rows are tokens of chunks, not requests. kUnlike: rows of a unit may
// see different keys (chunks, and requests shorter than the prefix that they share).
// kTree: of its sequence's last tokens a row sees those that its bits name. kKeep: the
// scores stay for a pass that weighs the keys. kFine: probabilities in two parts, which
// these two always have. None of them must cost a D of 64 one of the three
// workgroups of a CU that rows_target counts on: with a few registers too many, 16 FP32
// trees of 3 to 5 tokens after 500 to 4,000 keys took 42 us, not 32.
template <typename T, int D, bool kCap, bool kPaged16, bool kPrefill, bool kUnlike, bool kTree,
          bool kKeep, bool kFine>
__global__ __launch_bounds__(256, kFine && D <= 64 ? 3 : 1) void scored_rows_kernel(
    ScoredParams p) {
  static_assert(kFine || !(kTree || kKeep), "these are in two parts");
  // What an fp16 probability, at most 1, is scaled by in two parts.
  constexpr float kUp = kFine && std::is_same_v<T, f16_t> ? 32768.f : 1.f;
  constexpr int kVe = D / 16;  // elements of a row that a lane of P V holds
  constexpr int kE = 16 / sizeof(T);
  constexpr int kBatch = D * sizeof(T) <= 128 ? 4 : D * sizeof(T) <= 256 ? 2 : 1;
  using M = Tile<T, D>;
  __shared__ float s_m[kWavesWg][kRows], s_l[kWavesWg][kRows];
  __shared__ __align__(16) float s_acc[kWavesWg][kRows][D + 4];
  __shared__ int64_t s_keys[kWavesWg];
  __shared__ int s_count[kWavesWg], s_unit, s_split, s_of;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m16 = lane & 15, g = lane >> 4;

  // The cut: all keys, hence the split length; this thread's units and the
  // items before them. -1: a unit without rows. Without splits an item is a unit; the
  // variants that are never left whole do not ask (a load of an argument before all others
  // and a branch, 0.7 us of a decode's 9 to 21).
  const bool whole = kFine && p.whole;
  const int per = (p.units + 255) / 256;
  const int u_lo = min(tid * per, p.units), u_hi = min(u_lo + per, p.units);
  auto len_of = [&](int u) -> int64_t {
    const Unit t = unit_of(p, u, kRows);
    return t.r0 < t.rows ? unit_len(t) : -1;
  };
  int64_t len0 = -1;  // of the first; mostly there is no other
  auto items_at = [&](int u, int split) {
    const int64_t len = u == u_lo ? len0 : len_of(u);
    return len < 0 ? 0 : items_of(len, split);
  };
  int split = 0, own = 0, before = 0, items = p.units;
  if (!whole) {
    if (u_lo < u_hi) len0 = len_of(u_lo);
    int64_t keys = max(len0, int64_t(0));
    for (int u = u_lo + 1; u < u_hi; ++u) keys += max(len_of(u), int64_t(0));
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) keys += __shfl_xor(keys, o);
    if (lane == 0) s_keys[wv] = keys;
    __syncthreads();
    split = split_of(s_keys[0] + s_keys[1] + s_keys[2] + s_keys[3], p);
    for (int u = u_lo; u < u_hi; ++u) own += items_at(u, split);
    before = own;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int x = __shfl_up(before, o);
      if (lane >= o) before += x;
    }
    if (lane == 63) s_count[wv] = before;
    before -= own;
    __syncthreads();
    items = 0;
    for (int i = 0; i < kWavesWg; ++i) {
      if (i < wv) before += s_count[i];
      items += s_count[i];
    }
    if (blockIdx.x == 0 && p.first) {
      int at = before;
      for (int u = u_lo; u < u_hi; ++u) {
        p.first[u] = at;
        at += items_at(u, split);
      }
      if (tid == 255) p.first[p.units] = items;
    }
  }

  const float inv_cap = kCap ? 1.f / p.cap : 0.f;
  for (int w = blockIdx.x; w < items * p.hkv; w += gridDim.x) {
    const int item = w / p.hkv, kvh = w - item * p.hkv;
    int unit = item, part = 0, parts = 1;
    if (!whole) {
      if (item >= before && item < before + own) {
        int at = before;
        for (int u = u_lo; u < u_hi; ++u) {
          const int n = items_at(u, split);
          if (item < at + n) {
            s_unit = u;
            s_split = item - at;
            s_of = n;
            break;
          }
          at += n;
        }
      }
      __syncthreads();
      unit = __builtin_amdgcn_readfirstlane(s_unit);
      part = __builtin_amdgcn_readfirstlane(s_split);
      parts = __builtin_amdgcn_readfirstlane(s_of);
    }
    const bool alone = parts == 1 && !p.force_partial;
    const Unit t = unit_of(p, unit, kRows);
    if (kFine && t.r0 >= t.rows) continue;  // uniform: without splits, a unit without rows
    const int len = item_len(t, parts, 16);
    // Keys are below 2^31.
    const int64_t from = unit_base(t) + static_cast<int64_t>(part) * len;
    const int k0 = __builtin_amdgcn_readfirstlane(static_cast<int>(min(from, int64_t(0x7fffff00))));
    const int k1 = __builtin_amdgcn_readfirstlane(static_cast<int>(min(t.hi, from + len)));
    const int lo = __builtin_amdgcn_readfirstlane(static_cast<int>(t.lo));

    // The lane's row: its query, its position and the keys that it sees.
    const int r = t.r0 + m16;
    const bool live = r < t.rows;
    const int tok = live ? r / p.group : 0;
    const int head = kvh * p.group + (live ? r - tok * p.group : 0);
    const int64_t row = t.q0 + tok;
    int pos = static_cast<int>(t.ctx) - 1, limit = static_cast<int>(t.hi);
    if (kPrefill) {
      pos = static_cast<int>(t.pos0) + tok;
      limit = max(pos + 1, static_cast<int>(t.ahead));
    } else if (t.prefix) {
      // A request shorter than the prefix sees its own first positions.
      pos = static_cast<int>(clamp64(p.ctx[row], 0, 0x7fffffff)) - 1;
      limit = min(limit, pos + 1);
    }
    // The first key that the row does not see (kTree: may not see).
    const int tree0 = static_cast<int>(t.pos0);
    const int own_end = !live ? 0x7fffffff : kTree ? tree0 : limit;
    if (!live) limit = 0;
    const float slope = p.slopes ? p.slopes[head] : 0.f;
    uint4 q[M::kK];
    const T *qr = static_cast<const T *>(p.q) + row * p.q_st + head * p.q_sh;
#pragma unroll
    for (int j = 0; j < M::kK; ++j) {
      const int dim = 4 * kE * j + kE * g;
      q[j] = make_uint4(0, 0, 0, 0);
      if (live && dim < p.d) q[j] = *reinterpret_cast<const uint4 *>(qr + dim);
    }

    Rows<T, D, kPaged16> src{p, static_cast<const T *>(p.k), static_cast<const T *>(p.v),
                             table_of(p, t) + (kFine ? kvh * p.bt_sh : 0),
                             static_cast<int>((t.prefix ? p.prefix_width : p.bt_width) *
                                              p.block_size),
                             static_cast<int>(min(p.block_size, int64_t(0x7fffffff))), m16, g, kvh};
    f32x4_t acc[kVe];
#pragma unroll
    for (int n = 0; n < kVe; ++n) acc[n] = f32x4_t{0, 0, 0, 0};
    float mx = -INFINITY, l = 0.f;  // l: of this lane's keys only

    M tile[kBatch];
    uint32_t ok[kBatch];
    constexpr int step = 16 * kWavesWg;
    for (int b0 = k0 + 16 * wv; b0 < k1; b0 += step * kBatch) {
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const int key0 = b0 + b * step;
        ok[b] = 0;
        if (key0 < k1) ok[b] = src.load(tile[b], key0, lo, k1);
      }
      // Scores of the batch and their maximum.
      float x[kBatch][4];
      float top = mx;
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const int key0 = b0 + b * step;
        if (key0 >= k1) {
#pragma unroll
          for (int i = 0; i < 4; ++i) x[b][i] = -INFINITY;
          continue;
        }
        f32x4_t s = {0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < M::kK; ++j) {
          if constexpr (sizeof(T) == 2) {
            s = Mma16<T>::qk(tile[b].k[j], q[j], s);
          } else {
            const f32x4_t a = __builtin_bit_cast(f32x4_t, tile[b].k[j]);
            const f32x4_t c = __builtin_bit_cast(f32x4_t, q[j]);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              s = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], c[e], s, 0, 0, 0);
          }
        }
        float y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = s[i] * p.scale;
        if constexpr (kCap) cap_scores<T>(y, p.cap, inv_cap);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = key0 + 4 * g + i;
          y[i] -= slope * static_cast<float>(abs(pos - key));
          bool seen = (ok[b] >> i & 1) && key >= lo && key < limit;
          if (kTree && seen && key >= tree0) seen = bit_of(p, row, key - tree0);
          x[b][i] = seen ? y[i] : -INFINITY;
          top = fmaxf(top, x[b][i]);
        }
        if (kKeep && live)
          *reinterpret_cast<float4 *>(p.scores + (row * p.hq + head) * p.scores_st + key0 + 4 * g) =
              make_float4(x[b][0], x[b][1], x[b][2], x[b][3]);
      }
      top = max_groups(top);
      // A row that has seen no key yet keeps its reference point at 0.
      const float ref = top == -INFINITY ? 0.f : top;
      const float fall = __builtin_amdgcn_exp2f((mx - ref) * kLog2e);
      mx = top;
      l *= fall;
#pragma unroll
      for (int n = 0; n < kVe; ++n) acc[n] *= fall;
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        if (b0 + b * step >= k1) continue;
        float pr[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          pr[i] = __builtin_amdgcn_exp2f((x[b][i] - ref) * kLog2e);
          l += pr[i];
          pr[i] *= kUp;
        }
        bool plain = true;
        if (kUnlike && __builtin_expect(__any(own_end < min(b0 + b * step + 16, k1)), 0)) {
          // Keys that some row does not see: a V that is not finite must not
          // reach that row as 0 * V.
          bool bad = false;
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int c = 0; c < M::kV; ++c) {
              const uint32_t e = tile[b].v[i][c];
              if constexpr (sizeof(T) == 4) bad = bad || (e & 0x7f800000u) == 0x7f800000u;
              else if constexpr (std::is_same_v<T, bf16_t>)
                bad = bad || (e & 0x7f80u) == 0x7f80u || (e & 0x7f800000u) == 0x7f800000u;
              else bad = bad || (e & 0x7c00u) == 0x7c00u || (e & 0x7c000000u) == 0x7c000000u;
            }
          plain = __builtin_amdgcn_ballot_w64(bad) == 0;
        }
        if (__builtin_expect(plain, 1)) {
          uint4 parts = make_uint4(0, 0, 0, 0);  // (hi, hi, lo, lo) of the four keys
          if constexpr (kFine && sizeof(T) == 2) {
            two_parts<T>(pr[0], pr[1], parts.x, parts.z);
            two_parts<T>(pr[2], pr[3], parts.y, parts.w);
          }
#pragma unroll
          for (int n = 0; n < kVe; ++n) {
            if constexpr (sizeof(T) == 2) {
              // Element n of the four rows, packed as operand A.
              uint32_t w01, w23;
              if (n & 1) {
                w01 = __builtin_amdgcn_perm(tile[b].v[1][n / 2], tile[b].v[0][n / 2], 0x07060302);
                w23 = __builtin_amdgcn_perm(tile[b].v[3][n / 2], tile[b].v[2][n / 2], 0x07060302);
              } else {
                w01 = __builtin_amdgcn_perm(tile[b].v[1][n / 2], tile[b].v[0][n / 2], 0x05040100);
                w23 = __builtin_amdgcn_perm(tile[b].v[3][n / 2], tile[b].v[2][n / 2], 0x05040100);
              }
              if constexpr (kFine) {
                acc[n] = Mma16<T>::pv2(make_uint2(w01, w23), parts, acc[n]);
              } else {
                acc[n] = Mma16<T>::pv(make_uint2(w01, w23),
                                      make_uint2(pack2<T>(pr[0], pr[1]), pack2<T>(pr[2], pr[3])),
                                      acc[n]);
              }
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i)
                acc[n] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(tile[b].v[i][n]),
                                                              pr[i], acc[n], 0, 0, 0);
            }
          }
        } else {
          // Key by key, each row adding only the keys that it sees: the lane
          // holds elements kVe (4 g + e) + n of row m16.
          for (int j = 0; j < 16; ++j) {
            const int from = (j & 12) * 4 + m16;
            const float p0 = __shfl(pr[0], from), p1 = __shfl(pr[1], from);
            const float p2 = __shfl(pr[2], from), p3 = __shfl(pr[3], from);
            const float pj = (j & 2) ? ((j & 1) ? p3 : p2) : ((j & 1) ? p1 : p0);
            const int key = b0 + b * step + j;
            bool exists = key < k1;
            int64_t slot = 0;
            if (exists) slot = src.slot_of(key, exists);
            if (!exists || key < lo || key >= limit) continue;
            if (kTree && key >= tree0 && !bit_of(p, row, key - tree0)) continue;
            const T *vr = src.v + (slot * p.hkv + kvh) * p.d;
#pragma unroll
            for (int n = 0; n < kVe; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int dim = kVe * (4 * g + e) + n;
                if (dim < p.d) acc[n][e] += pj * Elem<T>::to_f32(vr[dim]);
              }
          }
        }
      }
    }
    l = sum_groups(l);
    if constexpr (kUp != 1.f) {
#pragma unroll
      for (int n = 0; n < kVe; ++n) acc[n] *= 1.f / kUp;
    }

    // Join the waves. acc[n][e] is element kVe (4 g + e) + n of row m16.
    if (g == 0) {
      s_m[wv][m16] = mx;
      s_l[wv][m16] = l;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int n = 0; n < kVe; n += 4) {
        const f32x4_t x = {acc[n][e], acc[n + 1][e], acc[n + 2][e], acc[n + 3][e]};
        *reinterpret_cast<f32x4_t *>(&s_acc[wv][m16][kVe * (4 * g + e) + n]) = x;
      }
    __syncthreads();
    const int rr = tid >> 4, d0 = (tid & 15) * kVe;
    float m_all = -INFINITY;
#pragma unroll
    for (int i = 0; i < kWavesWg; ++i) m_all = fmaxf(m_all, s_m[i][rr]);
    const float ref = m_all == -INFINITY ? 0.f : m_all;
    float sum = 0.f, o[kVe];
#pragma unroll
    for (int n = 0; n < kVe; ++n) o[n] = 0.f;
#pragma unroll
    for (int i = 0; i < kWavesWg; ++i) {
      const float f = __builtin_amdgcn_exp2f((s_m[i][rr] - ref) * kLog2e);
      sum += s_l[i][rr] * f;
#pragma unroll
      for (int n = 0; n < kVe; ++n) o[n] += s_acc[i][rr][d0 + n] * f;
    }
    const int orow = t.r0 + rr;
    const int64_t at = static_cast<int64_t>(w) * kRows + rr;
    if ((!alone || kKeep) && (tid & 15) == 0) {
      p.ml[2 * at] = m_all;
      p.ml[2 * at + 1] = sum;
    }
    if (!alone) {
#pragma unroll
      for (int n = 0; n < kVe; ++n) p.acc[at * D + d0 + n] = o[n];
    } else if (orow < t.rows) {
      const int otok = orow / p.group;
      const int ohead = kvh * p.group + orow - otok * p.group;
      const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
      T *dst = static_cast<T *>(p.out) + (t.q0 + otok) * p.o_st + ohead * p.o_sh;
#pragma unroll
      for (int n = 0; n < kVe; ++n)
        if (d0 + n < p.d) dst[d0 + n] = Elem<T>::from_f32(o[n] * inv);
    }
    __syncthreads();  // s_* are written again for the next item
  }
}

template <typename T, int D>
int launch_rows(const ScoredParams &p, unsigned grid, hipStream_t stream) {
  const bool paged16 = p.block_size % 16 == 0;
#define MLR_ROWS(C, B, F, U, R, K, E) \
  scored_rows_kernel<T, D, C, B, F, U, R, K, E><<<grid, 256, 0, stream>>>(p)
#define MLR_ROWS_B(C, B)                                                             \
  if (p.mode == kModePrefill && p.bits) MLR_ROWS(C, B, true, true, true, false, true);     \
  else if (p.mode == kModePrefill) MLR_ROWS(C, B, true, true, false, false, false);        \
  else if (p.mode == kModePrefix) MLR_ROWS(C, B, false, true, false, false, false);        \
  else if (p.scores) MLR_ROWS(C, B, false, false, false, true, true);                      \
  else if (p.fine) MLR_ROWS(C, B, false, false, false, false, true);                       \
  else MLR_ROWS(C, B, false, false, false, false, false);
  if (p.cap > 0) {
    if (paged16) { MLR_ROWS_B(true, true) } else { MLR_ROWS_B(true, false) }
  } else {
    if (paged16) { MLR_ROWS_B(false, true) } else { MLR_ROWS_B(false, false) }
  }
#undef MLR_ROWS_B
#undef MLR_ROWS
  return check_launch("scored_rows");
}

}  // namespace

int launch_scored_rows(const ScoredParams &p, int dtype, unsigned grid, hipStream_t stream) {
  const bool wide = p.d > 64;
  switch (dtype) {
    case MLR_DTYPE_F32:
      return wide ? launch_rows<float, 128>(p, grid, stream) : launch_rows<float, 64>(p, grid, stream);
    case MLR_DTYPE_F16:
      return wide ? launch_rows<f16_t, 128>(p, grid, stream) : launch_rows<f16_t, 64>(p, grid, stream);
    default:
      return wide ? launch_rows<bf16_t, 128>(p, grid, stream)
                  : launch_rows<bf16_t, 64>(p, grid, stream);
  }
}

}  // namespace mlr

// Paged attention with capped or biased scores, for many query rows per key
// (bf16, fp16): packed prompt chunks, trees of drafted tokens, and a decode batch over the
// prefix that its requests share. The scores are those of scored_rows.hip.
//
// A unit is 128 query rows of one KV head, a row being one (token, head of the
// group): the heads of a group share every K/V tile that is loaded. Eight
// waves: four groups of 32 rows, twice, for two halves of the unit's keys
// (joined through LDS at the end). Keys stream through LDS in tiles of 64,
// two stages per half, copied there from memory without registers on the way
// (buffer_load ... lds), one tile ahead of its use, one barrier per tile.
//
// Per tile and wave, v_mfma_f32_32x32x16:
//   S^T[64 keys x 32 rows] = K Q^T: operand A = K rows from LDS, B = Q^T in
//     registers. Lane l holds row l % 32 and, of each 32 keys, keys
//     8 (i / 4) + 4 (l / 32) + i % 4, i < 16.
//   scores in base 2, relative to the row's reference point m, which follows
//     the running maximum only when a tile exceeds it by 2^kLazy: probabilities
//     stay below 2^kLazy, numerator and sum share m, and most tiles rescale nothing.
//     (Trees in fp16: m lies kBelow below that maximum, so that the parts of a
//     probability use the type's range, up to 2^15.)
//   O^T[D x 32 rows] += V^T P^T: B = P^T straight from the S^T registers, rounded
//     to the 16-bit type (by at most 2^-8 of it in bf16, 2^-11 in fp16; see
//     scored_rows.hip), for trees in two parts, a product each (two_parts); A = V^T
//     by transposing LDS reads.
//
// Tiles are taken from the last to the first, as a bias by distance makes the last
// keys the heaviest, and the two key halves run their vector and matrix phases in
// turn, so that one's exponentials cover the other's products.
//
// What bounds it is the vector work per score beside the matrix work (D = 64:
// 16 cycles of MFMA per wave and score): 28 cycles plain, of which the
// exponential takes 16. The cap as exponential and reciprocal would add 40;
// tanh(y) = y P(y^2) with three terms beyond the first (relative error 5.1e-7
// for |y| <= 1/2) adds 16 and with two (4.0e-7 for |y| <= 1/4) 12, so a tile takes
// the shortest form that holds for all of its scores (with the order of the keys,
// 101 -> 92 us on the first of these); where none does, the exponential or the
// polynomial score by score. Measured: capped bf16, 8 chunks of 512 tokens after up to
// 3,584, 14/2 heads of 64: 36.0 GF in 76 us, 470 TF/s; biased fp16 prompts at head size
// 128: 52.7 GF in 89 us, 590 TF/s; 64 requests over 8,192 shared keys with their own:
// 20 us of the kernel; 32 over 24,000, head size 128: 29 us.
//
// Trees of drafted tokens are chunks of which a row sees the keys before them and
// those of its bits: tiles that reach past those keys are masked bit by bit. 16 trees
// of 20 to 48 tokens after 512 to 4,096 keys, 28/4 heads of 128: 24 GF, and 12 more for
// the second parts of the probabilities, in 71 us (60 with one part, whose rounding is
// 2^-8); at 14/2 heads of 64 33 us (28). Counted of the first, cycles of the shader clock:
// a CU has work in 112,000 of 173,000, and in these its matrix units work for 38,000, its
// vector units for 44,000 and LDS for 24,000 (6,000 of them bank conflicts). So no unit
// bounds it: planning and first loads of a workgroup, items of unlike ends, and two phases
// that wait for each other do.
//
// LDS rows are unpadded; the 16-byte chunk c of row r lies at c ^ swizzle(r),
// which keeps the row reads of K and the transposing reads of V free of bank
// conflicts.
#include "scored_attention.h"

namespace mlr {
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void_t;
typedef __attribute__((address_space(3))) s16x4_t lds_s16x4_t;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLazy = 8.f;
constexpr int kTile = 64;    // keys
constexpr int kHalves = 2;   // of the keys
constexpr int kThreads = 256 * kHalves;
constexpr int kRankUnits = 4096, kRankSeqs = 512;  // most that are ranked by their keys

template <typename T> struct Wide;
template <> struct Wide<bf16_t> {
  using v8 = bf16x8_t;
  using h = __bf16;
  __device__ static f32x16_t mfma(v8 a, v8 b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  // Bits 15 and 31: whether that half of w is an infinity or NaN.
  __device__ static uint32_t odd(uint32_t w) {
    return ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
  }
};
template <> struct Wide<f16_t> {
  using v8 = f16x8_t;
  using h = _Float16;
  __device__ static f32x16_t mfma(v8 a, v8 b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  __device__ static uint32_t odd(uint32_t w) {
    return ((w & 0x7c007c00u) + 0x04000400u) & 0x80008000u;
  }
};

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  typedef float f32x2_v __attribute__((ext_vector_type(2)));
  typedef typename Wide<T>::h h2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_v{a, b}, h2));
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c);
}
__device__ __forceinline__ float pair_max(float x) {  // lanes l and l ^ 32
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  return __builtin_elementwise_maximum(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float pair_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

template <int D>
__device__ __forceinline__ int swizzle(int r) {
  if (D == 64) return (((r >> 1) & 1) << 2) | (((r >> 2) & 1) << 1) | ((r >> 3) & 1);
  return ((r & 1) << 1) | (((r >> 1) & 3) << 2) | ((r >> 3) & 1);
}

// What the order of units needs of a sequence.
struct Seq {
  int rows, pos0, ahead;
};

// Units of a sequence that see more than `keys` keys: those whose last row
// belongs to token keys - pos0 or a later one.
__device__ __forceinline__ int units_past(const Seq &t, int group, int keys) {
  const int all = (t.rows + kTileRows - 1) / kTileRows;
  const int tok = keys - t.pos0;
  if (t.ahead > keys || tok <= 0) return all;
  return tok > (t.rows - 1) / group ? 0 : all - tok * group / kTileRows;
}

// kTree: of its sequence's last tokens a row sees those that its bits name.
template <typename T, int D, bool kCap, bool kBias, bool kTree>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(D == 64 ? 4 : 2)))
void scored_tiles_kernel(ScoredParams p) {
  using W = Wide<T>;
  using v8 = typename W::v8;
  constexpr int QS = D / 16, NB = D / 32, KB = kTile / 32;
  constexpr int kRowB = 2 * D, kChunks = D / 8;
  constexpr int kCopies = 16 * kRowB / 1024;  // 1 KB copies of a wave's 16 rows
  constexpr int kTileB = kTile * kRowB;
  constexpr float kBelow = kTree && std::is_same_v<T, f16_t> ? 7.f : 0.f;
  // Each stage is an object of its own, so that the compiler does not make reads
  // of one wait for copies into another.
  __shared__ __align__(1024) unsigned char ks0[kHalves][kTileB], ks1[kHalves][kTileB];
  __shared__ __align__(1024) unsigned char vs0[kHalves][kTileB], vs1[kHalves][kTileB];
  __shared__ int64_t s_keys[kThreads / 64];
  __shared__ int s_count[kThreads / 64], s_most[kThreads / 64], s_unit, s_part, s_of, s_all, s_odd;
  __shared__ float s_time[kTree ? 16 : 1];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int w = wave & 3, half = wave >> 2;
  const int m32 = lane & 31, hh = lane >> 5;

  // Which item this workgroup takes.
  int split = 0x7fffffc0;
  int64_t item;
  int kvh;
  if (p.whole) {
    // Heaviest units first, so that the last to start are short. Where two
    // workgroups fit a CU (D = 64), b and b + ncu share one: the second ncu go in
    // reverse, light beside heavy.
    const int n = gridDim.x;
    int b = blockIdx.x;
    if (D == 64 && b >= p.ncu && b < 2 * p.ncu) b = min(n, 2 * p.ncu) - 1 - (b - p.ncu);
    const int rank = b / p.hkv;
    kvh = b - rank * p.hkv;
    if (p.units > kRankUnits || p.seqs > kRankSeqs) {
      const int seq = rank / p.tiles;
      if (tid == 0) s_unit = seq * p.tiles + p.tiles - 1 - (rank - seq * p.tiles);
    } else {
      // By keys, then by sequence, then later rows first. The sequences' sizes
      // are read once, into what will be the first stage. Every workgroup does this,
      // in time units * sequences, which pays for some chunks but not for many short
      // ones: 32, 64 and 256 prompts of 128 tokens at 14/2 heads of 64 take 22, 63 and
      // 1,668 us, the plain prefill, whose units have no order, 16, 30 and 128 us.
      Seq *seqs = reinterpret_cast<Seq *>(&ks0[0][0]);
      static_assert(sizeof(ks0) >= kRankSeqs * sizeof(Seq), "the sizes fit a stage");
      for (int q = tid; q < p.seqs; q += kThreads) {
        const Unit t = unit_of(p, q * p.tiles, kTileRows);
        seqs[q] = Seq{t.rows, static_cast<int>(t.pos0), static_cast<int>(t.ahead)};
      }
      if (tid == 0) s_unit = -1;
      __syncthreads();
      for (int u = tid; u < p.units; u += kThreads) {
        const int seq = u / p.tiles, at = u - seq * p.tiles;
        const Seq t = seqs[seq];
        if (at * kTileRows >= t.rows) continue;
        const int last = min(t.rows, (at + 1) * kTileRows) - 1;
        const int hi = max(max(t.pos0 + last / p.group + 1, t.ahead), 0);
        int r = (t.rows + kTileRows - 1) / kTileRows - 1 - at;
        for (int q = 0; q < p.seqs; ++q) {
          const Seq o = seqs[q];
          if (q != seq && o.rows > 0) r += units_past(o, p.group, q < seq ? hi - 1 : hi);
        }
        if (r == rank) s_unit = u;
      }
    }
    if (tid == 0) {
      s_part = 0;
      s_of = 1;
    }
    item = rank;
  } else if (kTree) {
    // The cut. A thread has one sequence, whose units see the same keys. Of some splits,
    // from the one that would deal all keys evenly on and the longest unit cut in up to
    // eight, that whose items, in rounds over the CUs, take the shortest time; an item
    // costs as much as kStart keys more than its own (its planning, q and first tile). 16
    // trees of 20 to 48 tokens after 512 to 4,096 keys, 4 KV heads of 128, merge included: 69 us
    // with the cut of chunks, 63 us with this.
    constexpr int kStart = 400;
    int *lens = reinterpret_cast<int *>(&ks0[0][0]), *units = lens + kThreads;
    static_assert(kTreeSeqs <= kThreads && sizeof(ks0) >= 2 * kThreads * sizeof(int),
                  "a thread has one sequence");
    int own_units = 0, own_len = 0;
    if (tid < p.seqs) {
      const Unit t = unit_of(p, tid * p.tiles, kTileRows);
      own_units = min((t.rows + kTileRows - 1) / kTileRows, p.tiles);
      own_len = own_units > 0 ? static_cast<int>(unit_len(t)) : 0;
    }
    lens[tid] = own_len;
    units[tid] = own_units;
    int64_t keys = static_cast<int64_t>(own_len) * own_units;
    int most = own_len;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      keys += __shfl_xor(keys, o);
      most = max(most, __shfl_xor(most, o));
    }
    if (lane == 0) {
      s_keys[wave] = keys;
      s_most[wave] = most;
    }
    if (tid == 0) s_unit = -1;
    __syncthreads();
    keys = 0;
#pragma unroll
    for (int i = 0; i < kThreads / 64; ++i) {
      keys += s_keys[i];
      most = max(most, s_most[i]);
    }
    const int slots = D == 64 ? 2 * p.ncu : p.ncu;
    const float even = static_cast<float>(keys) * p.hkv / slots;
    auto cut_of = [&](int i) __attribute__((always_inline)) {
      const float x = i < 8 ? even * (1.f + 0.14f * i) : most / static_cast<float>(i - 7);
      const float y = fminf(fmaxf(fmaxf(x, even), static_cast<float>(kMinSplit)), 2.0e9f);
      return (static_cast<int>(y) + 64) & ~63;
    };
    for (int i = wave; i < 16; i += kThreads / 64) {
      const int cut = cut_of(i);
      int n = 0;
      for (int q = lane; q < p.seqs; q += 64) n += units[q] * items_of(lens[q], cut);
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o);
      const float rounds = static_cast<float>((n * p.hkv + slots - 1) / slots);
      if (lane == 0) s_time[i] = rounds * (min(cut, most) + kStart);
    }
    __syncthreads();
    int best = 0;
#pragma unroll
    for (int i = 1; i < 16; ++i) best = s_time[i] < s_time[best] ? i : best;
    const int own_parts = items_of(own_len, cut_of(best)), own = own_units * own_parts;
    int before = own;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int x = __shfl_up(before, o);
      if (lane >= o) before += x;
    }
    if (lane == 63) s_count[wave] = before;
    before -= own;
    __syncthreads();
    int items = 0;
#pragma unroll
    for (int i = 0; i < kThreads / 64; ++i) {
      if (i < wave) before += s_count[i];
      items += s_count[i];
    }
    item = blockIdx.x / p.hkv;
    kvh = blockIdx.x - static_cast<int>(item) * p.hkv;
    if (item >= before && item < before + own) {
      const int at = static_cast<int>(item) - before;
      s_unit = tid * p.tiles + at / own_parts;
      s_part = at % own_parts;
      s_of = own_parts;
    }
    if (blockIdx.x == 0 && tid < p.seqs) {
      for (int k = 0; k < p.tiles; ++k)
        p.first[tid * p.tiles + k] = before + min(k, own_units) * own_parts;
      if (tid == 0) p.first[p.units] = items;
    }
  } else {
    const int per = (p.units + kThreads - 1) / kThreads;
    const int u_lo = min(tid * per, p.units), u_hi = min(u_lo + per, p.units);
    int64_t keys = 0;
    int most = 0;
    for (int u = u_lo; u < u_hi; ++u) {
      const int64_t len = unit_len(unit_of(p, u, kTileRows));
      keys += len;
      most = max(most, static_cast<int>(len));
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      keys += __shfl_xor(keys, o);
      most = max(most, __shfl_xor(most, o));
    }
    if (lane == 0) {
      s_keys[wave] = keys;
      s_most[wave] = most;
    }
    __syncthreads();
    keys = 0;
    for (int i = 0; i < kThreads / 64; ++i) {
      keys += s_keys[i];
      most = max(most, s_most[i]);
    }
    // A prefill's units stay whole unless splits pay.
    if (p.mode != kModePrefill || splits_pay(static_cast<int64_t>(p.units) * p.hkv, most, p.ncu))
      split = split_of(keys, p);
    int own = 0;
    for (int u = u_lo; u < u_hi; ++u) own += unit_items(unit_of(p, u, kTileRows), split);
    int before = own;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int x = __shfl_up(before, o);
      if (lane >= o) before += x;
    }
    if (lane == 63) s_count[wave] = before;
    before -= own;
    if (tid == 0) s_unit = -1;
    __syncthreads();
    int items = 0;
    for (int i = 0; i < kThreads / 64; ++i) {
      if (i < wave) before += s_count[i];
      items += s_count[i];
    }
    item = blockIdx.x / p.hkv;
    kvh = blockIdx.x - static_cast<int>(item) * p.hkv;
    int at = before;
    for (int u = u_lo; u < u_hi; ++u) {
      const int n = unit_items(unit_of(p, u, kTileRows), split);
      if (blockIdx.x == 0) p.first[u] = at;
      if (item >= at && item < at + n) {
        s_unit = u;
        s_part = static_cast<int>(item) - at;
        s_of = n;
      }
      at += n;
    }
    if (blockIdx.x == 0 && tid == kThreads - 1) p.first[p.units] = items;
  }
  if (tid == 0) {
    s_all = 0x7fffffff;
    s_odd = 0;
  }
  __syncthreads();
  const int unit = __builtin_amdgcn_readfirstlane(s_unit);
  if (unit < 0) return;  // uniform: no item left for this workgroup
  const int part = __builtin_amdgcn_readfirstlane(s_part);
  const int parts = __builtin_amdgcn_readfirstlane(s_of);
  const bool alone = parts == 1 && !p.force_partial;
  const Unit t = unit_of(p, unit, kTileRows);
  if (t.r0 >= t.rows) return;
  const int len = item_len(t, parts, kTile);
  const int k_lo =
      __builtin_amdgcn_readfirstlane(static_cast<int>(unit_base(t) + static_cast<int64_t>(part) * len));
  const int low = __builtin_amdgcn_readfirstlane(static_cast<int>(t.lo));  // first key seen
  const int k_hi = __builtin_amdgcn_readfirstlane(
      static_cast<int>(min(t.hi, static_cast<int64_t>(k_lo) + len)));

  // This half's tiles [t_lo, t_hi) of the item's, taken from the last to the
  // first: a bias by distance makes the last keys the heaviest, and the running
  // maximum then stays where the first tile puts it.
  const int tiles = (k_hi - k_lo + kTile - 1) / kTile;
  const int chunk = (tiles + kHalves - 1) / kHalves;
  const int t_lo = half * chunk, t_hi = min(tiles, t_lo + chunk);

  // The lane's row: token, head, position, first key that it does not see.
  const int r_first = t.r0 + 32 * w, unit_rows = t.rows;
  const int64_t q_first = t.q0;
  const int r = r_first + m32;
  const bool live = r < unit_rows;
  const int rc = live ? r : t.rows - 1;
  const int tok = rc / p.group, head = kvh * p.group + rc - tok * p.group;
  const int64_t row = t.q0 + tok;
  int pos, limit;
  if (p.mode == kModePrefill) {
    pos = static_cast<int>(t.pos0) + tok;
    limit = max(pos + 1, static_cast<int>(t.ahead));
  } else {
    // A request shorter than the prefix sees its own first positions.
    const int64_t ctx = clamp64(p.ctx[row], 0, 0x7fffffff);
    pos = static_cast<int>(ctx) - 1;
    limit = static_cast<int>(min(t.hi, ctx));
  }
  if (!live) limit = 0;
  // Keys that all of the wave's rows see, and that any does.
  const int tree0 = static_cast<int>(t.pos0);
  int all = !live ? 0x7fffffff : kTree ? tree0 : limit, any = limit;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    all = min(all, __shfl_xor(all, o));
    any = max(any, __shfl_xor(any, o));
  }
  all = __builtin_amdgcn_readfirstlane(all);
  any = __builtin_amdgcn_readfirstlane(any);

  // Q^T fragments: Q[row][16 s + 8 hh ..]. A negative scale goes into Q's sign,
  // so that the factor of the scores is positive.
  const uint32_t flip = p.scale < 0 ? 0x80008000u : 0u;
  v8 qf[QS];
  const uint16_t *qr = static_cast<const uint16_t *>(p.q) + row * p.q_st + head * p.q_sh;
#pragma unroll
  for (int s = 0; s < QS; ++s) {
    const int e = 16 * s + 8 * hh;
    uint4 q = make_uint4(0, 0, 0, 0);
    if (live && e < p.d) q = *reinterpret_cast<const uint4 *>(qr + e);
    q.x ^= flip;
    q.y ^= flip;
    q.z ^= flip;
    q.w ^= flip;
    qf[s] = __builtin_bit_cast(v8, q);
  }
  // Score in base 2: c2 s, or with the cap s (b0 + s^2 (b1 + ...)). Uniform, so
  // held in scalar registers.
  auto uniform = [](float x) {
    return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(x)));
  };
  const float scale = fabsf(p.scale);
  const float c2 = uniform(scale * kLog2e);
  const float c1 = uniform(kCap ? fminf(scale / p.cap, 1e37f) : 0.f);  // y = c1 s
  const float top = uniform(kCap ? p.cap * kLog2e : 0.f);  // the cap in base 2
  // tanh(y) / y up to |y| = 1/2 (relative error 5.1e-7) and 1/4 (4.0e-7), the powers
  // of c1 in the factors. Scores whose square has no finite value take the
  // exponential; under a cap so small (some 1e-7 of the scale) that the factors
  // have none, all do, as a score of 0 times such a factor would be NaN.
  const float c3 = c1 * c1 * c2, c5 = c1 * c1 * c3, c7 = c1 * c1 * c5;
  const bool held = c7 < __FLT_MAX__;
  const float near = uniform(held ? fminf(0.5f / c1, 1.8e19f) : -1.f);
  const float near2 = uniform(held ? fminf(0.25f / c1, 1.8e19f) : -1.f);
  const float b0 = uniform(kTanh0 * c2), b1 = uniform(kTanh1 * c3);
  const float b2 = uniform(kTanh2 * c5), b3 = uniform(kTanh3 * c7);
  const float a0 = uniform(0.99999960f * c2), a1 = uniform(-0.33321908f * c3);
  const float a2 = uniform(0.12841613f * c5);
  const float slope = kBias ? p.slopes[head] * kLog2e : 0.f;

  // Copies: copy i of a wave's 16 rows moves chunk places [64 i, 64 i + 64);
  // lane l fills place 64 i + l, row rr, physical chunk pc, with the logical
  // chunk pc ^ swizzle(rr). Chunks past the head lie outside every resource.
  const uint32_t row_bytes = static_cast<uint32_t>(p.hkv) * p.d * 2;
  uint32_t src_off[kCopies];
#pragma unroll
  for (int i = 0; i < kCopies; ++i) {
    const int place = 64 * i + lane, rr = place / kChunks;
    const int c = (place % kChunks) ^ swizzle<D>(rr);
    src_off[i] = 8 * c < p.d ? rr * row_bytes + 16 * c : 0x7fffffffu;
  }
  typedef __attribute__((address_space(4))) const int64_t const_i64;
  const const_i64 *table = (const const_i64 *)table_of(p, t);
  const int bs_log2 = p.bs_log2, bs_mask = (1 << bs_log2) - 1;
  const uint32_t head_bytes = 2 * p.d, kv_bytes = static_cast<uint32_t>(kvh) * head_bytes;
  // Fewer than 2^31 blocks of fewer than 2^31 bytes.
  const uint32_t block_bytes = row_bytes << bs_log2, blocks = static_cast<uint32_t>(p.num_blocks);
  auto known = [&](int64_t id) __attribute__((always_inline)) {
    return static_cast<uint32_t>(static_cast<uint64_t>(id) >> 32) == 0u &&
           static_cast<uint32_t>(id) < blocks;
  };

  // Whether some block id of the item is out of range (then every tile asks).
  bool strange = false;
  for (int i = (k_lo >> bs_log2) + tid; k_hi > 0 && i <= (k_hi - 1) >> bs_log2; i += kThreads) {
    const int64_t id = table_of(p, t)[i];
    strange = strange || !known(id);
  }
  if (lane == 0) atomicMin(&s_all, all);
  strange = __syncthreads_or(strange);
  // Tiles that start in [low, whole_to] are seen whole by all rows of the wave,
  // those in [low, unit_to] by all rows of the unit.
  const int whole_to = min(all, k_hi) - kTile;
  const int unit_to = __builtin_amdgcn_readfirstlane(s_all) - kTile;

  // The wave's 16 rows of tile i: where they start, and how many bytes from there
  // on may be read (rows past k_hi and of blocks out of range arrive as zeros).
  struct Span {
    uint64_t at;
    uint32_t bytes;
  };
  const int first_key = k_lo + t_lo * kTile, last_key = k_lo + (t_hi - 1) * kTile;
  auto key_of = [&](int i) __attribute__((always_inline)) {  // first key of the i-th tile
    return last_key - i * kTile;
  };
  auto id_of = [&](int i) __attribute__((always_inline)) -> int64_t {
    return table[min(max(key_of(i) + 16 * w, 0), k_hi - 1) >> bs_log2];
  };
  auto span_of = [&](int i, int64_t id) __attribute__((always_inline)) -> Span {
    const int key = key_of(i) + 16 * w;
    const bool ok = key >= first_key && key < k_hi && known(id);
    Span x;
    x.bytes = ok ? static_cast<uint32_t>(min(k_hi - key, 16) - 1) * row_bytes + head_bytes : 0u;
    x.at = static_cast<uint64_t>(ok ? static_cast<uint32_t>(id) : 0u) * block_bytes +
           (static_cast<uint32_t>(key & bs_mask) * row_bytes + kv_bytes);
    return x;
  };
  auto copy = [&](const Span &x, const void *cache, unsigned char *dst)
      __attribute__((always_inline)) {
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<unsigned char *>(static_cast<const unsigned char *>(cache) + x.at), 0, x.bytes,
        0x00020000);
    dst += 16 * w * kRowB;
#pragma unroll
    for (int c = 0; c < kCopies; ++c) {
      const uint32_t off = src_off[c];
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void_t *)(dst + 1024 * c), 16, off, 0, 0, 0);
    }
  };
  // One bit per run of 16 keys from key0 on whose block is out of range.
  auto bad_of = [&](int key0) __attribute__((always_inline)) -> uint32_t {
    uint32_t bad = 0;
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      if (!known(table[min(key0 + 16 * b, k_hi - 1) >> bs_log2])) bad |= 1u << b;
    }
    return bad;
  };

  // Lane-constant LDS offsets, as XORs of the chunk index: K row m32 (+ 32 per
  // block), chunk 2 st + hh; V^T by two transposing reads per MFMA, where of a
  // group of 16 lanes lane li reads 8 bytes of row 4 (group / 2) + li / 4 (the
  // second: 8 rows on) at byte 64 n + 32 (group % 2) + 8 (li % 4).
  const int koff0 = m32 * kRowB + ((hh ^ swizzle<D>(m32)) << 4);
  const int grp = lane >> 4, li = lane & 15;
  const int vrow = 4 * (grp >> 1) + (li >> 2), vbyte = 32 * (grp & 1) + 8 * (li & 3);
  const int voff0 = vrow * kRowB + ((((vbyte >> 4) ^ swizzle<D>(vrow)) << 4) | (vbyte & 15));

  f32x16_t acc[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) acc[n] = f32x16_t{};
  float m = 0.f, l = 0.f;
  float thr = -__FLT_MAX__;  // a tile's maximum above this moves m; m is unset so far

  // Two phases per tile, a workgroup barrier after each, the halves one phase
  // apart: on every SIMD one wave's matrix work meets the other's vector work.
  //   M_i: O^T += V^T P^T of tile i - 1, S^T of tile i
  //   V_i: copies of K_{i+2} and V_{i+1} into the stages that M_i has read,
  //        then scores and probabilities of tile i, packed for M_{i+1}
  // A wave waits for its own copies of the phase before, the barrier for all.
  f32x16_t s[KB];
  uint32_t pk[KB][8], pl[KB][kTree ? 8 : 1];  // pl: the second parts
  auto active = [&](int i) __attribute__((always_inline)) {
    const int key0 = key_of(i);
    return key0 >= first_key && key0 < any;
  };
  auto add_values = [&](const unsigned char *vt) __attribute__((always_inline)) {
    int vo = voff0;
    asm volatile("" : "+v"(vo));
#pragma unroll
    for (int kb = 0; kb < 2 * KB; ++kb) {
      const uint32_t *x = &pk[kb >> 1][4 * (kb & 1)];
      const v8 pb = __builtin_bit_cast(v8, make_uint4(x[0], x[1], x[2], x[3]));
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        const uint2 lo = __builtin_bit_cast(
            uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                       (lds_s16x4_t *)(vt + 16 * kb * kRowB + (vo ^ (n << 6)))));
        const uint2 hi = __builtin_bit_cast(
            uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                       (lds_s16x4_t *)(vt + 16 * kb * kRowB + ((vo ^ 16 ^ (n << 6)) + 8 * kRowB))));
        const v8 va = __builtin_bit_cast(v8, make_uint4(lo.x, lo.y, hi.x, hi.y));
        acc[n] = W::mfma(va, pb, acc[n]);
        if constexpr (kTree) {
          const uint32_t *y = &pl[kb >> 1][4 * (kb & 1)];
          acc[n] = W::mfma(va, __builtin_bit_cast(v8, make_uint4(y[0], y[1], y[2], y[3])), acc[n]);
        }
      }
    }
    // Two fragments' V reads ahead of the MFMAs.
    constexpr int kFragments = 2 * KB * NB, kEach = kTree ? 2 : 1;
    __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
    for (int x = 0; x < kFragments - 2; ++x) {
      __builtin_amdgcn_sched_group_barrier(0x008, kEach, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, 2 * kEach, 0);
  };
  // Where some row does not see some key, a V that is not finite would reach
  // it as 0 * V. So in such tiles each wave looks through the 16 rows that it has
  // copied, turns what is not finite to zeros, and notes that the item has met
  // such values; they are given to the rows that see them after the loop.
  auto clean = [&](unsigned char *vt) __attribute__((always_inline)) {
#pragma unroll 1
    for (int c = 0; c < kCopies; ++c) {
      uint4 *at = reinterpret_cast<uint4 *>(vt + 16 * w * kRowB + 1024 * c) + lane;
      uint4 x = *at;
      const uint4 o = make_uint4(W::odd(x.x), W::odd(x.y), W::odd(x.z), W::odd(x.w));
      if ((o.x | o.y | o.z | o.w) != 0) {
        // A flag in bit 15 of a half to ones all over that half.
        x.x &= ~((o.x >> 15) * 0xffffu);
        x.y &= ~((o.y >> 15) * 0xffffu);
        x.z &= ~((o.z >> 15) * 0xffffu);
        x.w &= ~((o.w >> 15) * 0xffffu);
        *at = x;
        s_odd = 1;
      }
    }
  };
  auto scores = [&](const unsigned char *kt) __attribute__((always_inline)) {
    int ko = koff0;  // the offsets below are made here, not kept over the loop
    asm volatile("" : "+v"(ko));
#pragma unroll
    for (int j = 0; j < KB; ++j) {
      s[j] = f32x16_t{};
#pragma unroll
      for (int st = 0; st < QS; ++st) {
        const v8 a = *reinterpret_cast<const v8 *>(kt + 32 * j * kRowB + (ko ^ (st << 5)));
        s[j] = W::mfma(a, qf[st], s[j]);
      }
    }
    // Two K reads ahead of the MFMAs; more would only hold registers.
    __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
#pragma unroll
    for (int x = 0; x < KB * QS - 2; ++x) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
  };
  auto weigh = [&](int i) __attribute__((always_inline)) {
    const int key0 = key_of(i);
    const uint32_t bad = strange ? bad_of(key0) : 0u;
    const bool masked = key0 > whole_to || key0 < low || bad != 0;

    // Scores relative to m.
    if constexpr (kCap) {
      float big = 0.f;
#pragma unroll
      for (int j = 0; j < KB; ++j)
#pragma unroll
        for (int e = 0; e < 16; e += 2) big = max3(big, fabsf(s[j][e]), fabsf(s[j][e + 1]));
      if (!__any(!(big <= near2))) {
#pragma unroll
        for (int j = 0; j < KB; ++j)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float x = s[j][e], u = x * x;
            s[j][e] = fmaf(x, fmaf(u, fmaf(u, a2, a1), a0), -m);
          }
      } else if (__any(!(big <= near))) {
#pragma unroll
        for (int j = 0; j < KB; ++j)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            // Score by score: the exponential's error is some 4e-7 of the cap.
            const float x = s[j][e], u = x * x;
            const float w = __builtin_amdgcn_exp2f(x * (2.f * kLog2e * c1));
            const float far = top * (1.f - 2.f * __builtin_amdgcn_rcpf(w + 1.f));
            const float low = x * fmaf(u, fmaf(u, fmaf(u, b3, b2), b1), b0);
            s[j][e] = (fabsf(x) <= near ? low : far) - m;
          }
      } else {
#pragma unroll
        for (int j = 0; j < KB; ++j)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float x = s[j][e], u = x * x;
            s[j][e] = fmaf(x, fmaf(u, fmaf(u, fmaf(u, b3, b2), b1), b0), -m);
          }
      }
    } else {
#pragma unroll
      for (int j = 0; j < KB; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[j][e] = fmaf(s[j][e], c2, -m);
    }
    if constexpr (kBias) {
      const float d0 = static_cast<float>(pos - key0 - 4 * hh);
#pragma unroll
      for (int j = 0; j < KB; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          s[j][e] = fmaf(-slope, fabsf(d0 - static_cast<float>(32 * j + 8 * (e >> 2) + (e & 3))),
                         s[j][e]);
    }
    if (masked) {
      const float hidden = -INFINITY;
      if constexpr (kTree) {
        // Bit x: whether the row sees key key0 + x. The bits of place `from` on
        // of the drafted tokens, below which every key is seen, up to the end.
        const int from = key0 - tree0, left = min(limit, k_hi) - key0;
        auto word = [&](int i) __attribute__((always_inline)) -> uint64_t {
          return live && i < p.words ? static_cast<uint64_t>(p.bits[row * p.words + i]) : 0u;
        };
        uint64_t sees = ~uint64_t(0);
        if (from >= 0) {
          const int shift = from & 63;
          sees = word(from >> 6) >> shift;
          if (shift > 0) sees |= word((from >> 6) + 1) << (64 - shift);
        } else if (from > -64) {
          sees = (sees >> (64 + from)) | word(0) << -from;
        }
        if (left < 64) sees = left > 0 ? sees & ~uint64_t(0) >> (64 - left) : 0u;
        sees >>= 4 * hh;
#pragma unroll
        for (int j = 0; j < KB; ++j) {
          const uint32_t half = static_cast<uint32_t>(sees >> (32 * j));
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            // All ones where the key is seen.
            const int keep = static_cast<int>(half << (31 - 8 * (e >> 2) - (e & 3))) >> 31;
            s[j][e] = __int_as_float((__float_as_int(s[j][e]) & keep) |
                                     (__float_as_int(hidden) & ~keep));
          }
        }
      } else {
        // Key `at` of the tile is seen if at - from < lim - from, unsigned. One
        // compare and select at a time: 32 compares side by side would take 64
        // scalar registers, and every uniform value of the loop would be spilled.
        const int from = max(low - key0 - 4 * hh, -128);
        const int lim = min(min(limit, k_hi) - key0 - 4 * hh, 128);
        const uint32_t span = static_cast<uint32_t>(max(lim - from, 0));
#pragma unroll
        for (int j = 0; j < KB; ++j)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const uint32_t at = 32 * j + 8 * (e >> 2) + (e & 3) - from;
            float x = s[j][e];
            asm volatile("v_cmp_lt_u32 vcc, %1, %2\n\tv_cndmask_b32 %0, %3, %0, vcc"
                         : "+v"(x)
                         : "v"(at), "v"(span), "v"(hidden)
                         : "vcc");
            s[j][e] = x;
          }
      }
      if (bad != 0) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (bad >> r & 1) {
#pragma unroll
            for (int e = 0; e < 8; ++e) s[r >> 1][8 * (r & 1) + e] = hidden;
          }
      }
    }
    float mc[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const f32x16_t &x = s[c >> 1];
      const int b = 8 * (c & 1);
      mc[c] = max3(max3(x[b], x[b + 1], x[b + 2]), x[b + 3], x[b + 4]);
      mc[c] = __builtin_elementwise_maximum(max3(mc[c], x[b + 5], x[b + 6]), x[b + 7]);
    }
    const float rel = pair_max(__builtin_elementwise_maximum(
        max3(mc[0], mc[1], mc[2]), mc[3]));
    if (__any(rel > thr)) {
      // Rows below their threshold keep m: a factor of 1. A row without a key so
      // far has sums of 0, whatever the factor.
      const bool move = rel > thr;
      const float shift = move ? rel - kBelow : 0.f;
      const float fall = move && thr > 0.f ? __builtin_amdgcn_exp2f(-shift) : 1.f;
      l *= fall;
#pragma unroll
      for (int n = 0; n < NB; ++n) acc[n] *= fall;
      m += shift;
      if (move) thr = kLazy + kBelow;
#pragma unroll
      for (int j = 0; j < KB; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[j][e] -= shift;
    }
    float lsum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < KB; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s[j][e] = __builtin_amdgcn_exp2f(s[j][e]);
        lsum[e & 3] += s[j][e];
      }
    l += (lsum[0] + lsum[1]) + (lsum[2] + lsum[3]);

#pragma unroll
    for (int j = 0; j < KB; ++j)
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        if constexpr (kTree) two_parts<T>(s[j][2 * x], s[j][2 * x + 1], pk[j][x], pl[j][x]);
        else pk[j][x] = pack2<T>(s[j][2 * x], s[j][2 * x + 1]);
      }
  };
  // s_waitcnt: all but the newest batch of copies, and LDS; LDS and scalars alone.
  constexpr int kBatch = 2 * kCopies;
  constexpr int kWaitBatch = (kBatch & 15) | ((kBatch >> 4) << 14) | 0x70;
  constexpr int kWaitLds = 0xC07F;
  Span next_k{}, next_v{};
  int64_t id = 0;
  auto m_phase = [&](int i, const unsigned char *kt, const unsigned char *vt)
      __attribute__((always_inline)) {
    const int64_t id3 = id_of(i + 3);
    __builtin_amdgcn_s_setprio(3);
    if (i >= 1 && active(i - 1)) add_values(vt);
    __builtin_amdgcn_sched_barrier(0);
    if (active(i)) {
      scores(kt);
    } else {  // defined in every phase, so that it lives over none
#pragma unroll
      for (int j = 0; j < KB; ++j) asm volatile("" : "=v"(s[j]));
    }
    __builtin_amdgcn_s_setprio(0);
    next_v = next_k;
    next_k = span_of(i + 2, id);
    id = id3;
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(kWaitLds);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  // vt: the stage of V_{i+1}; vi: that of V_i, which has landed when the copies
  // of this phase are the only ones left.
  auto v_phase = [&](int i, unsigned char *kt, unsigned char *vt, unsigned char *vi)
      __attribute__((always_inline)) {
    copy(next_k, p.k, kt);
    copy(next_v, p.v, vt);
    if (active(i)) {
      weigh(i);
    } else {
#pragma unroll
      for (int j = 0; j < KB; ++j)
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          asm volatile("" : "=v"(pk[j][x]));
          if constexpr (kTree) asm volatile("" : "=v"(pl[j][x]));
        }
    }
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(kWaitBatch);
    if (key_of(i) > unit_to || key_of(i) < low) {  // uniform
      clean(vi);
      __builtin_amdgcn_s_waitcnt(kWaitBatch);
    }
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  if (chunk > 0) {  // uniform: without keys the table is not read
    const int64_t id0 = id_of(0), id1 = id_of(1);
    id = id_of(2);
    const Span first = span_of(0, id0);
    next_k = span_of(1, id1);
    copy(first, p.k, ks0[half]);
    copy(first, p.v, vs0[half]);
    copy(next_k, p.k, ks1[half]);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0);
    __builtin_amdgcn_s_barrier();
    if (half == 1) __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    for (int i = 0; i < chunk; i += 2) {
      m_phase(i, ks0[half], vs1[half]);
      v_phase(i, ks0[half], vs1[half], vs0[half]);
      m_phase(i + 1, ks1[half], vs0[half]);
      v_phase(i + 1, ks1[half], vs0[half], vs1[half]);
    }
    // The last tile's values; an odd count had them in the phase past its end.
    if ((chunk & 1) == 0) m_phase(chunk, ks0[half], vs1[half]);
    if (half == 0) __builtin_amdgcn_s_barrier();
    __syncthreads();
    if (s_odd) {  // rare: values that are not finite, for the rows that see them
      const int end = min(k_hi, k_lo + t_hi * kTile);
      for (int k = max(first_key, low); k < end; ++k) {
        // Only tiles that were looked through.
        const int key0 = k_lo + (k - k_lo) / kTile * kTile;
        if (key0 <= unit_to && key0 >= low) continue;
        const int64_t block = table[k >> bs_log2];
        if (!known(block) || k >= limit) continue;
        if (kTree && k >= tree0 && !bit_of(p, row, k - tree0)) continue;
        const uint16_t *v = static_cast<const uint16_t *>(p.v) +
                            ((block << bs_log2) + (k & bs_mask)) * (row_bytes / 2) + kv_bytes / 2;
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int dim = 32 * n + 8 * (e >> 2) + 4 * hh + (e & 3);
            const float x = dim < p.d ? Elem<T>::to_f32(T{v[dim]}) : 0.f;
            if (!__builtin_isfinite(x)) acc[n][e] += x;
          }
      }
    }
  }
  l = pair_sum(l);
  if (thr < 0.f) m = -INFINITY;

  // The second half hands (m, l, O^T) over through the stage buffers, word by
  // word, lanes side by side.
  constexpr int kWords = 16 * NB + 2;
  static_assert(sizeof(ks0) >= kWords * 64 * sizeof(float), "hand-over buffer");
  float *mine = reinterpret_cast<float *>(w == 0 ? &ks0[0][0] : w == 1 ? &ks1[0][0]
                                          : w == 2 ? &vs0[0][0] : &vs1[0][0]);
  auto word = [&](int a) __attribute__((always_inline)) -> float * {
    return mine + a * 64 + lane;
  };
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  if (half == 1) {
    *word(0) = m;
    *word(1) = l;
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int e = 0; e < 16; ++e) *word(2 + 16 * n + e) = acc[n][e];
  }
  __syncthreads();
  if (half == 1) return;
  const float m1 = *word(0), l1 = *word(1);
  const float all_m = fmaxf(m, m1), ref = all_m == -INFINITY ? 0.f : all_m;
  const float f0 = __builtin_amdgcn_exp2f(m - ref), f1 = __builtin_amdgcn_exp2f(m1 - ref);
  const float sum = l * f0 + l1 * f1;
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[n][e] = acc[n][e] * f0 + *word(2 + 16 * n + e) * f1;

  // What the end needs of the arguments is read again here, and the row made
  // again, rather than kept over the loop.
  typedef const __attribute__((address_space(4))) ScoredParams const_params;
  const_params *late = (const_params *)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(late));
  int lane2 = m32;
  asm volatile("" : "+v"(lane2));
  const int r2 = r_first + lane2;
  if (r2 >= unit_rows) return;
  if (!alone) {
    const int64_t at = (item * late->hkv + kvh) * kTileRows + 32 * w + lane2;
    if (hh == 0) {
      // Partial results are in units of the natural exponent.
      late->ml[2 * at] = all_m * 0.6931471805599453f;
      late->ml[2 * at + 1] = sum;
    }
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const float4 x = make_float4(acc[n][4 * g], acc[n][4 * g + 1], acc[n][4 * g + 2],
                                     acc[n][4 * g + 3]);
        *reinterpret_cast<float4 *>(late->acc + at * D + 32 * n + 8 * g + 4 * hh) = x;
      }
    return;
  }
  const int group = late->group, tok2 = r2 / group, head2 = kvh * group + r2 - tok2 * group;
  const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
  const int64_t o_st = late->o_st, o_sh = late->o_sh;
  uint16_t *o = static_cast<uint16_t *>(late->out) + (q_first + tok2) * o_st + head2 * o_sh;
  const bool wide =
      o_st % 4 == 0 && o_sh % 4 == 0 && reinterpret_cast<uintptr_t>(late->out) % 8 == 0;
  const int d = late->d;
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int e0 = 32 * n + 8 * g + 4 * hh;
      if (e0 >= d) continue;
      uint16_t x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        x[e] = __builtin_bit_cast(uint16_t, Elem<T>::from_f32(acc[n][4 * g + e] * inv));
      if (wide) {
        *reinterpret_cast<uint2 *>(o + e0) =
            make_uint2(x[0] | static_cast<uint32_t>(x[1]) << 16,
                       x[2] | static_cast<uint32_t>(x[3]) << 16);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e0 + e] = x[e];
      }
    }
}

template <typename T, int D>
int launch_tiles(const ScoredParams &p, unsigned grid, hipStream_t stream) {
#define MLR_TILES(C, B, R) scored_tiles_kernel<T, D, C, B, R><<<grid, kThreads, 0, stream>>>(p)
  if (p.bits) {
    if (p.cap > 0) MLR_TILES(true, false, true); else MLR_TILES(false, false, true);
  } else if (p.cap > 0) {
    if (p.slopes) MLR_TILES(true, true, false); else MLR_TILES(true, false, false);
  } else {
    if (p.slopes) MLR_TILES(false, true, false); else MLR_TILES(false, false, false);
  }
#undef MLR_TILES
  return check_launch("scored_tiles");
}

}  // namespace

int launch_scored_tiles(const ScoredParams &p, int dtype, unsigned grid, hipStream_t stream) {
  if (dtype == MLR_DTYPE_F16)
    return p.d > 64 ? launch_tiles<f16_t, 128>(p, grid, stream)
                    : launch_tiles<f16_t, 64>(p, grid, stream);
  return p.d > 64 ? launch_tiles<bf16_t, 128>(p, grid, stream)
                  : launch_tiles<bf16_t, 64>(p, grid, stream);
}

}  // namespace mlr

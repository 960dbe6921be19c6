// What the scored attention kernels, and those of drafted trees, weighed keys and selected
// blocks, share: a call's operands, the cut of its
// work into items, the scores, and the layout of partial results.
//
// A unit is a group of query rows that share their keys: kRows consecutive rows
// of one sequence and KV head, a row being one (token, query head of the KV
// head's group), tokens first. Its keys are cut into splits, alike in length;
// an item is one (unit, split, KV head). The longest split is chosen on the
// device from the lengths themselves: the whole call makes about `target`
// items whatever the table's width says, and the same lengths always give the
// same splits.
#pragma once

#include "mlr_common.h"

namespace mlr {

enum ScoredMode {
  kModePrefill = 0,  // packed chunks, causal, prefixes seen ahead
  kModeDecode = 1,   // one token a sequence
  kModePrefix = 2,   // one token a sequence, the keys [0, prefix) of one table
  kModeShared = 3,   // units of kModePrefix, then one unit per sequence of kModeDecode
};

constexpr int kMinSplit = 128;  // keys of the shortest split

// tanh(y) = y (kTanh0 + kTanh1 y^2 + kTanh2 y^4 + kTanh3 y^6) for |y| <= 1/2, with a
// relative error of 5.1e-7.
constexpr float kTanh0 = 0.99999949f, kTanh1 = -0.33326618f;
constexpr float kTanh2 = 0.13193061f, kTanh3 = -0.044465f;

struct ScoredParams {
  const void *q, *k, *v;
  int64_t q_st, q_sh;
  int64_t num_blocks, block_size;
  int hkv, group, d, hq;
  const int64_t *bt, *ctx, *qsl, *ahead;
  int64_t bt_st, bt_width;
  int64_t bt_sh;           // from one KV head's table to the next's; 0: one table for all
  int seqs, tiles;         // sequences; units of a sequence (kModePrefix: of the call)
  int64_t total_q;         // rows of q
  int64_t start;           // first key (kModeDecode), number of keys (kModePrefix), both
  const int64_t *prefix;   // kModePrefix, kModeShared: the prefix's table
  int64_t prefix_width;
  int prefix_units;        // kModeShared: units over the prefix
  float scale, cap;
  const float *slopes;
  const int64_t *bits;     // kModePrefill: what each row sees of its sequence's last tokens,
  int words;               // `words` words a row (null: causal)
  float *scores;           // kModeDecode: where to leave the scores (null: nowhere),
  int64_t scores_st;       // [seqs * hq][scores_st]
  bool fine;               // kModeDecode: probabilities in two parts (two_parts); trees and
                           // decodes that leave their scores always have them so
  void *out;
  int64_t o_st, o_sh;
  int mode, units;
  bool force_partial;      // results go to the workspace even of a single split
  int64_t target;          // items the call is cut into, about
  bool whole;              // no splits: an item is a unit
  int bs_log2, ncu;        // log2 of block_size (-1: no power of two); CUs of the GPU
  int *first;              // [units + 1]: items before each unit (of one KV head)
  float *ml, *acc;         // [items][kRows][2], [items][kRows][D] of partial results
};

// One unit's rows and keys.
struct Unit {
  int64_t q0;      // row of q of the sequence's first token
  int64_t pos0;    // position of that token (kModePrefill)
  int64_t ctx;     // keys of the sequence
  int64_t ahead;   // keys visible to every query
  int64_t lo, hi;  // keys [lo, hi) that some row sees
  int rows, r0;    // rows of the sequence; first of the unit
  int seq;
  bool prefix;     // over the shared prefix: keys by its table, rows of all sequences
};

__device__ __forceinline__ const int64_t *table_of(const ScoredParams &p, const Unit &t) {
  return t.prefix ? p.prefix : p.bt + t.seq * p.bt_st;
}

// Whether row `row` sees the key at place `node` >= 0 of its sequence's last tokens.
__device__ __forceinline__ bool bit_of(const ScoredParams &p, int64_t row, int node) {
  const int word = node >> 6;
  return word < p.words && (static_cast<uint64_t>(p.bits[row * p.words + word]) >> (node & 63) & 1);
}

// Two probabilities a and b as operands of 16 bits, hi + lo each, which a product with V adds
// up in FP32: hi is cut off, not rounded, and lo is more than 0 wherever hi is (in bf16 down
// to probabilities of 2^-103), so that an infinite V stays one: hi times it and lo times it
// have one sign, and neither is 0 times it. lo, up to 2^-7 of the probability in bf16 and
// 2^-10 in fp16, is rounded by 2^-8 and 2^-11 of itself: 2^-15 and 2^-21 of the probability.
// fp16 takes numbers scaled up to 2^15, of which it drops 2^-24 at most, 2^-39 of that.
template <typename T>
__device__ __forceinline__ void two_parts(float a, float b, uint32_t &hi, uint32_t &lo) {
  typedef float f32x2_v __attribute__((ext_vector_type(2)));
  if constexpr (std::is_same_v<T, bf16_t>) {
    typedef __bf16 h2 __attribute__((ext_vector_type(2)));
    const uint32_t ua = __float_as_uint(a), ub = __float_as_uint(b);
    constexpr float kMore = 1.f + 0x1p-23f;
    hi = __builtin_amdgcn_perm(ub, ua, 0x07060302);
    lo = __builtin_bit_cast(
        uint32_t, __builtin_convertvector(
                      f32x2_v{fmaf(a, kMore, -__uint_as_float(ua & 0xffff0000u)),
                              fmaf(b, kMore, -__uint_as_float(ub & 0xffff0000u))}, h2));
  } else {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const h2 cut = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_pkrtz(a, b));
    hi = __builtin_bit_cast(uint32_t, cut);
    const float la = a - static_cast<float>(cut[0]), lb = b - static_cast<float>(cut[1]);
    lo = __builtin_bit_cast(
        uint32_t, __builtin_convertvector(f32x2_v{fmaxf(la, fminf(a, 0x1p-24f)),
                                                  fmaxf(lb, fminf(b, 0x1p-24f))}, h2));
  }
}

__device__ __forceinline__ int64_t clamp64(int64_t x, int64_t lo, int64_t hi) {
  return x < lo ? lo : x > hi ? hi : x;
}

__device__ __forceinline__ Unit unit_of(const ScoredParams &p, int u, int kRows) {
  Unit t;
  const bool prefix =
      p.mode == kModePrefix || (p.mode == kModeShared && u < p.prefix_units);
  t.prefix = prefix;
  if (p.mode == kModeShared && !prefix) u -= p.prefix_units;
  t.seq = prefix ? 0 : u / p.tiles;
  t.r0 = (u - t.seq * p.tiles) * kRows;
  const int64_t covered = p.bt_width * p.block_size;
  t.pos0 = t.ahead = 0;
  t.lo = 0;
  if (p.mode == kModePrefill) {
    t.q0 = clamp64(p.qsl[t.seq], 0, p.total_q);
    const int64_t end = clamp64(p.qsl[t.seq + 1], t.q0, p.total_q);
    t.ctx = clamp64(p.ctx[t.seq], 0, covered);
    t.pos0 = t.ctx - (end - t.q0);
    // With bits, which keys a row sees of the last ones is up to them.
    t.ahead = p.bits ? t.ctx : p.ahead ? clamp64(p.ahead[t.seq], 0, t.ctx) : 0;
    // Rows past the declared longest chunk have no unit.
    const int64_t rows = (end - t.q0) * p.group, most = static_cast<int64_t>(p.tiles) * kRows;
    t.rows = static_cast<int>(rows < most ? rows : most);
    t.hi = 0;
    if (t.r0 < t.rows) {
      const int last = (t.rows < t.r0 + kRows ? t.rows : t.r0 + kRows) - 1;
      t.hi = t.pos0 + last / p.group + 1;
      if (t.hi < t.ahead) t.hi = t.ahead;
      if (t.hi < 0) t.hi = 0;
    }
  } else if (!prefix) {
    t.q0 = t.seq;
    t.ctx = clamp64(p.ctx[t.seq], 0, covered);
    t.rows = p.group;
    t.hi = t.ctx;
    t.lo = p.start;
  } else {
    t.q0 = 0;
    t.ctx = 0;
    t.rows = p.seqs * p.group;
    const int64_t most = p.prefix_width * p.block_size;
    t.hi = p.start < most ? p.start : most;
  }
  return t;
}

// Splits of a unit start at multiples of 16 keys.
__device__ __forceinline__ int64_t unit_base(const Unit &t) { return t.lo & ~int64_t(15); }
__device__ __forceinline__ int64_t unit_len(const Unit &t) {
  return t.hi > t.lo && t.r0 < t.rows ? t.hi - unit_base(t) : 0;
}
// A unit with rows but no key has one item, which writes what an empty sum gives.
// Lengths are below 2^31 and the split at least kMinSplit.
__device__ __forceinline__ int items_of(int64_t len, int split) {
  const uint32_t n = (static_cast<uint32_t>(len) + split - 1) / static_cast<uint32_t>(split);
  return n > 0 ? static_cast<int>(n) : 1;
}
__device__ __forceinline__ int unit_items(const Unit &t, int split) {
  return t.r0 < t.rows ? items_of(unit_len(t), split) : 0;
}
// Length of the n items of a unit: alike, up to `step` keys, a power of two that
// divides the split length; so none is longer than that, and none is empty.
__device__ __forceinline__ int item_len(const Unit &t, int n, int step) {
  const uint32_t len = static_cast<uint32_t>(unit_len(t));
  return static_cast<int>(((len + n - 1) / static_cast<uint32_t>(n) + step - 1) & -step);
}
// In floating point, as the 64-bit division takes longer; the same everywhere.
__device__ __forceinline__ int split_of(int64_t total_keys, const ScoredParams &p) {
  const double s = static_cast<double>(total_keys) * p.hkv / static_cast<double>(p.target);
  const int split = s < 2.0e9 ? static_cast<int>(s) + 1 : 0x7fffff80;  // past every length
  return ((split > kMinSplit ? split : kMinSplit) + 63) & ~63;
}

// Whether a prefill of `units` units of 128 rows over all KV heads, the longest of
// `keys` keys, gains from splits: whole it takes the time of its longest unit, split
// the partial results of all units take theirs. bf16, whole and split, us:
//   14 units of 1,024 and 4,096 keys, head size 64: 24 and 20, 65 and 24
//   56 units of 1,024, 2,048 and 4,096 keys: 25 and 27, 38 and 31, 66 and 46
//   32 units of 512, 1,024 and 2,048 keys, head size 128: 20 and 26, 28 and 28, 43 and 31
//   128 units of 2,048, 4,096 and 16,384 keys: 45 and 53, 75 and 71, 260 and 183
//   224 units of 4,096 and 16,384 keys, head size 64: 68 and 96, 250 and 245
__host__ __device__ inline bool splits_pay(int64_t units, int64_t keys, int cus) {
  return 2 * units <= cus && keys > 512 + units * units / 4;
}

int launch_scored_rows(const ScoredParams &p, int dtype, unsigned grid, hipStream_t stream);

// Rows of a unit of that kernel, and a call of it over single tokens: its operands, the
// checks that all entry points share, its cut into items and its workspace.
constexpr int kRows = 16;
struct Operands {
  const char *what;
  const void *q;
  int64_t q_st, q_sh;
  const void *k, *v;
  int64_t num_blocks, block_size, hkv, d;
  const int64_t *bt;
  int64_t bt_st, bt_width;
  const int64_t *ctx;
  int64_t seqs, hq;
  double scale, cap;
  const float *slopes;
  int dtype;
  const void *out;
  int64_t o_st, o_sh;
};
int check_operands(const Operands &o);
ScoredParams params_of(const Operands &o, int mode);
size_t decode_workspace(int64_t batch, int64_t hq, int64_t hkv, int64_t d, int64_t max_keys);
// Plans a decode and places its partial results; the number of its items.
int64_t plan_decode(ScoredParams &p, int64_t max_keys, char *workspace);
// Whether units of up to max_keys keys are better left whole on that kernel: cutting them
// costs each workgroup its planning and the call a launch to join the parts, some 8 us, and
// a workgroup takes 2.5 us for 32 KB of keys (FP32, head size 64, whole and cut: 320 keys
// 14.4 and 15.6 us, 640 keys 19.5 and 13.5 us).
inline bool short_keys(int64_t max_keys, int64_t d, int dtype) {
  return max_keys * (d > 64 ? 128 : 64) * dtype_size(dtype) <= 80 << 10;
}
unsigned grid_of(int64_t items);
int merge_decode(const ScoredParams &p, int dtype, hipStream_t stream);
size_t align256(size_t n);

// Units of 128 rows; bf16 and fp16, block_size a power of two from 16 on. Drafted trees
// that are not left whole: at most kTreeSeqs sequences.
constexpr int kTileRows = 128, kTreeSeqs = 512;
int launch_scored_tiles(const ScoredParams &p, int dtype, unsigned grid, hipStream_t stream);

}  // namespace mlr

// Entry points of paged attention with capped or biased scores, and the sum of
// the partial results that splits leave in the workspace.
#include "scored_attention.h"

#include <algorithm>

namespace mlr {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kRows = 16;

// out = sum_i e^{m_i - M} O_i / sum_i e^{m_i - M} l_i over a row's items: those
// of its unit u0 + u of `p` and, over a shared prefix, those of `x` too. One wave
// per row, 16 lanes side by side over its elements, four groups of lanes dealing
// the items among them, the groups' sums joined in a fixed order. A unit that has
// written its result itself is left alone. Rows from `used` on of a unit do not
// exist. Bound by latency: the row's m and l, then its sums, are each read in a few
// rounds (64 sequences of 14 heads of 64 and 10 items each: 4.3 us).
template <typename T, int D>
__global__ __launch_bounds__(256) void scored_merge(ScoredParams p, int u0, int p_rows, int used,
                                                    ScoredParams x, int x_rows, bool prefixed) {
  constexpr int kVe = D / 16;
  const int lane = threadIdx.x & 63;
  const int slots = (p.units - u0) * p.hkv * used;
  for (int slot = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); slot < slots;
       slot += gridDim.x * 4) {
    const int uk = slot / used, rr = slot - uk * used;
    const int u = u0 + uk / p.hkv, kvh = uk - uk / p.hkv * p.hkv;
    const int first = p.first[u], count = p.first[u + 1] - first;
    if (count == 0 || (count == 1 && !p.force_partial)) continue;
    const Unit t = unit_of(p, u, p_rows);
    const int r = t.r0 + rr;
    if (r >= t.rows) continue;
    const int d0 = (lane & 15) * kVe, group = lane >> 4;
    const int tok = r / p.group, g = r - tok * p.group;
    // Items of the row: `count` from p, then `more` from x.
    const int64_t at = (static_cast<int64_t>(first) * p.hkv + kvh) * p_rows + rr;
    int64_t x_at = 0;
    int more = 0;
    if (prefixed) {
      const int xr = t.seq * p.group + g;
      const int xu = xr / x_rows;
      const int x_first = x.first[xu];
      more = x.first[xu + 1] - x_first;
      x_at = (static_cast<int64_t>(x_first) * x.hkv + kvh) * x_rows + (xr - xu * x_rows);
    }
    const int64_t step = static_cast<int64_t>(p.hkv) * p_rows;
    const int64_t x_step = static_cast<int64_t>(p.hkv) * x_rows;
    float m = -INFINITY;
    for (int i = lane; i < count; i += 64) m = fmaxf(m, p.ml[2 * (at + i * step)]);
    for (int i = lane; i < more; i += 64) m = fmaxf(m, x.ml[2 * (x_at + i * x_step)]);
    m = wave_max(m);
    const float ref = m == -INFINITY ? 0.f : m;
    float sum = 0.f, acc[kVe];
#pragma unroll
    for (int n = 0; n < kVe; ++n) acc[n] = 0.f;
    auto add = [&](const ScoredParams &s, int64_t row) __attribute__((always_inline)) {
      const float f = __builtin_amdgcn_exp2f((s.ml[2 * row] - ref) * kLog2e);
      sum += s.ml[2 * row + 1] * f;
#pragma unroll
      for (int n = 0; n < kVe; n += 4) {
        const float4 v = *reinterpret_cast<const float4 *>(s.acc + row * D + d0 + n);
        acc[n] += v.x * f;
        acc[n + 1] += v.y * f;
        acc[n + 2] += v.z * f;
        acc[n + 3] += v.w * f;
      }
    };
#pragma unroll 8
    for (int i = group; i < count; i += 4) add(p, at + i * step);
#pragma unroll 8
    for (int i = group; i < more; i += 4) add(x, x_at + i * x_step);
    auto join = [](float v) {
      v += __shfl_xor(v, 16);
      return v + __shfl_xor(v, 32);
    };
    sum = join(sum);
#pragma unroll
    for (int n = 0; n < kVe; ++n) acc[n] = join(acc[n]);
    if (group != 0) continue;
    const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
    T *dst = static_cast<T *>(p.out) + (t.q0 + tok) * p.o_st + (kvh * p.group + g) * p.o_sh;
#pragma unroll
    for (int n = 0; n < kVe; ++n)
      if (d0 + n < p.d) dst[d0 + n] = Elem<T>::from_f32(acc[n] * inv);
  }
}

int launch_merge(const ScoredParams &p, int u0, int p_rows, const ScoredParams &x, int x_rows,
                 bool prefixed, int dtype, hipStream_t stream) {
  const int used = p.mode == kModePrefill ? p_rows : std::min(p_rows, p.group);
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(
      ceil_div(static_cast<int64_t>(p.units - u0) * p.hkv * used, 4), 1 << 20));
#define MLR_MERGE(T)                                                                         \
  if (p.d > 64)                                                                              \
    scored_merge<T, 128><<<grid, 256, 0, stream>>>(p, u0, p_rows, used, x, x_rows, prefixed);      \
  else                                                                                       \
    scored_merge<T, 64><<<grid, 256, 0, stream>>>(p, u0, p_rows, used, x, x_rows, prefixed)
  if (dtype == MLR_DTYPE_F32) {
    MLR_MERGE(float);
  } else if (dtype == MLR_DTYPE_F16) {
    MLR_MERGE(f16_t);
  } else {
    MLR_MERGE(bf16_t);
  }
#undef MLR_MERGE
  return check_launch("scored_merge");
}

int cus() {
  const int n = current_device_cus();
  return n > 0 ? n : 256;
}
// Items of the kernel of 16 rows a unit. `slots` workgroups run at once; units of
// different lengths make half an item each more than their keys ask for, and items
// past a full round cost a round. With too many units for one round, two rounds of
// shorter items even out better. 64 requests of 128 to 4,096 keys, us, this rule and
// two items for every CU: bf16, 14/2 heads of 64 25.1 and 27.6, 12/4 heads of 64 33.3
// and 37.9, 32/8 heads of 128 96 and 113; FP32, 32/8 heads of 128 193 and 256. (64
// requests of exactly 1,024 keys, 32/8 heads of 128: 51.5 and 44.9, as a unit for
// each of the 512 slots is a perfect round.)
int64_t rows_target(int64_t units, int64_t hkv, int64_t d) {
  const int64_t slots = (d > 64 ? 2 : 3) * static_cast<int64_t>(cus());
  const int64_t rounds = 3 * units * hkv <= 2 * slots ? 1 : 2;
  return std::max(slots / 2, rounds * slots - units * hkv / 2);
}

// Items of a call at most, over its KV heads, cut into about `target`.
int64_t max_items(int64_t units, int64_t hkv, int64_t max_keys, int64_t target) {
  const int64_t by_len = units * std::max<int64_t>(1, ceil_div(max_keys + 15, kMinSplit));
  return std::min(by_len, units + ceil_div(target, hkv) + 1) * hkv;
}

size_t align256(size_t n) { return (n + 255) & ~size_t(255); }

// Workspace of one kernel's partial results: [first | ml | acc].
size_t part_bytes(int64_t units, int64_t items, int64_t rows, int64_t d) {
  const int64_t wide = d > 64 ? 128 : 64;
  return align256((units + 1) * sizeof(int)) + align256(items * rows * 2 * sizeof(float)) +
         align256(items * rows * wide * sizeof(float));
}

char *place_parts(ScoredParams &p, char *ws, int64_t items, int64_t rows) {
  const int64_t wide = p.d > 64 ? 128 : 64;
  p.first = reinterpret_cast<int *>(ws);
  ws += align256((p.units + 1) * sizeof(int));
  p.ml = reinterpret_cast<float *>(ws);
  ws += align256(items * rows * 2 * sizeof(float));
  p.acc = reinterpret_cast<float *>(ws);
  return ws + align256(items * rows * wide * sizeof(float));
}

int64_t decode_units(int64_t batch, int64_t group) { return batch * ceil_div(group, kRows); }
int64_t prefill_units(int64_t seqs, int64_t max_q, int64_t group, int64_t rows) {
  return seqs * ceil_div(max_q * group, rows);
}
int64_t prefix_units(int64_t batch, int64_t group, int64_t rows) {
  return ceil_div(batch * group, rows);
}

// What the kernel of 128 rows a unit can run.
bool fits_tiles(int64_t block_size, int64_t hkv, int64_t d, int dtype) {
  return dtype != MLR_DTYPE_F32 && log2_if_pow2(block_size) >= 4 &&
         block_size < (int64_t(1) << 30) / (hkv * d);  // 32-bit offsets inside a block
}
// Whether a call with `rows` query rows per sequence and KV head goes to it: more
// than two of the other kernel's units (16 chunks after 4,096 keys, this kernel and
// the other: 28 rows 28.3 and 26.4 us, 35 rows 29.9 and 49.9 us at head size 64;
// 16 rows 81 and 65 us, 64 rows 87 and 175 us at 128).
bool takes_tiles(int64_t rows, int64_t block_size, int64_t hkv, int64_t d, int dtype) {
  return rows > 2 * kRows && fits_tiles(block_size, hkv, d, dtype);
}

// A shared prefix on the kernel of 128 rows a unit, with each request's own keys
// (all heads of a group in one unit) in the same launch: a launch less, also for
// few rows (8,192 keys shared by 2, 8 and 64 requests of 14/2 heads of 64: 16.4,
// 17.3 and 26.9 us, against 19.6, 22.9 and 29.6 us), and for long keys of the
// requests' own (2,000 shared and up to 4,000 own: 64 requests of 14/2 heads 29.1 and
// 38.3 us, 32 of 12/12 heads 65.8 and 75.3 us). At head sizes above 64 that
// kernel's stages take a whole CU, so a request's few keys would hold one each;
// there the requests' own keys go to the other kernel (16 and 64 requests of 32/8
// heads of 128: 33.9 and 45.1 us, in one launch 36.2 and 53.3 us).
// So they do where there are many of them: a unit's 128 rows of partial results hold
// one group only, 32 KB for each request and KV head, and from some four for every CU
// on reading and writing them takes longer than the launch saved. 4,096 shared and
// up to 300 own keys, one launch and two, us: 12/12 heads of 64, 64, 128 and 256
// requests 36.0 and 38.2, 53.7 and 47.4, 97.1 and 77.1; 32/32 heads, 32 and 128
// requests 42.6 and 52.2, 123.5 and 93.1; 8,192 shared and up to 1,000 own: 14/2 heads,
// 512 requests 83.0 and 86.1; 32/8 heads, 128 requests 65.0 and 69.5; but 2,000 shared
// and up to 100 own, 16/4 heads, 256 requests: 44.6 and 37.4.
bool shares_tiles(int64_t batch, int64_t group, int64_t block_size, int64_t hkv, int64_t d,
                  int dtype) {
  return d <= 64 && group <= kTileRows && batch * hkv <= 4 * static_cast<int64_t>(cus()) &&
         fits_tiles(block_size, hkv, d, dtype);
}
// Two workgroups fit a CU; the last split of each unit is half full on average, and
// a second round of workgroups would cost more than longer splits.
int64_t shared_target(int64_t units, int64_t hkv) {
  const int64_t slots = 2 * static_cast<int64_t>(cus());
  return std::max(slots / 2, slots - units * hkv / 2);
}
// For a prefix alone: items of equal length, one for each CU at most.
int64_t prefix_target(int64_t units, int64_t hkv) {
  return std::max<int64_t>(1, cus() / (units * hkv)) * units * hkv;
}

// Items of a prefill on that kernel: one for each CU, less the last splits of the
// units, half full on average.
int64_t tiles_target(int64_t units, int64_t hkv) {
  return std::max<int64_t>(cus() / 2, cus() - units * hkv / 2);
}

// A prefill's rows per unit, units, items, and whether units stay whole. Splits on
// the kernel of 128 rows cost a pass over FP32 partial results of every unit, so
// they pay only where units are few and their keys many (see splits_pay); the kernel
// decides that from the lengths, and what no lengths could change is decided here.
// On the other kernel a call of so many units that their partial results would pass
// kMostParts (a batch of one long prompt and many short ones has room for as many
// long ones) has enough items without splits.
constexpr size_t kMostParts = size_t(256) << 20;
struct PrefillPlan {
  int64_t rows, units, items, target;
  bool whole, parts;
};
PrefillPlan plan_prefill(int64_t seqs, int64_t max_q, int64_t max_keys, int64_t block_size,
                         int64_t hq, int64_t hkv, int64_t d, int dtype) {
  const int64_t group = hq / hkv;
  PrefillPlan n;
  const bool tiles = takes_tiles(max_q * group, block_size, hkv, d, dtype);
  n.rows = tiles ? kTileRows : kRows;
  n.units = prefill_units(seqs, max_q, group, n.rows);
  n.target = tiles ? tiles_target(n.units, hkv) : rows_target(n.units, hkv, d);
  n.items = max_items(n.units, hkv, max_keys, n.target);
  n.whole = tiles ? !splits_pay(n.units * hkv, max_keys, cus())
                  : part_bytes(n.units, n.items, kRows, d) > kMostParts;
  if (n.whole) {
    n.target = 1;  // a split as long as all keys
    n.items = n.units * hkv;
  }
  n.parts = !n.whole && max_keys > kMinSplit;
  return n;
}

bool head_dim_ok(int64_t d, int dtype) {
  return d > 0 && d <= 128 && d % (dtype == MLR_DTYPE_F32 ? 4 : 8) == 0;
}

// The kernels count positions in 32 bits, up to a few tiles past the last.
bool covers_less(int64_t blocks, int64_t block_size) {
  return blocks < (int64_t(1) << 31) / block_size &&
         blocks * block_size <= (int64_t(1) << 31) - 4096;
}

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

int check_operands(const Operands &o) {
  const char *w = o.what;
  MLR_REQUIRE(o.dtype == MLR_DTYPE_F32 || o.dtype == MLR_DTYPE_F16 || o.dtype == MLR_DTYPE_BF16,
              "%s: unsupported dtype %d", w, o.dtype);
  MLR_REQUIRE(o.seqs >= 0 && o.seqs < (1 << 24), "%s: number of sequences must be in [0, 2^24)", w);
  MLR_REQUIRE(o.hkv > 0 && o.hq > 0 && o.hq % o.hkv == 0 && o.hq < (1 << 16),
              "%s: query heads must be a positive multiple of the KV heads, below 2^16", w);
  MLR_REQUIRE(head_dim_ok(o.d, o.dtype),
              "%s: head_dim must be a multiple of %d up to 128, got %lld", w,
              o.dtype == MLR_DTYPE_F32 ? 4 : 8, static_cast<long long>(o.d));
  MLR_REQUIRE(o.num_blocks > 0 && o.num_blocks < (int64_t(1) << 31) && o.block_size > 0 && o.bt_width >= 0,
              "%s: the cache needs fewer than 2^31 blocks of a positive size", w);
  MLR_REQUIRE(covers_less(o.bt_width, o.block_size),
              "%s: a block table must cover fewer than 2^31 positions", w);
  // A cap so small that its inverse is infinite would make NaN of scores of 0.
  MLR_REQUIRE(o.cap == 0 || (o.cap >= 1e-30 && o.cap <= 1e30),
              "%s: softcap must be 0 (off) or in [1e-30, 1e30]", w);
  MLR_REQUIRE(o.scale == o.scale && o.scale - o.scale == 0, "%s: scale must be finite", w);
  const int64_t vec = 16 / dtype_size(o.dtype);
  MLR_REQUIRE(o.q_st % vec == 0 && o.q_sh % vec == 0 && reinterpret_cast<uintptr_t>(o.q) % 16 == 0,
              "%s: q rows must start at multiples of 16 bytes", w);
  MLR_REQUIRE((reinterpret_cast<uintptr_t>(o.k) | reinterpret_cast<uintptr_t>(o.v)) % 16 == 0,
              "%s: the cache must be 16-byte aligned", w);
  return MLR_OK;
}

ScoredParams params_of(const Operands &o, int mode) {
  ScoredParams p{};
  p.q = o.q;
  p.k = o.k;
  p.v = o.v;
  p.q_st = o.q_st;
  p.q_sh = o.q_sh;
  p.num_blocks = o.num_blocks;
  p.block_size = o.block_size;
  p.hkv = static_cast<int>(o.hkv);
  p.hq = static_cast<int>(o.hq);
  p.group = static_cast<int>(o.hq / o.hkv);
  p.d = static_cast<int>(o.d);
  p.bt = o.bt;
  p.bt_st = o.bt_st;
  p.bt_width = o.bt_width;
  p.ctx = o.ctx;
  p.seqs = static_cast<int>(o.seqs);
  p.total_q = o.seqs;
  p.scale = static_cast<float>(o.scale);
  p.cap = static_cast<float>(o.cap);
  p.slopes = o.slopes;
  p.out = const_cast<void *>(o.out);
  p.o_st = o.o_st;
  p.o_sh = o.o_sh;
  p.mode = mode;
  p.ncu = cus();
  p.bs_log2 = log2_if_pow2(o.block_size);
  return p;
}

unsigned grid_of(int64_t items) { return static_cast<unsigned>(std::min<int64_t>(items, 1024)); }

}  // namespace
}  // namespace mlr

using namespace mlr;

extern "C" size_t mlr_paged_decode_scored_workspace_size(int64_t batch, int64_t num_q_heads,
                                                         int64_t num_kv_heads, int64_t head_dim,
                                                         int64_t max_context) {
  if (batch <= 0 || num_kv_heads <= 0 || num_q_heads <= 0 || max_context <= kMinSplit) return 0;
  const int64_t units = decode_units(batch, num_q_heads / num_kv_heads);
  return part_bytes(units, max_items(units, num_kv_heads, max_context,
                                     rows_target(units, num_kv_heads, head_dim)),
                    kRows, head_dim);
}

extern "C" int mlr_paged_decode_scored(
    const void *q, int64_t q_stride_b, int64_t q_stride_h, const void *k_cache,
    const void *v_cache, int64_t num_blocks, int64_t block_size, int64_t num_kv_heads,
    int64_t head_dim, const int64_t *block_tables, int64_t bt_stride, int64_t max_blocks,
    const int64_t *seq_lens, int64_t batch, int64_t num_q_heads, double scale, double softcap,
    const float *alibi_slopes, int dtype, void *workspace, size_t workspace_bytes, void *out,
    int64_t out_stride_b, int64_t out_stride_h, void *stream) {
  clear_error();
  const Operands o{"mlr_paged_decode_scored", q, q_stride_b, q_stride_h, k_cache, v_cache,
                   num_blocks, block_size, num_kv_heads, head_dim, block_tables, bt_stride,
                   max_blocks, seq_lens, batch, num_q_heads, scale, softcap, alibi_slopes, dtype,
                   out, out_stride_b, out_stride_h};
  if (const int rc = check_operands(o)) return rc;
  if (batch == 0) return MLR_OK;
  MLR_REQUIRE(batch * num_q_heads < (int64_t(1) << 28), "%s: too many query rows", o.what);
  MLR_REQUIRE(q && k_cache && v_cache && (block_tables || max_blocks == 0) && seq_lens && out,
              "mlr_paged_decode_scored: null pointer");
  const int64_t max_keys = max_blocks * block_size;
  const size_t need = mlr_paged_decode_scored_workspace_size(batch, num_q_heads, num_kv_heads,
                                                             head_dim, max_keys);
  MLR_REQUIRE(need == 0 || (workspace && workspace_bytes >= need),
              "mlr_paged_decode_scored: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  ScoredParams p = params_of(o, kModeDecode);
  p.tiles = static_cast<int>(ceil_div(p.group, kRows));
  p.units = static_cast<int>(decode_units(batch, p.group));
  p.target = rows_target(p.units, p.hkv, p.d);
  const int64_t items = max_items(p.units, p.hkv, max_keys, p.target);
  if (need) place_parts(p, static_cast<char *>(workspace), items, kRows);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (const int rc = launch_scored_rows(p, dtype, grid_of(items), s)) return rc;
  return need ? launch_merge(p, 0, kRows, p, kRows, false, dtype, s) : MLR_OK;
}

extern "C" size_t mlr_paged_prefill_scored_workspace_size(int64_t num_seqs, int64_t max_query_len,
                                                          int64_t max_blocks, int64_t block_size,
                                                          int64_t num_q_heads,
                                                          int64_t num_kv_heads, int64_t head_dim,
                                                          int dtype) {
  if (num_seqs <= 0 || max_query_len <= 0 || num_kv_heads <= 0 || num_q_heads <= 0 ||
      head_dim <= 0 || block_size <= 0)
    return 0;
  const PrefillPlan n = plan_prefill(num_seqs, max_query_len, max_blocks * block_size, block_size,
                                     num_q_heads, num_kv_heads, head_dim, dtype);
  return n.parts ? part_bytes(n.units, n.items, n.rows, head_dim) : 0;
}

extern "C" int mlr_paged_prefill_scored(
    const void *q, int64_t q_stride_t, int64_t q_stride_h, const void *k_cache,
    const void *v_cache, int64_t num_blocks, int64_t block_size, int64_t num_kv_heads,
    int64_t head_dim, const int64_t *block_tables, int64_t bt_stride, int64_t max_blocks,
    const int64_t *query_start_loc, const int64_t *context_lens, const int64_t *prefix_lens,
    int64_t num_seqs, int64_t total_q, int64_t max_query_len, int64_t num_q_heads, double scale,
    double softcap, const float *alibi_slopes, int dtype, void *workspace, size_t workspace_bytes,
    void *out, int64_t out_stride_t, int64_t out_stride_h, void *stream) {
  clear_error();
  const Operands o{"mlr_paged_prefill_scored", q, q_stride_t, q_stride_h, k_cache, v_cache,
                   num_blocks, block_size, num_kv_heads, head_dim, block_tables, bt_stride,
                   max_blocks, context_lens, num_seqs, num_q_heads, scale, softcap, alibi_slopes,
                   dtype, out, out_stride_t, out_stride_h};
  if (const int rc = check_operands(o)) return rc;
  MLR_REQUIRE(total_q >= 0 && max_query_len >= 0,
              "mlr_paged_prefill_scored: token counts must be >= 0");
  if (num_seqs == 0 || total_q == 0 || max_query_len == 0) return MLR_OK;
  MLR_REQUIRE(q && k_cache && v_cache && (block_tables || max_blocks == 0) && query_start_loc &&
                  context_lens && out,
              "mlr_paged_prefill_scored: null pointer");
  max_query_len = std::min(max_query_len, total_q);
  const int64_t group = num_q_heads / num_kv_heads;
  MLR_REQUIRE(max_query_len < (int64_t(1) << 31) / group &&
                  prefill_units(num_seqs, max_query_len, group, kRows) * num_kv_heads <
                      (int64_t(1) << 25),
              "mlr_paged_prefill_scored: too many query rows");
  const int64_t max_keys = max_blocks * block_size;
  const PrefillPlan n = plan_prefill(num_seqs, max_query_len, max_keys, block_size, num_q_heads,
                                     num_kv_heads, head_dim, dtype);
  const size_t need = mlr_paged_prefill_scored_workspace_size(
      num_seqs, max_query_len, max_blocks, block_size, num_q_heads, num_kv_heads, head_dim, dtype);
  MLR_REQUIRE(need == 0 || (workspace && workspace_bytes >= need),
              "mlr_paged_prefill_scored: workspace of %zu bytes, %zu needed", workspace_bytes,
              need);
  ScoredParams p = params_of(o, kModePrefill);
  p.qsl = query_start_loc;
  p.ahead = prefix_lens;
  p.total_q = total_q;
  p.units = static_cast<int>(n.units);
  p.tiles = static_cast<int>(n.units / num_seqs);
  p.whole = n.whole;
  p.target = n.target;
  const int rows = static_cast<int>(n.rows);
  if (n.parts) place_parts(p, static_cast<char *>(workspace), n.items, rows);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int rc = rows == kTileRows
                     ? launch_scored_tiles(p, dtype, static_cast<unsigned>(n.items), s)
                     : launch_scored_rows(p, dtype, grid_of(n.items), s);
  if (rc) return rc;
  return n.parts ? launch_merge(p, 0, rows, p, rows, false, dtype, s) : MLR_OK;
}

extern "C" size_t mlr_paged_decode_shared_prefix_workspace_size(
    int64_t batch, int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim, int64_t prefix_len,
    int64_t max_blocks, int64_t block_size, int dtype) {
  if (batch <= 0 || num_kv_heads <= 0 || num_q_heads <= 0 || head_dim <= 0 || block_size <= 0)
    return 0;
  const int64_t group = num_q_heads / num_kv_heads, max_keys = max_blocks * block_size;
  if (shares_tiles(batch, group, block_size, num_kv_heads, head_dim, dtype)) {
    const int64_t units = prefix_units(batch, group, kTileRows) + batch;
    return part_bytes(units, max_items(units, num_kv_heads, std::max(prefix_len, max_keys),
                                       shared_target(units, num_kv_heads)), kTileRows, head_dim);
  }
  const int64_t rows =
      takes_tiles(batch * group, block_size, num_kv_heads, head_dim, dtype) ? kTileRows : kRows;
  const int64_t own = decode_units(batch, group), over = prefix_units(batch, group, rows);
  const int64_t target = rows == kTileRows ? prefix_target(over, num_kv_heads)
                                           : rows_target(over, num_kv_heads, head_dim);
  return part_bytes(own, max_items(own, num_kv_heads, max_keys,
                                   rows_target(own, num_kv_heads, head_dim)), kRows, head_dim) +
         part_bytes(over, max_items(over, num_kv_heads, prefix_len, target), rows, head_dim);
}

extern "C" int mlr_paged_decode_shared_prefix(
    const void *q, int64_t q_stride_b, int64_t q_stride_h, const void *k_cache,
    const void *v_cache, int64_t num_blocks, int64_t block_size, int64_t num_kv_heads,
    int64_t head_dim, const int64_t *prefix_table, int64_t prefix_blocks, int64_t prefix_len,
    const int64_t *block_tables, int64_t bt_stride, int64_t max_blocks, const int64_t *seq_lens,
    int64_t batch, int64_t num_q_heads, double scale, double softcap, const float *alibi_slopes,
    int dtype, void *workspace, size_t workspace_bytes, void *out, int64_t out_stride_b,
    int64_t out_stride_h, void *stream) {
  clear_error();
  const Operands o{"mlr_paged_decode_shared_prefix", q, q_stride_b, q_stride_h, k_cache, v_cache,
                   num_blocks, block_size, num_kv_heads, head_dim, block_tables, bt_stride,
                   max_blocks, seq_lens, batch, num_q_heads, scale, softcap, alibi_slopes, dtype,
                   out, out_stride_b, out_stride_h};
  if (const int rc = check_operands(o)) return rc;
  MLR_REQUIRE(prefix_len >= 0 && prefix_blocks >= 0 &&
                  covers_less(prefix_blocks, block_size) &&
                  prefix_len <= prefix_blocks * block_size,
              "mlr_paged_decode_shared_prefix: the prefix table does not cover the prefix");
  if (batch == 0) return MLR_OK;
  MLR_REQUIRE(batch * num_q_heads < (int64_t(1) << 28), "%s: too many query rows", o.what);
  MLR_REQUIRE(q && k_cache && v_cache && (prefix_table || prefix_len == 0) &&
                  (block_tables || max_blocks == 0) && seq_lens && out,
              "mlr_paged_decode_shared_prefix: null pointer");
  const int64_t max_keys = max_blocks * block_size;
  const size_t need = mlr_paged_decode_shared_prefix_workspace_size(
      batch, num_q_heads, num_kv_heads, head_dim, prefix_len, max_blocks, block_size, dtype);
  MLR_REQUIRE(workspace && workspace_bytes >= need,
              "mlr_paged_decode_shared_prefix: workspace of %zu bytes, %zu needed",
              workspace_bytes, need);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t group = num_q_heads / num_kv_heads;
  if (shares_tiles(batch, group, block_size, num_kv_heads, head_dim, dtype)) {
    ScoredParams p = params_of(o, kModeShared);
    p.prefix = prefix_table;
    p.prefix_width = prefix_blocks;
    p.prefix_units = static_cast<int>(prefix_units(batch, group, kTileRows));
    p.tiles = 1;
    p.units = static_cast<int>(p.prefix_units + batch);
    p.start = prefix_len;
    p.force_partial = true;
    p.target = shared_target(p.units, p.hkv);
    const int64_t items = max_items(p.units, p.hkv, std::max(prefix_len, max_keys), p.target);
    place_parts(p, static_cast<char *>(workspace), items, kTileRows);
    if (const int rc = launch_scored_tiles(p, dtype, static_cast<unsigned>(items), s)) return rc;
    return launch_merge(p, p.prefix_units, kTileRows, p, kTileRows, true, dtype, s);
  }
  ScoredParams own = params_of(o, kModeDecode);
  own.tiles = static_cast<int>(ceil_div(group, kRows));
  own.units = static_cast<int>(decode_units(batch, group));
  own.target = rows_target(own.units, own.hkv, own.d);
  own.start = prefix_len;
  own.force_partial = true;
  const int64_t own_items = max_items(own.units, own.hkv, max_keys, own.target);
  char *ws = place_parts(own, static_cast<char *>(workspace), own_items, kRows);
  ScoredParams over = params_of(o, kModePrefix);
  over.prefix = prefix_table;
  over.prefix_width = prefix_blocks;
  const bool tiles = takes_tiles(batch * group, block_size, over.hkv, over.d, dtype);
  const int rows = tiles ? kTileRows : kRows;
  over.units = over.tiles = static_cast<int>(prefix_units(batch, group, rows));
  over.start = prefix_len;
  over.force_partial = true;
  over.target = tiles ? prefix_target(over.units, over.hkv)
                      : rows_target(over.units, over.hkv, over.d);
  const int64_t over_items = max_items(over.units, over.hkv, prefix_len, over.target);
  place_parts(over, ws, over_items, rows);
  const int rc = tiles ? launch_scored_tiles(over, dtype, static_cast<unsigned>(over_items), s)
                       : launch_scored_rows(over, dtype, grid_of(over_items), s);
  if (rc) return rc;
  if (const int rc2 = launch_scored_rows(own, dtype, grid_of(own_items), s)) return rc2;
  return launch_merge(own, 0, kRows, over, rows, true, dtype, s);
}

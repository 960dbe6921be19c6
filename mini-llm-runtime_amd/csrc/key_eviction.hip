// Which keys a cache holds: a decode that adds up what attention each key gets, the
// choice of the keys that stay, and their move, in place, to the front.
//
//   weigh: w[j] += sum over the heads h of a KV group of softmax_j(x_hj); the newest
//          key's entry is set, as its slot may hold what an earlier owner left.
//   evict: the first `sinks`, the last `recent` and of the others the heaviest stay.
//   move:  row start + i <- row kept[i], in order.
#include "key_select.h"
#include "scored_attention.h"

#include <algorithm>

namespace mlr {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kChunk = 1024;  // keys of a workgroup of weigh_keys
constexpr int kHeads = 64;    // heads whose statistics it holds at a time

// The second pass of a weighing decode: scores, and (m, l) of each row's items, are in
// the workspace. A workgroup joins the statistics of its KV head's rows, then adds
// up the weights of its keys, four to a thread. Requests that share a block add to the
// same entry, hence the atomic; where blocks are a request's own each entry has one
// addend and the result does not depend on any order.
__global__ __launch_bounds__(256) void weigh_keys(ScoredParams p, float *weights) {
  __shared__ float s_m[kHeads], s_inv[kHeads];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t b = blockIdx.x;
  const int64_t seq = b % p.seqs;
  const int kvh = static_cast<int>(b / p.seqs % p.hkv);
  const int64_t chunk = b / p.seqs / p.hkv;
  const int64_t ctx = clamp64(p.ctx[seq], 0, p.bt_width * p.block_size);
  if (chunk * kChunk >= ctx) return;  // uniform
  const int64_t key0 = chunk * kChunk + 4 * tid;
  float w[4] = {0.f, 0.f, 0.f, 0.f};
  for (int h0 = 0; h0 < p.group; h0 += kHeads) {
    const int heads = min(kHeads, p.group - h0);
    for (int h = wave; h < heads; h += 4) {
      const int tile = (h0 + h) / kRows, rr = (h0 + h) - tile * kRows;
      const int64_t unit = seq * p.tiles + tile;
      const int first = p.first[unit], count = p.first[unit + 1] - first;
      const int64_t at = (static_cast<int64_t>(first) * p.hkv + kvh) * kRows + rr;
      const int64_t step = static_cast<int64_t>(p.hkv) * kRows;
      float m = -INFINITY, l = 0.f;
      for (int i = lane; i < count; i += 64) m = fmaxf(m, p.ml[2 * (at + i * step)]);
      m = wave_max(m);
      const float ref = m == -INFINITY ? 0.f : m;
      for (int i = lane; i < count; i += 64)
        l += p.ml[2 * (at + i * step) + 1] *
             __builtin_amdgcn_exp2f((p.ml[2 * (at + i * step)] - ref) * kLog2e);
      l = wave_sum(l);
      if (lane == 0) {
        s_m[h] = ref;
        s_inv[h] = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
      }
    }
    __syncthreads();
    if (key0 < ctx) {
      const float *row = p.scores + (seq * p.hq + kvh * p.group + h0) * p.scores_st + key0;
      for (int h = 0; h < heads; ++h) {
        const float4 x = *reinterpret_cast<const float4 *>(row + h * p.scores_st);
        w[0] += __builtin_amdgcn_exp2f((x.x - s_m[h]) * kLog2e) * s_inv[h];
        w[1] += __builtin_amdgcn_exp2f((x.y - s_m[h]) * kLog2e) * s_inv[h];
        w[2] += __builtin_amdgcn_exp2f((x.z - s_m[h]) * kLog2e) * s_inv[h];
        w[3] += __builtin_amdgcn_exp2f((x.w - s_m[h]) * kLog2e) * s_inv[h];
      }
    }
    __syncthreads();
  }
  const int64_t *table = p.bt + seq * p.bt_st;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t key = key0 + i;
    if (key >= ctx) break;
    const int64_t at = key / p.block_size;
    const int64_t block = table[at];
    if (block < 0 || block >= p.num_blocks) continue;
    float *entry = weights + (block * p.hkv + kvh) * p.block_size + (key - at * p.block_size);
    if (key == ctx - 1) *entry = w[i];
    else unsafeAtomicAdd(entry, w[i]);
  }
}

struct CacheParams {
  unsigned char *k, *v;  // [num_blocks, block_size, hkv, row_bytes]
  float *weights;        // [num_blocks, hkv, block_size]
  int64_t num_blocks, block_size, hkv, row_bytes;
  const int64_t *bt;
  int64_t bt_st, bt_width;
  int64_t seqs;
  int bs_log2;  // log2 of block_size, -1 if it is no power of two

  __device__ __forceinline__ int64_t covered() const { return bt_width * block_size; }
  // Slot of a position of a request, -1 if there is none.
  __device__ __forceinline__ int64_t slot(int64_t seq, int64_t pos) const {
    if (pos < 0 || pos >= covered()) return -1;
    const int64_t at = bs_log2 >= 0 ? pos >> bs_log2 : pos / block_size;
    const int64_t block = bt[seq * bt_st + at];
    return block < 0 || block >= num_blocks ? -1 : block * block_size + (pos - at * block_size);
  }
};

// A workgroup chooses the places of one request and KV head.
__global__ __launch_bounds__(kSelectThreads) void choose_keys(CacheParams c, const int64_t *ctx,
                                                              int sinks, int recent, int budget,
                                                              int64_t *kept, int64_t *lens) {
  __shared__ SelectShared s;
  const int64_t seq = blockIdx.x % c.seqs, kvh = blockIdx.x / c.seqs;
  const int n = static_cast<int>(clamp64(ctx[seq], 0, c.covered()));
  int64_t *list = kept + (seq * c.hkv + kvh) * budget;
  const int chosen = select_places<uint32_t, 16>(
      s, n, sinks, recent, budget,
      [&](int i) __attribute__((always_inline)) {
        const int64_t at = c.slot(seq, i);
        if (at < 0) return order_key(-INFINITY);
        const int64_t block = c.bs_log2 >= 0 ? at >> c.bs_log2 : at / c.block_size;
        return order_key(
            c.weights[(block * c.hkv + kvh) * c.block_size + (at - block * c.block_size)]);
      },
      [&](int r, int i) __attribute__((always_inline)) { list[r] = i; });
  for (int i = chosen + threadIdx.x; i < budget; i += kSelectThreads) list[i] = -1;
  if (kvh == 0 && threadIdx.x == 0) lens[seq] = chosen;
}

// Rows start + i <- row kept[i]. Lists ascend and kept[i] >= start + i, so a row is
// written only after, or together with, the reading of the row that lay there, if a
// list is gone through in order: a wave takes 64 bytes of every row of a list, of K or of
// V, 16 rows at a time and kBatch of those between their reads and their writes.
// Columns never meet, so nothing but the wave's own wait orders them.
constexpr int kBatch = 8;
struct Lists {
  const int64_t *kept, *start;
  int64_t st_b, st_h, n;
};

__global__ __launch_bounds__(256) void move_rows(CacheParams c, Lists l, int columns) {
  const int lane = threadIdx.x & 63;
  const int64_t task =
      blockIdx.x * 4 + static_cast<int64_t>(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6));
  // Columns of K, of V, then the weights.
  const int per = 2 * columns + (c.weights ? 1 : 0);
  const int64_t pair = task / per;
  if (pair >= c.seqs * c.hkv) return;
  const int column = static_cast<int>(task - pair * per);
  const int64_t seq = pair / c.hkv, kvh = pair - seq * c.hkv;
  const int64_t *list = l.kept + seq * l.st_b + kvh * l.st_h;
  const int64_t start = l.start ? l.start[seq] : 0;
  if (column == 2 * columns) {
    for (int64_t i0 = 0; i0 < l.n; i0 += 64 * kBatch) {
      float x[kBatch];
      int64_t to[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int64_t i = i0 + 64 * u + lane;
        to[u] = -1;
        const int64_t from = i < l.n ? list[i] : -1;
        if (from < 0 || from == start + i) continue;
        const int64_t src = c.slot(seq, from), dst = c.slot(seq, start + i);
        if (src < 0 || dst < 0) continue;
        const int64_t sb = src / c.block_size, db = dst / c.block_size;
        x[u] = c.weights[(sb * c.hkv + kvh) * c.block_size + (src - sb * c.block_size)];
        to[u] = (db * c.hkv + kvh) * c.block_size + (dst - db * c.block_size);
      }
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_waitcnt(0);
      asm volatile("" ::: "memory");
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
        if (to[u] >= 0) c.weights[to[u]] = x[u];
    }
    return;
  }
  unsigned char *cache = column < columns ? c.k : c.v;
  const int64_t byte = 64 * (column < columns ? column : column - columns) + 16 * (lane & 3);
  const bool mine = byte < c.row_bytes;
  for (int64_t i0 = 0; i0 < l.n; i0 += 16 * kBatch) {
    uint4 x[kBatch];
    int64_t to[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int64_t i = i0 + 16 * u + (lane >> 2);
      to[u] = -1;
      const int64_t from = i < l.n && mine ? list[i] : -1;
      if (from < 0 || from == start + i) continue;
      const int64_t src = c.slot(seq, from), dst = c.slot(seq, start + i);
      if (src < 0 || dst < 0) continue;
      x[u] = *reinterpret_cast<const uint4 *>(cache + (src * c.hkv + kvh) * c.row_bytes + byte);
      to[u] = (dst * c.hkv + kvh) * c.row_bytes + byte;
    }
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0);
    asm volatile("" ::: "memory");
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
      if (to[u] >= 0) *reinterpret_cast<uint4 *>(cache + to[u]) = x[u];
  }
}

int launch_move(const CacheParams &c, const Lists &l, hipStream_t stream) {
  if (l.n == 0) return MLR_OK;
  const int columns = static_cast<int>(ceil_div(c.row_bytes, 64));
  const int64_t waves = c.seqs * c.hkv * (2 * columns + (c.weights ? 1 : 0));
  move_rows<<<static_cast<unsigned>(ceil_div(waves, 4)), 256, 0, stream>>>(c, l, columns);
  return check_launch("move_rows");
}

int check_cache(const char *w, const void *k, const void *v, int64_t num_blocks,
                int64_t block_size, int64_t hkv, int64_t d, const int64_t *bt, int64_t width,
                int64_t seqs, int dtype) {
  MLR_REQUIRE(dtype == MLR_DTYPE_F32 || dtype == MLR_DTYPE_F16 || dtype == MLR_DTYPE_BF16,
              "%s: unsupported dtype %d", w, dtype);
  MLR_REQUIRE(seqs >= 0 && seqs < (1 << 24), "%s: number of sequences must be in [0, 2^24)", w);
  MLR_REQUIRE(hkv > 0 && hkv < (1 << 16), "%s: KV heads must be in [1, 2^16)", w);
  MLR_REQUIRE(d > 0 && d <= 1024 && d * dtype_size(dtype) % 16 == 0,
              "%s: rows must be multiples of 16 bytes, of at most 1024 elements", w);
  MLR_REQUIRE(num_blocks > 0 && num_blocks < (int64_t(1) << 31) && block_size > 0 && width >= 0,
              "%s: the cache needs fewer than 2^31 blocks of a positive size", w);
  MLR_REQUIRE(width < (int64_t(1) << 31) / block_size &&
                  width * block_size <= (int64_t(1) << 31) - 4096,
              "%s: a block table must cover fewer than 2^31 positions", w);
  if (seqs == 0) return MLR_OK;
  MLR_REQUIRE(k && v && (bt || width == 0), "%s: null pointer", w);
  MLR_REQUIRE((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % 16 == 0,
              "%s: the cache must be 16-byte aligned", w);
  return MLR_OK;
}

CacheParams cache_of(void *k, void *v, float *weights, int64_t num_blocks, int64_t block_size,
                     int64_t hkv, int64_t d, const int64_t *bt, int64_t bt_st, int64_t width,
                     int64_t seqs, int dtype) {
  return CacheParams{static_cast<unsigned char *>(k), static_cast<unsigned char *>(v), weights,
                     num_blocks, block_size, hkv, d * dtype_size(dtype), bt, bt_st, width, seqs,
                     log2_if_pow2(block_size)};
}

size_t scores_bytes(int64_t batch, int64_t hq, int64_t max_keys) {
  return align256(batch * hq * ((max_keys + 15) & ~int64_t(15)) * sizeof(float));
}

}  // namespace
}  // namespace mlr

using namespace mlr;

extern "C" size_t mlr_paged_decode_weighted_workspace_size(int64_t batch, int64_t num_q_heads,
                                                           int64_t num_kv_heads, int64_t head_dim,
                                                           int64_t max_context) {
  if (batch <= 0 || num_kv_heads <= 0 || num_q_heads <= 0 || max_context <= 0) return 0;
  return scores_bytes(batch, num_q_heads, max_context) +
         decode_workspace(batch, num_q_heads, num_kv_heads, head_dim, max_context);
}

extern "C" int mlr_paged_decode_weighted(
    const void *q, int64_t q_stride_b, int64_t q_stride_h, const void *k_cache,
    const void *v_cache, float *key_weights, int64_t num_blocks, int64_t block_size,
    int64_t num_kv_heads, int64_t head_dim, const int64_t *block_tables, int64_t bt_stride,
    int64_t max_blocks, const int64_t *seq_lens, int64_t batch, int64_t num_q_heads, double scale,
    double softcap, int dtype, void *workspace, size_t workspace_bytes, void *out,
    int64_t out_stride_b, int64_t out_stride_h, void *stream) {
  clear_error();
  const Operands o{"mlr_paged_decode_weighted", q, q_stride_b, q_stride_h, k_cache, v_cache,
                   num_blocks, block_size, num_kv_heads, head_dim, block_tables, bt_stride,
                   max_blocks, seq_lens, batch, num_q_heads, scale, softcap, nullptr, dtype,
                   out, out_stride_b, out_stride_h};
  if (const int rc = check_operands(o)) return rc;
  if (batch == 0) return MLR_OK;
  MLR_REQUIRE(batch * num_q_heads < (int64_t(1) << 28), "%s: too many query rows", o.what);
  MLR_REQUIRE(q && k_cache && v_cache && key_weights && (block_tables || max_blocks == 0) &&
                  seq_lens && out, "%s: null pointer", o.what);
  const int64_t max_keys = max_blocks * block_size;
  const size_t need = mlr_paged_decode_weighted_workspace_size(batch, num_q_heads, num_kv_heads,
                                                               head_dim, max_keys);
  const int64_t groups = batch * num_kv_heads * ceil_div(std::max<int64_t>(max_keys, 1), kChunk);
  MLR_REQUIRE(groups < (int64_t(1) << 31), "%s: too many keys", o.what);
  MLR_REQUIRE(need == 0 || (workspace && workspace_bytes >= need),
              "%s: workspace of %zu bytes, %zu needed", o.what, workspace_bytes, need);
  ScoredParams p = params_of(o, kModeDecode);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (need == 0) {  // tables without a column: every result is zeros
    return launch_scored_rows(p, dtype, grid_of(plan_decode(p, 0, nullptr)), s);
  }
  char *ws = static_cast<char *>(workspace);
  p.scores = reinterpret_cast<float *>(ws);
  p.scores_st = (max_keys + 15) & ~int64_t(15);
  p.force_partial = true;
  const int64_t items = plan_decode(p, max_keys, ws + scores_bytes(batch, num_q_heads, max_keys));
  if (const int rc = launch_scored_rows(p, dtype, grid_of(items), s)) return rc;
  weigh_keys<<<static_cast<unsigned>(groups), 256, 0, s>>>(p, key_weights);
  if (const int rc = check_launch("weigh_keys")) return rc;
  return merge_decode(p, dtype, s);
}

extern "C" int mlr_evict_keys(void *k_cache, void *v_cache, float *key_weights,
                              int64_t num_blocks, int64_t block_size, int64_t num_kv_heads,
                              int64_t head_dim, const int64_t *block_tables, int64_t bt_stride,
                              int64_t max_blocks, const int64_t *seq_lens, int64_t batch,
                              int64_t budget, int64_t sinks, int64_t recent, int dtype,
                              int64_t *kept, int64_t *new_lens, void *stream) {
  clear_error();
  const char *w = "mlr_evict_keys";
  if (const int rc = check_cache(w, k_cache, v_cache, num_blocks, block_size, num_kv_heads,
                                 head_dim, block_tables, max_blocks, batch, dtype))
    return rc;
  MLR_REQUIRE(sinks >= 0 && recent >= 0 && budget < (int64_t(1) << 31) && sinks <= budget &&
                  recent <= budget - sinks,
              "%s: budget must cover sinks and recent", w);
  if (batch == 0) return MLR_OK;
  MLR_REQUIRE(batch * num_kv_heads < (int64_t(1) << 25), "%s: too many lists", w);
  MLR_REQUIRE(key_weights && seq_lens && new_lens && (kept || budget == 0), "%s: null pointer", w);
  const CacheParams c = cache_of(k_cache, v_cache, key_weights, num_blocks, block_size,
                                 num_kv_heads, head_dim, block_tables, bt_stride, max_blocks,
                                 batch, dtype);
  hipStream_t s = static_cast<hipStream_t>(stream);
  choose_keys<<<static_cast<unsigned>(batch * num_kv_heads), kSelectThreads, 0, s>>>(
      c, seq_lens, static_cast<int>(sinks), static_cast<int>(recent), static_cast<int>(budget),
      kept, new_lens);
  if (const int rc = check_launch("choose_keys")) return rc;
  return launch_move(c, Lists{kept, nullptr, num_kv_heads * budget, budget,
                              std::min(budget, max_blocks * block_size)}, s);
}

extern "C" int mlr_compact_keys(void *k_cache, void *v_cache, float *key_weights,
                                int64_t num_blocks, int64_t block_size, int64_t num_kv_heads,
                                int64_t head_dim, const int64_t *block_tables, int64_t bt_stride,
                                int64_t max_blocks, const int64_t *kept, int64_t kept_stride_b,
                                int64_t kept_stride_h, int64_t num_kept, const int64_t *start,
                                int64_t batch, int dtype, void *stream) {
  clear_error();
  const char *w = "mlr_compact_keys";
  if (const int rc = check_cache(w, k_cache, v_cache, num_blocks, block_size, num_kv_heads,
                                 head_dim, block_tables, max_blocks, batch, dtype))
    return rc;
  MLR_REQUIRE(num_kept >= 0 && num_kept < (int64_t(1) << 31), "%s: bad number of kept keys", w);
  if (batch == 0 || num_kept == 0) return MLR_OK;
  MLR_REQUIRE(batch * num_kv_heads < (int64_t(1) << 25), "%s: too many lists", w);
  MLR_REQUIRE(kept, "%s: null pointer", w);
  const CacheParams c = cache_of(k_cache, v_cache, key_weights, num_blocks, block_size,
                                 num_kv_heads, head_dim, block_tables, bt_stride, max_blocks,
                                 batch, dtype);
  return launch_move(c, Lists{kept, start, kept_stride_b, kept_stride_h, num_kept},
                     static_cast<hipStream_t>(stream));
}

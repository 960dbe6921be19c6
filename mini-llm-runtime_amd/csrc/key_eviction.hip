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
constexpr int kChunk = 256;  // keys of a wave of weigh_keys
constexpr int kHeads = 64;   // heads whose statistics it holds at a time

// out = sum_i e^{m_i - M} O_i / sum_i e^{m_i - M} l_i over the items of row (sequence,
// head) of a decode: 16 lanes side by side over its elements, four groups of lanes dealing
// the items among them, joined in a fixed order.
template <typename T, int D>
__device__ __forceinline__ void join_row(const ScoredParams &p, int64_t row) {
  constexpr int kVe = D / 16;
  const int lane = threadIdx.x & 63, d0 = (lane & 15) * kVe, quarter = lane >> 4;
  const int64_t seq = row / p.hq;
  const int head = static_cast<int>(row - seq * p.hq), kvh = head / p.group;
  const int in_group = head - kvh * p.group, tile = in_group / kRows;
  const int64_t unit = seq * p.tiles + tile;
  const int first = p.first[unit], count = p.first[unit + 1] - first;
  const int64_t at = (static_cast<int64_t>(first) * p.hkv + kvh) * kRows + in_group - tile * kRows;
  const int64_t step = static_cast<int64_t>(p.hkv) * kRows;
  float m = -INFINITY;
  for (int i = lane; i < count; i += 64) m = fmaxf(m, p.ml[2 * (at + i * step)]);
  m = wave_max(m);
  const float ref = m == -INFINITY ? 0.f : m;
  float sum = 0.f, acc[kVe];
#pragma unroll
  for (int n = 0; n < kVe; ++n) acc[n] = 0.f;
#pragma unroll 4
  for (int i = quarter; i < count; i += 4) {
    const float2 ml = *reinterpret_cast<const float2 *>(p.ml + 2 * (at + i * step));
    const float f = __builtin_amdgcn_exp2f((ml.x - ref) * kLog2e);
    sum += ml.y * f;
#pragma unroll
    for (int n = 0; n < kVe; n += 4) {
      const float4 v = *reinterpret_cast<const float4 *>(p.acc + (at + i * step) * D + d0 + n);
      acc[n] += v.x * f;
      acc[n + 1] += v.y * f;
      acc[n + 2] += v.z * f;
      acc[n + 3] += v.w * f;
    }
  }
  auto join = [](float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
  };
  sum = join(sum);
#pragma unroll
  for (int n = 0; n < kVe; ++n) acc[n] = join(acc[n]);
  if (quarter != 0) return;
  const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
  T *dst = static_cast<T *>(p.out) + seq * p.o_st + head * p.o_sh;
#pragma unroll
  for (int n = 0; n < kVe; ++n)
    if (d0 + n < p.d) dst[d0 + n] = Elem<T>::from_f32(acc[n] * inv);
}

// The second pass of a weighing decode: the scores, and (m, l) of each row's items, are
// in the workspace. A wave joins the statistics of its KV head's rows and adds up the
// weights of 256 keys, four to a lane. Requests that share a block add to the same
// entry, hence the atomic; where blocks are a request's own each entry has one addend
// and the result does not depend on any order.
// Bound by latency, as the scores of 64 requests are 8 MB: what does not depend on the
// statistics (table, scores of up to kAhead heads) is read before them, and the weights change
// lanes, so that the lanes' atomics go to neighbouring entries. 64 requests of 128 to 4,096
// keys, 14 heads over 2 of 64: 7.2 us, with the join of the results (four neighbours a lane:
// 9.0); 500 to 2,000 keys, 12 over 12: 11.2 us (20). A wave past its request's end leaves
// before it reads scores, which nobody wrote there: 64 requests of 500 to 1,024 keys in tables of
// 32,768 9.2 us, 22.4 with the work of all waves, 6.3 in tables of 1,024.
constexpr int kAhead = 8;
__device__ __forceinline__ void weigh_keys(const ScoredParams &p, float *weights, int64_t task,
                                           float (*s_ml)[2], float *s_w) {
  const int lane = threadIdx.x & 63;
  const int64_t seq = task % p.seqs;
  const int kvh = static_cast<int>(task / p.seqs % p.hkv);
  const int64_t covered = p.bt_width * p.block_size;
  const int64_t base = task / p.seqs / p.hkv * kChunk, key0 = base + 4 * lane;
  const int64_t ctx = clamp64(p.ctx[seq], 0, covered);
  if (base >= ctx) return;  // uniform
  const float *row = p.scores + (seq * p.hq + kvh * p.group) * p.scores_st +
                     min(key0, p.scores_st - 4);
  float4 x[kAhead];
#pragma unroll
  for (int h = 0; h < kAhead; ++h)
    x[h] = *reinterpret_cast<const float4 *>(row + min(h, p.group - 1) * p.scores_st);
  const uint32_t bs = static_cast<uint32_t>(p.block_size);
  auto block_of = [&](uint32_t key) __attribute__((always_inline)) {
    return p.bs_log2 >= 0 ? key >> p.bs_log2 : key / bs;
  };
  // For the sums a lane has every 64th key, so that the lanes' entries are neighbours.
  int64_t block[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    block[i] = p.bt[seq * p.bt_st +
                    block_of(static_cast<uint32_t>(min(base + 64 * i + lane, covered - 1)))];
  float w[4] = {0.f, 0.f, 0.f, 0.f};
  for (int h0 = 0; h0 < p.group; h0 += kHeads) {
    const int heads = min(kHeads, p.group - h0);
    // Eight lanes a head, its items dealt among them.
    for (int h8 = 0; h8 < heads; h8 += 8) {
      const int h = min(h8 + (lane >> 3), heads - 1);
      const int tile = (h0 + h) / kRows, rr = (h0 + h) - tile * kRows;
      const int64_t unit = seq * p.tiles + tile;
      const int first = p.whole ? static_cast<int>(unit) : p.first[unit];
      const int count = p.whole ? 1 : p.first[unit + 1] - first;
      const int64_t at = (static_cast<int64_t>(first) * p.hkv + kvh) * kRows + rr;
      const int64_t step = static_cast<int64_t>(p.hkv) * kRows;
      float m = -INFINITY, l = 0.f;
#pragma unroll 4
      for (int i = lane & 7; i < count; i += 8) {
        const float2 ml = *reinterpret_cast<const float2 *>(p.ml + 2 * (at + i * step));
        const float top = fmaxf(m, ml.x), ref = top == -INFINITY ? 0.f : top;
        l = l * __builtin_amdgcn_exp2f((m - ref) * kLog2e) +
            ml.y * __builtin_amdgcn_exp2f((ml.x - ref) * kLog2e);
        m = top;
      }
      float top = m;
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
      const float ref = top == -INFINITY ? 0.f : top;
      l *= __builtin_amdgcn_exp2f((m - ref) * kLog2e);
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) l += __shfl_xor(l, o);
      if ((lane & 7) == 0) {
        s_ml[h][0] = ref;
        s_ml[h][1] = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
      }
    }
    // One wave's own part of LDS, here and below: in order without a barrier.
    asm volatile("" ::: "memory");
    auto add = [&](const float4 &v, int h) __attribute__((always_inline)) {
      const float m = s_ml[h][0], inv = s_ml[h][1];
      w[0] += __builtin_amdgcn_exp2f((v.x - m) * kLog2e) * inv;
      w[1] += __builtin_amdgcn_exp2f((v.y - m) * kLog2e) * inv;
      w[2] += __builtin_amdgcn_exp2f((v.z - m) * kLog2e) * inv;
      w[3] += __builtin_amdgcn_exp2f((v.w - m) * kLog2e) * inv;
    };
    int h = 0;
    if (h0 == 0) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        if (i < heads) add(x[i], i);
      h = min(kAhead, heads);
    }
    for (; h < heads; ++h)
      add(*reinterpret_cast<const float4 *>(row + (h0 + h) * p.scores_st), h);
  }
  *reinterpret_cast<float4 *>(s_w + 4 * lane) = make_float4(w[0], w[1], w[2], w[3]);
  asm volatile("" ::: "memory");
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t at = base + 64 * i + lane;
    const float sum = s_w[64 * i + lane];
    if (at >= ctx || block[i] < 0 || block[i] >= p.num_blocks) continue;
    const uint32_t key = static_cast<uint32_t>(at);
    float *entry = weights + (block[i] * p.hkv + kvh) * p.block_size + (key - block_of(key) * bs);
    if (at == ctx - 1) *entry = sum;
    else unsafeAtomicAdd(entry, sum);
  }
}

// Both ends of a weighing decode that was cut into items: its results joined, a wave a
// row, and its keys weighed, a wave for 256 of them.
template <typename T, int D>
__global__ __launch_bounds__(256) void weigh_and_join(ScoredParams p, float *weights,
                                                      int64_t rows, int64_t tasks) {
  __shared__ float s_ml[4][kHeads][2];
  __shared__ __align__(16) float s_w[4][kChunk];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  for (int64_t task = blockIdx.x * int64_t(4) + wave; task < rows + tasks;
       task += gridDim.x * int64_t(4)) {
    if (task < rows) join_row<T, D>(p, task);
    else weigh_keys(p, weights, task - rows, s_ml[wave], s_w[wave]);
  }
}

int launch_weigh(const ScoredParams &p, float *weights, int64_t max_keys, int dtype,
                 hipStream_t stream) {
  const int64_t rows = p.whole ? 0 : static_cast<int64_t>(p.seqs) * p.hq;
  const int64_t tasks = static_cast<int64_t>(p.seqs) * p.hkv * ceil_div(max_keys, kChunk);
  const unsigned grid =
      static_cast<unsigned>(std::min<int64_t>(ceil_div(rows + tasks, 4), 1 << 20));
#define MLR_WEIGH(T)                                                                          \
  if (p.d > 64) weigh_and_join<T, 128><<<grid, 256, 0, stream>>>(p, weights, rows, tasks);    \
  else weigh_and_join<T, 64><<<grid, 256, 0, stream>>>(p, weights, rows, tasks)
  if (dtype == MLR_DTYPE_F32) {
    MLR_WEIGH(float);
  } else if (dtype == MLR_DTYPE_F16) {
    MLR_WEIGH(f16_t);
  } else {
    MLR_WEIGH(bf16_t);
  }
#undef MLR_WEIGH
  return check_launch("weigh_and_join");
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
  // Positions and block sizes are below 2^31.
  __device__ __forceinline__ uint32_t block_of(uint32_t at) const {
    return bs_log2 >= 0 ? at >> bs_log2 : at / static_cast<uint32_t>(block_size);
  }
  // Slot of a position of a request, -1 if there is none.
  __device__ __forceinline__ int64_t slot(int64_t seq, int64_t pos) const {
    if (pos < 0 || pos >= covered()) return -1;
    const int64_t at = block_of(static_cast<uint32_t>(pos));
    const int64_t block = bt[seq * bt_st + at];
    return block < 0 || block >= num_blocks ? -1 : block * block_size + (pos - at * block_size);
  }
};

// A workgroup chooses the places of one request and KV head. Bound by latency: the keys'
// two loads (a table, then four neighbouring weights where a block holds a multiple of
// four), the selection's histogram, the list. 32 lists of 16,384 keys 17 us to 20, of which the
// histogram's atomics are 6; 128 lists of 1,040 keys 8 us.
template <int kThreads, int kHeld>
__global__ __launch_bounds__(kThreads) void choose_keys(CacheParams c, const int64_t *ctx,
                                                        int sinks, int recent, int budget,
                                                        int64_t *kept, int64_t *lens) {
  __shared__ SelectShared s;
  const int64_t seq = blockIdx.x % c.seqs, kvh = blockIdx.x / c.seqs;
  const int n = static_cast<int>(clamp64(ctx[seq], 0, c.covered()));
  int64_t *list = kept + (seq * c.hkv + kvh) * budget;
  const int64_t *table = c.bt + seq * c.bt_st;
  const bool fours = c.block_size % 4 == 0 && reinterpret_cast<uintptr_t>(c.weights) % 16 == 0;
  // A weight's place; block ids out of range count as -infinity.
  auto entry = [&](int64_t block, uint32_t i) __attribute__((always_inline)) {
    return c.weights + (block * c.hkv + kvh) * c.block_size + i;
  };
  const uint32_t bs = static_cast<uint32_t>(c.block_size);
  const int chosen = select_places<uint32_t, kThreads, kHeld>(
      s, n, sinks, recent, budget,
      [&](auto &keys, auto place) __attribute__((always_inline)) {
        constexpr int kMany = sizeof(keys) / sizeof(keys[0]);
        int64_t block[kMany];
        if (fours) {
#pragma unroll
          for (int j = 0; j < kMany; ++j) block[j] = table[c.block_of(min(place(j), n - 1))];
#pragma unroll
          for (int j = 0; j < kMany; ++j) {
            const bool ok = block[j] >= 0 && block[j] < c.num_blocks;
            const uint32_t at = min(place(j), n - 1), in = at - c.block_of(at) * bs;
            const float4 w = *reinterpret_cast<const float4 *>(entry(ok ? block[j] : 0, in & ~3u));
            keys[j][0] = order_key(ok ? w.x : -INFINITY);
            keys[j][1] = order_key(ok ? w.y : -INFINITY);
            keys[j][2] = order_key(ok ? w.z : -INFINITY);
            keys[j][3] = order_key(ok ? w.w : -INFINITY);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
#pragma unroll
            for (int j = 0; j < kMany; ++j) block[j] = table[c.block_of(min(place(j) + e, n - 1))];
#pragma unroll
            for (int j = 0; j < kMany; ++j) {
              const bool ok = block[j] >= 0 && block[j] < c.num_blocks;
              const uint32_t at = min(place(j) + e, n - 1), in = at - c.block_of(at) * bs;
              const float w = *entry(ok ? block[j] : 0, in);
              keys[j][e] = order_key(ok ? w : -INFINITY);
            }
          }
        }
      },
      [&](int r, int i, int) __attribute__((always_inline)) { list[r] = i; });
  for (int i = chosen + threadIdx.x; i < budget; i += kThreads) list[i] = -1;
  if (kvh == 0 && threadIdx.x == 0) lens[seq] = chosen;
}

// Rows start + i <- row kept[i]. Lists ascend and kept[i] >= start + i: what is written
// in place i lies at or before the row that is read for it, so a row is overwritten by
// its own place in the list or a later one. A workgroup that goes through a list in
// order, a batch of rows at a time, may therefore read the next batch before it has
// written this one; it only has to have read all of a batch before it writes any of it:
// one barrier a batch. Columns of 64 bytes of K and of V never meet, so each is a
// workgroup of its own and nothing else orders them.
//
// Bound by what is in flight: each wave has two batches of 16 loads, one landing while the
// other is written. The rows' places are made a batch ahead, from the list, which is read
// two ahead, and the request's block table, which lies in LDS. 4 lists of 6,144 rows for each of
// 8 heads of 128, 201 MB read and written: 55 us, 3.7 TB/s.
constexpr int kLanes = 4;    // of 16 bytes, of a row of a column
constexpr int kLoads = 16;   // of a wave and batch
constexpr int kWaveRows = 64 / kLanes * kLoads;
constexpr int kTable = 4096;  // block ids that lie in LDS; the others are read again
struct Lists {
  const int64_t *kept, *start;
  int64_t st_b, st_h, n;
};

// What a row of a column is: `step` bytes apart from `base` on, row(block, i) of them for
// place i of a block.
template <typename Unit, int kPer, int kWaves, class Row>
__device__ __forceinline__ void move_list(const CacheParams &c, const int64_t *list, int64_t n,
                                          int64_t start, int64_t seq, bool mine,
                                          int64_t (*places)[2][kWaveRows], uint32_t *table,
                                          unsigned char *base, int64_t step, Row row) {
  constexpr int kRowsLoad = 64 / kPer;            // rows of a load
  constexpr int kCount = kWaveRows / kRowsLoad;   // loads
  constexpr int kBatch = kWaveRows * kWaves;      // rows of the workgroup's batch
  const int lane = threadIdx.x & 63, sub = lane / kPer;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t *ids = c.bt + seq * c.bt_st;
  constexpr uint32_t kNone = ~0u;  // block ids are below 2^31
  auto known = [&](int64_t id) __attribute__((always_inline)) {
    return id >= 0 && id < c.num_blocks ? static_cast<uint32_t>(id) : kNone;
  };
  auto id_of = [&](uint32_t at) __attribute__((always_inline)) {
    return at < kTable ? table[at] : known(ids[at]);
  };
  int from[kWaveRows / 64];  // positions are below 2^31; -1: nothing to move
  auto read_list = [&](int64_t batch) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < kWaveRows / 64; ++j) {
      const int64_t i = batch * kBatch + wave * kWaveRows + 64 * j + lane;
      const int64_t x = list[min(i, n - 1)];
      from[j] = i < n && x >= 0 && x < c.covered() ? static_cast<int>(x) : -1;
    }
  };
  // Byte offsets of a batch's rows: a source of 0 and a target of -1 where nothing moves.
  auto make_places = [&](int64_t batch) __attribute__((always_inline)) {
    const uint32_t bs = static_cast<uint32_t>(c.block_size);
#pragma unroll
    for (int j = 0; j < kWaveRows / 64; ++j) {
      const int64_t to = start + batch * kBatch + wave * kWaveRows + 64 * j + lane;
      bool ok = from[j] >= 0 && from[j] != to && to >= 0 && to < c.covered();
      const uint32_t src = ok ? from[j] : 0, dst = ok ? static_cast<uint32_t>(to) : 0;
      const uint32_t sa = c.block_of(src), da = c.block_of(dst);
      const uint32_t sb = id_of(sa), db = id_of(da);
      ok = ok && sb != kNone && db != kNone;
      places[batch & 1][0][64 * j + lane] = ok ? row(sb, src - sa * bs) * step : 0;
      places[batch & 1][1][64 * j + lane] = ok ? row(db, dst - da * bs) * step : -1;
    }
  };
  // Batches are whole: rows past the list read row 0 and are not written.
  Unit x0[kCount], x1[kCount];
  auto read = [&](Unit (&to)[kCount], int64_t batch) __attribute__((always_inline)) {
    int64_t at[kCount];
#pragma unroll
    for (int u = 0; u < kCount; ++u) at[u] = places[batch & 1][0][u * kRowsLoad + sub];
#pragma unroll
    for (int u = 0; u < kCount; ++u) to[u] = *reinterpret_cast<const Unit *>(base + at[u]);
  };
  auto write = [&](const Unit (&of)[kCount], int64_t batch) __attribute__((always_inline)) {
    int64_t at[kCount];
#pragma unroll
    for (int u = 0; u < kCount; ++u) at[u] = places[batch & 1][1][u * kRowsLoad + sub];
#pragma unroll
    for (int u = 0; u < kCount; ++u)
      if (at[u] >= 0 && mine) *reinterpret_cast<Unit *>(base + at[u]) = of[u];
  };
  read_list(0);
  const int held = static_cast<int>(min(c.bt_width, int64_t(kTable)));
#pragma unroll 4
  for (int i = threadIdx.x; i < held; i += 64 * kWaves) table[i] = known(ids[i]);
  __syncthreads();
  make_places(0);
  const int64_t batches = (n + kBatch - 1) / kBatch;
  read(x0, 0);
  if (batches > 1) read_list(1);
  // Writes batch b, which `of` holds, with the next one on its way to `to`.
  auto step_of = [&](Unit (&of)[kCount], Unit (&to)[kCount], int64_t b)
      __attribute__((always_inline)) {
    if (b + 1 < batches) {
      make_places(b + 1);
      if (b + 2 < batches) read_list(b + 2);
      asm volatile("" ::: "memory");
      read(to, b + 1);
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_waitcnt(0x0f70 | (kCount & 15) | (kCount >> 4) << 14);
    } else {
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_waitcnt(0x0f70);
    }
    if (kWaves > 1) __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    write(of, b);
    asm volatile("" ::: "memory");
  };
  for (int64_t b = 0; b < batches; b += 2) {
    step_of(x0, x1, b);
    if (b + 1 < batches) step_of(x1, x0, b + 1);
  }
}

// A workgroup's task: a column of K, of V, or the weights, of one request and KV head.
template <int kWaves>
__global__ __launch_bounds__(64 * kWaves) void move_rows(CacheParams c, Lists l, int columns) {
  __shared__ int64_t places[kWaves][2][2][kWaveRows];
  __shared__ uint32_t table[kTable];
  // The columns of a line of 128 bytes on one XCD, and on each lines of all heads.
  constexpr int kPerLine = 8 / kLanes;
  const int64_t pairs = c.seqs * c.hkv;
  const int lines = (columns + kPerLine - 1) / kPerLine;
  const int64_t i = blockIdx.x / 8, k = i / kPerLine;
  const int64_t at = 8 * k + ((blockIdx.x - k - k / 8) & 7);
  const int64_t line = at / pairs, pair = at - line * pairs;
  if (line > 2 * lines || (line == 2 * lines && (!c.weights || i % kPerLine != 0))) return;
  const int64_t column = (line % lines) * kPerLine + i % kPerLine;
  if (line < 2 * lines && column >= columns) return;
  const int64_t seq = pair / c.hkv, kvh = pair - seq * c.hkv;
  const int64_t *list = l.kept + seq * l.st_b + kvh * l.st_h;
  const int64_t start = l.start ? l.start[seq] : 0;
  int64_t(*mine)[2][kWaveRows] = places[threadIdx.x >> 6];
  if (line == 2 * lines) {
    move_list<float, 1, kWaves>(c, list, l.n, start, seq, true, mine, table,
                                reinterpret_cast<unsigned char *>(c.weights), sizeof(float),
                                [&](int64_t block, int64_t i) __attribute__((always_inline)) {
                                  return (block * c.hkv + kvh) * c.block_size + i;
                                });
    return;
  }
  typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
  unsigned char *cache = line < lines ? c.k : c.v;
  const int64_t byte = 16 * kLanes * column + 16 * (threadIdx.x % kLanes);
  const bool in_row = byte < c.row_bytes;
  move_list<u32x4_t, kLanes, kWaves>(
      c, list, l.n, start, seq, in_row, mine, table,
      cache + kvh * c.row_bytes + (in_row ? byte : 0), c.hkv * c.row_bytes,
      [&](int64_t block, int64_t i) __attribute__((always_inline)) {
        return block * c.block_size + i;
      });
}

int64_t cus() {
  const int n = current_device_cus();
  return n > 0 ? n : 256;
}

int launch_move(const CacheParams &c, const Lists &l, hipStream_t stream) {
  if (l.n == 0 || c.bt_width == 0) return MLR_OK;
  const int columns = static_cast<int>(ceil_div(c.row_bytes, 16 * kLanes));
  const int64_t lines = 2 * ceil_div(columns, 8 / kLanes) + (c.weights ? 1 : 0);
  const int64_t groups = ceil_div(c.seqs * c.hkv * lines, 8) * 8 * (8 / kLanes);
  MLR_REQUIRE(groups < (int64_t(1) << 31), "move_rows: too many rows");
  const unsigned grid = static_cast<unsigned>(groups);
  // As many waves a column as the list fills, up to some nine for every CU: more would run
  // one after the other. us by 2, 4 and 8: 4 lists of 6,144 rows for each of 8 heads of 128
  // (256 columns) 69, 59, 55; 64 of 1,024 for 2 heads of 64 (640 columns) 15, 17, 24.
  const int64_t active = c.seqs * c.hkv * (2 * columns + (c.weights ? 1 : 0));
  const int64_t most = std::min(ceil_div(l.n, kWaveRows), 9 * cus() / active);
  if (most >= 8) move_rows<8><<<grid, 512, 0, stream>>>(c, l, columns);
  else if (most >= 4) move_rows<4><<<grid, 256, 0, stream>>>(c, l, columns);
  else if (most >= 2) move_rows<2><<<grid, 128, 0, stream>>>(c, l, columns);
  else move_rows<1><<<grid, 64, 0, stream>>>(c, l, columns);
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
  p.whole = short_keys(max_keys, head_dim, dtype);
  p.force_partial = !p.whole;
  const int64_t items = plan_decode(p, max_keys, ws + scores_bytes(batch, num_q_heads, max_keys));
  if (const int rc = launch_scored_rows(p, dtype, grid_of(items), s)) return rc;
  return launch_weigh(p, key_weights, max_keys, dtype, s);
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
  const unsigned lists = static_cast<unsigned>(batch * num_kv_heads);
#define MLR_CHOOSE(T, H)                                                                   \
  choose_keys<T, H><<<lists, T, 0, s>>>(c, seq_lens, static_cast<int>(sinks),              \
                                        static_cast<int>(recent), static_cast<int>(budget), \
                                        kept, new_lens)
  // As many waves as hold the longest row's keys in registers: fewer meet sooner. us of the
  // three: 128 lists of 1,040 keys 7.8, 11.1, 14.0 and of 2,047 10.7, 13.2, 16.2; 32 lists of
  // 16,384 81, 20.0, 22.6 and of 32,760 145, 51, 26.7.
  const int64_t most = max_blocks * block_size;
  if (most <= 2048) MLR_CHOOSE(256, 2);
  else if (most <= 16384) MLR_CHOOSE(1024, 4);
  else MLR_CHOOSE(1024, 8);
#undef MLR_CHOOSE
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

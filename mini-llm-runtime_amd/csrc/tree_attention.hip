// Ancestors of drafted tokens as bits, from their parents.
//
// Bit j of a token's row: whether token j of its sequence is the token itself or one of
// its ancestors. A thread walks one token's path to its root for four words of its row;
// parents are read through LDS. A path ends at a parent that is no token of the
// sequence, and after as many steps as there are tokens, so that it ends where
// parents form a circle too.
//
// Bound by latency: a path of depth 16 is 16 dependent reads of LDS, 0.1 us each. A sequence
// of more than 256 rows of four words has several workgroups, so that no thread walks a long
// chain for many tokens one after the other. 16 sequences of 48 tokens 3.1 us, 4 of 500 3.8
// us; a chain of 500 47 us, one of 4,096 0.37 ms, 64 of 4,096 4.05 ms.
#include "mlr_common.h"

#include <algorithm>

namespace mlr {
namespace {

constexpr int kMostNodes = 4096;  // tokens of a sequence that are nodes

__global__ __launch_bounds__(256) void tree_ancestors(const int64_t *parents, const int64_t *qsl,
                                                      int64_t total, int64_t words,
                                                      int64_t *ancestors) {
  __shared__ int s_parent[kMostNodes];
  const int64_t seq = blockIdx.x;
  const int64_t q0 = min(max(qsl[seq], int64_t(0)), total);
  const int n = static_cast<int>(
      min(min(max(qsl[seq + 1], q0), total) - q0, static_cast<int64_t>(kMostNodes)));
  for (int i = threadIdx.x; i < n; i += 256) {
    const int64_t up = parents[q0 + i];
    s_parent[i] = up >= 0 && up < n ? static_cast<int>(up) : -1;
  }
  __syncthreads();
  // Four words of a token's row at a time; its path is walked once for these.
  const int fours = static_cast<int>((words + 3) / 4);
  for (int at = blockIdx.y * 256 + threadIdx.x; at < n * fours; at += gridDim.y * 256) {
    const int token = at / fours, word = 4 * (at - token * fours);
    uint64_t bits[4] = {0, 0, 0, 0};
    int up = token;
    for (int steps = 0; steps < n && up >= 0; ++steps) {
      const int next = s_parent[up], w = (up >> 6) - word;
      const uint64_t bit = uint64_t(1) << (up & 63);
#pragma unroll
      for (int i = 0; i < 4; ++i) bits[i] |= w == i ? bit : 0;
      up = next;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (word + i < words) ancestors[(q0 + token) * words + word + i] = static_cast<int64_t>(bits[i]);
  }
}

}  // namespace
}  // namespace mlr

using namespace mlr;

extern "C" int mlr_tree_ancestors(const int64_t *parents, const int64_t *query_start_loc,
                                  int64_t num_seqs, int64_t total_q, int64_t words,
                                  int64_t *ancestors, void *stream) {
  clear_error();
  MLR_REQUIRE(num_seqs >= 0 && num_seqs < (1 << 24) && total_q >= 0 &&
                  total_q < (int64_t(1) << 31) && words > 0 && words <= kMostNodes / 64,
              "mlr_tree_ancestors: bad sizes (a row of ancestors has 1 to %d words)",
              kMostNodes / 64);
  if (num_seqs == 0 || total_q == 0) return MLR_OK;
  MLR_REQUIRE(parents && query_start_loc && ancestors, "mlr_tree_ancestors: null pointer");
  const int64_t nodes = std::min(total_q, 64 * words);
  const dim3 grid(static_cast<unsigned>(num_seqs),
                  static_cast<unsigned>(ceil_div(nodes * ceil_div(words, 4), 256)));
  tree_ancestors<<<grid, 256, 0, static_cast<hipStream_t>(stream)>>>(parents, query_start_loc,
                                                                     total_q, words, ancestors);
  return check_launch("tree_ancestors");
}

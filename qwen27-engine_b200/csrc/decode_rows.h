// Parameters of the decode attention over part of a cache (decode_rows.cu).
#pragma once
#include "cache_ref.h"

#include <algorithm>

namespace q27b {

constexpr int MAX_SEL = 16384;  // blocks in a list

struct RowsParams {
  CacheRef c;
  const float* qn;       // [B][T][nqh][256]
  const float* qg;       // [B][T][nqh][512], the gate in the second half
  const void* kcache;
  const void* vcache;
  void* o;               // f16 [B][T][nqh][256], or
  int8_t* xq;            // q8_1
  float* xd;
  const uint64_t* mask;  // tree: [B][T], bit j: draft j is visible
  const int* sel;        // blocks: [B][T][nkvh][k], -1 = none; null: tree
  int k;
  float kq_scale;
  float* part_o;         // unnormalised O of a row of a part, 256 floats each: [row][nsplit] (blocks) or [part][128 rows] (tree)
  float2* part_ml;       // (max, sum) of the same; tree: the sum's sign is set where V values of drafts are left to the merge
  int nsplit;            // parts of a list, or of a row tile of one sequence
  int64_t* plan;         // tree, paged: [0] tiles of a part, [1 + b] parts of a unit summed over the sequences before b (tree_parts)
};

// The tensor-core kernel of the tree (decode_tree.cu).
constexpr int TREE_ROWS = 128;         // (draft, head) rows of a KV head in a CTA
constexpr int TREE_MAX_TILES = 65536;  // position tiles of a sequence over pages
__host__ __device__ inline int tree_row_tiles(int T) { return (T * GQA + TREE_ROWS - 1) / TREE_ROWS; }
__host__ __device__ inline int tree_tiles(int n) { return n > 0 ? (n + BLK - 1) / BLK : 0; }
// A unit is a row tile of a KV head of a sequence. Its ntot position tiles are cut into parts of equal length, at most `share`.
__host__ __device__ inline int tree_parts(int ntot, int share) { return (ntot + share - 1) / share; }
// A batch: `share` so that the parts of all units come to w rounds of the SMs, for the w of the least time: a part takes some 9 us
// and 1.3 us a tile. N tiles and U units that are not empty: N / share + U / 2 parts or so. At most tree_grid(U, n_sm) of them.
__host__ __device__ inline int64_t tree_rounds(int64_t U, int n_sm) { return (6 * U / 10) / n_sm + 1; }
__host__ __device__ inline int64_t tree_share_of(int64_t N, int64_t U, int64_t w, int n_sm) {
  const int64_t d = w * n_sm - (55 * U + 99) / 100;
  return d < 1 ? N + 1 : (N + d - 1) / d;
}
__host__ __device__ inline int64_t tree_grid(int64_t U, int n_sm) { return (tree_rounds(U, n_sm) + 2) * n_sm + U / 2 + 1; }
__host__ __device__ inline int tree_share(int64_t N, int64_t U, int n_sm) {
  const int64_t w0 = tree_rounds(U, n_sm);
  int64_t best = 0, cost = 0;
  for (int64_t w = w0; w <= w0 + 2; w++) {
    const int64_t s = tree_share_of(N, U, w, n_sm), c = w * (13 * s + 90);
    if (w == w0 || c < cost) best = s, cost = c;
  }
  return (int)(best < 1 ? 1 : best < TREE_MAX_TILES ? best : TREE_MAX_TILES);
}
int launch_tree(const RowsParams& p, int n_sm, cudaStream_t s);

}  // namespace q27b

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
  int nsplit;
  int share;             // tree, paged: position tiles of a split; 0: an equal share of the sequence's
  float* part_o;         // [row][nsplit][256], unnormalised
  float2* part_ml;       // [row][nsplit] (max, sum)
};

// The tensor-core kernel of the tree (decode_tree.cu): grid (splits, row tiles x KV heads, sequences).
constexpr int TREE_ROWS = 128;       // (draft, head) rows of a KV head in a CTA
constexpr int TREE_MAX_SHARE = 2048;  // position tiles of a split with pages
__host__ __device__ inline int tree_row_tiles(int T) { return (T * GQA + TREE_ROWS - 1) / TREE_ROWS; }
__host__ __device__ inline int tree_tiles(int n) { return n > 0 ? (n + BLK - 1) / BLK : 0; }
// Tiles of a split of a sequence of ntot tiles; split z holds tiles z * share .. of them.
__host__ __device__ inline int tree_share(const RowsParams& p, int ntot) { return p.share ? p.share : (ntot + p.nsplit - 1) / p.nsplit; }
int launch_tree(const RowsParams& p, cudaStream_t s);

}  // namespace q27b

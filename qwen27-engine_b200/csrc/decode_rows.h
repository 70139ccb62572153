// Parameters of the decode attention over part of a cache (decode_rows.cu).
#pragma once
#include "cache_ref.h"
#include "rows_plan.h"

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
int launch_tree(const RowsParams& p, int n_sm, cudaStream_t s);

}  // namespace q27b

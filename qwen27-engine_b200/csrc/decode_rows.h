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
  int max_len;           // no sequence is longer
  float kq_scale;
  int nsplit;
  float* part_o;         // [row][nsplit][256], unnormalised
  float2* part_ml;       // [row][nsplit] (max, sum)
};

}  // namespace q27b

// The part of a list of blocks that a CTA of the decode kernels attends.
#pragma once
#include "common.cuh"
#include "decode_params.h"
#include "rows_plan.h"

namespace q27b {
namespace {

// Position of the token that grid slot z (sequence b, token t) stands for.
__device__ __forceinline__ int sel_pos(const ListParams& p, bool paged, int z) {
  return (paged ? p.seq_len[z / p.sel_T] - p.sel_T : *p.pos0) + z % p.sel_T;
}

// Entries [i0, i1) of the list of (z, kh) that have a row below n, in order, into `list` (shared memory); one warp, returns
// how many. An entry that is no block, or whose page is none, is flagged and left out.
__device__ __forceinline__ int collect_blocks(const ListParams& p, bool paged, int z, int kh, int i0, int i1, int n, int* list) {
  const int lane = threadIdx.x & 31;
  const int* src = p.sel + ((size_t)z * p.nkvh + kh) * p.sel_k;
  int count = 0;
  for (int i = i0; i < i1; i += 32) {
    const int blk = i + lane < i1 ? src[i + lane] : -1;
    if (blk < -1 || blk > (p.n_ctx - 1) / 64) atomicOr(p.status, ST_BAD_INDEX);
    bool ok = blk >= 0 && blk <= (n - 1) / 64 && n > 0;
    if (paged && ok) {
      const int pg = p.page_table[(size_t)(z / p.sel_T) * p.max_pages + blk / (Q27B_PAGE / 64)];
      if (pg < 0 || pg >= p.n_pages) {
        atomicOr(p.status, ST_BAD_PAGE);
        ok = false;
      }
    }
    const uint32_t m = __ballot_sync(0xffffffffu, ok);
    if (ok) list[count + __popc(m & ((1u << lane) - 1))] = blk;
    count += __popc(m);
  }
  return count;
}

}  // namespace
}  // namespace q27b

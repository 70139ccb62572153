// Where the rows of a KV cache lie: one sequence in a contiguous cache, or sequences over a page pool.
#pragma once
#include "common.cuh"
#include "host.h"

namespace q27b {

constexpr int BLK = 64;                  // positions per block of the block-sparse operators (= a tile of the kernels)
constexpr int BLK_PER_PAGE = Q27B_PAGE / BLK;
constexpr int MAX_TREE_T = Q27B_MAX_TREE_T;

struct CacheRef {
  int nkvh, n_ctx;        // paged: n_ctx = max_pages * 256
  int q8;
  int B, T;               // T new tokens of each of B sequences (contiguous: B = 1)
  const int* pos0;        // contiguous: position of the first new token
  const int* page_table;  // paged: [B][max_pages], else null
  const int* seq_len;     // paged: [B], the new tokens included
  int max_pages, n_pages;
  int* status;
};

// Rows of a whole cache or pool (the scales of a q8_0 cache lie behind that many rows of values).
__host__ __device__ inline size_t cache_rows(const CacheRef& c) {
  return (size_t)c.nkvh * (c.page_table ? (size_t)c.n_pages * Q27B_PAGE : (size_t)c.n_ctx);
}
// Position of the first new token of sequence b.
__device__ __forceinline__ int first_pos(const CacheRef& c, int b) { return c.page_table ? c.seq_len[b] - c.T : *c.pos0; }
// Row of position pos of head kh, or -1 (outside the cache; or a page index outside the pool, which is flagged).
__device__ __forceinline__ int64_t cache_row(const CacheRef& c, int b, int kh, int pos) {
  if (pos < 0 || pos >= c.n_ctx) return -1;
  if (!c.page_table) return (int64_t)kh * c.n_ctx + pos;
  const int pg = c.page_table[(size_t)b * c.max_pages + pos / Q27B_PAGE];
  if (pg < 0 || pg >= c.n_pages) {
    atomicOr(c.status, ST_BAD_PAGE);
    return -1;
  }
  return ((int64_t)pg * c.nkvh + kh) * Q27B_PAGE + pos % Q27B_PAGE;
}
// The bounds of block blk (64 positions) of head kh: [2][256] f16 at this block index, or -1.
__device__ __forceinline__ int64_t bounds_index(const CacheRef& c, int b, int kh, int blk) {
  if (!c.page_table) return (int64_t)kh * ((c.n_ctx + BLK - 1) / BLK) + blk;
  const int64_t row = cache_row(c, b, kh, blk * BLK);
  return row < 0 ? -1 : row / BLK;
}

// Fills the contiguous (paged) form; the caller has checked the arguments.
inline CacheRef contiguous_ref(const DeviceCtx* ctx, const int* pos0, int T, int nkvh, int n_ctx, int q8) {
  CacheRef c = {};
  c.nkvh = nkvh; c.n_ctx = n_ctx; c.q8 = q8 != 0; c.B = 1; c.T = T; c.pos0 = pos0; c.status = ctx->status;
  return c;
}
inline CacheRef paged_ref(const DeviceCtx* ctx, const int* page_table, const int* seq_len, int B, int T, int nkvh, int n_pages,
                          int max_pages) {
  CacheRef c = {};
  c.nkvh = nkvh; c.n_ctx = max_pages * Q27B_PAGE; c.q8 = 1; c.B = B; c.T = T; c.page_table = page_table; c.seq_len = seq_len;
  c.max_pages = max_pages; c.n_pages = n_pages; c.status = ctx->status;
  return c;
}
// Shape checks that the entry points share. Row and page counts stay within what an int holds.
inline bool bad_contiguous(int T, int max_T, int nkvh, int n_ctx) {
  return T < 1 || T > max_T || nkvh < 1 || nkvh > 16384 || n_ctx < 1 || (int64_t)nkvh * n_ctx > 0x7fffffff;
}
inline bool bad_paged(int B, int T, int max_T, int nkvh, int n_pages, int max_pages) {
  return B < 1 || B > 65535 || T < 1 || T > max_T || nkvh < 1 || nkvh > 16384 || n_pages < 1 || max_pages < 1 ||
         max_pages > (1 << 22) || (int64_t)n_pages * nkvh * Q27B_PAGE > 0x7fffffff;
}

}  // namespace q27b

// Cache bookkeeping around tree verification and block-sparse drafting: rows of the accepted path moved to the front
// of the drafted rows (commit), per-block bounds of the keys (bounds), choice of the blocks to attend (select).
#include "cache_ref.h"

#include <mutex>

namespace q27b {
namespace {

// ---------------------------------------------------------------- commit
// Row first + i <- row first + path[i] for i < count, K and V, every head. A CTA owns one (head, K or V, sequence): it
// holds all moved rows in registers (up to 64 rows of 272 or 512 bytes in 256 threads) before it writes the first, so a
// path may name rows in any order. Launch and latency bound: 64 rows of 4 heads are 0.3 MB.
constexpr int COMMIT_WARPS = 8, COMMIT_ROWS = MAX_TREE_T / COMMIT_WARPS;

__global__ void __launch_bounds__(32 * COMMIT_WARPS) commit_kernel(const CacheRef c, void* kcache, void* vcache, const int* path,
                                                                   const int* count) {
  pdl_trigger();
  const int kh = blockIdx.x, b = blockIdx.z, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* base = (uint8_t*)(blockIdx.y ? vcache : kcache);
  const size_t scales = cache_rows(c) * AD;
  pdl_wait();
  const int n = min(max(count[b], 0), c.T), first = first_pos(c, b);
  int64_t dst[COMMIT_ROWS];
  uint4 val[COMMIT_ROWS];
  uint32_t sc[COMMIT_ROWS];
#pragma unroll
  for (int j = 0; j < COMMIT_ROWS; j++) {
    const int i = warp + j * COMMIT_WARPS;
    dst[j] = -1;
    if (i >= n) continue;
    const int from = path[(size_t)b * c.T + i];
    if (from < 0 || from >= c.T) {  // not a drafted row: flag it and leave row i as it is
      atomicOr(c.status, ST_BAD_INDEX);
      continue;
    }
    if (from == i) continue;
    const int64_t src = cache_row(c, b, kh, first + from);
    if (src >= 0) dst[j] = cache_row(c, b, kh, first + i);
    if (dst[j] < 0) continue;
    if (c.q8) {
      const uint2 v = *(const uint2*)(base + src * AD + 8 * lane);
      val[j] = make_uint4(v.x, v.y, 0, 0);
      if (lane < 4) sc[j] = *(const uint32_t*)(base + scales + src * 16 + 4 * lane);
    } else {
      val[j] = *(const uint4*)(base + src * 2 * AD + 16 * lane);
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < COMMIT_ROWS; j++) {
    if (dst[j] < 0) continue;
    if (c.q8) {
      *(uint2*)(base + dst[j] * AD + 8 * lane) = make_uint2(val[j].x, val[j].y);
      if (lane < 4) *(uint32_t*)(base + scales + dst[j] * 16 + 4 * lane) = sc[j];
    } else {
      *(uint4*)(base + dst[j] * 2 * AD + 16 * lane) = val[j];
    }
  }
}

int launch_commit(const CacheRef& c, void* kcache, void* vcache, const int* path, const int* count, cudaStream_t s) {
  Q27B_CK(launch_step(commit_kernel, dim3(c.nkvh, 2, c.B), dim3(32 * COMMIT_WARPS), 0, s, c, kcache, vcache, path, count));
  return Q27B_OK;
}

// ---------------------------------------------------------------- bounds
// Per (block of 64 positions, head, dim) the smallest and the largest key as attention reads it (f16; q8_0: value times
// scale, rounded once), over the rows of the block below the sequence's end. NaN stays NaN. One CTA a block and head: 16
// lanes hold a row, 16 row groups take four rows each, all loaded before the first is used.
constexpr int BND_THREADS = 256;

__device__ __forceinline__ void widen(__half2 (&lo)[8], __half2 (&hi)[8], const uint32_t (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i++) {
    lo[i] = __hmin2_nan(lo[i], u32_as_h2(x[i]));
    hi[i] = __hmax2_nan(hi[i], u32_as_h2(x[i]));
  }
}
// 16 int8 values times their block scale, as f16 pairs in order.
__device__ __forceinline__ void dequant16(const uint4& v, __half d, uint32_t (&x)[8]) {
  const __half2 dd = __half2half2(d);
  const uint32_t w[4] = {v.x ^ 0x80808080u, v.y ^ 0x80808080u, v.z ^ 0x80808080u, v.w ^ 0x80808080u};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    x[2 * i] = dq_pair(__byte_perm(w[i], 0x64646464u, 0x4140), dd);
    x[2 * i + 1] = dq_pair(__byte_perm(w[i], 0x64646464u, 0x4342), dd);
  }
}

__global__ void __launch_bounds__(BND_THREADS) bounds_kernel(const CacheRef c, const void* kcache, __half* bounds) {
  __shared__ uint32_t red[BND_THREADS / 32][2][AD / 2];
  pdl_trigger();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, c16 = tid & 15, rg = tid >> 4;
  const int kh = blockIdx.y, b = blockIdx.z;
  pdl_wait();
  const int first = first_pos(c, b), end = min(first + c.T, c.n_ctx);
  const int blk = max(first, 0) / BLK + blockIdx.x, p0 = blk * BLK;
  if (first >= end || p0 >= end) return;
  const int64_t row0 = cache_row(c, b, kh, p0);
  const int64_t at = bounds_index(c, b, kh, blk);
  if (row0 < 0) return;
  const int n = min(BLK, end - p0);
  const __half2 inf = __half2half2(__ushort_as_half((unsigned short)0x7C00)), ninf = __hneg2(inf);
  __half2 lo[8], hi[8];
#pragma unroll
  for (int i = 0; i < 8; i++) lo[i] = inf, hi[i] = ninf;
  uint4 v[4], w[4];
  __half d[4];
  const uint8_t* base = (const uint8_t*)kcache;
  const size_t scales = cache_rows(c) * AD;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const int r = rg + 16 * j;
    if (r >= n) continue;
    const size_t row = (size_t)row0 + r;
    if (c.q8) {
      v[j] = *(const uint4*)(base + row * AD + 16 * c16);
      d[j] = *(const __half*)(base + scales + row * 16 + (c16 >> 1) * 2);
    } else {
      v[j] = *(const uint4*)(base + row * 2 * AD + 32 * c16);
      w[j] = *(const uint4*)(base + row * 2 * AD + 32 * c16 + 16);
    }
  }
#pragma unroll
  for (int j = 0; j < 4; j++) {
    if (rg + 16 * j >= n) continue;
    uint32_t x[8];
    if (c.q8) {
      dequant16(v[j], d[j], x);
    } else {
      x[0] = v[j].x, x[1] = v[j].y, x[2] = v[j].z, x[3] = v[j].w;
      x[4] = w[j].x, x[5] = w[j].y, x[6] = w[j].z, x[7] = w[j].w;
    }
    widen(lo, hi, x);
  }
#pragma unroll
  for (int i = 0; i < 8; i++) {
    lo[i] = __hmin2_nan(lo[i], u32_as_h2(__shfl_xor_sync(0xffffffffu, h2_as_u32(lo[i]), 16)));
    hi[i] = __hmax2_nan(hi[i], u32_as_h2(__shfl_xor_sync(0xffffffffu, h2_as_u32(hi[i]), 16)));
    if (lane < 16) {
      red[warp][0][c16 * 8 + i] = h2_as_u32(lo[i]);
      red[warp][1][c16 * 8 + i] = h2_as_u32(hi[i]);
    }
  }
  __syncthreads();
  const int which = tid >> 7, pair = tid & 127;
  __half2 m = u32_as_h2(red[0][which][pair]);
#pragma unroll
  for (int k = 1; k < BND_THREADS / 32; k++) {
    const __half2 x = u32_as_h2(red[k][which][pair]);
    m = which ? __hmax2_nan(m, x) : __hmin2_nan(m, x);
  }
  ((uint32_t*)bounds)[(size_t)at * AD + tid] = h2_as_u32(m);
}

int launch_bounds(const CacheRef& c, const void* kcache, void* bounds, cudaStream_t s) {
  const unsigned blocks = (unsigned)((c.T + BLK - 2) / BLK + 1);  // as many as T rows can touch
  Q27B_CK(launch_step(bounds_kernel, dim3(blocks, c.nkvh, c.B), dim3(BND_THREADS), 0, s, c, kcache, (__half*)bounds));
  return Q27B_OK;
}

// ---------------------------------------------------------------- select
// score(block) = max over the six query heads of the KV head of sum_d max(q_d lo_d, q_d hi_d): no key of the block has a
// larger q.k. The order of scores decides what is attended, so they are sums in 64 bits (the products of f32 and f16
// values are exact there): which block wins does not depend on the order of a sum, short of differences of 1e-16.
struct SelectParams {
  CacheRef c;
  const float* qn;        // [B][T][6 nkvh][256]
  const __half* bounds;
  int* sel;               // [B][T][nkvh][k]
  int k, n_sink, n_recent;
};
constexpr int SEL_THREADS = 512;
constexpr int SEL_MAX_BLOCKS = 16384;

// Keys in the order of the scores: larger score, larger key; NaN above all.
__device__ __forceinline__ unsigned long long score_key(double s) {
  if (s != s) return ~0ull;
  const long long bits = __double_as_longlong(s + 0.0);
  return bits < 0 ? ~(unsigned long long)bits : (unsigned long long)bits | 0x8000000000000000ull;
}
// Exclusive sum over the block of x (two counts, 32 bits each); *total of all threads.
__device__ __forceinline__ unsigned long long block_scan(unsigned long long x, unsigned long long* sums, unsigned long long* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned long long v = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  if (lane == 31) sums[warp] = v;
  __syncthreads();
  unsigned long long before = 0, all = 0;
  for (int w = 0; w < SEL_THREADS / 32; w++) {
    if (w < warp) before += sums[w];
    all += sums[w];
  }
  __syncthreads();
  *total = all;
  return before + v - x;
}

__global__ void __launch_bounds__(SEL_THREADS) select_kernel(const SelectParams p) {
  extern __shared__ unsigned long long keys[];
  __shared__ double q[GQA][AD];
  __shared__ unsigned long long sums[SEL_THREADS / 32];
  __shared__ unsigned int hist[256];
  __shared__ unsigned long long s_prefix;
  __shared__ int s_need, s_done;
  pdl_trigger();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int kh = blockIdx.x, t = blockIdx.y, b = blockIdx.z, nqh = p.c.nkvh * GQA;
  int* out = p.sel + (((size_t)b * p.c.T + t) * p.c.nkvh + kh) * p.k;
  pdl_wait();
  const int last_pos = min(first_pos(p.c, b) + t, p.c.n_ctx - 1);
  const int nb = last_pos < 0 ? 0 : last_pos / BLK + 1;  // blocks up to the token's own
  const int sink = min(p.n_sink, nb), recent = min(p.n_recent, nb - sink), lo = sink, hi = nb - recent;
  const int want = p.k - sink - recent;  // of the blocks [lo, hi)
  if (nb <= p.k) {
    for (int i = tid; i < p.k; i += SEL_THREADS) out[i] = i < nb ? i : -1;
    return;
  }
  const float* qn = p.qn + (((size_t)b * p.c.T + t) * nqh + kh * GQA) * AD;
  for (int i = tid; i < GQA * AD; i += SEL_THREADS) (&q[0][0])[i] = (double)qn[i];
  __syncthreads();
  for (int blk = lo + warp; blk < hi; blk += SEL_THREADS / 32) {
    const int64_t at = bounds_index(p.c, b, kh, blk);
    double s[GQA] = {};
    if (at >= 0) {
      const uint4 l4 = *(const uint4*)(p.bounds + at * 2 * AD + 8 * lane), h4 = *(const uint4*)(p.bounds + at * 2 * AD + AD + 8 * lane);
      const uint32_t lw[4] = {l4.x, l4.y, l4.z, l4.w}, hw[4] = {h4.x, h4.y, h4.z, h4.w};
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const float2 lf = __half22float2(u32_as_h2(lw[i >> 1])), hf = __half22float2(u32_as_h2(hw[i >> 1]));
        const double l = i & 1 ? lf.y : lf.x, h = i & 1 ? hf.y : hf.x;
#pragma unroll
        for (int g = 0; g < GQA; g++) {
          const double x = q[g][8 * lane + i];
          s[g] = fma(x, x < 0.0 ? l : h, s[g]);
        }
      }
    }
    double best = -INFINITY;
    bool nan = false;
#pragma unroll
    for (int g = 0; g < GQA; g++) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s[g] += __shfl_xor_sync(0xffffffffu, s[g], o);
      nan |= s[g] != s[g];
      best = fmax(best, s[g]);
    }
    if (lane == 0) keys[blk - lo] = at < 0 ? 0ull : nan ? ~0ull : score_key(best);
  }
  __syncthreads();
  // The want-th largest key, eight bits at a time from the top; done early when a bin holds just what is still wanted.
  const int n = hi - lo;
  if (tid == 0) s_prefix = 0, s_need = want, s_done = 0;
  int shift = 56;
  unsigned long long mask = 0;
  __syncthreads();
  if (want > 0) {
    for (; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += SEL_THREADS) hist[i] = 0;
      __syncthreads();
      const unsigned long long prefix = s_prefix;
      for (int i = tid; i < n; i += SEL_THREADS)
        if ((keys[i] & mask) == prefix) atomicAdd(&hist[(unsigned)(keys[i] >> shift) & 255u], 1u);
      __syncthreads();
      if (tid == 0) {
        int need = s_need, d = 255;
        while ((int)hist[d] < need) need -= (int)hist[d--];
        s_need = need;
        s_prefix = prefix | ((unsigned long long)d << shift);
        s_done = (int)hist[d] == need;
      }
      __syncthreads();
      mask |= 255ull << shift;
      if (s_done) break;
    }
  }
  // Blocks above the prefix are in; of those that share it all (done early) or the first s_need.
  const unsigned long long prefix = s_prefix;
  const int need = want > 0 ? s_need : 0;
  const int per = (nb + SEL_THREADS - 1) / SEL_THREADS, b0 = min(nb, tid * per), b1 = min(nb, b0 + per);
  auto rank_of = [&](int blk) {  // 2: in, 1: shares the prefix, 0: out
    if (blk < lo || blk >= hi) return 2;
    if (want <= 0) return 0;
    const unsigned long long k = keys[blk - lo] & mask;
    return k > prefix ? 2 : k == prefix ? 1 : 0;
  };
  unsigned long long mine = 0, total;
  for (int blk = b0; blk < b1; blk++) {
    const int r = rank_of(blk);
    mine += r == 2 ? 1ull << 32 : r == 1 ? 1ull : 0ull;
  }
  const unsigned long long before = block_scan(mine, sums, &total);
  int above = (int)(before >> 32), equal = (int)(before & 0xffffffffu);
  for (int blk = b0; blk < b1; blk++) {
    const int r = rank_of(blk);
    if (r == 2 || (r == 1 && equal < need)) out[above + min(equal, need)] = blk;
    above += r == 2;
    equal += r == 1;
  }
}

int launch_select(const SelectParams& p, int max_len, cudaStream_t s) {
  static bool attr[64] = {};
  static std::mutex attr_mu;
  int dev;
  Q27B_CK(cudaGetDevice(&dev));
  {
    std::lock_guard<std::mutex> lock(attr_mu);
    if (!attr[dev]) {
      Q27B_CK(cudaFuncSetAttribute(select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SEL_MAX_BLOCKS * 8));
      attr[dev] = true;
    }
  }
  const size_t smem = (size_t)((max_len + BLK - 1) / BLK) * 8;
  Q27B_CK(launch_step(select_kernel, dim3(p.c.nkvh, p.c.T, p.c.B), dim3(SEL_THREADS), smem, s, p));
  return Q27B_OK;
}

int check_select(const char* who, int T, int k, int n_sink, int n_recent, int nqh, int nkvh, int64_t max_len) {
  if (T > Q27B_MAX_T || nqh != nkvh * GQA || k < 1 || k > SEL_MAX_BLOCKS || n_sink < 0 || n_recent < 1 || n_sink > k ||
      n_recent > k - n_sink)
    return fail(Q27B_BAD_SHAPE, std::string(who) + ": bad shape");
  if (max_len > (int64_t)SEL_MAX_BLOCKS * BLK)
    return fail(Q27B_UNSUPPORTED, std::string(who) + ": sequences of more than " + std::to_string(SEL_MAX_BLOCKS * BLK) + " positions");
  return Q27B_OK;
}

}  // namespace
}  // namespace q27b

using namespace q27b;

extern "C" {

int q27b_kv_commit(void* kcache, void* vcache, const int* pos0, const int* path, const int* count, int T, int nkvh, int n_ctx,
                   int q8, void* stream) {
  if (!kcache || !vcache || !pos0 || !path || !count) return fail(Q27B_BAD_SHAPE, "kv_commit: null pointer");
  if (bad_contiguous(T, MAX_TREE_T, nkvh, n_ctx)) return fail(Q27B_BAD_SHAPE, "kv_commit: bad shape");
  DeviceCtx* ctx;
  if (int rc = device_ctx(&ctx)) return rc;
  return launch_commit(contiguous_ref(ctx, pos0, T, nkvh, n_ctx, q8), kcache, vcache, path, count, (cudaStream_t)stream);
}

int q27b_kv_commit_paged(void* kpool, void* vpool, const int* page_table, const int* seq_len, const int* path, const int* count,
                         int B, int T, int nkvh, int n_pages, int max_pages, void* stream) {
  if (!kpool || !vpool || !page_table || !seq_len || !path || !count) return fail(Q27B_BAD_SHAPE, "kv_commit_paged: null pointer");
  if (bad_paged(B, T, MAX_TREE_T, nkvh, n_pages, max_pages)) return fail(Q27B_BAD_SHAPE, "kv_commit_paged: bad shape");
  DeviceCtx* ctx;
  if (int rc = device_ctx(&ctx)) return rc;
  return launch_commit(paged_ref(ctx, page_table, seq_len, B, T, nkvh, n_pages, max_pages), kpool, vpool, path, count,
                       (cudaStream_t)stream);
}

uint64_t q27b_kv_bounds_bytes(int nkvh, int n_ctx) {
  return nkvh < 1 || n_ctx < 1 ? 0 : (uint64_t)nkvh * (((uint64_t)n_ctx + BLK - 1) / BLK) * 2 * AD * 2;
}
uint64_t q27b_kv_bounds_pool_bytes(int nkvh, int n_pages) {
  return nkvh < 1 || n_pages < 1 ? 0 : (uint64_t)n_pages * nkvh * BLK_PER_PAGE * 2 * AD * 2;
}

int q27b_kv_bounds(const void* kcache, void* bounds, const int* pos0, int T, int nkvh, int n_ctx, int q8, void* stream) {
  if (!kcache || !bounds || !pos0) return fail(Q27B_BAD_SHAPE, "kv_bounds: null pointer");
  if (bad_contiguous(T, 0x7fffffff, nkvh, n_ctx) || T > n_ctx) return fail(Q27B_BAD_SHAPE, "kv_bounds: bad shape");
  DeviceCtx* ctx;
  if (int rc = device_ctx(&ctx)) return rc;
  return launch_bounds(contiguous_ref(ctx, pos0, T, nkvh, n_ctx, q8), kcache, bounds, (cudaStream_t)stream);
}

int q27b_kv_bounds_paged(const void* kpool, void* bounds, const int* page_table, const int* seq_len, int B, int T, int nkvh,
                         int n_pages, int max_pages, void* stream) {
  if (!kpool || !bounds || !page_table || !seq_len) return fail(Q27B_BAD_SHAPE, "kv_bounds_paged: null pointer");
  if (bad_paged(B, T, 0x7fffffff, nkvh, n_pages, max_pages) || T > max_pages * Q27B_PAGE)
    return fail(Q27B_BAD_SHAPE, "kv_bounds_paged: bad shape");
  DeviceCtx* ctx;
  if (int rc = device_ctx(&ctx)) return rc;
  return launch_bounds(paged_ref(ctx, page_table, seq_len, B, T, nkvh, n_pages, max_pages), kpool, bounds, (cudaStream_t)stream);
}

int q27b_select_blocks(const float* qn, const void* bounds, int* sel, const int* pos0, int T, int k, int n_sink, int n_recent,
                       int nqh, int nkvh, int n_ctx, void* stream) {
  if (!qn || !bounds || !sel || !pos0) return fail(Q27B_BAD_SHAPE, "select_blocks: null pointer");
  if (bad_contiguous(T, Q27B_MAX_T, nkvh, n_ctx)) return fail(Q27B_BAD_SHAPE, "select_blocks: bad shape");
  if (int rc = check_select("select_blocks", T, k, n_sink, n_recent, nqh, nkvh, n_ctx)) return rc;
  DeviceCtx* ctx;
  if (int rc = device_ctx(&ctx)) return rc;
  SelectParams p = {};
  p.c = contiguous_ref(ctx, pos0, T, nkvh, n_ctx, 1);
  p.qn = qn; p.bounds = (const __half*)bounds; p.sel = sel; p.k = k; p.n_sink = n_sink; p.n_recent = n_recent;
  return launch_select(p, n_ctx, (cudaStream_t)stream);
}

int q27b_select_blocks_paged(const float* qn, const void* bounds, int* sel, const int* page_table, const int* seq_len, int B,
                             int T, int k, int n_sink, int n_recent, int nqh, int nkvh, int n_pages, int max_pages,
                             int max_seq_len, void* stream) {
  if (!qn || !bounds || !sel || !page_table || !seq_len) return fail(Q27B_BAD_SHAPE, "select_blocks_paged: null pointer");
  if (bad_paged(B, T, Q27B_MAX_T, nkvh, n_pages, max_pages) || max_seq_len < T || max_seq_len > max_pages * Q27B_PAGE)
    return fail(Q27B_BAD_SHAPE, "select_blocks_paged: bad shape");
  if (int rc = check_select("select_blocks_paged", T, k, n_sink, n_recent, nqh, nkvh, max_seq_len)) return rc;
  DeviceCtx* ctx;
  if (int rc = device_ctx(&ctx)) return rc;
  SelectParams p = {};
  p.c = paged_ref(ctx, page_table, seq_len, B, T, nkvh, n_pages, max_pages);
  p.c.n_ctx = max_seq_len;  // a longer sequence than the caller said is cut there: the scores have room for no more
  p.qn = qn; p.bounds = (const __half*)bounds; p.sel = sel; p.k = k; p.n_sink = n_sink; p.n_recent = n_recent;
  return launch_select(p, max_seq_len, (cudaStream_t)stream);
}

}  // extern "C"

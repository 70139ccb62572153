// Decode attention over part of a cache: T drafted tokens of a tree (every draft sees the prefix and the drafts of its
// mask), and T tokens that each attend their own list of 64-position blocks.
//
// y = sigmoid(gate) * sum_p P_p v_p with P the softmax of kq_scale * q.k over the visible rows p, in f32; 0 where a row
// sees nothing. Rows that are not visible are not read, whatever they hold.
//
// One CTA takes the six query rows of a (token, KV head) over one share of its positions: a warp per position, eight
// dims a lane; m, l and O of each warp are merged at the end and written as a partial, and a second kernel merges the
// partials of a row.
#include "cache_ref.h"
#include "decode_rows.h"

namespace q27b {
namespace {

constexpr int WARPS = 8;

// Eight values of a stored row as f32.
__device__ __forceinline__ void load8(const uint8_t* base, size_t scales, bool q8, size_t row, int lane, float (&x)[8]) {
  if (q8) {
    const uint2 v = *(const uint2*)(base + row * AD + 8 * lane);
    const float d = __half2float(*(const __half*)(base + scales + row * 16 + (lane >> 2) * 2));
    const int8_t* b = (const int8_t*)&v;
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = (float)b[i] * d;
  } else {
    const uint4 v = *(const uint4*)(base + row * 2 * AD + 16 * lane);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float2 f = __half22float2(u32_as_h2(w[i]));
      x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
  }
}

__global__ void __launch_bounds__(32 * WARPS) blocks_kernel(const RowsParams p) {
  __shared__ float sm[WARPS][GQA], sl[WARPS][GQA], so[WARPS][AD];
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int z = blockIdx.x, kh = blockIdx.y, b = blockIdx.z / p.c.T, t = blockIdx.z % p.c.T, nqh = p.c.nkvh * GQA;
  pdl_wait();
  const int first = first_pos(p.c, b), n = max(0, min(first + p.c.T, p.c.n_ctx));
  const int share = (p.k + p.nsplit - 1) / p.nsplit;
  const int* list = p.sel + (((size_t)b * p.c.T + t) * p.c.nkvh + kh) * p.k;
  const size_t row0 = ((size_t)b * p.c.T + t) * nqh + kh * GQA;  // the first of the six output rows
  float q[GQA][8], o[GQA][8], m[GQA], l[GQA];
#pragma unroll
  for (int g = 0; g < GQA; g++) {
    const float* src = p.qn + (row0 + g) * AD + 8 * lane;
#pragma unroll
    for (int i = 0; i < 8; i++) q[g][i] = src[i] * p.kq_scale, o[g][i] = 0.f;
    m[g] = M_INIT;
    l[g] = 0.f;
  }
  const size_t scales = cache_rows(p.c) * AD;
  for (int i = z * share; i < min(p.k, (z + 1) * share); i++) {
    const int tile = list[i];
    if (tile == -1) continue;
    if (tile < -1 || tile > (p.c.n_ctx - 1) / BLK) {
      if (threadIdx.x == 0) atomicOr(p.c.status, ST_BAD_INDEX);
      continue;
    }
    if (tile * BLK >= n) continue;
    const int64_t base = cache_row(p.c, b, kh, tile * BLK);
    if (base < 0) continue;
    for (int r = warp; r < BLK; r += WARPS) {
      const int pos = tile * BLK + r;
      if (pos >= n || pos > first + t) continue;
      float x[8], s[GQA];
      load8((const uint8_t*)p.kcache, scales, p.c.q8, base + r, lane, x);
#pragma unroll
      for (int g = 0; g < GQA; g++) {
        s[g] = 0.f;
#pragma unroll
        for (int e = 0; e < 8; e++) s[g] = fmaf(q[g][e], x[e], s[g]);
#pragma unroll
        for (int e = 16; e > 0; e >>= 1) s[g] += __shfl_xor_sync(0xffffffffu, s[g], e);
      }
      load8((const uint8_t*)p.vcache, scales, p.c.q8, base + r, lane, x);
#pragma unroll
      for (int g = 0; g < GQA; g++) {
        const float mn = fmaxf(m[g], s[g]), f = ex2((m[g] - mn) * LOG2E), e = ex2((s[g] - mn) * LOG2E);
        m[g] = mn;
        l[g] = l[g] * f + e;
#pragma unroll
        for (int k = 0; k < 8; k++) o[g][k] = fmaf(e, x[k], o[g][k] * f);
      }
    }
  }
  if (lane == 0)
#pragma unroll
    for (int g = 0; g < GQA; g++) sm[warp][g] = m[g], sl[warp][g] = l[g];
#pragma unroll
  for (int g = 0; g < GQA; g++) {
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 8; k++) so[warp][8 * lane + k] = o[g][k];
    __syncthreads();
    float M = M_INIT, L = 0.f, A = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; w++) M = fmaxf(M, sm[w][g]);
#pragma unroll
    for (int w = 0; w < WARPS; w++) {
      const float f = ex2((sm[w][g] - M) * LOG2E);
      L += sl[w][g] * f;
      A += so[w][threadIdx.x] * f;
    }
    const size_t at = (row0 + g) * p.nsplit + z;
    p.part_o[at * AD + threadIdx.x] = A;
    if (threadIdx.x == 0) p.part_ml[at] = make_float2(M, L);
  }
}

// Merges the partials of a row, applies the gate and writes f16, or q8_1. One CTA a row, four groups of 64 threads that
// take every fourth partial; a row without a visible position is 0.
__global__ void __launch_bounds__(256) rows_merge_kernel(const RowsParams p) {
  __shared__ float4 sa[3][64];
  __shared__ float sl[4];
  const size_t row = blockIdx.x;
  const int grp = threadIdx.x >> 6, c = threadIdx.x & 63;
  pdl_wait();
  pdl_trigger();
  const float2* ml = p.part_ml + row * p.nsplit;
  int np = p.nsplit;  // partials that were written
  if (!p.sel) {
    const int b = (int)(row / ((size_t)p.c.T * p.c.nkvh * GQA)), ntot = tree_tiles(min(first_pos(p.c, b) + p.c.T, p.c.n_ctx));
    np = ntot ? (ntot - 1) / tree_share(p, ntot) + 1 : 0;
  }
  float M = M_INIT;
  for (int z = 0; z < np; z++) M = fmaxf(M, ml[z].x);
  float L = 0.f;
  float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int z = grp; z < np; z += 4) {
    const float2 v = ml[z];
    if (v.y == 0.f) continue;  // holds nothing
    const float f = ex2((v.x - M) * LOG2E);
    const float4 x = *(const float4*)(p.part_o + (row * p.nsplit + z) * AD + 4 * c);
    L += v.y * f;
    A.x += x.x * f, A.y += x.y * f, A.z += x.z * f, A.w += x.w * f;
  }
  if (grp > 0) sa[grp - 1][c] = A;
  if (c == 0) sl[grp] = L;
  __syncthreads();
  if (grp > 0) return;
#pragma unroll
  for (int k = 0; k < 3; k++) {
    const float4 x = sa[k][c];
    A.x += x.x, A.y += x.y, A.z += x.z, A.w += x.w;
    L += sl[k + 1];
  }
  const float inv = L == 0.f ? 0.f : 1.0f / L;
  const float4 g = *(const float4*)(p.qg + row * 2 * AD + AD + 4 * c);
  float y[4] = {A.x * inv, A.y * inv, A.z * inv, A.w * inv};
  const float gv[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
  for (int i = 0; i < 4; i++) y[i] *= 1.0f / (1.0f + expf(-gv[i]));
  if (!p.xq) {
    *(uint2*)((__half*)p.o + row * AD + 4 * c) = make_uint2(pack_h2(y[0], y[1]), pack_h2(y[2], y[3]));
    return;
  }
  // q8_1 of 32 dims = eight lanes, as the merge of attn_decode writes it
  float amax = fmaxf(fmaxf(fabsf(y[0]), fabsf(y[1])), fmaxf(fabsf(y[2]), fabsf(y[3])));
#pragma unroll
  for (int o = 1; o <= 4; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  const float d = __fdiv_rn(amax, 127.0f);
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; i++) w |= (uint32_t)((amax == 0.0f ? 0 : (int)roundf(__fdiv_rn(y[i], d))) & 0xFF) << (8 * i);
  *(uint32_t*)(p.xq + row * AD + 4 * c) = w;
  if ((c & 7) == 0) p.xd[(row * AD + 4 * c) / 32] = __half2float(__float2half_rn(d));
}

// Rounds a workspace of `floats` down to the splits that it holds of `rows` rows.
int64_t splits_that_fit(size_t floats, int64_t rows) { return (int64_t)(floats / ((size_t)rows * (AD + 2))); }

// Partials of `rows` rows in *nsplit splits: in the prefill workspace, whose size is fixed (fewer splits where it holds no
// more), or, for a batch, in the paged workspace.
int place_partials(DeviceCtx* ctx, RowsParams& p, int64_t rows, int64_t nsplit, const char* who) {
  float* part;
  if (p.c.page_table) {
    if (int rc = paged_ws(ctx, (size_t)rows * nsplit * (AD + 2), &part)) return rc;
  } else {
    size_t cap;
    if (int rc = prefill_ws(ctx, &part, &cap)) return rc;
    const int64_t fit = splits_that_fit(cap, rows);
    if (fit < 1)
      return fail(Q27B_UNSUPPORTED, std::string(who) + ": the prefill workspace (" + std::to_string(cap * sizeof(float)) +
                                        " bytes) is too small for the partials of this call (" +
                                        std::to_string((size_t)rows * (AD + 2) * sizeof(float)) + " bytes)");
    nsplit = std::min(nsplit, fit);
  }
  p.nsplit = (int)nsplit;
  p.part_o = part;
  p.part_ml = (float2*)(part + (size_t)rows * nsplit * AD);
  return Q27B_OK;
}

int run_blocks(DeviceCtx* ctx, RowsParams& p, const char* who, cudaStream_t s) {
  const int64_t rows = (int64_t)p.c.B * p.c.T * p.c.nkvh * GQA, ctas = (int64_t)p.c.B * p.c.T * p.c.nkvh;
  const int64_t ns = std::max<int64_t>(1, std::min<int64_t>({p.k, 64, (8 * (int64_t)ctx->n_sm + ctas - 1) / ctas}));
  if (int rc = place_partials(ctx, p, rows, ns, who)) return rc;
  Q27B_CK(launch_step(blocks_kernel, dim3(p.nsplit, p.c.nkvh, p.c.B * p.c.T), dim3(32 * WARPS), 0, s, p));
  Q27B_CK(launch_step(rows_merge_kernel, dim3((unsigned)rows), dim3(256), 0, s, p));
  return Q27B_OK;
}

// One sequence: a CTA per SM, the positions of every row tile in equal shares. A batch: shares of equal length, so that the
// sequences' CTAs come to about four rounds of the SMs if all are of the largest length.
int run_tree(DeviceCtx* ctx, RowsParams& p, const char* who, cudaStream_t s) {
  const int64_t rows = (int64_t)p.c.B * p.c.T * p.c.nkvh * GQA, ctas = (int64_t)p.c.B * p.c.nkvh * tree_row_tiles(p.c.T);
  const int64_t tiles = tree_tiles(p.c.n_ctx);
  int64_t ns;
  if (p.c.page_table) {
    const int64_t share = std::min<int64_t>(TREE_MAX_SHARE, std::max<int64_t>(8, ctas * tiles / (4 * ctx->n_sm)));
    p.share = (int)share;
    ns = (tiles + share - 1) / share;
  } else {
    ns = std::max<int64_t>(1, std::min(tiles, ctx->n_sm / ctas));
  }
  if (int rc = place_partials(ctx, p, rows, ns, who)) return rc;
  if (int rc = launch_tree(p, s)) return rc;
  Q27B_CK(launch_step(rows_merge_kernel, dim3((unsigned)rows), dim3(256), 0, s, p));
  return Q27B_OK;
}

}  // namespace
}  // namespace q27b

using namespace q27b;

extern "C" {

int q27b_tree_plan(const int* parent, int T, uint64_t* mask, int* depth) {
  if (!parent || !mask) return fail(Q27B_BAD_SHAPE, "tree_plan: null pointer");
  if (T < 1 || T > Q27B_MAX_TREE_T) return fail(Q27B_BAD_SHAPE, "tree_plan: bad shape");
  for (int t = 0; t < T; t++)
    if (parent[t] < -1 || parent[t] >= t)
      return fail(Q27B_BAD_SHAPE, "tree_plan: the parent of draft " + std::to_string(t) + " is " + std::to_string(parent[t]) +
                                      ", neither -1 nor an earlier draft");
  int d[Q27B_MAX_TREE_T];
  for (int t = 0; t < T; t++) {
    mask[t] = (parent[t] < 0 ? 0 : mask[parent[t]]) | (uint64_t)1 << t;
    d[t] = parent[t] < 0 ? 0 : d[parent[t]] + 1;
    if (depth) depth[t] = d[t];
  }
  return Q27B_OK;
}

int q27b_attn_decode_tree(const float* qn, const float* qg, const void* kcache, const void* vcache, void* o, int8_t* xq, float* xd,
                          const int* pos0, const uint64_t* mask, int T, float kq_scale, int nqh, int nkvh, int n_ctx, int q8,
                          void* stream) {
  if (bad_contiguous(T, MAX_TREE_T, nkvh, n_ctx) || nqh != nkvh * GQA || T > n_ctx)
    return fail(Q27B_BAD_SHAPE, "attn_decode_tree: bad shape");
  if (!qn || !qg || !kcache || !vcache || !pos0 || !mask || (!o && !xq) || (xq && !xd))
    return fail(Q27B_BAD_SHAPE, "attn_decode_tree: null pointer");
  DeviceCtx* ctx;
  if (int rc = device_ctx(&ctx)) return rc;
  RowsParams p = {};
  p.c = contiguous_ref(ctx, pos0, T, nkvh, n_ctx, q8);
  p.qn = qn; p.qg = qg; p.kcache = kcache; p.vcache = vcache; p.o = o; p.xq = xq; p.xd = xd; p.mask = mask; p.kq_scale = kq_scale;
  return run_tree(ctx, p, "attn_decode_tree", (cudaStream_t)stream);
}

int q27b_attn_decode_tree_paged(const float* qn, const float* qg, const void* kpool, const void* vpool, const int* page_table,
                                const int* seq_len, const uint64_t* mask, void* o, int8_t* xq, float* xd, int B, int T,
                                float kq_scale, int nqh, int nkvh, int n_pages, int max_pages, int max_seq_len, void* stream) {
  if (bad_paged(B, T, MAX_TREE_T, nkvh, n_pages, max_pages) || nqh != nkvh * GQA || max_seq_len < T ||
      max_seq_len > max_pages * Q27B_PAGE || (int64_t)B * T > 65535)
    return fail(Q27B_BAD_SHAPE, "attn_decode_tree_paged: bad shape");
  if (!qn || !qg || !kpool || !vpool || !page_table || !seq_len || !mask || (!o && !xq) || (xq && !xd))
    return fail(Q27B_BAD_SHAPE, "attn_decode_tree_paged: null pointer");
  DeviceCtx* ctx;
  if (int rc = device_ctx(&ctx)) return rc;
  RowsParams p = {};
  p.c = paged_ref(ctx, page_table, seq_len, B, T, nkvh, n_pages, max_pages);
  p.c.n_ctx = max_seq_len;  // a longer sequence is cut there
  p.qn = qn; p.qg = qg; p.kcache = kpool; p.vcache = vpool; p.o = o; p.xq = xq; p.xd = xd; p.mask = mask; p.kq_scale = kq_scale;
  return run_tree(ctx, p, "attn_decode_tree_paged", (cudaStream_t)stream);
}

int q27b_attn_decode_blocks(const float* qn, const float* qg, const void* kcache, const void* vcache, void* o, int8_t* xq,
                            float* xd, const int* pos0, const int* sel, int T, int k, float kq_scale, int nqh, int nkvh, int n_ctx,
                            int q8, void* stream) {
  if (bad_contiguous(T, Q27B_MAX_T, nkvh, n_ctx) || nqh != nkvh * GQA || k < 1 || k > MAX_SEL)
    return fail(Q27B_BAD_SHAPE, "attn_decode_blocks: bad shape");
  if (!qn || !qg || !kcache || !vcache || !pos0 || !sel || (!o && !xq) || (xq && !xd))
    return fail(Q27B_BAD_SHAPE, "attn_decode_blocks: null pointer");
  DeviceCtx* ctx;
  if (int rc = device_ctx(&ctx)) return rc;
  RowsParams p = {};
  p.c = contiguous_ref(ctx, pos0, T, nkvh, n_ctx, q8);
  p.qn = qn; p.qg = qg; p.kcache = kcache; p.vcache = vcache; p.o = o; p.xq = xq; p.xd = xd; p.sel = sel; p.k = k;
  p.kq_scale = kq_scale;
  return run_blocks(ctx, p, "attn_decode_blocks", (cudaStream_t)stream);
}

int q27b_attn_decode_blocks_paged(const float* qn, const float* qg, const void* kpool, const void* vpool, const int* page_table,
                                  const int* seq_len, const int* sel, void* o, int8_t* xq, float* xd, int B, int T, int k,
                                  float kq_scale, int nqh, int nkvh, int n_pages, int max_pages, void* stream) {
  if (bad_paged(B, T, Q27B_MAX_T, nkvh, n_pages, max_pages) || nqh != nkvh * GQA || k < 1 || k > MAX_SEL ||
      (int64_t)B * T > 65535)
    return fail(Q27B_BAD_SHAPE, "attn_decode_blocks_paged: bad shape");
  if (!qn || !qg || !kpool || !vpool || !page_table || !seq_len || !sel || (!o && !xq) || (xq && !xd))
    return fail(Q27B_BAD_SHAPE, "attn_decode_blocks_paged: null pointer");
  DeviceCtx* ctx;
  if (int rc = device_ctx(&ctx)) return rc;
  RowsParams p = {};
  p.c = paged_ref(ctx, page_table, seq_len, B, T, nkvh, n_pages, max_pages);
  p.qn = qn; p.qg = qg; p.kcache = kpool; p.vcache = vpool; p.o = o; p.xq = xq; p.xd = xd; p.sel = sel; p.k = k;
  p.kq_scale = kq_scale;
  return run_blocks(ctx, p, "attn_decode_blocks_paged", (cudaStream_t)stream);
}

}  // extern "C"

// Decode attention over part of a cache: T drafted tokens of a tree (every draft sees the prefix and the drafts of its
// mask), and T tokens that each attend their own list of 64-position blocks.
//
// y = sigmoid(gate) * sum_p P_p v_p with P the softmax of kq_scale * q.k over the visible rows p, in f32; 0 where a row
// sees nothing. Rows that are not visible may be loaded (tiles of 64), but have no influence, whatever they hold.
//
// The split kernels leave the partials (m, l, O) of a row for every part of its positions; the kernels here merge them. Trees:
// decode_tree.cu, or for up to four drafts the kernels of q27b_attn_decode over the prefix. Lists of blocks: the split-K kernels
// of decode_ws.cu (q8_0) and decode.cu (f16), a chunk of a list a CTA, every (token, KV head) for itself.
#include "cache_ref.h"
#include "decode_params.h"
#include "decode_rows.h"

namespace q27b {
namespace {

// Dims 4 c .. 4 c + 3 of a row (c = 0..63, two whole warps): A / L times the gate, as f16 or q8_1.
__device__ __forceinline__ void write_row(const RowsParams& p, size_t row, int c, const float4& A, float L, const float4& g) {
  const float inv = L == 0.f ? 0.f : 1.0f / L;
  float out[4] = {A.x * inv, A.y * inv, A.z * inv, A.w * inv};
  const float gv[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
  for (int i = 0; i < 4; i++) out[i] *= 1.0f / (1.0f + expf(-gv[i]));
  if (!p.xq) {
    *(uint2*)((__half*)p.o + row * AD + 4 * c) = make_uint2(pack_h2(out[0], out[1]), pack_h2(out[2], out[3]));
    return;
  }
  // q8_1 of 32 dims = eight lanes, as the merge of attn_decode writes it
  float amax = fmaxf(fmaxf(fabsf(out[0]), fabsf(out[1])), fmaxf(fabsf(out[2]), fabsf(out[3])));
#pragma unroll
  for (int o = 1; o <= 4; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  const float d = __fdiv_rn(amax, 127.0f);
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; i++) w |= (uint32_t)((amax == 0.0f ? 0 : (int)roundf(__fdiv_rn(out[i], d))) & 0xFF) << (8 * i);
  *(uint32_t*)(p.xq + row * AD + 4 * c) = w;
  if ((c & 7) == 0) p.xd[(row * AD + 4 * c) / 32] = __half2float(__float2half_rn(d));
}

// Dims 4 c .. 4 c + 3 of a row of head kh of a cache, in f32.
__device__ __forceinline__ float4 four_of(const CacheRef& ref, const void* cache, int64_t at, int c) {
  const uint8_t* base = (const uint8_t*)cache;
  if (!ref.q8) {
    const uint2 w = *(const uint2*)(base + at * 2 * AD + 8 * c);
    const float2 lo = __half22float2(u32_as_h2(w.x)), hi = __half22float2(u32_as_h2(w.y));
    return make_float4(lo.x, lo.y, hi.x, hi.y);
  }
  const uint32_t w = *(const uint32_t*)(base + at * AD + 4 * c);
  const float d = __half2float(*(const __half*)(base + cache_rows(ref) * AD + at * 16 + (c >> 3) * 2));
  return make_float4((float)(int8_t)w * d, (float)(int8_t)(w >> 8) * d, (float)(int8_t)(w >> 16) * d, (float)(int8_t)(w >> 24) * d);
}

// What the tree kernel leaves out of dims 4 c .. of a row: the V values, not finite in f16, of the drafts that the row sees, times
// their weights relative to M. Rare, and kept out of line.
__device__ __noinline__ float4 left_out(const RowsParams& p, size_t row, int c, float M) {
  const int T = p.c.T, nqh = p.c.nkvh * GQA, b = (int)(row / ((size_t)T * nqh)), t = (int)(row / nqh % T), kh = (int)(row % nqh) / GQA;
  uint64_t left = p.mask[(size_t)b * T + t];
  if (T < 64) left &= ((uint64_t)1 << T) - 1;
  float A[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
  for (; left; left &= left - 1) {
    const int64_t at = cache_row(p.c, b, kh, first_pos(p.c, b) + __ffsll((long long)left) - 1);
    if (at < 0) continue;
    const float4 v4 = four_of(p.c, p.vcache, at, c);
    const float v[4] = {v4.x, v4.y, v4.z, v4.w};
    bool any = false;
#pragma unroll
    for (int i = 0; i < 4; i++) any |= !(fabsf(v[i]) < 65520.f);  // (from there on a value rounds to infinity in f16)
    if (!any) continue;
    float s = 0.f;
#pragma unroll 1
    for (int i = 0; i < AD / 4; i++) {
      const float4 q = *(const float4*)(p.qn + row * AD + 4 * i), k = four_of(p.c, p.kcache, at, i);
      s += q.x * k.x + q.y * k.y + q.z * k.z + q.w * k.w;
    }
    const float f = ex2((s * p.kq_scale - M) * LOG2E);
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (!(fabsf(v[i]) < 65520.f)) A[i] += f * v[i];
  }
  return make_float4(A[0], A[1], A[2], A[3]);
}

// Merges the partials of a row, applies the gate and writes f16, or q8_1; a row without a visible position is 0. 64 threads to
// a row, four dims each, or four times as many that take every fourth partial; PRE partials of a thread are requested at a time, the
// first before the maxima are known. 72 rows of 148 partials: PRE = 10 and two CTAs on an SM 18.4 us a call, 6 and three 20.1;
// 384 rows of 49, which fill the SMs more than once with two CTAs: 29.0 and 26.4. Many rows have few partials each (a batch): a
// CTA takes four rows then (6,144 rows of a few partials: 151.8 and 134.3 us a call, a CTA for every row 224).
template <bool TREE, int GROUPS, int PRE, int CTAS>
__global__ void __launch_bounds__(256, CTAS) rows_merge_kernel(const __grid_constant__ RowsParams p, int64_t rows) {
  constexpr int ROWS = 4 / GROUPS;  // of a CTA
  __shared__ float4 sa[GROUPS > 1 ? GROUPS - 1 : 1][64];
  __shared__ float sl[4], sm[8];
  const int tid = threadIdx.x, grp = GROUPS > 1 ? tid >> 6 : 0, c = tid & 63;
  const size_t row = (size_t)blockIdx.x * ROWS + (GROUPS > 1 ? 0 : tid >> 6);
  const bool mine = (int64_t)row < rows;
  // The split kernel ran right before and lets its dependents start only when everything before it has completed: what it does
  // not write may be read before the wait.
  int b = 0, y = 0, r = 0, tiles = 0;  // tree: sequence, unit in it and row in that; its tiles
  const int nqh = p.c.nkvh * GQA;
  float4 g = make_float4(0.f, 0.f, 0.f, 0.f);
  if (mine) {
    g = *(const float4*)(p.qg + row * 2 * AD + AD + 4 * c);
    if (TREE) {
      b = (int)(row / ((size_t)p.c.T * nqh));
      const int h = (int)(row % nqh), gr = (int)(row / nqh % p.c.T) * GQA + h % GQA;
      y = gr / TREE_ROWS * p.c.nkvh + h / GQA;
      r = gr % TREE_ROWS;
      tiles = tree_tiles(min(first_pos(p.c, b) + p.c.T, p.c.n_ctx));
    }
  }
  pdl_wait();
  pdl_trigger();
  int np = 0;        // partials of the row: first, first + step, ..
  size_t first = 0, step = 1;
  if (mine && !TREE) {
    np = p.nsplit;
    first = row * p.nsplit;
  } else if (mine && tiles > 0) {
    const int units = p.c.nkvh * tree_row_tiles(p.c.T);
    if (p.c.page_table) {
      np = tree_parts(tiles, (int)p.plan[0]);
      first = (size_t)p.plan[1 + b] * units + (size_t)y * np;
    } else {
      np = min(p.nsplit, tiles);
      first = (size_t)y * p.nsplit;
    }
    first = first * TREE_ROWS + r;
    step = TREE_ROWS;
  }
  const float2* ml = p.part_ml + first;
  const float* po = p.part_o + first * AD + 4 * c;
  float4 x[PRE];  // every GROUPS-th partial, PRE at a time
  float2 xml[PRE];
  auto fetch = [&](int z0) {
#pragma unroll
    for (int i = 0; i < PRE; i++)
      if (z0 + GROUPS * i < np) {
        x[i] = *(const float4*)(po + (size_t)(z0 + GROUPS * i) * step * AD);
        xml[i] = ml[(size_t)(z0 + GROUPS * i) * step];
      }
  };
  fetch(grp);
  float M = M_INIT;
  for (int z = GROUPS > 1 ? tid : c; z < np; z += 64 * GROUPS) M = fmaxf(M, ml[(size_t)z * step].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  if ((tid & 31) == 0) sm[tid >> 5] = M;
  __syncthreads();
  if (GROUPS > 1) {
#pragma unroll
    for (int w = 0; w < 8; w++) M = fmaxf(M, sm[w]);
  } else {
    M = fmaxf(sm[tid >> 6 << 1], sm[(tid >> 6 << 1) + 1]);
  }
  float L = 0.f;
  float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
  uint32_t signs = 0;  // of the sums: the tree kernel left something out
  auto add = [&](const float2& v, const float4& x) {
    if (TREE) signs |= __float_as_uint(v.y);
    if (v.y == 0.f) return;  // holds nothing
    const float f = ex2((v.x - M) * LOG2E);
    L += (TREE ? fabsf(v.y) : v.y) * f;
    A.x += x.x * f, A.y += x.y * f, A.z += x.z * f, A.w += x.w * f;
  };
  for (int z0 = grp; z0 < np; z0 += GROUPS * PRE) {
    if (z0 > grp) fetch(z0);
#pragma unroll
    for (int i = 0; i < PRE; i++)
      if (z0 + GROUPS * i < np) add(xml[i], x[i]);
  }
  if (GROUPS > 1) {
    if (grp > 0) sa[grp - 1][c] = A;
    if (c == 0) sl[grp] = TREE ? __uint_as_float(__float_as_uint(L) | (signs & 0x80000000u)) : L;
    __syncthreads();
    if (grp > 0) return;
#pragma unroll
    for (int k = 0; k < GROUPS - 1; k++) {
      const float4 x = sa[k][c];
      A.x += x.x, A.y += x.y, A.z += x.z, A.w += x.w;
      L += TREE ? fabsf(sl[k + 1]) : sl[k + 1];
      if (TREE) signs |= __float_as_uint(sl[k + 1]);
    }
  }
  if (!mine) return;
  if (TREE && signs >> 31) {
    const float4 x = left_out(p, row, c, M);
    A.x += x.x, A.y += x.y, A.z += x.z, A.w += x.w;
  }
  write_row(p, row, c, A, L, g);
}

// Up to four drafts: the partials of the prefix, and the drafts themselves, merged. 64 threads to a row, four dims each, or four
// times as many (GROUPS) that share the drafts and the partials out. A draft that the row sees is scored, and its V row taken as a
// partial (score, 1, v), in f32 and before the partials are there. 24 rows of 148 partials: 25.1 us a call with groups and ten in
// flight, 27.5 with six and three CTAs on an SM, 38 without groups; 384 rows of up to 32 76.2, 74.0 and 77; 6,144 rows of up to four 157,
// 133 and 99.9 (without groups, four in flight).
template <int GROUPS, int PRE, int CTAS>
__global__ void __launch_bounds__(256, CTAS) draft_merge_kernel(const RowsParams p, const PrefixPartials pre, int64_t rows) {
  constexpr int ROWS = 4 / GROUPS, DRAFTS = 4 / GROUPS;  // rows of a CTA, drafts of a thread
  __shared__ float4 sa[GROUPS > 1 ? GROUPS - 1 : 1][64];
  __shared__ float sl[4], sm[8], sd[8][DRAFTS];
  const int tid = threadIdx.x, warp = tid >> 5, c = tid & 63, grp = GROUPS > 1 ? tid >> 6 : 0;
  const size_t row = min((int64_t)blockIdx.x * ROWS + (GROUPS > 1 ? 0 : tid >> 6), rows - 1);  // rows beyond the last do its work again
  const int T = p.c.T, nqh = p.c.nkvh * GQA;
  const int b = (int)(row / ((size_t)T * nqh)), t = (int)(row / nqh % T), h = (int)(row % nqh), kh = h / GQA;
  const int first = first_pos(p.c, b), n = max(0, min(first, p.c.n_ctx));  // drafts, prefix
  const float4 g = *(const float4*)(p.qg + row * 2 * AD + AD + 4 * c), q = *(const float4*)(p.qn + row * AD + 4 * c);
  const uint64_t mask = p.mask[(size_t)b * T + t];
  float4 k[DRAFTS], v[DRAFTS];
  bool seen[DRAFTS];
#pragma unroll
  for (int d = 0; d < DRAFTS; d++) {
    const int j = grp + d;
    const int64_t at = j < T && ((mask >> j) & 1) ? cache_row(p.c, b, kh, first + j) : -1;
    k[d] = v[d] = make_float4(0.f, 0.f, 0.f, 0.f);
    seen[d] = at >= 0;
    if (seen[d]) k[d] = four_of(p.c, p.kcache, at, c), v[d] = four_of(p.c, p.vcache, at, c);
  }
#pragma unroll
  for (int d = 0; d < DRAFTS; d++) {
    float s = q.x * k[d].x + q.y * k[d].y + q.z * k[d].z + q.w * k[d].w;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if ((tid & 31) == 0) sd[warp][d] = seen[d] ? s * p.kq_scale : M_INIT / 2;
  }
  const int np = pre.chunk_len ? (n + pre.chunk_len - 1) / pre.chunk_len : n > 0 ? filled_chunks(n, pre.nch) : 0;
  const float* po = pre.part + (((size_t)b * p.c.nkvh + kh) * pre.nch * MAXR + t * GQA + h % GQA) * PROW;  // chunks MAXR rows apart
  pdl_wait();
  pdl_trigger();
  float2 x[PRE][2], ml[PRE];  // every GROUPS-th partial, PRE at a time
  auto fetch = [&](int z0) {
#pragma unroll
    for (int i = 0; i < PRE; i++)
      if (z0 + GROUPS * i < np) {
        const float* r = po + (size_t)(z0 + GROUPS * i) * MAXR * PROW;
        ml[i] = *(const float2*)r;
        x[i][0] = *(const float2*)(r + 2 + 4 * c);
        x[i][1] = *(const float2*)(r + 4 + 4 * c);
      }
  };
  fetch(grp);
  float M = M_INIT;
  for (int z = GROUPS > 1 ? tid : c; z < np; z += 64 * GROUPS) M = fmaxf(M, po[(size_t)z * MAXR * PROW]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  if ((tid & 31) == 0) sm[warp] = M;
  __syncthreads();
  const int pair = warp & ~1;  // the two warps of this group
  if (GROUPS > 1) {
#pragma unroll
    for (int w = 0; w < 8; w++) M = fmaxf(M, sm[w]);
#pragma unroll
    for (int w = 0; w < 8; w += 2) M = fmaxf(M, sd[w][0] + sd[w + 1][0]);
  } else {
    M = fmaxf(sm[pair], sm[pair + 1]);
#pragma unroll
    for (int d = 0; d < DRAFTS; d++) M = fmaxf(M, sd[pair][d] + sd[pair + 1][d]);
  }
  float L = 0.f;
  float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](float m, float l, float ax, float ay, float az, float aw) {
    if (l == 0.f) return;  // holds nothing
    const float f = ex2((m - M) * LOG2E);
    L += l * f;
    A.x += ax * f, A.y += ay * f, A.z += az * f, A.w += aw * f;
  };
#pragma unroll
  for (int d = 0; d < DRAFTS; d++)
    if (seen[d]) add(sd[pair][d] + sd[pair + 1][d], 1.f, v[d].x, v[d].y, v[d].z, v[d].w);
  for (int z0 = grp; z0 < np; z0 += GROUPS * PRE) {
    if (z0 > grp) fetch(z0);
#pragma unroll
    for (int i = 0; i < PRE; i++)
      if (z0 + GROUPS * i < np) add(ml[i].x, ml[i].y, x[i][0].x, x[i][0].y, x[i][1].x, x[i][1].y);
  }
  if (GROUPS > 1) {
    if (grp > 0) sa[grp - 1][c] = A;
    if (c == 0) sl[grp] = L;
    __syncthreads();
    if (grp > 0) return;
#pragma unroll
    for (int i = 0; i < GROUPS - 1; i++) {
      const float4 y = sa[i][c];
      A.x += y.x, A.y += y.y, A.z += y.z, A.w += y.w;
      L += sl[i + 1];
    }
  }
  write_row(p, row, c, A, L, g);
}

template <bool TREE>
int launch_rows_merge(const RowsParams& p, int64_t rows, int n_sm, cudaStream_t s) {
  const bool split = rows < 8 * (int64_t)n_sm;  // a row's partials among the groups of a CTA
  auto* k = !split ? rows_merge_kernel<TREE, 1, 6, 3>
            : rows > 2 * (int64_t)n_sm ? rows_merge_kernel<TREE, 4, 6, 3> : rows_merge_kernel<TREE, 4, 10, 2>;
  Q27B_CK(launch_step(k, dim3((unsigned)(split ? rows : (rows + 3) / 4)), dim3(256), 0, s, p, rows));
  return Q27B_OK;
}

// Room for the partials of `rows` rows (and `more` floats behind them): in the prefill workspace, whose size is fixed, or, for a
// batch, in the paged workspace. *fit: as many of `rows` as there is room for (a batch: all).
int place_partials(DeviceCtx* ctx, RowsParams& p, int64_t rows, int64_t more, int64_t* fit, float** part, const char* who) {
  const size_t floats = (size_t)rows * (AD + 2) + (size_t)more;
  *fit = rows;
  if (p.c.page_table) return paged_ws(ctx, floats, part, who);
  size_t cap;
  if (int rc = prefill_ws(ctx, part, &cap)) return rc;
  if (cap < floats) *fit = cap < (size_t)more ? 0 : (int64_t)((cap - (size_t)more) / (AD + 2));
  return Q27B_OK;
}
int no_room(const char* who) { return fail(Q27B_UNSUPPORTED, std::string(who) + ": the prefill workspace is too small for the partials of this call"); }

int run_blocks(DeviceCtx* ctx, RowsParams& p, const char* who, cudaStream_t s) {
  const CacheRef& c = p.c;
  const int64_t lists = (int64_t)c.B * c.T * c.nkvh, rows = lists * GQA;
  const BlocksPlan plan = plan_blocks(lists, p.k, ctx->n_sm, c.q8);
  float* part;
  int64_t fit;
  if (int rc = place_partials(ctx, p, rows * plan.nch, 0, &fit, &part, who)) return rc;
  if (fit < rows) return no_room(who);
  const int chunk = (p.k + (int)(fit / rows) - 1) / (int)(fit / rows);
  if (chunk > SEL_CHUNK) return no_room(who);
  p.nsplit = (p.k + chunk - 1) / chunk;
  p.part_o = part;
  p.part_ml = (float2*)(part + rows * p.nsplit * AD);
  ListParams d = {};
  d.qn = p.qn; d.pos0 = c.pos0; d.status = c.status; d.T = 1; d.nqh = c.nkvh * GQA; d.nkvh = c.nkvh; d.n_ctx = c.n_ctx;
  d.nch = p.nsplit; d.kq_scale = p.kq_scale; d.n_local = -1; d.page_table = c.page_table; d.seq_len = c.seq_len;
  d.max_pages = c.max_pages; d.n_pages = c.n_pages; d.chunk_len = chunk; d.sel = p.sel; d.sel_k = p.k; d.sel_T = c.T;
  d.part_o = p.part_o; d.part_ml = p.part_ml;
  CUtensorMap kv, ks, vv, vs;
  const uint64_t cache = cache_rows(c);
  if (c.q8) {
    if (int rc = q8_tmaps(p.kcache, cache, &kv, &ks)) return rc;
    if (int rc = q8_tmaps(p.vcache, cache, &vv, &vs)) return rc;
    if (int rc = launch_blocks_ws(&kv, &ks, &vv, &vs, d, c.B * c.T, s, plan.pairs)) return rc;
  } else {
    if (int rc = cached_tmap_2d(&kv, p.kcache, cache, 2 * AD, 2 * AD, 128, BLK, true)) return rc;
    if (int rc = cached_tmap_2d(&vv, p.vcache, cache, 2 * AD, 2 * AD, 128, BLK, true)) return rc;
    if (int rc = launch_blocks_f16(&kv, &vv, d, c.B * c.T, s)) return rc;
  }
  return launch_rows_merge<false>(p, rows, ctx->n_sm, s);
}

int run_tree(DeviceCtx* ctx, RowsParams& p, const char* who, cudaStream_t s) {
  const CacheRef& c = p.c;
  if (c.T <= Q27B_MAX_T && c.nkvh <= ctx->n_sm && (c.q8 || (int64_t)c.nkvh * c.n_ctx <= 32768)) {
    // Up to four drafts are 24 rows of a KV head. The decode kernels, made for those, take the prefix, and the merge the drafts:
    // four behind 1,000 positions 8.8 us against 9.9 with the 128-row tiles of decode_tree.cu, behind 150,000 70 against 84 (cool), a
    // single one 58 against 85; four each behind 16 sequences of up to 16,384 80 against 101, of 64 to 4,096 39 against 40. An f16
    // cache has nothing to convert there and is bound by its reads earlier: four behind 8,000 positions of four heads 13.5 against
    // 15.2, behind 16,000 17.5 against 18.5, behind 32,000 36 against 32, behind 150,000 137 against 104 (a single one: 16,000 12 against
    // 18, 150,000 112 against 101). Only the allocated rows are known here; a long cache is taken to be a full one.
    PrefixPartials pre;
    if (c.page_table) {
      if (int rc = launch_prefix_paged(ctx, p.qn, p.kcache, p.vcache, c.page_table, c.seq_len, c.B, c.T, p.kq_scale, c.nkvh, c.n_pages,
                                       c.max_pages, c.n_ctx, who, &pre, s))
        return rc;
    } else if (int rc = launch_prefix(ctx, p.qn, p.kcache, p.vcache, c.pos0, c.T, p.kq_scale, c.nkvh, c.n_ctx, c.q8, &pre, s)) {
      return rc;
    }
    const int64_t rows = (int64_t)c.B * c.T * c.nkvh * GQA;
    const bool split = rows <= 4 * (int64_t)ctx->n_sm;
    auto* k = !split ? draft_merge_kernel<1, 4, 3> : rows > 2 * (int64_t)ctx->n_sm ? draft_merge_kernel<4, 6, 3> : draft_merge_kernel<4, 10, 2>;
    Q27B_CK(launch_step(k, dim3((unsigned)(split ? rows : (rows + 3) / 4)), dim3(256), 0, s, p, pre, rows));
    return Q27B_OK;
  }
  const int64_t rows = (int64_t)p.c.B * p.c.T * p.c.nkvh * GQA, units = (int64_t)p.c.B * p.c.nkvh * tree_row_tiles(p.c.T);
  const bool paged = p.c.page_table != nullptr;
  const int64_t head = paged ? (2 * (p.c.B + 1) + 3) / 4 * 4 : 0;  // the plan, in floats
  // One sequence: a CTA per SM (its shared and tensor memory take one), the same number for every unit.
  int64_t parts = std::max<int64_t>(1, std::min<int64_t>(ctx->n_sm / units, tree_tiles(p.c.n_ctx))), fit;
  int64_t slots = paged ? tree_grid(units, ctx->n_sm) : units * parts;
  float* part;
  if (int rc = place_partials(ctx, p, slots * TREE_ROWS, head, &fit, &part, who)) return rc;
  if (fit < slots * TREE_ROWS) {
    parts = fit / (units * TREE_ROWS);
    if (parts < 1) return no_room(who);
    slots = units * parts;
  }
  p.nsplit = (int)parts;
  p.plan = (int64_t*)part;
  p.part_o = part + head;
  p.part_ml = (float2*)(p.part_o + slots * TREE_ROWS * AD);
  if (int rc = launch_tree(p, ctx->n_sm, s)) return rc;
  return launch_rows_merge<true>(p, rows, ctx->n_sm, s);
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
  if (misaligned({qn, qg, kcache, vcache, o, xq})) return fail(Q27B_BAD_SHAPE, "attn_decode_tree: pointers must be 16-byte aligned");
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
  if (misaligned({qn, qg, kpool, vpool, o, xq})) return fail(Q27B_BAD_SHAPE, "attn_decode_tree_paged: pointers must be 16-byte aligned");
  DeviceCtx* ctx;
  if (int rc = device_ctx(&ctx)) return rc;
  RowsParams p = {};
  p.c = paged_ref(ctx, page_table, seq_len, B, T, nkvh, n_pages, max_pages);
  p.c.n_ctx = max_seq_len;  // a longer sequence is cut there
  if (tree_tiles(max_seq_len) > TREE_MAX_TILES)
    return fail(Q27B_UNSUPPORTED, "attn_decode_tree_paged: sequences of more than " + std::to_string(TREE_MAX_TILES * BLK) + " positions");
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
  if (misaligned({qn, qg, kcache, vcache, o, xq})) return fail(Q27B_BAD_SHAPE, "attn_decode_blocks: pointers must be 16-byte aligned");
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
  if (misaligned({qn, qg, kpool, vpool, o, xq})) return fail(Q27B_BAD_SHAPE, "attn_decode_blocks_paged: pointers must be 16-byte aligned");
  DeviceCtx* ctx;
  if (int rc = device_ctx(&ctx)) return rc;
  RowsParams p = {};
  p.c = paged_ref(ctx, page_table, seq_len, B, T, nkvh, n_pages, max_pages);
  p.qn = qn; p.qg = qg; p.kcache = kpool; p.vcache = vpool; p.o = o; p.xq = xq; p.xd = xd; p.sel = sel; p.k = k;
  p.kq_scale = kq_scale;
  return run_blocks(ctx, p, "attn_decode_blocks_paged", (cudaStream_t)stream);
}

}  // extern "C"

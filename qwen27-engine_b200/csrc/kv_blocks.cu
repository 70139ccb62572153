// Cache bookkeeping around tree verification and block-sparse drafting: rows of the accepted path moved to the front
// of the drafted rows (commit), per-block bounds of the keys (bounds), choice of the blocks to attend (select).
#include "cache_ref.h"

#include <algorithm>
#include <mutex>

namespace q27b {
namespace {

// ---------------------------------------------------------------- commit
// Row first + i <- row first + path[i] for i < count, K and V, every head. A CTA owns one (head, K or V, sequence): it
// holds all moved rows in registers (up to 64 rows of 272 or 512 bytes in 256 threads) before it writes the first, so a
// path may name rows in any order. Launch and latency bound: 16 drafts of one sequence 3.2 to 3.7 us a call, 64 of each of 64 sequences 4.1.
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
// lanes hold a row, 16 row groups take four rows each, all loaded before the first is used. The block of one token: 3.6 to 4.0 us a
// call, launch and two trips to memory.
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

// The same for a q8_0 cache with a warp per block and head: two rows at a time, eight of a lane requested together, no barrier. For
// many blocks: the 2,345 of 150,000 positions times four heads take 32.1 us (5.4 TB/s) against 45.3 with a CTA each, 513 times
// four 11.9 against 12.2, 257 times four 10.5 against 6.3. (f16, 60,000 positions of four heads: 25.4 against 23.8 us.)
__global__ void __launch_bounds__(BND_THREADS) bounds_warp_kernel(const CacheRef c, const void* kcache, __half* bounds, int blocks) {
  pdl_trigger();
  const int lane = threadIdx.x & 31, c16 = lane & 15, kh = blockIdx.y, b = blockIdx.z, i0 = blockIdx.x * (BND_THREADS / 32) + (threadIdx.x >> 5);
  pdl_wait();
  const int first = first_pos(c, b), end = min(first + c.T, c.n_ctx);
  const int blk = max(first, 0) / BLK + i0, p0 = blk * BLK;
  if (i0 >= blocks || first >= end || p0 >= end) return;
  const int64_t row0 = cache_row(c, b, kh, p0), at = bounds_index(c, b, kh, blk);
  if (row0 < 0) return;
  const int n = min(BLK, end - p0);
  const uint8_t* src = (const uint8_t*)kcache + (row0 + (lane >> 4)) * AD + 16 * c16;
  const uint8_t* sc = (const uint8_t*)kcache + cache_rows(c) * AD + (row0 + (lane >> 4)) * 16 + (c16 >> 1) * 2;
  const __half2 inf = __half2half2(__ushort_as_half((unsigned short)0x7C00)), ninf = __hneg2(inf);
  __half2 lo[8], hi[8];
#pragma unroll
  for (int i = 0; i < 8; i++) lo[i] = inf, hi[i] = ninf;
  constexpr int G = 8;  // rows of this lane that are requested together
  for (int r = 0; r < n; r += 2 * G) {
    uint4 v[G];
    __half d[G];
#pragma unroll
    for (int j = 0; j < G; j++) {
      const int k = r + 2 * j;
      if (k + (lane >> 4) >= n) continue;
      v[j] = *(const uint4*)(src + k * AD);
      d[j] = *(const __half*)(sc + k * 16);
    }
#pragma unroll
    for (int j = 0; j < G; j++) {
      if (r + 2 * j + (lane >> 4) >= n) continue;
      uint32_t x[8];
      dequant16(v[j], d[j], x);
      widen(lo, hi, x);
    }
  }
  uint32_t l[8], h[8];
#pragma unroll
  for (int i = 0; i < 8; i++) {
    l[i] = h2_as_u32(__hmin2_nan(lo[i], u32_as_h2(__shfl_xor_sync(0xffffffffu, h2_as_u32(lo[i]), 16))));
    h[i] = h2_as_u32(__hmax2_nan(hi[i], u32_as_h2(__shfl_xor_sync(0xffffffffu, h2_as_u32(hi[i]), 16))));
  }
  uint4* out = (uint4*)(bounds + (size_t)at * 2 * AD + (lane >> 4) * AD + 16 * c16);  // the first 16 lanes write lo, the others hi
  out[0] = lane < 16 ? make_uint4(l[0], l[1], l[2], l[3]) : make_uint4(h[0], h[1], h[2], h[3]);
  out[1] = lane < 16 ? make_uint4(l[4], l[5], l[6], l[7]) : make_uint4(h[4], h[5], h[6], h[7]);
}

int launch_bounds(const CacheRef& c, const void* kcache, void* bounds, int n_sm, cudaStream_t s) {
  const int blocks = (int)(((int64_t)c.T + BLK - 2) / BLK + 1);  // as many as T rows can touch
  constexpr int WARPS = BND_THREADS / 32;
  if (!c.q8 || (int64_t)blocks * c.nkvh * c.B < 12 * (int64_t)n_sm)
    Q27B_CK(launch_step(bounds_kernel, dim3(blocks, c.nkvh, c.B), dim3(BND_THREADS), 0, s, c, kcache, (__half*)bounds));
  else
    Q27B_CK(launch_step(bounds_warp_kernel, dim3((blocks + WARPS - 1) / WARPS, c.nkvh, c.B),
                        dim3(BND_THREADS), 0, s, c, kcache, (__half*)bounds, blocks));
  return Q27B_OK;
}

// ---------------------------------------------------------------- select
// score(block) = max over the six query heads of the KV head of sum_d max(q_d lo_d, q_d hi_d) = sum_d (q+_d hi_d + q-_d lo_d):
// no key of the block has a larger q.k. The order of scores decides what is attended, so it is that of sums in 64 bits,
// in which the products of f32 and f16 values are exact: which block wins does not depend on the order of a sum, short of
// differences of 1e-16. Two kernels:
//  * score_kernel: every score to about 15 bits on the tensor cores, with a bound of its error;
//  * select_kernel: what the bounds leave open around the border (a few blocks) again in 64 bits, and the choice.
// All scores in 64 bits take ten times as long as reading the bounds (32 sequences of up to 131,072 positions, two tokens:
// 222 us): two selects and an FMA at half rate per dim and head.
struct SelectParams {
  CacheRef c;
  const float* qn;        // [B][T][6 nkvh][256]
  const __half* bounds;
  int* sel;               // [B][T][nkvh][k]
  float2* score;          // [B][T][nkvh][max_blocks] (score, error)
  int k, n_sink, n_recent, max_blocks;
};
constexpr int SEL_MAX_BLOCKS = 16384;

// Blocks up to the own one of token t of sequence b.
__device__ __forceinline__ int blocks_of(const CacheRef& c, int b, int t) {
  const int last = min(first_pos(c, b) + t, c.n_ctx - 1);
  return last < 0 ? 0 : last / BLK + 1;
}

// A warp scores 16 blocks of a (KV head, sequence) for all its T tokens with m16n8k16 MMAs: the bounds are the A operand as they
// lie in memory (a lane's 16 bytes are two k-steps; the order of the dims is free), all of them in registers at once (one token) or half, the
// query heads are six of the eight columns of B. q times a power of two, so that its largest value is below 2^10, is the sum
// of two f16 values, off by at most 2^-22 of itself or 2^-25. Four accumulators: q+ hi and q- lo, with the larger parts and with
// the smaller ones, 16 MMAs each. With A = sum |q| max(|lo|, |hi|) (a fifth one, of |q| + 2^-6): the PTX ISA promises an MMA of f16
// into f32 products and sums of at least single precision, and what is published of tensor cores (Fasi, Higham, Mikaitis, Pranesh,
// "Numerical behavior of NVIDIA tensor cores", PeerJ Computer Science 7:e330, 2021) is exact products whose sum with the accumulator
// is cut at 2^-23 of the largest addend or below. With each of 17 addends cut there the error is below 16 * 18 * 2^-23 A +
// 2^-22 A < 2^-14.7 A; 2^-14 A is what is passed on. Measured against 64 bits over 45 million sums (signs that cancel, magnitudes
// of 14 binades, one product among 255 of 2^-24 of it): at most 2^-17.5 A. 32 sequences of up to 131,072 positions, two tokens: 45 us for 147 MB of bounds, between the latency of their loads
// (a quarter of the issue slots and of the tensor pipe is used; more warps would need the registers that hold loads in flight) and
// memory; one token behind 150,000 positions: one trip to memory, 4 us.
constexpr int SCORE_WARPS = 4, SCORE_GROUP = 16 * SCORE_WARPS, Q_STRIDE = 2 * AD + 64;  // bytes between staged query rows: 16-byte reads without conflicts
enum { QP_HI, QM_HI, QP_LO, QM_LO, QABS, Q_PARTS };
constexpr int Q_TOKEN = Q_PARTS * 8 * Q_STRIDE;  // bytes of a staged token

template <int T>
__global__ void __launch_bounds__(32 * SCORE_WARPS, T == 2 ? 3 : 2) score_kernel(const SelectParams p) {
  constexpr int TURNS = T == 1 ? 1 : 2, PER = 8 / TURNS;  // the dims in one or two turns of 32 PER
  extern __shared__ __align__(16) uint8_t sq[];  // [T][Q_PARTS][8 columns][Q_STRIDE]
  __shared__ float unit[T][8];          // 1 / scale of a head
  pdl_trigger();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, tg = lane & 3;
  const int kh = blockIdx.y, b = blockIdx.z, nqh = p.c.nkvh * GQA;
  for (int i = tid; i < T * Q_PARTS * 2 * Q_STRIDE / 4; i += 32 * SCORE_WARPS)  // the two columns that are no head
    *(uint32_t*)&sq[i / (2 * Q_STRIDE / 4) * (8 * Q_STRIDE) + 6 * Q_STRIDE + i % (2 * Q_STRIDE / 4) * 4] = 0;
  pdl_wait();
  const int nb = blocks_of(p.c, b, T - 1), ngroups = (nb + SCORE_GROUP - 1) / SCORE_GROUP;
  if (nb <= p.k || (int)blockIdx.x >= ngroups) return;  // every block is taken; or no block of this sequence
  uint4 lo[2][PER], hi[2][PER];  // a turn's dims of rows g and g + 8, 32 dims each: 8 of them in this lane
  int64_t at[2];
  auto aim = [&](int group) {
#pragma unroll
    for (int e = 0; e < 2; e++) {
      const int blk = group * SCORE_GROUP + 16 * warp + g + 8 * e;
      at[e] = blk < nb ? bounds_index(p.c, b, kh, blk) : -1;
    }
  };
  auto load = [&](int turn) {
#pragma unroll
    for (int e = 0; e < 2; e++)
#pragma unroll
      for (int j = 0; j < PER; j++) {
        lo[e][j] = hi[e][j] = make_uint4(0, 0, 0, 0);
        if (at[e] >= 0) {
          lo[e][j] = *(const uint4*)(p.bounds + at[e] * 2 * AD + 32 * PER * turn + 32 * j + 8 * tg);
          hi[e][j] = *(const uint4*)(p.bounds + at[e] * 2 * AD + AD + 32 * PER * turn + 32 * j + 8 * tg);
        }
      }
  };
  aim(blockIdx.x);
  load(0);
  for (int i = warp; i < T * GQA; i += SCORE_WARPS) {
    const int t = i / GQA, h = i % GQA;
    const float* src = p.qn + (((size_t)b * T + t) * nqh + kh * GQA + h) * AD + 8 * lane;
    float x[8], amax = 0.f;
#pragma unroll
    for (int k = 0; k < 8; k++) x[k] = src[k], amax = fmaxf(amax, fabsf(x[k]));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    const int e = (int)(__float_as_uint(amax) >> 23) - 127;  // amax < 2^(e + 1)
    const int up = min(9 - e, 100);
    const float scale = __uint_as_float((uint32_t)(127 + up) << 23);
    if (lane == 0) unit[t][h] = __uint_as_float((uint32_t)(127 - up) << 23);
    uint32_t w[Q_PARTS][4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const float a = x[2 * k] * scale, c = x[2 * k + 1] * scale;
      const __half2 h2 = __floats2half2_rn(a, c);
      const float2 f = __half22float2(h2);
      const __half2 l2 = __floats2half2_rn(a - f.x, c - f.y);
      const uint32_t pos = (a < 0.f ? 0u : 0xFFFFu) | (c < 0.f ? 0u : 0xFFFF0000u);  // by the sign of q itself
      w[QP_HI][k] = h2_as_u32(h2) & pos;
      w[QM_HI][k] = h2_as_u32(h2) & ~pos;
      w[QP_LO][k] = h2_as_u32(l2) & pos;
      w[QM_LO][k] = h2_as_u32(l2) & ~pos;
      w[QABS][k] = h2_as_u32(__hadd2(__habs2(h2), __half2half2(__ushort_as_half((unsigned short)0x2400))));  // + 2^-6
    }
#pragma unroll
    for (int k = 0; k < Q_PARTS; k++)
      *(uint4*)&sq[t * Q_TOKEN + (k * 8 + h) * Q_STRIDE + 16 * lane] = make_uint4(w[k][0], w[k][1], w[k][2], w[k][3]);
  }
  __syncthreads();
#pragma unroll 1
  for (int group = blockIdx.x; group < ngroups; group += gridDim.x) {
    if (group != (int)blockIdx.x) {
      aim(group);
      load(0);
    }
    const int ahead = (group + gridDim.x) * SCORE_GROUP + 16 * warp + (lane >> 1);  // the next group's bounds into L2, half a block a lane
    if (ahead < nb) {
      const int64_t next = bounds_index(p.c, b, kh, ahead);
      if (next >= 0)
#pragma unroll
        for (int i = 0; i < 4; i++) prefetch_l2(p.bounds + next * 2 * AD + (lane & 1) * AD + 64 * i);
    }
    float sp[T][4] = {}, sm[T][4] = {}, sl[T][4] = {}, sn[T][4] = {}, sa[T][4] = {};
#pragma unroll 1
    for (int turn = 0; turn < TURNS; turn++) {
      if (turn) load(turn);
#pragma unroll
      for (int j = 0; j < PER; j++) {
        const uint4 l0 = lo[0][j], l1 = lo[1][j], h0 = hi[0][j], h1 = hi[1][j];
        const auto widest = [](uint32_t x, uint32_t y) { return h2_as_u32(__hmax2_nan(__habs2(u32_as_h2(x)), __habs2(u32_as_h2(y)))); };
        const uint4 w0 = make_uint4(widest(l0.x, h0.x), widest(l0.y, h0.y), widest(l0.z, h0.z), widest(l0.w, h0.w));
        const uint4 w1 = make_uint4(widest(l1.x, h1.x), widest(l1.y, h1.y), widest(l1.z, h1.z), widest(l1.w, h1.w));
#pragma unroll
        for (int t = 0; t < T; t++) {
          const uint8_t* qt = sq + t * Q_TOKEN + g * Q_STRIDE + 16 * tg + 64 * PER * turn + 64 * j;
          uint4 q[Q_PARTS];
#pragma unroll
          for (int k = 0; k < Q_PARTS; k++) q[k] = *(const uint4*)(qt + k * 8 * Q_STRIDE);
          mma16816(sp[t], h0.x, h1.x, h0.y, h1.y, q[QP_HI].x, q[QP_HI].y);
          mma16816(sm[t], l0.x, l1.x, l0.y, l1.y, q[QM_HI].x, q[QM_HI].y);
          mma16816(sl[t], h0.x, h1.x, h0.y, h1.y, q[QP_LO].x, q[QP_LO].y);
          mma16816(sn[t], l0.x, l1.x, l0.y, l1.y, q[QM_LO].x, q[QM_LO].y);
          mma16816(sa[t], w0.x, w1.x, w0.y, w1.y, q[QABS].x, q[QABS].y);
          mma16816(sp[t], h0.z, h1.z, h0.w, h1.w, q[QP_HI].z, q[QP_HI].w);
          mma16816(sm[t], l0.z, l1.z, l0.w, l1.w, q[QM_HI].z, q[QM_HI].w);
          mma16816(sl[t], h0.z, h1.z, h0.w, h1.w, q[QP_LO].z, q[QP_LO].w);
          mma16816(sn[t], l0.z, l1.z, l0.w, l1.w, q[QM_LO].z, q[QM_LO].w);
          mma16816(sa[t], w0.z, w1.z, w0.w, w1.w, q[QABS].z, q[QABS].w);
        }
      }
    }
#pragma unroll
    for (int t = 0; t < T; t++) {
      // rows g and g + 8, heads 2 tg and 2 tg + 1
#pragma unroll
      for (int e = 0; e < 2; e++) {
        float best = -INFINITY, err = 0.f;
        bool odd = false;  // something is no finite number
        if (tg < 3) {
#pragma unroll
          for (int i = 0; i < 2; i++) {
            const float u = unit[t][2 * tg + i], v = (sp[t][2 * e + i] + sm[t][2 * e + i] + (sl[t][2 * e + i] + sn[t][2 * e + i])) * u, a = sa[t][2 * e + i] * u * 6.2e-5f;
            odd |= !(fabsf(v) <= 3e38f) || !(a <= 3e38f);
            best = fmaxf(best, v);
            err = fmaxf(err, a);
          }
        }
        if (odd) err = INFINITY;
#pragma unroll
        for (int o = 1; o <= 2; o <<= 1) {
          best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
          err = fmaxf(err, __shfl_xor_sync(0xffffffffu, err, o));
        }
        const int blk = group * SCORE_GROUP + 16 * warp + g + 8 * e;
        if (tg == 0 && blk < nb)
          p.score[(((size_t)b * T + t) * p.c.nkvh + kh) * p.max_blocks + blk] = at[e] >= 0 ? make_float2(best, err) : make_float2(-3e38f, 0.f);
      }
    }
  }
}

constexpr int SEL_THREADS = 512, SEL_WARPS = SEL_THREADS / 32, SEL_BITS = 11, SEL_BINS = 1 << SEL_BITS;
static_assert(SEL_MAX_BLOCKS <= 32 * SEL_THREADS, "a word of 32 blocks per thread");

struct SelShared {
  unsigned int hist[SEL_BINS];
  unsigned long long sums[SEL_WARPS];
  uint64_t key_red[2][SEL_WARPS];
  float red[3][SEL_WARPS];
  int bin, need, inside, n_in, n_open;
  alignas(16) float q[GQA][AD];
  uint32_t in[SEL_MAX_BLOCKS / 32], edge[SEL_MAX_BLOCKS / 32];  // a bit per block: is chosen; is chosen while there is room
};

// Exclusive sum over the block of x (two counts, 32 bits each).
__device__ __forceinline__ unsigned long long block_scan(unsigned long long x, unsigned long long* sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned long long v = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  if (lane == 31) sums[warp] = v;
  __syncthreads();
  unsigned long long before = 0;
#pragma unroll
  for (int w = 0; w < SEL_WARPS; w++) before += w < warp ? sums[w] : 0;
  __syncthreads();
  return before + v - x;
}

// Keys whose order is that of the numbers: larger number, larger key; -0 as 0; NaN (64 bits) above all.
__device__ __forceinline__ uint32_t order_key(float s) {
  const uint32_t bits = __float_as_uint(s + 0.f);
  return bits >> 31 ? ~bits : bits | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k >> 31 ? k & 0x7FFFFFFFu : ~k); }
__device__ __forceinline__ uint64_t order_key(double s) {
  if (s != s) return ~0ull;
  const uint64_t bits = (uint64_t)__double_as_longlong(s + 0.0);
  return bits >> 63 ? ~bits : bits | 0x8000000000000000ull;
}

// The bin of the histogram (2,048 bins, filled before a barrier) in which the count from the top reaches `want`, all 512 threads:
// how many of its entries belong to the want largest, and how many it has. Leaves the histogram at zero.
__device__ __forceinline__ int find_bin(int want, SelShared& sh, int* need, int* inside) {
  constexpr int PER = SEL_BINS / SEL_THREADS;
  const int tid = threadIdx.x, top = SEL_BINS - 1 - PER * tid;  // thread i looks at the four bins from 2047 - 4 i down
  unsigned int h[PER], mine = 0;
#pragma unroll
  for (int j = 0; j < PER; j++) {
    mine += h[j] = sh.hist[top - j];
    sh.hist[top - j] = 0;
  }
  int above = (int)block_scan(mine, sh.sums);
#pragma unroll
  for (int j = 0; j < PER; j++) {
    if (above < want && above + (int)h[j] >= want) {
      sh.bin = top - j;
      sh.need = want - above;
      sh.inside = (int)h[j];
    }
    above += (int)h[j];
  }
  __syncthreads();
  const int bin = sh.bin;
  *need = sh.need;
  *inside = sh.inside;
  __syncthreads();
  return bin;
}

// Where the want-th largest (1 <= want <= n) of key(0) .. key(n - 1) lies, all 512 threads: eleven bits at a time from the
// highest bit in which keys differ, until at most `few` keys share its leading bits. Returns those bits; *mask_out which they
// are, *need_out how many of the keys that share them belong to the want largest. hist is zero on entry and on return.
template <typename K, typename F>
__device__ K nth_largest(F key, int n, int want, int few, SelShared& sh, K* mask_out, int* need_out) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int BITS = 8 * sizeof(K);
  K mn = ~(K)0, mx = 0;
  for (int i = tid; i < n; i += SEL_THREADS) mn = min(mn, key(i)), mx = max(mx, key(i));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    mn = min(mn, __shfl_xor_sync(0xffffffffu, mn, o));
    mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  }
  if (lane == 0) sh.key_red[0][warp] = mn, sh.key_red[1][warp] = mx;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < SEL_WARPS; w++) mn = min(mn, (K)sh.key_red[0][w]), mx = max(mx, (K)sh.key_red[1][w]);
  const int top = 64 - __clzll((long long)(uint64_t)(K)(mn ^ mx));  // keys agree above the lowest `top` bits
  int need = want, shift = max(0, top - SEL_BITS), inside = n;
  K mask = top >= BITS ? (K)0 : (K)(~(K)0 << top), prefix = mn & mask;
  while (mask != ~(K)0 && inside > few) {
    for (int i = tid; i < n; i += SEL_THREADS) {
      const K x = key(i);
      if ((x & mask) == prefix) atomicAdd(&sh.hist[(unsigned)(x >> shift) & (SEL_BINS - 1)], 1u);
    }
    __syncthreads();
    prefix |= (K)find_bin(need, sh, &need, &inside) << shift;
    mask |= (K)(SEL_BINS - 1) << shift;
    shift = max(0, shift - SEL_BITS);
  }
  *mask_out = mask;
  *need_out = need;
  return prefix;
}

// The choice of one (token, KV head, sequence). With s the score to 15 bits, e its error, E the largest e and [t0, t1] an interval
// that holds the want-th largest s: want blocks or more have a score of at least t0 - E, so a block of s + e < t0 - E is
// out; the scores of the blocks with s <= t1 are at most t1 + E, and fewer than want have a larger s, so a block of s - e > t1 + E
// is in. The blocks between are scored again in 64 bits, a warp each, and the best of them fill up the list; of equal ones the
// lower. Where something is not finite, or everything alike, these are all blocks. Bound by the latency of a dozen barriers and of
// the trips to memory (scores, then the bounds of the open blocks): about 8 of the 13 us of a call on 2,344 blocks of four heads,
// k = 128. Counting by the bits of the scores, three turns instead of one, took 2.6 us longer.
__global__ void __launch_bounds__(SEL_THREADS, 2) select_kernel(const SelectParams p) {
  extern __shared__ uint64_t dyn[];  // [max_blocks] (score, error), then the 64-bit keys of the open blocks; then their numbers
  __shared__ SelShared sh;
  pdl_trigger();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int kh = blockIdx.x, t = blockIdx.y, b = blockIdx.z, nqh = p.c.nkvh * GQA;
  const size_t tok = (size_t)b * p.c.T + t, row = tok * p.c.nkvh + kh;
  int* out = p.sel + row * p.k;
  for (int i = tid; i < SEL_BINS; i += SEL_THREADS) sh.hist[i] = 0;
  if (tid == 0) sh.n_open = 0, sh.n_in = 0;
  pdl_wait();
  const int nb = blocks_of(p.c, b, t);
  if (nb <= p.k) {
    for (int i = tid; i < p.k; i += SEL_THREADS) out[i] = i < nb ? i : -1;
    return;
  }
  const int lo = p.n_sink, hi = nb - p.n_recent, n = hi - lo;  // k < nb: both ends are whole and apart
  const int want = p.k - p.n_sink - p.n_recent;                // of the blocks [lo, hi); fewer than n
  const int words = (nb + 31) / 32;
  float2* score = (float2*)dyn;
  uint16_t* open = (uint16_t*)(dyn + p.max_blocks);
  float above = INFINITY, below = INFINITY;  // want = 0: nothing between the ends
  if (want > 0) {
    const float2* src = p.score + row * p.max_blocks + lo;
    const float* qn = p.qn + (tok * nqh + kh * GQA) * AD;
    float E = 0.f, mn = INFINITY, mx = -INFINITY;
#pragma unroll 4
    for (int i = tid; i < n; i += SEL_THREADS) {
      const float2 v = src[i];
      score[i] = v;
      E = fmaxf(E, v.y);
      mn = fminf(mn, v.x);
      mx = fmaxf(mx, v.x);
    }
#pragma unroll
    for (int i = 0; i < GQA * AD / SEL_THREADS; i++) (&sh.q[0][0])[tid + i * SEL_THREADS] = qn[tid + i * SEL_THREADS];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      E = fmaxf(E, __shfl_xor_sync(0xffffffffu, E, o));
      mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    }
    if (lane == 0) sh.red[0][warp] = E, sh.red[1][warp] = mn, sh.red[2][warp] = mx;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < SEL_WARPS; w++) {
      E = fmaxf(E, sh.red[0][w]);
      mn = fminf(mn, sh.red[1][w]);
      mx = fmaxf(mx, sh.red[2][w]);
    }
    if (E <= 3e38f) {
      // The scores in 2,048 steps from the smallest to the largest: the want-th largest lies in the step where the count from the top
      // reaches want. The step's ends are moved out by more than the roundings of the arithmetic. Where the scores are too far
      // apart or too close for that, or many lie in the step, by their bits.
      const float width = mx - mn, scale = (float)SEL_BINS / width;
      int inside = n;
      const bool steps = width > 1e-30f && width < 1e30f;
      if (steps) {
        for (int i = tid; i < n; i += SEL_THREADS) atomicAdd(&sh.hist[min(SEL_BINS - 1, (int)((score[i].x - mn) * scale))], 1u);
        __syncthreads();
        int need;
        const int bin = find_bin(want, sh, &need, &inside);
        const float step = width / SEL_BINS, slack = 1e-6f * (fabsf(mn) + fabsf(mx));
        above = mn + (float)(bin + 1) * step + slack + E;
        below = mn + (float)bin * step - slack - E;
      }
      if (!steps || inside > 64) {
        uint32_t mask;
        int ignored;
        const uint32_t lead = nth_largest<uint32_t>([&](int i) { return order_key(score[i].x); }, n, want, 16, sh, &mask, &ignored);
        above = key_value(lead | ~mask) + E;
        below = key_value(lead) - E;
      }
    } else {
      below = -INFINITY;  // all are open (no s - e is above infinity)
    }
  }
  int n_in = 0;
  for (int w = warp; w < words; w += SEL_WARPS) {
    const int blk = 32 * w + lane;
    bool in = blk < lo || (blk >= hi && blk < nb), maybe = false;
    if (blk >= lo && blk < hi && want > 0) {
      const float2 v = score[blk - lo];
      in = v.x - v.y > above;
      maybe = !in && !(v.x + v.y < below);
    }
    const uint32_t wi = __ballot_sync(0xffffffffu, in), wo = __ballot_sync(0xffffffffu, maybe);
    n_in += __popc(wi);
    if (lane == 0) sh.in[w] = wi, sh.edge[w] = 0;
    if (wo) {
      int at = 0;
      if (lane == 0) at = atomicAdd(&sh.n_open, __popc(wo));
      at = __shfl_sync(0xffffffffu, at, 0);
      if (maybe) open[at + __popc(wo & ((1u << lane) - 1))] = (uint16_t)blk;
    }
  }
  if (lane == 0 && n_in) atomicAdd(&sh.n_in, n_in);
  __syncthreads();
  const int n_open = sh.n_open, room = p.k - sh.n_in;  // 0 <= room <= n_open, by the above
  int need = 0;
  if (room == n_open) {
    for (int c = tid; c < n_open; c += SEL_THREADS) atomicOr(&sh.in[open[c] >> 5], 1u << (open[c] & 31));
    __syncthreads();
  } else {
    uint64_t* key = dyn;  // the scores to 15 bits are no longer used
    for (int c = warp; c < n_open; c += SEL_WARPS) {
      const int64_t idx = bounds_index(p.c, b, kh, open[c]);
      double s[GQA] = {};
      if (idx >= 0) {
        const uint4 l4 = *(const uint4*)(p.bounds + idx * 2 * AD + 8 * lane), h4 = *(const uint4*)(p.bounds + idx * 2 * AD + AD + 8 * lane);
        const uint32_t lw[4] = {l4.x, l4.y, l4.z, l4.w}, hw[4] = {h4.x, h4.y, h4.z, h4.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float2 lf = __half22float2(u32_as_h2(lw[i])), hf = __half22float2(u32_as_h2(hw[i]));
#pragma unroll
          for (int g = 0; g < GQA; g++) {
            const float2 x = *(const float2*)&sh.q[g][8 * lane + 2 * i];
            s[g] = fma((double)x.x, (double)(x.x < 0.f ? lf.x : hf.x), s[g]);
            s[g] = fma((double)x.y, (double)(x.y < 0.f ? lf.y : hf.y), s[g]);
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
      if (lane == 0) key[c] = idx < 0 ? 0ull : nan ? ~0ull : order_key(best);
    }
    __syncthreads();
    if (n_open <= SEL_THREADS) {  // few: each counts those before it
      if (tid < n_open) {
        const uint64_t k = key[tid];
        const int blk = open[tid];
        int rank = 0;
        for (int c = 0; c < n_open; c++) rank += key[c] > k || (key[c] == k && open[c] < blk);
        if (rank < room) atomicOr(&sh.in[blk >> 5], 1u << (blk & 31));
      }
    } else {
      uint64_t mask;
      const uint64_t border = nth_largest<uint64_t>([&](int i) { return key[i]; }, n_open, room, 0, sh, &mask, &need);
      for (int c = tid; c < n_open; c += SEL_THREADS)
        if (key[c] >= border) atomicOr(key[c] > border ? &sh.in[open[c] >> 5] : &sh.edge[open[c] >> 5], 1u << (open[c] & 31));
    }
    __syncthreads();
  }
  // The list in order: what is in, and the first `need` on the edge.
  uint32_t in = tid < words ? sh.in[tid] : 0u, edge = tid < words ? sh.edge[tid] : 0u;
  const unsigned long long before = block_scan((unsigned long long)__popc(in) << 32 | (unsigned)__popc(edge), sh.sums);
  int on = (int)(before & 0xffffffffu), at = (int)(before >> 32) + min(on, need);
  for (uint32_t m = in | edge; m; m &= m - 1) {
    const int bit = __ffs((int)m) - 1;
    if ((edge >> bit) & 1 && on++ >= need) continue;
    out[at++] = 32 * tid + bit;
  }
}

int launch_select(DeviceCtx* ctx, SelectParams& p, int max_len, const char* who, cudaStream_t s) {
  static bool attr[64] = {};
  static std::mutex attr_mu;
  auto smem_of = [](int blocks) { return (size_t)blocks * 10; };  // a 64-bit key and a number of every block
  {
    std::lock_guard<std::mutex> lock(attr_mu);
    if (!attr[ctx->dev]) {
      Q27B_CK(cudaFuncSetAttribute(select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_of(SEL_MAX_BLOCKS)));
      Q27B_CK(cudaFuncSetAttribute(score_kernel<1>, cudaFuncAttributeMaxDynamicSharedMemorySize, 1 * Q_TOKEN));
      Q27B_CK(cudaFuncSetAttribute(score_kernel<2>, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * Q_TOKEN));
      Q27B_CK(cudaFuncSetAttribute(score_kernel<3>, cudaFuncAttributeMaxDynamicSharedMemorySize, 3 * Q_TOKEN));
      Q27B_CK(cudaFuncSetAttribute(score_kernel<4>, cudaFuncAttributeMaxDynamicSharedMemorySize, 4 * Q_TOKEN));
      attr[ctx->dev] = true;
    }
  }
  p.max_blocks = (max_len + BLK - 1) / BLK;
  const bool scored = p.max_blocks > p.k;
  if (scored) {
    const size_t floats = (size_t)p.c.B * p.c.T * p.c.nkvh * p.max_blocks * 2;
    float* scratch;
    if (p.c.page_table) {
      if (int rc = paged_ws(ctx, floats, &scratch, who)) return rc;
    } else {
      size_t cap;
      if (int rc = prefill_ws(ctx, &scratch, &cap)) return rc;
      if (cap < floats)
        return fail(Q27B_UNSUPPORTED, std::string(who) + ": the prefill workspace (" + std::to_string(cap * sizeof(float)) +
                                          " bytes) is too small for the scores of this call (" +
                                          std::to_string(floats * sizeof(float)) + " bytes)");
    }
    p.score = (float2*)scratch;
    // Two CTAs fit an SM; twice as many as that, where the blocks suffice, even out sequences of different length. A CTA
    // goes through several groups of 64 blocks with the queries staged once.
    const int64_t pairs = (int64_t)p.c.nkvh * p.c.B, groups = (p.max_blocks + SCORE_GROUP - 1) / SCORE_GROUP;
    const int64_t ctas = std::max<int64_t>(1, std::min<int64_t>(groups, (4 * (int64_t)ctx->n_sm + pairs - 1) / pairs));
    auto* score = p.c.T == 1 ? score_kernel<1> : p.c.T == 2 ? score_kernel<2> : p.c.T == 3 ? score_kernel<3> : score_kernel<4>;
    Q27B_CK(launch_step(score, dim3((unsigned)ctas, p.c.nkvh, p.c.B), dim3(32 * SCORE_WARPS), p.c.T * Q_TOKEN, s, p));
  }
  Q27B_CK(launch_step(select_kernel, dim3(p.c.nkvh, p.c.T, p.c.B), dim3(SEL_THREADS), scored ? smem_of(p.max_blocks) : 0, s, p));
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
  if (misaligned({kcache, vcache})) return fail(Q27B_BAD_SHAPE, "kv_commit: pointers must be 16-byte aligned");
  if (bad_contiguous(T, MAX_TREE_T, nkvh, n_ctx)) return fail(Q27B_BAD_SHAPE, "kv_commit: bad shape");
  DeviceCtx* ctx;
  if (int rc = device_ctx(&ctx)) return rc;
  return launch_commit(contiguous_ref(ctx, pos0, T, nkvh, n_ctx, q8), kcache, vcache, path, count, (cudaStream_t)stream);
}

int q27b_kv_commit_paged(void* kpool, void* vpool, const int* page_table, const int* seq_len, const int* path, const int* count,
                         int B, int T, int nkvh, int n_pages, int max_pages, void* stream) {
  if (!kpool || !vpool || !page_table || !seq_len || !path || !count) return fail(Q27B_BAD_SHAPE, "kv_commit_paged: null pointer");
  if (misaligned({kpool, vpool})) return fail(Q27B_BAD_SHAPE, "kv_commit_paged: pointers must be 16-byte aligned");
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
  if (misaligned({kcache, bounds})) return fail(Q27B_BAD_SHAPE, "kv_bounds: pointers must be 16-byte aligned");
  if (bad_contiguous(T, 0x7fffffff, nkvh, n_ctx) || T > n_ctx) return fail(Q27B_BAD_SHAPE, "kv_bounds: bad shape");
  DeviceCtx* ctx;
  if (int rc = device_ctx(&ctx)) return rc;
  return launch_bounds(contiguous_ref(ctx, pos0, T, nkvh, n_ctx, q8), kcache, bounds, ctx->n_sm, (cudaStream_t)stream);
}

int q27b_kv_bounds_paged(const void* kpool, void* bounds, const int* page_table, const int* seq_len, int B, int T, int nkvh,
                         int n_pages, int max_pages, void* stream) {
  if (!kpool || !bounds || !page_table || !seq_len) return fail(Q27B_BAD_SHAPE, "kv_bounds_paged: null pointer");
  if (misaligned({kpool, bounds})) return fail(Q27B_BAD_SHAPE, "kv_bounds_paged: pointers must be 16-byte aligned");
  if (bad_paged(B, T, 0x7fffffff, nkvh, n_pages, max_pages) || T > max_pages * Q27B_PAGE)
    return fail(Q27B_BAD_SHAPE, "kv_bounds_paged: bad shape");
  DeviceCtx* ctx;
  if (int rc = device_ctx(&ctx)) return rc;
  return launch_bounds(paged_ref(ctx, page_table, seq_len, B, T, nkvh, n_pages, max_pages), kpool, bounds, ctx->n_sm,
                       (cudaStream_t)stream);
}

int q27b_select_blocks(const float* qn, const void* bounds, int* sel, const int* pos0, int T, int k, int n_sink, int n_recent,
                       int nqh, int nkvh, int n_ctx, void* stream) {
  if (!qn || !bounds || !sel || !pos0) return fail(Q27B_BAD_SHAPE, "select_blocks: null pointer");
  if (misaligned({bounds})) return fail(Q27B_BAD_SHAPE, "select_blocks: pointers must be 16-byte aligned");
  if (bad_contiguous(T, Q27B_MAX_T, nkvh, n_ctx)) return fail(Q27B_BAD_SHAPE, "select_blocks: bad shape");
  if (int rc = check_select("select_blocks", T, k, n_sink, n_recent, nqh, nkvh, n_ctx)) return rc;
  DeviceCtx* ctx;
  if (int rc = device_ctx(&ctx)) return rc;
  SelectParams p = {};
  p.c = contiguous_ref(ctx, pos0, T, nkvh, n_ctx, 1);
  p.qn = qn; p.bounds = (const __half*)bounds; p.sel = sel; p.k = k; p.n_sink = n_sink; p.n_recent = n_recent;
  return launch_select(ctx, p, n_ctx, "select_blocks", (cudaStream_t)stream);
}

int q27b_select_blocks_paged(const float* qn, const void* bounds, int* sel, const int* page_table, const int* seq_len, int B,
                             int T, int k, int n_sink, int n_recent, int nqh, int nkvh, int n_pages, int max_pages,
                             int max_seq_len, void* stream) {
  if (!qn || !bounds || !sel || !page_table || !seq_len) return fail(Q27B_BAD_SHAPE, "select_blocks_paged: null pointer");
  if (misaligned({bounds})) return fail(Q27B_BAD_SHAPE, "select_blocks_paged: pointers must be 16-byte aligned");
  if (bad_paged(B, T, Q27B_MAX_T, nkvh, n_pages, max_pages) || max_seq_len < T || max_seq_len > max_pages * Q27B_PAGE)
    return fail(Q27B_BAD_SHAPE, "select_blocks_paged: bad shape");
  if (int rc = check_select("select_blocks_paged", T, k, n_sink, n_recent, nqh, nkvh, max_seq_len)) return rc;
  DeviceCtx* ctx;
  if (int rc = device_ctx(&ctx)) return rc;
  SelectParams p = {};
  p.c = paged_ref(ctx, page_table, seq_len, B, T, nkvh, n_pages, max_pages);
  p.c.n_ctx = max_seq_len;  // a longer sequence than the caller said is cut there: the scores have room for no more
  p.qn = qn; p.bounds = (const __half*)bounds; p.sel = sel; p.k = k; p.n_sink = n_sink; p.n_recent = n_recent;
  return launch_select(ctx, p, max_seq_len, "select_blocks_paged", (cudaStream_t)stream);
}

}  // extern "C"

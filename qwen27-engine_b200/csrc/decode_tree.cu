// Attention of a tree of T drafts over a KV cache on the tensor cores (q27b_attn_decode_tree*).
//
// Both contractions on tcgen05.mma kind::f16 as in the f16-QK prefill kernel: S = (Q kq_scale) K^T with Q in tensor memory,
// P = exp(S - m) in f16, O += P V with O in tensor memory, f32 accumulation, the reference maximum m of a row moved only
// when the true one has outgrown it by TAU. Q kq_scale, K and V (q8_0: value times scale) and P are rounded to f16, the
// operand type; m, the row sums and O are f32.
//
// A unit is 128 of the 6 T (draft, head) rows of a KV head of a sequence: the prefix belongs to all rows, so up to 21 drafts cost
// one pass over the cache. One CTA takes one part of a unit's position tiles and writes m, l and O as a partial. One sequence: a
// CTA per SM, the same number for every unit. A batch: every CTA adds up the lengths, from which the length of a part follows
// (tree_share), and finds its own part. A tile that reaches into
// the drafted rows gets a 64-bit word of visible columns per row: the row's mask, shifted to the tile.
// Weights of columns that a row does not see are 0, and so that 0 times what lies there is 0, V rows that no row
// may see (past the sequence, on a page that does not exist) are cleared on the way to the tensor core, and so are drafted V
// values that are not finite in f16: the rows that see such a draft say so with the sign of their sum, and the merge adds weight times
// value to them in f32.
//
// Warps 0-3 softmax of the even tiles and 4-7 of the odd ones, a thread a row; warp 8 issues the Q K^T MMAs, warp 9 the P V MMAs.
// f16 cache: warp 10 brings the tiles by TMA as the tensor core reads them. q8_0 cache: warps 10-13 turn K and 14-17 V into f16
// operands, from registers that they load straight from the cache, a tile ahead: through shared
// memory, which 64 KB of operands a tile written and read again keep busy already, the int8 tile would cost another 68 KB.
// TMEM: columns 0-255 O (f32), 256-383 two buffers of 64 columns for S (f32) and over it P (f16), 384-511 the Q tile.
//
// Drafted V values that are not finite: f16 rows are cleaned by the softmax warps, q8_0 rows by the warp that issues P V, while the
// softmax is at the tile. (In the converters, whose registers are all taken, a batch of 16 sequences took 124 to 138 us instead of
// 114; the values added in this kernel's epilogue instead of the merge: 138.)
//
// Measured (events, 16 drafts behind 150,000 positions of four heads, 327 MB and 59 GFLOP): 91 to 94 us with the GPU cool, 115 in a long
// run, in which it draws 970 W and lowers its clock to 1.54 GHz: 2.8 TB/s, 0.51 PFLOP/s. At full clock a tile takes 2,600 cycles of an SM;
// the MMAs are 1,000 of them, MMAs and softmax without the int8 tiles 1,780 (65 us). The following left it at 93 to 98 us and
// are not in: the next tiles brought into L2 ahead, int8 tiles through TMA into shared memory two ahead, all loads of a tile in a burst,
// 32-byte loads, no exponentials, 16 converter warps (101). P in shared memory instead of over S: 98 cool and 117 long, a batch of 16
// sequences 128 long instead of 122. Both warpgroups on every tile, 32 columns a thread: the same at 150,000, 18.2 instead of
// 19.3 us for 12 drafts behind 20,000 of one f16 head, where a CTA has three tiles.
#include "cache_ref.h"
#include "decode_rows.h"
#include "f16_tile.cuh"

#include <mutex>

namespace q27b {
namespace {

constexpr int QT = TREE_ROWS;    // query rows per CTA
constexpr float TAU = 5.0f;
constexpr int NWG = 2, OW = AD / NWG;  // softmax threads per row: of the even and of the odd tiles; their columns of Q and O
constexpr int NSW = 4 * NWG, MMA_WARP = NSW, PV_WARP = NSW + 1, TMA_WARP = NSW + 2, KCONV_WARP0 = NSW + 2, VCONV_WARP0 = NSW + 6;
constexpr int N_CONV_WARPS = 4, NK = 3, NV = 3;  // f16 K and V buffers
enum { B_QFULL = 0, B_KFULL = 1, B_KEMPTY = 4, B_VFULL = 7, B_VEMPTY = 10, B_SFULL = 13, B_PFULL = 15, B_PVDONE = 17, B_ODONE = 19, NBAR = 20 };
// Shared memory
constexpr int OFF_K = 0;
constexpr int OFF_V = OFF_K + NK * KV_BYTES;
constexpr int OFF_STAGE = OFF_V + NV * KV_BYTES;          // the Q tile on its way to tensor memory, 2 KB a softmax warp
constexpr int OFF_XCH = OFF_STAGE + NSW * 2048;           // f32: [128] reference maxima, [NWG][128] sums
constexpr int OFF_BAR = OFF_XCH + (1 + NWG) * QT * 4;
constexpr int OFF_BAD = OFF_BAR + NBAR * 8;               // [2 words]: drafts of whose V rows something was cleared
constexpr int OFF_SKIP = OFF_BAD + 8;                     // [TREE_MAX_TILES / 32] words: tiles on pages that do not exist
constexpr int OFF_SCAN = OFF_SKIP + TREE_MAX_TILES / 8;   // [32] 64-bit sums
constexpr int OFF_MISC = OFF_SCAN + 32 * 8;
constexpr int SMEM_BYTES = OFF_MISC + 16 + 1024;
static_assert(SMEM_BYTES <= 232448, "shared memory budget of one CTA");
constexpr int threads(bool q8) { return (NSW + 2 + (q8 ? 2 * N_CONV_WARPS : 1)) * 32; }
constexpr uint32_t TMEM_COLS = 512;
constexpr uint32_t TM_O = 0, TM_S = 256, TM_Q = 384;  // O f32 256 columns, S 2 x 64 f32, Q 128 columns of f16 pairs
constexpr uint32_t IDESC_QK = umma_idesc(1, 0, 0, 0, 0, QT, PT);   // f32 += f16 * f16, both K-major, M128 N64
constexpr uint32_t IDESC_PV = umma_idesc(1, 0, 0, 0, 1, QT, AD);   // B (V) MN-major, M128 N256

// One lane of a converged warp, the same one every time; in code that the compiler knows to be one lane's, the operands of
// an MMA stay in uniform registers.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(one));
  return one != 0;
}
// The two threads of a query row sit in warp q of either softmax warpgroup. Between them: the reference maximum after a tile is there.
__device__ __forceinline__ void ref_ready(int q, int parity) { asm volatile("bar.arrive %0, %1;" ::"r"(1 + 2 * q + parity), "n"(64) : "memory"); }
__device__ __forceinline__ void ref_wait(int q, int parity) { asm volatile("bar.sync %0, %1;" ::"r"(1 + 2 * q + parity), "n"(64) : "memory"); }
__device__ __forceinline__ void row_sync(int q) { asm volatile("bar.sync %0, %1;" ::"r"(9 + q), "n"(64) : "memory"); }
__device__ __forceinline__ bool not_finite(uint32_t h2) { return (h2 & 0x7C00u) == 0x7C00u || (h2 & 0x7C000000u) == 0x7C000000u; }

__device__ __forceinline__ uint32_t finite_of(uint32_t h2) {  // 0 for a half that is none
  return h2 & (((h2 & 0x7C00u) == 0x7C00u ? 0u : 0xFFFFu) | ((h2 & 0x7C000000u) == 0x7C000000u ? 0u : 0xFFFF0000u));
}

// Clears what may not reach the tensor core of row r of a swizzled f16 V tile, dims 64 sg .. 64 sg + 63: all of a row that no draft
// has (draft < 0), else the values that are not finite, noted in bad[draft].
__device__ __forceinline__ void clean_v_row(uint8_t* vrow, int r, int draft, uint32_t* bad) {
  uint4 x[8];
  bool odd = draft < 0;
#pragma unroll
  for (int c = 0; c < 8; c++) x[c] = *(const uint4*)(vrow + ((c ^ (r & 7)) << 4));
#pragma unroll
  for (int c = 0; c < 8; c++) odd |= not_finite(x[c].x) || not_finite(x[c].y) || not_finite(x[c].z) || not_finite(x[c].w);
  if (!odd) return;
  if (draft >= 0) atomicOr(&bad[draft >> 5], 1u << (draft & 31));
#pragma unroll
  for (int c = 0; c < 8; c++)
    *(uint4*)(vrow + ((c ^ (r & 7)) << 4)) =
        draft < 0 ? make_uint4(0, 0, 0, 0) : make_uint4(finite_of(x[c].x), finite_of(x[c].y), finite_of(x[c].z), finite_of(x[c].w));
}

// 16 bytes of the cache, read once.
__device__ __forceinline__ uint4 load16(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

template <bool Q8, bool PAGED>
__global__ void __launch_bounds__(threads(Q8), 1)
tree_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const RowsParams p, int n_sm) {
  constexpr int THREADS = threads(Q8);
  extern __shared__ uint8_t smem_raw[];
  const uint32_t sbase = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* sgen = smem_raw + (sbase - smem_u32(smem_raw));
  uint64_t* bar = (uint64_t*)(sgen + OFF_BAR);
  uint32_t* bad = (uint32_t*)(sgen + OFF_BAD);
  uint32_t* skip = (uint32_t*)(sgen + OFF_SKIP);
  uint32_t* tmem_slot = (uint32_t*)(sgen + OFF_MISC);
  volatile int* abort_flag = (volatile int*)(sgen + OFF_MISC + 4);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int T = p.c.T, nkvh = p.c.nkvh, nqh = nkvh * GQA, units = nkvh * tree_row_tiles(T);  // units of a sequence
  int64_t* scan = (int64_t*)(sgen + OFF_SCAN);

  // What needs no memory of the call runs while the previous kernel of the stream drains.
  if (tid == 0) {
    *abort_flag = 0;
    if (!Q8) {
      tma_prefetch_desc(&tm_k);
      tma_prefetch_desc(&tm_v);
    }
  }
  pdl_wait();
  pdl_trigger();
  // The part of this CTA: tiles it0 .. it0 + nt - 1 of unit y (a row tile of a KV head) of sequence b
  auto end_of = [&](int b) { return min(first_pos(p.c, b) + T, p.c.n_ctx); };
  int b = 0, y = 0, it0 = 0, nt = 0;
  if (!PAGED) {
    const int ntot = tree_tiles(end_of(0)), parts = min(p.nsplit, ntot), z = blockIdx.x % p.nsplit;
    y = blockIdx.x / p.nsplit;
    if (z < parts) it0 = (int)((int64_t)ntot * z / parts), nt = (int)((int64_t)ntot * (z + 1) / parts) - it0;
  } else {  // every thread looks at some sequences: the tiles of all of them, then their parts
    const int per = (p.c.B + THREADS - 1) / THREADS, b0 = min(p.c.B, tid * per), b1 = min(p.c.B, b0 + per);
    int64_t mine = 0, all = 0;
    auto sum = [&](int64_t v) {  // -> the sum before this thread's; `all`: of all
      int64_t x = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t t = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += t;
      }
      if (lane == 31) scan[warp] = x;
      __syncthreads();
      int64_t before = 0;
      all = 0;
      for (int w = 0; w < THREADS / 32; w++) {
        if (w < warp) before += scan[w];
        all += scan[w];
      }
      __syncthreads();
      return before + x - v;
    };
    for (int i = b0; i < b1; i++) {
      const int n = tree_tiles(end_of(i));
      mine += n ? ((int64_t)1 << 40) + n : 0;  // sequences that are not empty, and their tiles
    }
    sum(mine);
    const int share = tree_share((all & (((int64_t)1 << 40) - 1)) * units, (all >> 40) * units, n_sm);
    mine = 0;
    for (int i = b0; i < b1; i++) mine += tree_parts(tree_tiles(end_of(i)), share);
    int64_t at = sum(mine);
    if (tid == 0) scan[0] = -1;
    __syncthreads();
    for (int i = b0; i < b1; i++) {
      const int n = tree_parts(tree_tiles(end_of(i)), share);
      if (blockIdx.x == 0) p.plan[1 + i] = at;
      if (at * units <= blockIdx.x && blockIdx.x < (at + n) * units) scan[0] = i, scan[1] = at;
      at += n;
    }
    if (blockIdx.x == 0 && tid == 0) p.plan[0] = share;
    __syncthreads();
    b = (int)scan[0];
    if (b >= 0) {
      const int ntot = tree_tiles(end_of(b)), parts = tree_parts(ntot, share), k = (int)(blockIdx.x - scan[1] * units), z = k % parts;
      y = k / parts;
      it0 = (int)((int64_t)ntot * z / parts), nt = (int)((int64_t)ntot * (z + 1) / parts) - it0;
    }
  }
  if (nt > 0 && warp == 0) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (nt <= 0) return;  // the merge knows which parts there are
  const uint32_t tmem = *tmem_slot;
  const int first = first_pos(p.c, b);  // of the drafts
  const int n_end = end_of(b), zone = min(first, n_end);  // rows from `zone` on are not for everybody
  const int kh = y % nkvh, row0 = y / nkvh * QT;
  const int64_t slot0 = (int64_t)blockIdx.x * QT;  // its rows among the partials
  // Softmax warps q, q + 4 have rows 32 q ..; those past the last row have nothing to do (what the tensor core makes of their rows
  // of Q and P reaches no other row).
  const int n_active = min(4, (T * GQA - row0 + 31) / 32);  // of either warpgroup
  if (tid == 0) {
    mbar_init(&bar[B_QFULL], NWG * n_active);
    for (int s = 0; s < 3; s++) {
      mbar_init(&bar[B_KFULL + s], Q8 ? N_CONV_WARPS : 1);  // q8_0: the converter warps fill the buffers
      mbar_init(&bar[B_KEMPTY + s], 1);
      mbar_init(&bar[B_VFULL + s], Q8 ? N_CONV_WARPS : 1);
      mbar_init(&bar[B_VEMPTY + s], 1);
    }
    for (int s = 0; s < 2; s++) {  // the buffers of S and P
      mbar_init(&bar[B_SFULL + s], 1);
      mbar_init(&bar[B_PFULL + s], n_active);
      mbar_init(&bar[B_PVDONE + s], 1);
    }
    mbar_init(&bar[B_ODONE], 2);
    mbar_fence_init();
  }
  if (tid < 2) bad[tid] = 0;
  if (PAGED) {  // the pages of this part: what lies on one that is none is not visible
    for (int j = tid; j < (nt + 31) / 32; j += THREADS) skip[j] = 0;
    __syncthreads();
    for (int j = tid; j < nt; j += THREADS)
      if (cache_row(p.c, b, kh, (it0 + j) * PT) < 0) atomicOr(&skip[j >> 5], 1u << (j & 31));
  }
  __syncthreads();
  auto skipped = [&](int j) { return PAGED && ((((volatile uint32_t*)skip)[j >> 5] >> (j & 31)) & 1); };

  if (warp < NSW && (warp & 3) >= n_active) {
    // no rows
  } else if (warp < NSW) {
    // ================================================================ softmax warps
    const int wg = warp >> 2, q = warp & 3;
    const int r = q * 32 + lane;       // query row = TMEM lane
    const int t = (row0 + r) / GQA;
    float* xch = (float*)(sgen + OFF_XCH);
    const uint32_t tlane = tmem + ((uint32_t)(q * 32) << 16);
    // output row of row gr of the KV head
    auto out_row = [&](int gr) { return ((size_t)b * T + gr / GQA) * nqh + kh * GQA + gr % GQA; };
    {
      // Q tile -> tensor memory, lane = row, column c = dims 2c, 2c + 1 as f16: this warp writes dims OW wg .. of its 32
      // rows, scaled and rounded; rows past 6 T are zero. 32 dims at a time, loaded with eight lanes to 128 contiguous bytes of
      // a row and turned to a row per thread in shared memory (64 bytes a row, 16-byte chunk c of row r at c ^ (r / 2 % 4)).
      constexpr int LD = 2;  // turns whose loads are requested together
      uint8_t* stage = sgen + OFF_STAGE + warp * 2048;
#pragma unroll 1
      for (int c = 0; c < OW / 32; c += LD) {
        float4 x[LD][8];
#pragma unroll
        for (int u = 0; u < LD; u++)
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const int gr = row0 + q * 32 + 4 * i + (lane >> 3);
            x[u][i] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (gr < T * GQA) x[u][i] = *(const float4*)(p.qn + out_row(gr) * AD + OW * wg + (c + u) * 32 + 4 * (lane & 7));
          }
#pragma unroll
        for (int u = 0; u < LD; u++) {
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const int rr = 4 * i + (lane >> 3), ch = ((lane & 7) >> 1) ^ ((rr >> 1) & 3);
            const float4 v = x[u][i];
            *(uint2*)(stage + rr * 64 + ch * 16 + (lane & 1) * 8) =
                make_uint2(pack_h2(v.x * p.kq_scale, v.y * p.kq_scale), pack_h2(v.z * p.kq_scale, v.w * p.kq_scale));
          }
          __syncwarp();
          uint32_t w[16];
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const uint4 v = *(const uint4*)(stage + lane * 64 + ((i ^ ((lane >> 1) & 3)) << 4));
            w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
          }
          tmem_st16(tlane + TM_Q + wg * (OW / 2) + (c + u) * 16, w);
          __syncwarp();
        }
      }
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar[B_QFULL]);
    }
    uint64_t mine = t < T ? p.mask[(size_t)b * T + t] : 0;
    if (T < 64) mine &= ((uint64_t)1 << T) - 1;

    // The warpgroups take turns at the tiles, so that one's wait for S, its maxima and its exponentials lie under the other's. O
    // belongs to both: the reference maximum of a row goes from tile to tile, each tile's thread leaves it to the next.
    float m_ref = M_INIT;  // what l2 is relative to
    uint64_t l2 = pack2(0.f, 0.f);
    const uint64_t log2e2 = pack2(LOG2E, LOG2E);
    auto refer_to = [&](float m) {
      if (__any_sync(0xffffffffu, m != m_ref)) {
        const float f = ex2((m_ref - m) * LOG2E);  // 0 on the first move (m_ref = -1e30)
        l2 = mul2(l2, pack2(f, f));
        m_ref = m;
      }
    };
#pragma unroll 1
    for (int j = wg; j < nt; j += NWG) {
      const int ph = (j >> 1) & 1;
      const int p_tile = (it0 + j) * PT;
      mbar_wait(&bar[B_SFULL + wg], ph, abort_flag, p.c.status);
      tc_fence_after();
      // Columns of the tile that this row sees; only tiles that reach past the prefix (or lie on no page) have others.
      const bool partly = p_tile + PT > zone || skipped(j);
      uint64_t vis = ~(uint64_t)0;
      if (partly) {
        const int j0 = p_tile - first;  // the draft in column 0
        vis = j0 <= -PT ? ~(uint64_t)0 : j0 < 0 ? (mine << -j0) | (((uint64_t)1 << -j0) - 1) : j0 < 64 ? mine >> j0 : 0;
        if (n_end - p_tile < PT) vis &= ((uint64_t)1 << (n_end - p_tile)) - 1;
        if (skipped(j)) vis = 0;
      }
      uint32_t v[32];
      float mt = -INFINITY;
      auto load_s = [&](int half) {
        tmem_ld32(tlane + TM_S + wg * PT + 32 * half, v);
        tc_wait_ld();
        if (partly) {
          const uint32_t seen = (uint32_t)(vis >> (32 * half));
#pragma unroll
          for (int i = 0; i < 32; i++)
            if (!((seen >> i) & 1)) v[i] = 0xFF800000u;
        }
      };
#pragma unroll
      for (int half = 1; half >= 0; half--) {
        load_s(half);
        float mq[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 32; i++) mq[i & 3] = fmaxf(mq[i & 3], __uint_as_float(v[i]));
        mt = fmaxf(mt, fmaxf(fmaxf(mq[0], mq[1]), fmaxf(mq[2], mq[3])));
      }

      // The reference of a row moves when the maximum has run away from it (and on the first tile with a visible column).
      if (j > 0) ref_wait(q, wg ^ 1);
      float m = j > 0 ? xch[r] : M_INIT;
      if (__any_sync(0xffffffffu, mt > m + TAU)) {
        const float f = ex2((m - fmaxf(m, mt)) * LOG2E);
        m = fmaxf(m, mt);
        if (j > 0) {
          // O holds the sum of tiles < j once the P V of tile j-1 has completed
          mbar_wait(&bar[B_PVDONE + (wg ^ 1)], ((j - 1) >> 1) & 1, abort_flag, p.c.status);
          tc_fence_after();
          rescale_o_f16(tlane + TM_O, f, AD / 32);
          tc_wait_st();
          tc_fence_before();
        }
      }
      xch[r] = m;
      if (j + 1 < nt) ref_ready(q, wg);
      refer_to(m);

      // P = exp(s - m): f32 row sum, f16 for the P V MMA
      const float nmb = -m * LOG2E;
      const uint64_t nmb2 = pack2(nmb, nmb);
#pragma unroll
      for (int half = 0; half < 2; half++) {
        if (half) load_s(half);
        uint32_t w[16];
#pragma unroll
        for (int c = 0; c < 4; c++) {
#pragma unroll
          for (int k = 0; k < 4; k++) {
            float a0, a1;
            unpack2(fma2(pack2(__uint_as_float(v[c * 8 + 2 * k]), __uint_as_float(v[c * 8 + 2 * k + 1])), log2e2, nmb2), a0, a1);
            const float e0 = ex2(a0), e1 = ex2(a1);
            l2 = add2(l2, pack2(e0, e1));
            w[4 * c + k] = pack_h2(e0, e1);
          }
        }
        tmem_st16(tlane + TM_S + wg * PT + 16 * half, w);  // over the scores that it was made of
      }
      if (!Q8 && p_tile + PT > zone) {  // rows of drafts, and, as they came, rows behind the sequence (q8_0: the P V issuer sees to them)
        const int vb = j % NV, r0 = max(0, zone - p_tile);
        mbar_wait(&bar[B_VFULL + vb], (j / NV) & 1, abort_flag, p.c.status);
        for (int u = q * 32 + lane; u < 4 * PT; u += 32 * n_active)  // (segment, row)
          if ((u & 63) >= r0)
            clean_v_row(sgen + OFF_V + vb * KV_BYTES + (u >> 6) * SEGK + (u & 63) * 128, u & 63,
                        p_tile + (u & 63) < n_end ? p_tile + (u & 63) - first : -1, bad);
      }
      if (!Q8) fence_proxy_async();
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar[B_PFULL + wg]);
    }

    // ---- epilogue: the unnormalised partial of this part
    row_sync(q);
    refer_to(xch[r]);  // as the last tile left it
    float la, lb;
    unpack2(l2, la, lb);
    float l = la + lb;
    xch[(1 + wg) * QT + r] = l;
    row_sync(q);
    l += xch[(1 + (wg ^ 1)) * QT + r];
    mbar_wait(&bar[B_ODONE], 0, abort_flag, p.c.status);
    if (wg == 0 && t < T) {
      if (((uint64_t)bad[0] | (uint64_t)bad[1] << 32) & mine) l = __uint_as_float(__float_as_uint(l) | 0x80000000u);
      p.part_ml[slot0 + r] = make_float2(m_ref, l);
    }
    tc_fence_after();
    // 32 columns at a time through shared memory (the K buffers are free now): TMEM gives a thread a row, and a row per
    // thread would touch 32 lines with every store; read back, eight lanes share 128 contiguous bytes of a row.
    uint8_t* stage = sgen + OFF_K + warp * 4096;
#pragma unroll 1
    for (int c = 0; c < OW / 32; c++) {
      const int d0 = wg * OW + c * 32;
      {
        uint32_t v[32];
        tmem_ld32(tlane + TM_O + d0, v);
        tc_wait_ld();
#pragma unroll
        for (int i = 0; i < 8; i++) *(uint4*)(stage + swz128(lane, i)) = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
      }
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const int rr = 4 * i + (lane >> 3), gr = row0 + q * 32 + rr;
        if (gr >= T * GQA) continue;
        *(float4*)(p.part_o + (slot0 + q * 32 + rr) * AD + d0 + 4 * (lane & 7)) = *(const float4*)(stage + swz128(rr, lane & 7));
      }
      __syncwarp();
    }
    tc_fence_before();
  } else if (warp == MMA_WARP) {
    // ================================================================ Q K^T issuer
    mbar_wait(&bar[B_QFULL], 0, abort_flag, p.c.status);
    const bool issuer = elect_one();
    const uint64_t desc = umma_desc_sw128(sbase + OFF_K, 16, 1024);
    int st = 0, ph = 0;  // K buffer and its phase
#pragma unroll 1
    for (int j = 0; j < nt; j++) {
      const int ss = j & 1, sph = (j >> 1) & 1;                         // S buffer
      mbar_wait(&bar[B_KFULL + st], ph, abort_flag, p.c.status);
      mbar_wait(&bar[B_PVDONE + ss], sph ^ 1, abort_flag, p.c.status);  // P V of tile j-2 has read P there
      tc_fence_after();
      if (issuer) {
#pragma unroll
        for (int kk = 0; kk < AD / 16; kk++)  // (addresses of a descriptor are in units of 16 bytes)
          tc_mma_f16_ts(tmem + TM_S + ss * PT, tmem + TM_Q + kk * 8, desc + (uint64_t)(st * (KV_BYTES / 16) + ((kk >> 2) * SEGK + (kk & 3) * 32) / 16),
                        IDESC_QK, kk > 0 ? 1u : 0u);
        tc_commit(&bar[B_SFULL + ss]);
        tc_commit(&bar[B_KEMPTY + st]);
      }
      __syncwarp();
      if (++st == NK) st = 0, ph ^= 1;
    }
  } else if (warp == PV_WARP) {
    // ================================================================ P V issuer
    const bool issuer = elect_one();
    const uint64_t desc_v = umma_desc_sw128(sbase + OFF_V, SEGK, 1024);
    int st = 0, ph = 0;  // V buffer and its phase
#pragma unroll 1
    for (int j = 0; j < nt; j++) {
      const int pb = j & 1, p_tile = (it0 + j) * PT;
      mbar_wait(&bar[B_VFULL + st], ph, abort_flag, p.c.status);
      if (Q8 && p_tile + PT > zone) {  // rows of drafts, while the softmax warps are at this tile
        const int r0 = max(0, zone - p_tile), rows = min(PT, n_end - p_tile) - r0;
#pragma unroll 1
        for (int u = lane; u < 4 * rows; u += 32) {  // (segment, row): neighbouring lanes on neighbouring rows have no bank conflicts
          const int vr = r0 + u % rows;
          clean_v_row(sgen + OFF_V + st * KV_BYTES + u / rows * SEGK + vr * 128, vr, p_tile + vr - first, bad);
        }
        fence_proxy_async();
        __syncwarp();
      }
      mbar_wait(&bar[B_PFULL + pb], (j >> 1) & 1, abort_flag, p.c.status);
      tc_fence_after();
      if (issuer) {
#pragma unroll
        for (int kk = 0; kk < PT / 16; kk++)
          tc_mma_f16_ts(tmem + TM_O, tmem + TM_S + pb * PT + kk * 8, desc_v + (uint64_t)(st * (KV_BYTES / 16) + kk * 128),
                     IDESC_PV, (j > 0 || kk > 0) ? 1u : 0u);
        tc_commit(&bar[B_PVDONE + pb]);
        tc_commit(&bar[B_VEMPTY + st]);
        if (j == nt - 1) tc_commit(&bar[B_ODONE]);
      }
      __syncwarp();
      if (++st == NV) st = 0, ph ^= 1;
    }
    if (lane == 0) mbar_arrive(&bar[B_ODONE]);  // with it `bad` is there
  } else if constexpr (!Q8) {
    // ================================================================ TMA producer (f16 cache)
    if (lane == 0) {
#pragma unroll 1
      for (int j = 0; j < nt; j++) {
        const int row = kh * p.c.n_ctx + (it0 + j) * PT, kb = j % NK, vb = j % NV;
        uint8_t* ks = sgen + OFF_K + kb * KV_BYTES;
        uint8_t* vs = sgen + OFF_V + vb * KV_BYTES;
        mbar_wait(&bar[B_KEMPTY + kb], ((j / NK) & 1) ^ 1, abort_flag, p.c.status);
        mbar_expect_tx(&bar[B_KFULL + kb], KV_BYTES);
#pragma unroll
        for (int sg = 0; sg < 4; sg++) tma_load_2d(ks + sg * SEGK, &tm_k, sg * 128, row, &bar[B_KFULL + kb]);
        mbar_wait(&bar[B_VEMPTY + vb], ((j / NV) & 1) ^ 1, abort_flag, p.c.status);
        mbar_expect_tx(&bar[B_VFULL + vb], KV_BYTES);
#pragma unroll
        for (int sg = 0; sg < 4; sg++) tma_load_2d(vs + sg * SEGK, &tm_v, sg * 128, row, &bar[B_VFULL + vb]);
      }
    }
  } else {
    // ================================================================ converter warps (q8_0 cache)
    // Thread ct: 16 dims (chunk c16) of rows a.row0, a.row0 + 8, .. of every tile, in registers a tile ahead.
    const bool is_v = warp >= VCONV_WARP0;
    const int ct = tid - (is_v ? VCONV_WARP0 : KCONV_WARP0) * 32, c16 = (ct & 3) + 4 * ((ct >> 3) & 3);
    const int b_full = is_v ? B_VFULL : B_KFULL, b_empty = is_v ? B_VEMPTY : B_KEMPTY;
    const ConvAddr a = conv_addr(ct);
    const uint8_t* vals = (const uint8_t*)(is_v ? p.vcache : p.kcache);
    const uint8_t* scales = vals + cache_rows(p.c) * AD;
    // first row of tile j, and how many of its rows are there (past them, and on no page, nothing is read)
    auto tile_row = [&](int j) -> int64_t {
      const int pos = (it0 + j) * PT;
      if (!PAGED) return (int64_t)kh * p.c.n_ctx + pos;
      if (skipped(j)) return 0;
      return ((int64_t)p.c.page_table[(size_t)b * p.c.max_pages + pos / Q27B_PAGE] * nkvh + kh) * Q27B_PAGE + pos % Q27B_PAGE;
    };
    auto tile_rows = [&](int j) { return skipped(j) ? 0 : min(PT, n_end - (it0 + j) * PT); };
    uint4 x[8];
    uint32_t d[8];
    const uint8_t *src = nullptr, *ssrc = nullptr;  // this thread's first chunk of the tile that is fetched, and its scale
    int there = 0;                                  // rows of that tile from a.row0 on
    auto aim = [&](int j) {
      const int64_t row = tile_row(j) + a.row0;
      src = vals + row * AD + 16 * c16;
      ssrc = scales + row * 16 + (c16 >> 1) * 2;
      there = tile_rows(j) - a.row0;
    };
    // Rows that are not there: the bytes of the tile's first row (or the pool's) times 0.
    auto fetch = [&](int k, bool whole) {
      const int r = whole || 8 * k < there ? 8 * k : -a.row0;
      x[k] = load16(src + r * AD);
      d[k] = whole || 8 * k < there ? *(const uint16_t*)(ssrc + r * 16) : 0;
    };
    // Item k of the tile in registers into the f16 buffer, and the same item of the next tile fetched in its place.
    auto convert = [&](int k, uint8_t* dst, bool more, bool whole) {
      const __half2 dd = u32_as_h2(__byte_perm(d[k], d[k], 0x1010));
      const uint32_t xw[4] = {x[k].x ^ 0x80808080u, x[k].y ^ 0x80808080u, x[k].z ^ 0x80808080u, x[k].w ^ 0x80808080u};
      uint32_t o[8];
#pragma unroll
      for (int w = 0; w < 4; w++) {
        o[2 * w] = dq_pair(__byte_perm(xw[w], 0x64646464u, 0x4140), dd);
        o[2 * w + 1] = dq_pair(__byte_perm(xw[w], 0x64646464u, 0x4342), dd);
      }
      if (more) fetch(k, whole);
      *(uint4*)(dst + a.dst + k * 1024) = make_uint4(o[0], o[1], o[2], o[3]);
      *(uint4*)(dst + (a.dst ^ 16u) + k * 1024) = make_uint4(o[4], o[5], o[6], o[7]);
    };
    aim(0);
#pragma unroll
    for (int k = 0; k < 8; k++) fetch(k, false);
    const int nbuf = is_v ? NV : NK;
    int fb = 0, ph = 1;
#pragma unroll 1
    for (int j = 0; j < nt; j++) {
      const int p_tile = (it0 + j) * PT;
      const bool more = j + 1 < nt;
      if (more) aim(j + 1);
      mbar_wait(&bar[b_empty + fb], ph, abort_flag, p.c.status);  // the MMAs of the tile before it have read the buffer
      uint8_t* dst = sgen + (is_v ? OFF_V : OFF_K) + fb * KV_BYTES;
      if (more && tile_rows(j + 1) == PT) {
#pragma unroll
        for (int k = 0; k < 8; k++) convert(k, dst, true, true);
      } else {
#pragma unroll
        for (int k = 0; k < 8; k++) convert(k, dst, more, false);
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar[b_full + fb]);
      if (++fb == nbuf) fb = 0, ph ^= 1;
    }
  }

  drain_after_abort(abort_flag);
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }
}

template <bool Q8, bool PAGED>
int tree_attr() {
  Q27B_CK(cudaFuncSetAttribute(tree_kernel<Q8, PAGED>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES));
  return Q27B_OK;
}

}  // namespace

int launch_tree(const RowsParams& p, int n_sm, cudaStream_t s) {
  static bool attr[64] = {};
  static std::mutex attr_mu;
  int dev;
  Q27B_CK(cudaGetDevice(&dev));
  {
    std::lock_guard<std::mutex> lock(attr_mu);
    if (!attr[dev]) {
      if (int rc = tree_attr<true, false>()) return rc;
      if (int rc = tree_attr<true, true>()) return rc;
      if (int rc = tree_attr<false, false>()) return rc;
      attr[dev] = true;
    }
  }
  const int64_t units = (int64_t)p.c.B * p.c.nkvh * tree_row_tiles(p.c.T);
  const dim3 grid((unsigned)(p.c.page_table ? tree_grid(units, n_sm) : units * p.nsplit));
  CUtensorMap tk = {}, tv = {};  // f16 only
  if (p.c.page_table) {
    Q27B_CK(launch_step(tree_kernel<true, true>, grid, dim3(threads(true)), SMEM_BYTES, s, tk, tv, p, n_sm));
  } else if (p.c.q8) {
    Q27B_CK(launch_step(tree_kernel<true, false>, grid, dim3(threads(true)), SMEM_BYTES, s, tk, tv, p, n_sm));
  } else {
    const uint64_t rows = cache_rows(p.c);
    if (int rc = cached_tmap_2d(&tk, p.kcache, rows, 2 * AD, 2 * AD, 128, PT, true)) return rc;
    if (int rc = cached_tmap_2d(&tv, p.vcache, rows, 2 * AD, 2 * AD, 128, PT, true)) return rc;
    Q27B_CK(launch_step(tree_kernel<false, false>, grid, dim3(threads(false)), SMEM_BYTES, s, tk, tv, p, n_sm));
  }
  return Q27B_OK;
}

}  // namespace q27b

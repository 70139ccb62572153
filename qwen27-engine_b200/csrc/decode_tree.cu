// Attention of a tree of T drafts over a KV cache on the tensor cores (q27b_attn_decode_tree*).
//
// Both contractions on tcgen05.mma kind::f16 as in the f16-QK prefill kernel: S = (Q kq_scale) K^T with Q in tensor memory,
// P = exp(S - m) in f16, O += P V with O in tensor memory, f32 accumulation, the reference maximum m of a row moved only
// when the true one has outgrown it by TAU. Q kq_scale, K and V (q8_0: value times scale) and P are rounded to f16, the
// operand type; m, the row sums and O are f32.
//
// One CTA takes 128 of the 6 T (draft, head) rows of a KV head over one share of the position tiles, and writes its m, l
// and O as a partial: the prefix belongs to all rows, so up to 21 drafts cost one pass over the cache. A tile that reaches into
// the drafted rows gets a 64-bit word of visible columns per row: the row's mask, shifted to the tile.
// Weights of columns that a row does not see are 0, and so that 0 times what lies there is 0, V rows that no row
// may see (past the sequence, on a page that does not exist) are cleared on the way to the tensor core, and drafted V
// chunks of 16 dims that are not finite are cleared and remembered: the rows that see such a draft get NaN in these dims.
//
// Warps 0-7 softmax (two threads a row, 32 columns of a tile each), warp 8 TMA producer, warp 9 issues the Q K^T MMAs, warp
// 10 the P V MMAs; on a q8_0 cache warps 11-14 turn K and 15-18 V from int8 into f16 operands.
#include "cache_ref.h"
#include "decode_rows.h"
#include "f16_tile.cuh"

#include <mutex>

namespace q27b {
namespace {

constexpr int QT = TREE_ROWS;    // query rows per CTA
constexpr float TAU = 5.0f;
constexpr int P_BYTES = QT * 128;           // f16 P: [128][64 positions]
constexpr int NWG = 2, CW = PT / NWG, OW = AD / NWG;  // softmax threads per row; their columns of a tile and of O
constexpr int NSW = 4 * NWG, TMA_WARP = NSW, MMA_WARP = NSW + 1, PV_WARP = NSW + 2, KCONV_WARP0 = NSW + 3, VCONV_WARP0 = NSW + 7;
constexpr int N_CONV_WARPS = 4;
enum { B_QFULL = 0, B_KFULL = 1, B_KEMPTY = 4, B_VFULL = 7, B_VEMPTY = 10, B_SFULL = 13, B_SEMPTY = 15, B_PFULL = 17, B_PEMPTY = 18, B_ODONE = 19,
       B_RKFULL = 20, B_RKEMPTY = 22, B_RVFULL = 24, B_RVEMPTY = 26, NBAR = 28 };
template <bool Q8>
struct Lay {
  static constexpr int NKF = Q8 ? 2 : 3;                   // f16 K buffers, and as many f16 V buffers
  static constexpr int OFF_K = 0;
  static constexpr int OFF_V = OFF_K + NKF * KV_BYTES;
  static constexpr int OFF_P = OFF_V + NKF * KV_BYTES;
  static constexpr int OFF_RAW = OFF_P + P_BYTES;          // q8_0: K stage 0, 1, V stage 0, 1
  static constexpr int OFF_XCH = OFF_RAW + (Q8 ? 4 * RAW_BYTES : 0);  // [tile parity][NWG][128] f32
  static constexpr int OFF_BAR = OFF_XCH + 2 * NWG * QT * 4;
  static constexpr int OFF_BAD = OFF_BAR + NBAR * 8;       // [16 chunks of 16 dims][2 words]: drafts whose V chunk is not finite
  static constexpr int OFF_SKIP = OFF_BAD + 16 * 8;        // [TREE_MAX_SHARE / 32] words: tiles on pages that do not exist
  static constexpr int OFF_MISC = OFF_SKIP + TREE_MAX_SHARE / 8;
  static constexpr int SMEM_BYTES = OFF_MISC + 16 + 1024;
  static constexpr int THREADS = (NSW + 3 + (Q8 ? 2 * N_CONV_WARPS : 0)) * 32;
  static_assert(OFF_P % 1024 == 0 && OFF_RAW % 1024 == 0 && RAW_BYTES % 1024 == 0, "swizzled tiles need 1024-byte alignment");
  static_assert(SMEM_BYTES <= 232448, "shared memory budget of one CTA");
};
constexpr uint32_t TMEM_COLS = 512;
constexpr uint32_t TM_O = 0, TM_S = 256, TM_Q = 384;  // O f32 256 columns, S 2 x 64 f32, Q 128 columns of f16 pairs
constexpr uint32_t IDESC_QK = umma_idesc(1, 0, 0, 0, 0, QT, PT);   // f32 += f16 * f16, both K-major, M128 N64
constexpr uint32_t IDESC_PV = umma_idesc(1, 0, 0, 0, 1, QT, AD);   // B (V) MN-major, M128 N256

// the threads of a query row sit in warp q of every softmax warpgroup
__device__ __forceinline__ void row_sync(int q) { asm volatile("bar.sync %0, %1;" ::"r"(1 + q), "n"(32 * NWG) : "memory"); }
__device__ __forceinline__ bool not_finite(uint32_t h2) { return (h2 & 0x7C00u) == 0x7C00u || (h2 & 0x7C000000u) == 0x7C000000u; }

// Clears the 16-byte chunks of a swizzled f16 V tile that may not reach the tensor core: position p (row r of the tile),
// dims 64 sg .. 64 sg + 63. Rows from `end` on go entirely; chunks of drafted rows (from `zone` on) that are not finite go
// and are noted in bad[chunk of 16 dims][draft].
__device__ __noinline__ void clean_v_row(uint8_t* vrow, int r, int sg, int zone, int end, int draft, uint32_t* bad) {
#pragma unroll 1
  for (int c = 0; c < 8; c++) {
    uint4* at = (uint4*)(vrow + ((c ^ (r & 7)) << 4));
    if (r >= end) {
      *at = make_uint4(0, 0, 0, 0);
    } else if (r >= zone) {
      const uint4 x = *at;
      if (not_finite(x.x) || not_finite(x.y) || not_finite(x.z) || not_finite(x.w)) {
        *at = make_uint4(0, 0, 0, 0);
        atomicOr(&bad[2 * (4 * sg + c / 2) + (draft >> 5)], 1u << (draft & 31));
      }
    }
  }
}

template <bool Q8, bool PAGED>
__global__ void __launch_bounds__(Lay<Q8>::THREADS, 1)
tree_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
            const __grid_constant__ CUtensorMap tm_ks, const __grid_constant__ CUtensorMap tm_vs, const RowsParams p) {
  using LY = Lay<Q8>;
  constexpr int NKF = LY::NKF, OFF_K = LY::OFF_K, OFF_V = LY::OFF_V, OFF_P = LY::OFF_P, OFF_RAW = LY::OFF_RAW, OFF_XCH = LY::OFF_XCH;
  constexpr bool ROOM = LY::THREADS <= 384;  // registers for more loads in flight: 168 a thread; with 19 warps 96
  extern __shared__ uint8_t smem_raw[];
  const uint32_t sbase = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* sgen = smem_raw + (sbase - smem_u32(smem_raw));
  uint64_t* bar = (uint64_t*)(sgen + LY::OFF_BAR);
  uint32_t* bad = (uint32_t*)(sgen + LY::OFF_BAD);
  uint32_t* skip = (uint32_t*)(sgen + LY::OFF_SKIP);
  uint32_t* tmem_slot = (uint32_t*)(sgen + LY::OFF_MISC);
  volatile int* abort_flag = (volatile int*)(sgen + LY::OFF_MISC + 4);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int T = p.c.T, nkvh = p.c.nkvh, nqh = nkvh * GQA, z = blockIdx.x, kh = blockIdx.y % nkvh, row0 = (blockIdx.y / nkvh) * QT,
            b = blockIdx.z;

  // What needs no memory of the call runs while the previous kernel of the stream drains.
  if (tid == 0) {
    mbar_init(&bar[B_QFULL], NSW);
    for (int s = 0; s < 3; s++) {
      mbar_init(&bar[B_KFULL + s], Q8 ? N_CONV_WARPS : 1);  // q8_0: the converter warps fill the buffers
      mbar_init(&bar[B_KEMPTY + s], 1);
      mbar_init(&bar[B_VFULL + s], Q8 ? N_CONV_WARPS : 1);
      mbar_init(&bar[B_VEMPTY + s], 1);
    }
    for (int s = 0; s < 2; s++) {
      mbar_init(&bar[B_SFULL + s], 1);
      mbar_init(&bar[B_SEMPTY + s], NSW);
      mbar_init(&bar[B_RKFULL + s], 1);
      mbar_init(&bar[B_RKEMPTY + s], N_CONV_WARPS);
      mbar_init(&bar[B_RVFULL + s], 1);
      mbar_init(&bar[B_RVEMPTY + s], N_CONV_WARPS);
    }
    mbar_init(&bar[B_PFULL], NSW);
    mbar_init(&bar[B_PEMPTY], 1);
    mbar_init(&bar[B_ODONE], 1);
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
    if (Q8) {
      tma_prefetch_desc(&tm_ks);
      tma_prefetch_desc(&tm_vs);
    }
  }
  if (tid < 32) bad[tid] = 0;
  if (PAGED && tid >= 32 && tid < 32 + TREE_MAX_SHARE / 32) skip[tid - 32] = 0;
  pdl_wait();
  pdl_trigger();
  const int first = first_pos(p.c, b);  // of the drafts
  const int n_end = min(first + T, p.c.n_ctx), zone = min(first, n_end);  // rows from `zone` on are not for everybody
  const int ntot = tree_tiles(n_end), share = tree_share(p, ntot);
  const int it0 = min(ntot, z * share), nt = min(ntot, it0 + share) - it0;
  if (nt <= 0) return;  // the merge knows which shares hold tiles
  if (warp == MMA_WARP) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  if (PAGED) {  // the pages of this share: what lies on one that is none is not visible
    for (int j = tid; j < nt; j += LY::THREADS)
      if (cache_row(p.c, b, kh, (it0 + j) * PT) < 0) atomicOr(&skip[j >> 5], 1u << (j & 31));
    __syncthreads();
  }
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  auto skipped = [&](int j) { return PAGED && ((((volatile uint32_t*)skip)[j >> 5] >> (j & 31)) & 1); };

  if (warp < NSW) {
    // ================================================================ softmax warps
    const int wg = warp >> 2, q = warp & 3;
    const int r = q * 32 + lane;       // query row = TMEM lane
    const int t = (row0 + r) / GQA;
    float* xch = (float*)(sgen + OFF_XCH);
    const uint32_t tlane = tmem + ((uint32_t)(q * 32) << 16);
    // output row of row gr of the KV head
    auto out_row = [&](int gr) { return ((size_t)b * T + gr / GQA) * nqh + kh * GQA + gr % GQA; };
    uint64_t mine = t < T ? p.mask[(size_t)b * T + t] : 0;
    if (T < 64) mine &= ((uint64_t)1 << T) - 1;
    {
      constexpr int LD = ROOM ? 2 : 1;  // turns whose loads are requested together
      // Q tile -> tensor memory, lane = row, column c = dims 2c, 2c + 1 as f16: this warp writes dims OW wg .. of its 32
      // rows, scaled and rounded; rows past 6 T are zero. 32 dims at a time, loaded with eight lanes to 128 contiguous bytes of
      // a row and turned to a row per thread in the P buffer (64 bytes a row, 16-byte chunk c of row r at c ^ (r / 2 % 4)).
      uint8_t* stage = sgen + OFF_P + warp * 2048;
      static_assert(NSW * 2048 <= P_BYTES, "staging of the Q tile");
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

    const int col0 = wg * CW;          // this thread's positions of a tile
    float m_run = M_INIT, m_ref = M_INIT;
    uint64_t l2 = pack2(0.f, 0.f);
    const uint64_t log2e2 = pack2(LOG2E, LOG2E);

#pragma unroll 1
    for (int j = 0; j < nt; j++) {
      const int slot = j & 1;
      const int p_tile = (it0 + j) * PT;
      mbar_wait(&bar[B_SFULL + slot], (j >> 1) & 1, abort_flag, p.c.status);
      tc_fence_after();
      float s[CW];
      {
        uint32_t v[CW];
        tmem_ld(tlane + TM_S + slot * PT + col0, v);
        tc_wait_ld();
#pragma unroll
        for (int i = 0; i < CW; i++) s[i] = __uint_as_float(v[i]);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar[B_SEMPTY + slot]);  // the buffer is in registers: it can be overwritten

      // Columns of the tile that this row sees; only tiles that reach past the prefix (or lie on no page) have others.
      if (p_tile + PT > zone || skipped(j)) {
        const int j0 = p_tile - first;  // the draft in column 0
        uint64_t vis = j0 <= -PT ? ~(uint64_t)0 : j0 < 0 ? (mine << -j0) | (((uint64_t)1 << -j0) - 1) : j0 < 64 ? mine >> j0 : 0;
        if (n_end - p_tile < PT) vis &= ((uint64_t)1 << (n_end - p_tile)) - 1;
        if (skipped(j)) vis = 0;
        const uint32_t seen = (uint32_t)(vis >> col0);
#pragma unroll
        for (int i = 0; i < CW; i++)
          if (!((seen >> i) & 1)) s[i] = -INFINITY;
      }
      float mq[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < CW; i += 4) {
        mq[0] = fmaxf(mq[0], s[i]);
        mq[1] = fmaxf(mq[1], s[i + 1]);
        mq[2] = fmaxf(mq[2], s[i + 2]);
        mq[3] = fmaxf(mq[3], s[i + 3]);
      }
      float mt = fmaxf(fmaxf(mq[0], mq[1]), fmaxf(mq[2], mq[3]));
      // row maximum over the threads of the row; the buffer alternates with the tile
      xch[(slot * NWG + wg) * QT + r] = mt;
      row_sync(q);
#pragma unroll
      for (int o = 1; o < NWG; o++) mt = fmaxf(mt, xch[(slot * NWG + ((wg + o) % NWG)) * QT + r]);
      m_run = fmaxf(m_run, mt);

      // Move the reference max when the true max has run away from it (and on the first tile with a visible column). The
      // threads of a row hold the same m_run and m_ref, so their warps take the same branch.
      const bool want = m_run > m_ref + TAU;
      if (__any_sync(0xffffffffu, want)) {
        const float f = ex2((m_ref - m_run) * LOG2E);  // 0 on the first move (m_ref = -1e30)
        m_ref = m_run;
        l2 = mul2(l2, pack2(f, f));
        if (j > 0) {
          // O holds the sum of tiles < j once the P V of tile j-1 has completed
          mbar_wait(&bar[B_PEMPTY], (j - 1) & 1, abort_flag, p.c.status);
          tc_fence_after();
          rescale_o_f16(tlane + TM_O + wg * OW, f, OW / 32);
          tc_wait_st();
          tc_fence_before();
        }
      }

      // P = exp(s - m_ref): f32 row sum, f16 for the P V MMA (16-byte chunks CW/8 wg .. of the row)
      mbar_wait(&bar[B_PEMPTY], (j & 1) ^ 1, abort_flag, p.c.status);  // P V of tile j-1 has read the buffer
      uint8_t* sP = sgen + OFF_P;
      const float nmb = -m_ref * LOG2E;
      const uint64_t nmb2 = pack2(nmb, nmb);
#pragma unroll
      for (int c = 0; c < CW / 8; c++) {
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
          float a0, a1;
          unpack2(fma2(pack2(s[c * 8 + 2 * k], s[c * 8 + 2 * k + 1]), log2e2, nmb2), a0, a1);
          const float e0 = ex2(a0), e1 = ex2(a1);
          l2 = add2(l2, pack2(e0, e1));
          w[k] = pack_h2(e0, e1);
        }
        *(uint4*)(sP + swz128(r, CW / 8 * wg + c)) = make_uint4(w[0], w[1], w[2], w[3]);
      }
      if (!Q8 && p_tile + PT > zone) {  // f16 cache: V lies in the operand buffer as it came (the converters do this for q8_0)
        const int vb = j % NKF;
        mbar_wait(&bar[B_VFULL + vb], (j / NKF) & 1, abort_flag, p.c.status);
        static_assert(32 * NSW == 4 * PT, "a thread per (segment, row)");
        const int sg = tid >> 6, row = tid & 63;
        clean_v_row(sgen + OFF_V + vb * KV_BYTES + sg * SEGK + row * 128, row, sg, zone - p_tile, n_end - p_tile, p_tile + row - first, bad);
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar[B_PFULL]);
    }

    // ---- epilogue: the unnormalised partial of this share
    float la, lb;
    unpack2(l2, la, lb);
    float l = la + lb;
    xch[((nt & 1) * NWG + wg) * QT + r] = l;
    row_sync(q);
#pragma unroll
    for (int o = 1; o < NWG; o++) l += xch[((nt & 1) * NWG + ((wg + o) % NWG)) * QT + r];
    if (wg == 0 && t < T) p.part_ml[out_row(row0 + r) * p.nsplit + z] = make_float2(m_ref, l);
    mbar_wait(&bar[B_ODONE], 0, abort_flag, p.c.status);
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
        for (int h = 0; h < 2; h++) {  // chunks of 16 dims in which a draft that this row sees is not finite
          const uint64_t nf = (uint64_t)bad[2 * (d0 / 16 + h)] | (uint64_t)bad[2 * (d0 / 16 + h) + 1] << 32;
          if (nf & mine)
#pragma unroll
            for (int i = 0; i < 16; i++) v[16 * h + i] = 0x7FFFFFFFu;
        }
#pragma unroll
        for (int i = 0; i < 8; i++) *(uint4*)(stage + swz128(lane, i)) = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
      }
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const int rr = 4 * i + (lane >> 3), gr = row0 + q * 32 + rr;
        if (gr >= T * GQA) continue;
        *(float4*)(p.part_o + (out_row(gr) * p.nsplit + z) * AD + d0 + 4 * (lane & 7)) = *(const float4*)(stage + swz128(rr, lane & 7));
      }
      __syncwarp();
    }
    tc_fence_before();
  } else if (warp == TMA_WARP) {
    // ================================================================ TMA producer
    if (lane == 0) {
#pragma unroll 1
      for (int j = 0; j < nt; j++) {
        const int pos = (it0 + j) * PT;
        int row = kh * p.c.n_ctx + pos;
        if (PAGED)  // a tile never straddles a page; one that lies on none is fetched from the pool's first page and not seen
          row = skipped(j) ? 0 : (p.c.page_table[(size_t)b * p.c.max_pages + pos / Q27B_PAGE] * nkvh + kh) * Q27B_PAGE + pos % Q27B_PAGE;
        if constexpr (Q8) {
          const int st = j & 1, ph = (j >> 1) & 1;  // raw stages
          uint8_t* kr = sgen + OFF_RAW + st * RAW_BYTES;
          uint8_t* vr = sgen + OFF_RAW + (2 + st) * RAW_BYTES;
          mbar_wait(&bar[B_RKEMPTY + st], ph ^ 1, abort_flag, p.c.status);
          mbar_expect_tx(&bar[B_RKFULL + st], RAW_BYTES);
          tma_load_2d(kr, &tm_k, 0, row, &bar[B_RKFULL + st]);
          tma_load_2d(kr + PT * 128, &tm_k, 128, row, &bar[B_RKFULL + st]);
          tma_load_2d(kr + 2 * PT * 128, &tm_ks, 0, row, &bar[B_RKFULL + st]);
          mbar_wait(&bar[B_RVEMPTY + st], ph ^ 1, abort_flag, p.c.status);
          mbar_expect_tx(&bar[B_RVFULL + st], RAW_BYTES);
          tma_load_2d(vr, &tm_v, 0, row, &bar[B_RVFULL + st]);
          tma_load_2d(vr + PT * 128, &tm_v, 128, row, &bar[B_RVFULL + st]);
          tma_load_2d(vr + 2 * PT * 128, &tm_vs, 0, row, &bar[B_RVFULL + st]);
        } else {
          const int st = j % NKF, ph = (j / NKF) & 1;
          uint8_t* ks = sgen + OFF_K + st * KV_BYTES;
          uint8_t* vs = sgen + OFF_V + st * KV_BYTES;
          mbar_wait(&bar[B_KEMPTY + st], ph ^ 1, abort_flag, p.c.status);
          mbar_expect_tx(&bar[B_KFULL + st], KV_BYTES);
#pragma unroll
          for (int sg = 0; sg < 4; sg++) tma_load_2d(ks + sg * SEGK, &tm_k, sg * 128, row, &bar[B_KFULL + st]);
          mbar_wait(&bar[B_VEMPTY + st], ph ^ 1, abort_flag, p.c.status);
          mbar_expect_tx(&bar[B_VFULL + st], KV_BYTES);
#pragma unroll
          for (int sg = 0; sg < 4; sg++) tma_load_2d(vs + sg * SEGK, &tm_v, sg * 128, row, &bar[B_VFULL + st]);
        }
      }
    }
  } else if (Q8 && warp >= KCONV_WARP0) {
    // ================================================================ converter warps (q8_0 cache)
    const bool is_v = warp >= VCONV_WARP0;
    const int ct = tid - (is_v ? VCONV_WARP0 : KCONV_WARP0) * 32;
    const int b_rfull = is_v ? B_RVFULL : B_RKFULL, b_rempty = is_v ? B_RVEMPTY : B_RKEMPTY;
    const int b_full = is_v ? B_VFULL : B_KFULL, b_empty = is_v ? B_VEMPTY : B_KEMPTY;
    const ConvAddr ca = conv_addr(ct);
#pragma unroll 1
    for (int j = 0; j < nt; j++) {
      const int st = j & 1, fb = j % NKF, p_tile = (it0 + j) * PT;
      mbar_wait(&bar[b_rfull + st], (j >> 1) & 1, abort_flag, p.c.status);
      mbar_wait(&bar[b_empty + fb], ((j / NKF) & 1) ^ 1, abort_flag, p.c.status);  // the MMAs of tile j-NKF have read the buffer
      uint8_t* dst = sgen + (is_v ? OFF_V : OFF_K) + fb * KV_BYTES;
      convert_q8_tile(sgen + OFF_RAW + ((is_v ? 2 : 0) + st) * RAW_BYTES, dst, ca, is_v ? (skipped(j) ? 0 : n_end - p_tile) : PT);
      if (is_v && p_tile + PT > zone) {  // drafted rows: see clean_v_row
        asm volatile("bar.sync %0, %1;" ::"n"(1 + 4), "n"(32 * N_CONV_WARPS) : "memory");
#pragma unroll 1
        for (int u = ct; u < 4 * PT; u += 32 * N_CONV_WARPS)
          clean_v_row(dst + (u >> 6) * SEGK + (u & 63) * 128, u & 63, u >> 6, zone - p_tile, skipped(j) ? 0 : n_end - p_tile,
                      p_tile + (u & 63) - first, bad);
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&bar[b_full + fb]);
        mbar_arrive(&bar[b_rempty + st]);
      }
    }
  } else if (warp == PV_WARP) {
    // ================================================================ P V issuer
    if (lane == 0) {
#pragma unroll 1
      for (int j = 0; j < nt; j++) {
        const int st = j % NKF, ph = (j / NKF) & 1;
        mbar_wait(&bar[B_PFULL], j & 1, abort_flag, p.c.status);
        mbar_wait(&bar[B_VFULL + st], ph, abort_flag, p.c.status);
        tc_fence_after();
#pragma unroll
        for (int kk = 0; kk < PT / 16; kk++) {
          const uint64_t da = umma_desc_sw128(sbase + OFF_P + kk * 32, 16, 1024);
          const uint64_t db = umma_desc_sw128(sbase + OFF_V + st * KV_BYTES + kk * 2048, SEGK, 1024);
          tc_mma_f16(tmem + TM_O, da, db, IDESC_PV, (j > 0 || kk > 0) ? 1u : 0u);
        }
        tc_commit(&bar[B_PEMPTY]);
        tc_commit(&bar[B_VEMPTY + st]);
      }
      tc_commit(&bar[B_ODONE]);
    }
  } else if (warp == MMA_WARP) {
    // ================================================================ Q K^T issuer
    if (lane == 0) {
      mbar_wait(&bar[B_QFULL], 0, abort_flag, p.c.status);
      tc_fence_after();
#pragma unroll 1
      for (int j = 0; j < nt; j++) {
        const int ss = j & 1, sph = (j >> 1) & 1;                         // S buffer
        const int st = j % NKF, ph = (j / NKF) & 1;                       // K buffer
        mbar_wait(&bar[B_KFULL + st], ph, abort_flag, p.c.status);
        mbar_wait(&bar[B_SEMPTY + ss], sph ^ 1, abort_flag, p.c.status);
        tc_fence_after();
#pragma unroll
        for (int kk = 0; kk < AD / 16; kk++) {
          const uint64_t db = umma_desc_sw128(sbase + OFF_K + st * KV_BYTES + (kk >> 2) * SEGK + (kk & 3) * 32, 16, 1024);
          tc_mma_f16_ts(tmem + TM_S + ss * PT, tmem + TM_Q + kk * 8, db, IDESC_QK, kk > 0 ? 1u : 0u);
        }
        tc_commit(&bar[B_SFULL + ss]);
        tc_commit(&bar[B_KEMPTY + st]);
      }
    }
  }

  drain_after_abort(abort_flag);
  tc_fence_before();
  __syncthreads();
  if (warp == MMA_WARP) {
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }
}

template <bool Q8, bool PAGED>
int tree_attr() {
  Q27B_CK(cudaFuncSetAttribute(tree_kernel<Q8, PAGED>, cudaFuncAttributeMaxDynamicSharedMemorySize, Lay<Q8>::SMEM_BYTES));
  return Q27B_OK;
}

}  // namespace

int launch_tree(const RowsParams& p, cudaStream_t s) {
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
  CUtensorMap tk, tv, tks, tvs;
  const uint64_t rows = cache_rows(p.c);
  if (p.c.q8) {
    if (int rc = q8_tmaps(p.kcache, rows, &tk, &tks)) return rc;
    if (int rc = q8_tmaps(p.vcache, rows, &tv, &tvs)) return rc;
  } else {
    if (int rc = cached_tmap_2d(&tk, p.kcache, rows, 2 * AD, 2 * AD, 128, PT, true)) return rc;
    if (int rc = cached_tmap_2d(&tv, p.vcache, rows, 2 * AD, 2 * AD, 128, PT, true)) return rc;
    tks = tk;  // not read
    tvs = tv;
  }
  const dim3 grid(p.nsplit, p.c.nkvh * tree_row_tiles(p.c.T), p.c.B);
  if (p.c.page_table)
    Q27B_CK(launch_step(tree_kernel<true, true>, grid, dim3(Lay<true>::THREADS), Lay<true>::SMEM_BYTES, s, tk, tv, tks, tvs, p));
  else if (p.c.q8)
    Q27B_CK(launch_step(tree_kernel<true, false>, grid, dim3(Lay<true>::THREADS), Lay<true>::SMEM_BYTES, s, tk, tv, tks, tvs, p));
  else
    Q27B_CK(launch_step(tree_kernel<false, false>, grid, dim3(Lay<false>::THREADS), Lay<false>::SMEM_BYTES, s, tk, tv, tks, tvs, p));
  return Q27B_OK;
}

}  // namespace q27b

// Tiles of 64 positions as f16 operands of tcgen05.mma, shared by the f16-QK prefill kernel and the tree kernel: layout of
// a tile in shared memory, dequantisation of a q8_0 tile into it, rescaling of an accumulator in tensor memory.
#pragma once
#include "common.cuh"

namespace q27b {
namespace {

constexpr int PT = 64;           // positions per tile
constexpr int SEGK = PT * 128;   // one 64-dim segment of a K or V tile: [64 positions][128 B]
constexpr int KV_BYTES = 4 * SEGK;          // 32 KB
constexpr int RAW_BYTES = 2 * PT * 128 + PT * 16;  // q8_0 tile: two 128-dim int8 segments [64][128 B], then [64][8] f16 scales

// Rare, and kept out of line: inlined, its 32 registers of payload would sit on the loop's state.
__device__ __noinline__ void rescale_o_f16(uint32_t taddr, float f, int chunks) {
#pragma unroll 1
  for (int c = 0; c < chunks; c++) {
    uint32_t v[32];
    tmem_ld32(taddr + c * 32, v);
    tc_wait_ld();
#pragma unroll
    for (int i = 0; i < 32; i++) v[i] = __float_as_uint(__uint_as_float(v[i]) * f);
    tmem_st32(taddr + c * 32, v);
  }
}

// One tile of a q8_0 cache, raw stage -> f16 operand buffer. 128 threads; item = (row, 16-dim chunk);
// eight neighbouring lanes take 4 chunks of rows rho and rho ^ 5, which keeps both the swizzled
// 16-byte loads and the swizzled 16-byte stores free of bank conflicts. Thread ct owns the same chunk
// of rows row0, row0 + 8, .., row0 + 56: rows 8 apart share their swizzle phase, so every address is
// a per-thread base (ConvAddr, computed once per kernel) plus a constant. Rows >= zero_from are
// cleared (rows past the sequence may hold anything: P is 0 there, V must be too).
struct ConvAddr {
  int row0;       // first row of this thread
  uint32_t src;   // byte offset of its 16 int8 values of row0 in the raw stage
  uint32_t sc;    // ... of their f16 scale
  uint32_t dst;   // ... of the first of its two 16-byte chunks in the f16 buffer
};
__device__ __forceinline__ ConvAddr conv_addr(int ct) {
  ConvAddr a;
  a.row0 = (2 * (ct >> 5)) ^ (5 * ((ct >> 2) & 1));
  const int c16 = (ct & 3) + 4 * ((ct >> 3) & 3);
  a.src = (c16 >> 3) * (PT * 128) + swz128(a.row0, c16 & 7);
  a.sc = 2 * PT * 128 + a.row0 * 16 + (c16 >> 1) * 2;
  a.dst = (c16 >> 2) * SEGK + swz128(a.row0, 2 * (c16 & 3));
  return a;
}
__device__ __forceinline__ void convert_q8_tile(const uint8_t* raw, uint8_t* dst_tile, const ConvAddr& a, int zero_from) {
#pragma unroll 1
  for (int k0 = 0; k0 < 8; k0 += 4) {
    // loads of four items first: a shared-memory load is never moved above an earlier store
    uint4 x[4];
    __half d[4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
      x[k] = *(const uint4*)(raw + a.src + (k0 + k) * 1024);
      d[k] = *(const __half*)(raw + a.sc + (k0 + k) * 128);
    }
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const __half2 dd = __half2half2(d[k]);
      const uint32_t xw[4] = {x[k].x ^ 0x80808080u, x[k].y ^ 0x80808080u, x[k].z ^ 0x80808080u, x[k].w ^ 0x80808080u};
      uint32_t o[8];
#pragma unroll
      for (int w = 0; w < 4; w++) {
        o[2 * w] = dq_pair(__byte_perm(xw[w], 0x64646464u, 0x4140), dd);
        o[2 * w + 1] = dq_pair(__byte_perm(xw[w], 0x64646464u, 0x4342), dd);
      }
      if (a.row0 + 8 * (k0 + k) >= zero_from) {
#pragma unroll
        for (int w = 0; w < 8; w++) o[w] = 0;
      }
      uint8_t* dst = dst_tile + (k0 + k) * 1024;
      *(uint4*)(dst + a.dst) = make_uint4(o[0], o[1], o[2], o[3]);
      *(uint4*)(dst + (a.dst ^ 16u)) = make_uint4(o[4], o[5], o[6], o[7]);
    }
  }
}

}  // namespace
}  // namespace q27b
